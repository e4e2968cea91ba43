// C ABI: drafted decoding over a paged key/value cache (device pointers,
// caller's stream): page operations, tree attention, draft verification.
#include "cuda_util.cuh"
#include "kernels/draft_verify.cuh"
#include "kernels/paged_cache.cuh"
#include "kernels/tree_attention.cuh"

#include <algorithm>
#include <bit>
#include <cmath>
#include <utility>

namespace
{
using namespace tsacb;

constexpr size_t max_pool_pages = size_t{1} << 24, max_table = size_t{1} << 20;

// The cache's description, checked; what the checks cannot see (whether the
// buffers are as large as stated) is the caller's word.
dev::CacheView view(const tsac_cuda_paged_cache* cache)
{
    require(cache, "null argument");
    const tsac_cuda_paged_cache& c = *cache;
    require(c.pool && c.tables && c.counts && c.lengths && c.refs, "null paged cache buffer");
    require(c.type == TSAC_CUDA_BF16 || c.type == TSAC_CUDA_FP16, "paged cache type must be bf16 or fp16");
    require(c.page_size >= 1 && c.page_size <= 1024 && std::has_single_bit(c.page_size),
            "page size must be a power of two up to 1024");
    require(c.layers >= 1 && c.layers <= 4096, "paged cache layer count out of range");
    require(c.pages >= 1 && c.pages <= max_pool_pages, "paged cache page count out of range");
    require(c.kv_heads >= 1 && c.head_dim >= 1 && c.kv_heads <= 65536 && c.head_dim <= 65536 &&
                c.kv_heads * c.head_dim <= 65536 && c.kv_heads * c.head_dim % 8 == 0,
            "kv_heads * head_dim must be a multiple of 8 up to 65536");
    require(c.sequences >= 1 && c.sequences <= TSAC_CUDA_MAX_SEQUENCES, "paged cache sequence count out of range");
    require(c.max_pages >= 1 && c.max_pages <= max_table, "paged cache table width out of range");
    require(aligned16(c.pool), "paged cache pool must be 16-byte aligned");
    dev::CacheView v;
    v.pool = static_cast<unsigned char*>(c.pool);
    v.tables = c.tables;
    v.counts = c.counts;
    v.lengths = c.lengths;
    v.refs = c.refs;
    v.planes = static_cast<int>(2 * c.layers);
    v.pages = static_cast<int>(c.pages);
    v.page_shift = std::countr_zero(c.page_size);
    v.row_bytes = static_cast<int>(2 * c.kv_heads * c.head_dim);
    v.plane_bytes = static_cast<long long>(c.pages) * v.page_bytes();
    v.sequences = static_cast<int>(c.sequences);
    v.max_pages = static_cast<int>(c.max_pages);
    return v;
}

void require_list(const dev::CacheView& v, const int32_t* sequences, size_t count)
{
    require(count <= TSAC_CUDA_MAX_LIST, "too many sequences in one call");
    require(sequences || count <= static_cast<size_t>(v.sequences), "more entries than the cache has sequences");
}

// Strides of [entry][node][head] rows, in elements.
void require_strides(const ptrdiff_t strides[3], const char* what)
{
    require(strides, "null argument");
    for (int k = 0; k < 3; ++k)
        require(strides[k] % 8 == 0, what);
}

// Whether no two of the [entry][node][head] rows of `row` elements share one: each
// dimension, taken from the smallest stride up, steps over all that lies inside it.
bool rows_apart(const ptrdiff_t strides[3], const size_t sizes[3], size_t row)
{
    std::pair<size_t, size_t> steps[3]; // (stride, size)
    for (int k = 0; k < 3; ++k)
        steps[k] = {sizes[k] > 1 ? (strides[k] < 0 ? size_t{0} - static_cast<size_t>(strides[k]) : static_cast<size_t>(strides[k])) : SIZE_MAX,
                    sizes[k]};
    std::sort(steps, steps + 3);
    size_t span = row;
    for (const auto& [stride, size] : steps)
    {
        if (size <= 1)
            continue;
        if (stride < span || stride > SIZE_MAX / 4 / size)
            return false;
        span += stride * (size - 1);
    }
    return true;
}

bool overlap(const int32_t* a, size_t m, const int32_t* b, size_t n)
{
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + n * sizeof(int32_t) && y < x + m * sizeof(int32_t);
}
} // namespace

extern "C"
{
size_t tsac_cuda_cache_reserve_scratch_bytes(size_t count, size_t slots)
{
    return count <= TSAC_CUDA_MAX_LIST && slots <= max_table ? dev::cache_reserve_scratch(count, slots) : 0;
}

int tsac_cuda_cache_reserve(const tsac_cuda_paged_cache* cache, const int32_t* sequences, const int32_t* positions,
                            size_t count, size_t slots, void* scratch, size_t scratch_bytes, unsigned* error_word,
                            void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require_list(v, sequences, count);
            require(positions || count == 0, "null argument");
            require(slots >= 1 && slots <= cache->max_pages && count * slots <= 0x7fffffffu,
                    "slots of a reservation out of range");
            require(scratch && scratch_bytes >= dev::cache_reserve_scratch(count, slots) && aligned16(scratch),
                    "reservation scratch too small or not 16-byte aligned");
            require_device();
            if (count == 0)
                return;
            dev::cache_reserve(v, sequences, positions, static_cast<int>(count), static_cast<int>(slots), scratch,
                               error_word, static_cast<cudaStream_t>(stream));
            cuda_check(cudaGetLastError(), "cache reserve launch");
        });
}

int tsac_cuda_cache_fork(const tsac_cuda_paged_cache* cache, const int32_t* parents, const int32_t* children,
                         size_t count, unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require((parents && children) || count == 0, "null argument");
            require(count <= TSAC_CUDA_MAX_LIST, "too many sequences in one call");
            require_device();
            if (count == 0)
                return;
            dev::cache_fork(v, parents, children, static_cast<int>(count), error_word,
                            static_cast<cudaStream_t>(stream));
            cuda_check(cudaGetLastError(), "cache fork launch");
        });
}

int tsac_cuda_cache_release(const tsac_cuda_paged_cache* cache, const int32_t* sequences, const int32_t* positions,
                            size_t count, unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require_list(v, sequences, count);
            require_device();
            if (count == 0)
                return;
            dev::cache_release(v, sequences, positions, static_cast<int>(count), error_word,
                               static_cast<cudaStream_t>(stream));
            cuda_check(cudaGetLastError(), "cache release launch");
        });
}

int tsac_cuda_cache_append(const tsac_cuda_paged_cache* cache, size_t layer, const void* keys,
                           const ptrdiff_t key_strides[3], const void* values, const ptrdiff_t value_strides[3],
                           const int32_t* sequences, const int32_t* nodes, const int32_t* starts, size_t count,
                           size_t max_nodes, unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require_list(v, sequences, count);
            require((keys && values) || count == 0, "null argument");
            require(layer < cache->layers, "layer out of range");
            require(max_nodes >= 1 && max_nodes <= 0x7fffffffu, "row count out of range");
            require(cache->head_dim % 8 == 0, "appended rows need a head_dim that is a multiple of 8");
            require_strides(key_strides, "row strides must be multiples of 8 elements");
            require_strides(value_strides, "row strides must be multiples of 8 elements");
            require(aligned16(keys) && aligned16(values), "rows must be 16-byte aligned");
            require_device();
            if (count == 0)
                return;
            dev::AppendRows rows;
            rows.source[0] = static_cast<const unsigned char*>(keys);
            rows.source[1] = static_cast<const unsigned char*>(values);
            for (int k = 0; k < 2; ++k)
            {
                const ptrdiff_t* s = k ? value_strides : key_strides;
                rows.batch_bytes[k] = 2 * s[0];
                rows.node_bytes[k] = 2 * s[1];
                rows.head_bytes[k] = 2 * s[2];
            }
            rows.heads = static_cast<int>(cache->kv_heads);
            rows.head_chunks = static_cast<int>(cache->head_dim / 8);
            dev::cache_append(v, static_cast<int>(layer), rows, sequences, nodes, starts, static_cast<int>(count),
                              static_cast<int>(max_nodes), error_word, static_cast<cudaStream_t>(stream));
            cuda_check(cudaGetLastError(), "cache append launch");
        });
}

int tsac_cuda_cache_keep(const tsac_cuda_paged_cache* cache, const int32_t* sequences, const int32_t* path,
                         const int32_t* accepted, const int32_t* starts, int32_t* lengths_out, size_t count,
                         size_t width, unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require_list(v, sequences, count);
            require((path && accepted && lengths_out) || count == 0, "null argument");
            require(width >= 1 && width <= 0x7fffffffu, "path width out of range");
            require(!lengths_out || lengths_out == v.lengths || !overlap(lengths_out, cache->sequences, v.lengths, cache->sequences),
                    "new lengths overlap the cache's lengths");
            require(!starts || !overlap(lengths_out, cache->sequences, starts, count),
                    "new lengths overlap the starts");
            // Other CTAs still read these when the first new length is written.
            require(!(sequences && overlap(lengths_out, cache->sequences, sequences, count)) &&
                        !overlap(lengths_out, cache->sequences, path, count * width) &&
                        !overlap(lengths_out, cache->sequences, accepted, count) &&
                        (lengths_out == v.lengths || (!overlap(lengths_out, cache->sequences, v.counts, cache->sequences) &&
                                                      !overlap(lengths_out, cache->sequences, v.refs, cache->pages) &&
                                                      !overlap(lengths_out, cache->sequences, v.tables, cache->sequences * cache->max_pages))),
                    "new lengths overlap another argument");
            require_device();
            if (count == 0)
                return;
            dev::cache_keep(v, sequences, path, accepted, starts, lengths_out, static_cast<int>(count),
                            static_cast<int>(width), error_word, static_cast<cudaStream_t>(stream));
            cuda_check(cudaGetLastError(), "cache keep launch");
        });
}

size_t tsac_cuda_cache_compact_scratch_bytes(size_t pages)
{
    return pages <= max_pool_pages ? dev::cache_compact_scratch(pages) : 0;
}

int tsac_cuda_cache_compact(const tsac_cuda_paged_cache* cache, int32_t* tables_out, int32_t* refs_out, int32_t* live,
                            void* scratch, size_t scratch_bytes, unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require(tables_out && refs_out && live, "null argument");
            const size_t entries = cache->sequences * cache->max_pages;
            require(tables_out == v.tables || !overlap(tables_out, entries, v.tables, entries),
                    "new tables overlap the cache's tables");
            require(refs_out == v.refs || !overlap(refs_out, cache->pages, v.refs, cache->pages),
                    "new reference counts overlap the cache's");
            require(scratch && scratch_bytes >= dev::cache_compact_scratch(cache->pages) && aligned16(scratch),
                    "compaction scratch too small or not 16-byte aligned");
            require_device();
            dev::cache_compact(v, tables_out, refs_out, live, scratch, error_word, static_cast<cudaStream_t>(stream));
            cuda_check(cudaGetLastError(), "cache compact launch");
        });
}

size_t tsac_cuda_tree_attention_scratch_bytes(const tsac_cuda_paged_cache* cache, size_t heads, size_t max_nodes)
{
    if (!cache || (cache->head_dim != 64 && cache->head_dim != 128) || cache->kv_heads == 0 || heads > 65536 ||
        max_nodes > TSAC_CUDA_MAX_NODES)
        return 0;
    return dev::tree_attention_scratch(static_cast<int>(cache->head_dim),
                                       static_cast<int>(heads / cache->kv_heads * max_nodes));
}

int tsac_cuda_tree_attention(const tsac_cuda_paged_cache* cache, size_t layer, const int32_t* sequences,
                             const int32_t* parents, const int32_t* nodes, const void* query,
                             const ptrdiff_t query_strides[3], void* out, const ptrdiff_t out_strides[3], float* lse,
                             size_t heads, size_t count, size_t max_nodes, float scale, void* scratch,
                             size_t scratch_bytes, unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            const dev::CacheView v = view(cache);
            require_list(v, sequences, count);
            require((parents && query && out) || count == 0, "null argument");
            require(layer < cache->layers, "layer out of range");
            require(cache->head_dim == 64 || cache->head_dim == 128, "tree attention needs a head_dim of 64 or 128");
            require(heads >= 1 && heads <= 65536 && heads % cache->kv_heads == 0,
                    "query heads must be a multiple of the key heads");
            require(max_nodes >= 1 && max_nodes <= TSAC_CUDA_MAX_NODES, "tree node count out of range");
            const float scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
            require(std::isfinite(scale_log2), "softmax scale must be finite, times log2(e) too");
            require_strides(query_strides, "query strides must be multiples of 8 elements");
            require_strides(out_strides, "output strides must be multiples of 8 elements");
            require(aligned16(query) && aligned16(out), "query and output must be 16-byte aligned");
            const size_t sizes[3] = {count, max_nodes, heads};
            require(count == 0 || rows_apart(out_strides, sizes, cache->head_dim), "output rows overlap one another");
            for (int k = 0; k < 3 && count; ++k)
                require(out != query || sizes[k] == 1 || out_strides[k] == query_strides[k],
                        "output in place of the query needs the query's strides");
            require_device();
            require(scratch && aligned16(scratch) &&
                        scratch_bytes >= tsac_cuda_tree_attention_scratch_bytes(cache, heads, max_nodes),
                    "tree attention scratch too small or not 16-byte aligned");
            if (count == 0)
                return;
            dev::TreeArgs a;
            a.cache = v;
            a.layer = static_cast<int>(layer);
            a.heads = static_cast<int>(cache->kv_heads);
            a.group = static_cast<int>(heads / cache->kv_heads);
            a.head_dim = static_cast<int>(cache->head_dim);
            a.sequences = sequences;
            a.parents = parents;
            a.nodes = nodes;
            a.query = static_cast<const std::uint16_t*>(query);
            a.out = static_cast<std::uint16_t*>(out);
            a.query_batch = query_strides[0];
            a.query_node = query_strides[1];
            a.query_head = query_strides[2];
            a.out_batch = out_strides[0];
            a.out_node = out_strides[1];
            a.out_head = out_strides[2];
            a.lse = lse;
            a.count = static_cast<int>(count);
            a.max_nodes = static_cast<int>(max_nodes);
            a.scale_log2 = scale_log2;
            a.error_word = error_word;
            cuda_check(dev::tree_attention(a, static_cast<dev::ValueType>(cache->type), scratch,
                                           static_cast<cudaStream_t>(stream)),
                       "tree attention launch");
        });
}

int tsac_cuda_draft_verify(const void* target, const ptrdiff_t target_strides[2], const void* draft,
                           const ptrdiff_t draft_strides[2], int type, const int32_t* tokens, const int32_t* parents,
                           const float* coins, const float* draws, const int32_t* nodes, size_t batch,
                           size_t max_nodes, size_t vocab, int32_t* accepted, int32_t* path, int32_t* token,
                           unsigned* error_word, void* stream)
{
    return guarded(
        [&]
        {
            require(type == TSAC_CUDA_BF16 || type == TSAC_CUDA_FP16 || type == TSAC_CUDA_FP32,
                    "probabilities must be bf16, fp16 or fp32");
            require(batch == 0 || (target && target_strides && tokens && parents && coins && draws && accepted && path &&
                                   token && (!draft || draft_strides)),
                    "null argument");
            require(batch <= (1u << 20), "batch out of range");
            require(max_nodes >= 1 && max_nodes <= TSAC_CUDA_MAX_NODES, "tree node count out of range");
            require(vocab >= 1 && vocab <= (1u << 28), "vocabulary size out of range");
            const size_t size = type == TSAC_CUDA_FP32 ? 4 : 2;
            require(reinterpret_cast<uintptr_t>(target) % size == 0 && reinterpret_cast<uintptr_t>(draft) % size == 0,
                    "probabilities must be aligned to their type");
            require_device();
            if (batch == 0)
                return;
            dev::VerifyArgs a;
            a.target = target;
            a.draft = draft;
            a.target_batch = target_strides[0];
            a.target_node = target_strides[1];
            a.draft_batch = draft ? draft_strides[0] : 0;
            a.draft_node = draft ? draft_strides[1] : 0;
            a.tokens = tokens;
            a.parents = parents;
            a.coins = coins;
            a.draws = draws;
            a.nodes = nodes;
            a.accepted = accepted;
            a.path = path;
            a.token = token;
            a.vocab = static_cast<int>(vocab);
            a.max_nodes = static_cast<int>(max_nodes);
            a.error_word = error_word;
            cuda_check(dev::draft_verify(a, static_cast<dev::ValueType>(type), static_cast<int>(batch),
                                         static_cast<cudaStream_t>(stream)),
                       "draft verification launch");
        });
}
}
