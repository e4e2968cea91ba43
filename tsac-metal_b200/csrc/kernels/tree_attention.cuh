// Attention of trees of drafted tokens over a paged key/value cache: arguments,
// the division of the work over CTAs, and the launches (tree_attention.cu).
// The definition is stated in include/tsac_cuda.h.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels/draft_verify.cuh"
#include "kernels/error_bits.hpp"
#include "kernels/paged_cache.cuh"

namespace tsacb::dev
{
struct TreeArgs
{
    CacheView cache;
    int layer, heads, group, head_dim; // key heads, query heads per key head
    const int* sequences;              // [count] or null
    const int* parents;                // [count][max_nodes]
    const int* nodes;                  // [count] or null
    const std::uint16_t* query;        // strides in elements
    std::uint16_t* out;
    long long query_batch, query_node, query_head, out_batch, out_node, out_head;
    float* lse;                        // [count][max_nodes][heads * group] or null
    int count, max_nodes;
    float scale_log2;                  // softmax scale x log2(e)
    unsigned* error_word;
};

// The work is measured in units: one key tile of one item, an item being the
// query rows [first, first + ROWS) (node-major, then query head of the group)
// of one list entry and key head.  An item's last tile begins at last_base and
// holds the last committed keys and, behind them, all drafted nodes: last_base
// is the last multiple of KEYS where they fit, else of 64.  Before it lie
// ceil(last_base / KEYS) tiles, the last of them half full in that second case.
// So only the last tile needs the tree's mask, and a half-full one before it a
// limit.  Each item counts START units more than its tiles, in front of them:
// what it costs to begin and end one, in tiles (measured).  CTA c of the first
// g = min(grid, U) takes the units [U c / g, U (c + 1) / g): equal shares, none
// of them empty, whatever the lengths, with at most two items of each CTA shared
// with its neighbours.  A share that ends before an item's first tile leaves the
// item to the next CTA.
template <int KEYS, int ROWS, int START> struct TreeWork
{
    static constexpr int keys_per_tile = KEYS, rows_per_item = ROWS;

    struct Entry
    {
        int sequence, held, length, nodes, tiles, row_items;
        int last_base; // first position of the last tile
        long long units;
    };

    // Tiles and items of list entry i; one that is invalid (reported) or empty has none.
    static __device__ __forceinline__ Entry entry(const TreeArgs& a, int i)
    {
        Entry e;
        e.sequence = cache_sequence(a.cache, a.sequences, i);
        // All reads at once: a caller waits for one round trip.
        const int s = e.sequence < 0 ? 0 : e.sequence;
        e.nodes = a.nodes ? a.nodes[i] : a.max_nodes;
        e.held = cache_held(a.cache, s);
        e.length = a.cache.lengths[s];
        e.nodes = e.nodes < a.max_nodes ? e.nodes : a.max_nodes;
        e.tiles = e.row_items = e.last_base = 0;
        e.units = 0;
        const bool valid = e.sequence >= 0 && e.length >= 0 && static_cast<long long>(e.length) + e.nodes <= static_cast<long long>(e.held) << a.cache.page_shift;
        if (e.nodes <= 0 || !valid)
        {
            if (e.nodes > 0 && a.error_word)
                atomicOr(a.error_word, error_cache);
            return e;
        }
        // 64 nodes behind a multiple of 64 fit in a tile of 128, whose boxes then start on that multiple.
        const int behind = e.length % KEYS;
        e.last_base = e.length - (behind + e.nodes <= KEYS ? behind : e.length % (KEYS > 64 ? KEYS - 64 : 1));
        e.tiles = (e.last_base + KEYS - 1) / KEYS + 1;
        e.row_items = (e.nodes * a.group + ROWS - 1) / ROWS;
        e.units = static_cast<long long>(START + e.tiles) * e.row_items * a.heads;
        return e;
    }

    // By 32-bit division where it serves: the 64-bit one is a long routine.
    static __device__ __forceinline__ long long quotient(long long n, long long d)
    {
        if (static_cast<unsigned long long>(n | d) >> 32)
            return n / d;
        return static_cast<unsigned>(n) / static_cast<unsigned>(d);
    }
    // units * cta / ctas
    static __device__ __forceinline__ long long first_unit(long long units, int cta, int ctas)
    {
        const long long q = quotient(units, ctas);
        return q * cta + quotient((units - q * ctas) * cta, ctas);
    }
    // The CTA whose share holds unit u.
    static __device__ __forceinline__ int owner(long long units, long long u, int ctas)
    {
        return static_cast<int>(((u + 1) * ctas - 1) / units);
    }

    struct Start
    {
        long long units;  // of the whole call
        long long before; // units of the list entries before `entry`
        int entry;        // list entry that holds the CTA's first unit
        int ctas;         // CTAs that have a share
        long long first, last; // the CTA's share
    };

    static __device__ __forceinline__ long long warp_inclusive(long long v)
    {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1)
        {
            const long long up = __shfl_up_sync(0xffffffffu, v, d);
            v += (threadIdx.x & 31) >= d ? up : 0;
        }
        return v;
    }

    // The CTA's first list entry, by the whole CTA (THREADS threads, a multiple of 32).
    template <int THREADS>
    static __device__ Start find(const TreeArgs& a, int cta, int ctas, long long* warp_sums, Start* found)
    {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (a.count <= 32) // each warp for itself, without a barrier
        {
            const long long mine = lane < a.count ? entry(a, lane).units : 0;
            const long long until = warp_inclusive(mine);
            Start s;
            s.units = __shfl_sync(0xffffffffu, until, 31);
            s.ctas = s.units < ctas ? static_cast<int>(s.units) : ctas;
            s.first = cta < s.ctas ? first_unit(s.units, cta, s.ctas) : s.units;
            s.last = cta < s.ctas ? first_unit(s.units, cta + 1, s.ctas) : s.units;
            const unsigned behind = __ballot_sync(0xffffffffu, until > s.first); // entries that end behind the first unit
            s.entry = behind ? __ffs(static_cast<int>(behind)) - 1 : a.count;
            s.before = __shfl_sync(0xffffffffu, until - mine, s.entry & 31);
            return s;
        }
        const int each = (a.count + THREADS - 1) / THREADS;
        const int begin = min(a.count, static_cast<int>(threadIdx.x) * each), end = min(a.count, begin + each);
        long long mine = 0;
        for (int i = begin; i < end; ++i)
            mine += entry(a, i).units;
        const long long inclusive = warp_inclusive(mine);
        if (lane == 31)
            warp_sums[warp] = inclusive;
        if (threadIdx.x == 0)
            *found = Start{0, 0, a.count, 0, 0, 0};
        __syncthreads();
        long long before = 0, units = 0;
        for (int w = 0; w < THREADS / 32; ++w)
        {
            before += w < warp ? warp_sums[w] : 0;
            units += warp_sums[w];
        }
        before += inclusive - mine;
        const int sharing = units < ctas ? static_cast<int>(units) : ctas;
        const long long u = cta < sharing ? first_unit(units, cta, sharing) : units;
        const long long last = cta < sharing ? first_unit(units, cta + 1, sharing) : units;
        if (u >= before && u < before + mine)
        {
            for (int i = begin; i < end; ++i)
            {
                const long long n = entry(a, i).units;
                if (u < before + n)
                {
                    *found = Start{units, before, i, sharing, u, last};
                    break;
                }
                before += n;
            }
        }
        __syncthreads();
        Start s = *found;
        s.units = units;
        s.ctas = sharing;
        return s;
    }

    // A CTA's part of one item: tiles [tile_begin, tile_end) of its e.tiles.
    struct Segment
    {
        Entry e;
        int list_entry, head, first_row, rows, tile_begin, tile_end;
        long long item_start; // the item's first unit
    };

    // Walks the segments of a CTA's share; every thread of the CTA may keep its own.
    struct Cursor
    {
        long long unit, last_unit, before;
        int list_entry;

        __device__ __forceinline__ explicit Cursor(const Start& s)
            : unit(s.first), last_unit(s.last), before(s.before), list_entry(s.entry)
        {
        }
        __device__ __forceinline__ bool next(const TreeArgs& a, Segment& s)
        {
            while (unit < last_unit)
            {
                s.e = entry(a, list_entry);
                if (unit >= before + s.e.units)
                {
                    before += s.e.units;
                    ++list_entry;
                    continue;
                }
                const int item = static_cast<int>(quotient(unit - before, START + s.e.tiles));
                s.list_entry = list_entry;
                s.head = item / s.e.row_items;
                s.first_row = (item - s.head * s.e.row_items) * ROWS;
                s.rows = s.e.nodes * a.group;
                s.item_start = before + static_cast<long long>(item) * (START + s.e.tiles) + START; // its first tile's unit
                s.tile_begin = static_cast<int>(max(unit - s.item_start, 0ll));
                s.tile_end = static_cast<int>(min(static_cast<long long>(s.e.tiles), last_unit - s.item_start));
                unit = s.item_start + max(s.tile_end, 0);
                if (s.tile_begin >= s.tile_end) // the share ends before the item's first tile
                    continue;
                return true;
            }
            return false;
        }
    };

    static __device__ __forceinline__ bool is_last(const Segment& s, int tile) { return tile == s.e.tiles - 1; }
    // Position of a tile's first key, and the position behind the last that it may hold.
    static __device__ __forceinline__ int base(const Segment& s, int tile)
    {
        return is_last(s, tile) ? s.e.last_base : tile * KEYS;
    }
    static __device__ __forceinline__ int limit(const Segment& s, int tile)
    {
        return is_last(s, tile) ? s.e.length + s.e.nodes : s.e.last_base;
    }
    // Whether some of a tile's keys are not seen by every row.
    static __device__ __forceinline__ bool is_masked(const Segment& s, int tile)
    {
        return is_last(s, tile) || (tile + 1) * KEYS > s.e.last_base;
    }
    // Keys 32 c to 32 c + 31 of a tile that a row sees, one bit each; `sees` are its drafted nodes.
    static __device__ __forceinline__ std::uint32_t visible(const Segment& s, int tile, int c, unsigned long long sees)
    {
        const int committed = (is_last(s, tile) ? s.e.length : s.e.last_base) - base(s, tile) - 32 * c; // of these keys
        std::uint32_t bits = committed >= 32 ? ~0u : (committed <= 0 ? 0u : (1u << committed) - 1u);
        if (is_last(s, tile))
            bits |= static_cast<std::uint32_t>(committed >= 32    ? 0ull
                                               : committed >= 0   ? sees << committed
                                               : committed > -64  ? sees >> -committed
                                                                  : 0ull);
        return bits;
    }

    // Byte offset in a plane of key row `in_tile` of a tile, for one key head; -1: no such key.
    static __device__ __forceinline__ long long key_row(const TreeArgs& a, const Segment& s, int tile, int in_tile)
    {
        const int position = base(s, tile) + in_tile;
        if (tile >= s.tile_end || position >= limit(s, tile))
            return -1;
        const int page = cache_page(a.cache, s.e.sequence, s.e.held, position >> a.cache.page_shift);
        if (page < 0)
        {
            if (a.error_word)
                atomicOr(a.error_word, error_cache);
            return -1;
        }
        return page * a.cache.page_bytes() +
               static_cast<long long>(position & (a.cache.page_size() - 1)) * a.cache.row_bytes +
               2ll * s.head * a.head_dim;
    }
};

// Bit a of masks[n]: node a is node n or one of its ancestors.  By one warp, two
// nodes per lane, with pointer doubling: log2(64) rounds in place of a walk of
// up to 64 dependent steps.  A parent below -1 makes a node that sees no
// drafted node, not even itself; one that is not before its child is reported
// and treated as such.
__device__ __forceinline__ void ancestor_masks(const int* parents, int nodes, unsigned long long* masks,
                                               unsigned* error_word, int lane)
{
    unsigned long long mask[2];
    int above[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
    {
        const int n = lane + 32 * k;
        const int parent = n < nodes ? parents[n] : -2;
        const bool wrong = parent >= n;
        if (wrong && error_word)
            atomicOr(error_word, error_cache);
        mask[k] = parent < -1 || wrong ? 0ull : 1ull << n;
        above[k] = wrong || parent < 0 ? -1 : parent;
    }
    for (int round = 0; round < 6; ++round)
    {
        unsigned long long more[2];
        int next[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            const int from = above[k] & 31;
            const unsigned long long low = __shfl_sync(0xffffffffu, mask[0], from), high = __shfl_sync(0xffffffffu, mask[1], from);
            const int low_above = __shfl_sync(0xffffffffu, above[0], from), high_above = __shfl_sync(0xffffffffu, above[1], from);
            more[k] = above[k] < 0 ? 0ull : (above[k] < 32 ? low : high);
            next[k] = above[k] < 0 ? -1 : (above[k] < 32 ? low_above : high_above);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            mask[k] |= more[k];
            above[k] = next[k];
        }
    }
    masks[lane] = mask[0];
    masks[lane + 32] = mask[1];
}

// What a CTA leaves for the combining launch: the item it began and did not finish.
struct TreeShared
{
    int entry, head, first_row, pieces; // pieces of the item, the first by this CTA; 0 = none
    int nodes;
};

// A piece's row: the number that its weights are powers of two from, near the
// running maximum of scores x log2(e), and the sum and output of those weights.
constexpr int TREE_PIECE_HEAD = 4; // floats before a row's outputs, 16-byte aligned: maximum, sum
inline __host__ __device__ long long tree_piece_floats(int rows, int head_dim)
{
    return static_cast<long long>(rows) * (head_dim + TREE_PIECE_HEAD);
}

// The launches by rows per key head (max_nodes * group): tree_attention.cu
// for few, tree_attention_tc.cu for many.
bool tree_attention_many(int rows);
size_t tree_attention_scratch(int head_dim, int rows);
cudaError_t tree_attention(const TreeArgs& a, ValueType type, void* scratch, cudaStream_t stream);
cudaError_t tree_attention_tc(const TreeArgs& a, ValueType type, int ctas, float* pieces, TreeShared* shared_items,
                              cudaStream_t stream);
int tree_attention_tc_rows(int rows); // rows of one of its items
} // namespace tsacb::dev
