// Pages of a key/value cache: reserve (allocate, and copy what is shared),
// fork, release, append, keep and compact, all on the device, so that a
// decode step never waits for the host.
//
// The allocator's whole state is the reference count of each page: a page is
// free when no table entry names it, and allocation takes the lowest free
// pages in list order.  Every result therefore depends on the inputs alone,
// not on the order in which CTAs run (reference counts change by commutative
// integer atomics), and the state can be saved, restored or built by a caller
// as three integer tensors.
#include "kernels/error_bits.hpp"
#include "kernels/launch_count.hpp"
#include "kernels/paged_cache.cuh"
#include "kernels/pdl.cuh"

namespace tsacb::dev
{
namespace
{
constexpr int PLAN_THREADS = 1024;
constexpr int COPY_THREADS = 256;
constexpr int COPY_AHEAD = 8;                          // loads in flight per thread
constexpr int COPY_CHUNKS = COPY_AHEAD * COPY_THREADS; // 16-byte chunks of one copy unit

__device__ __forceinline__ void raise(unsigned* error_word, unsigned bit)
{
    if (error_word)
        atomicOr(error_word, bit);
}

// Exclusive sum over the block (1,024 threads) and the total.
__device__ __forceinline__ int block_exclusive(int value, int* warp_sums, int& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inclusive = value;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
    {
        const int up = __shfl_up_sync(0xffffffffu, inclusive, d);
        inclusive += lane >= d ? up : 0;
    }
    if (lane == 31)
        warp_sums[warp] = inclusive;
    __syncthreads();
    if (warp == 0)
    {
        int w = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1)
        {
            const int up = __shfl_up_sync(0xffffffffu, w, d);
            w += lane >= d ? up : 0;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    const int before = warp ? warp_sums[warp - 1] : 0;
    total = warp_sums[31];
    __syncthreads();
    return before + inclusive - value;
}

// Writes the lowest `limit` pages of [begin, end) whose reference count
// passes `test` to out, ascending; returns how many there are (at most limit).
// One pass of the block covers up to 32,768 pages: each warp owns a contiguous
// run, reads it coalesced with all loads in flight, keeps one ballot per 32
// pages (lane k the k-th), and the block scans the warps' totals once.
template <class Test>
__device__ int select_pages(const int* refs, int begin, int end, int limit, int* out, int* warp_sums, Test test)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int found = 0;
    for (int tile = begin; tile < end && found < limit; tile += PLAN_THREADS * 32)
    {
        const int left = end - tile;
        const int groups = left >= PLAN_THREADS * 32 ? 32 : (left + PLAN_THREADS - 1) / PLAN_THREADS;
        const int first = tile + warp * groups * 32;
        unsigned mine = 0;
#pragma unroll 8
        for (int k = 0; k < groups; ++k)
        {
            const int page = first + k * 32 + lane;
            const bool hit = page < end && test(refs[page]);
            const unsigned mask = __ballot_sync(0xffffffffu, hit);
            if (lane == k)
                mine = mask;
        }
        int total;
        const int before = found + block_exclusive(__popc(mine), warp_sums, total);
        for (int k = 0; k < groups; ++k)
        {
            const unsigned mask = __shfl_sync(0xffffffffu, mine, k);
            const int at = __shfl_sync(0xffffffffu, before, k) + __popc(mask & ((1u << lane) - 1u));
            if ((mask >> lane & 1u) && at < limit)
                out[at] = first + k * 32 + lane;
        }
        found += total;
    }
    __syncthreads();
    return found < limit ? found : limit;
}

// ------------------------------------------------------------------ reserve --
struct ReserveScratch
{
    int* copies_count;    // page copies to make
    int2* copies;         // (from, to)
    int2* shared;         // held pages of a write range that others hold too: (page, item)
    int* free_pages;      // lowest free pages
    unsigned char* flags; // [count][slots]: the held page of this slot is to be copied
};

ReserveScratch reserve_layout(void* scratch, size_t items)
{
    auto* base = static_cast<unsigned char*>(scratch);
    ReserveScratch s;
    s.copies_count = reinterpret_cast<int*>(base);
    s.copies = reinterpret_cast<int2*>(base + 16);
    s.shared = s.copies + items;
    s.free_pages = reinterpret_cast<int*>(s.shared + items);
    s.flags = reinterpret_cast<unsigned char*>(s.free_pages + items);
    return s;
}

struct WriteRange
{
    int sequence, held, first, last; // table entries [first, last]; empty when last < first
};

// The table entries that positions [length, length + more) of a list entry
// fall into; false when the entry is invalid.
__device__ __forceinline__ bool write_range(const CacheView& c, const int* sequences, const int* positions, int i,
                                            int slots, WriteRange& w)
{
    w.sequence = cache_sequence(c, sequences, i);
    if (w.sequence < 0)
        return false;
    w.held = cache_held(c, w.sequence);
    const long long length = c.lengths[w.sequence], more = positions[i];
    if (length < 0 || more < 0 || length > static_cast<long long>(w.held) << c.page_shift ||
        (length + more + c.page_size() - 1) >> c.page_shift > c.max_pages)
        return false;
    w.first = static_cast<int>(length >> c.page_shift);
    w.last = more == 0 ? w.first - 1 : static_cast<int>((length + more - 1) >> c.page_shift);
    return w.last - w.first < slots;
}

// A shared page is copied for each list entry that writes to it, except for
// the last of them when no other sequence holds it.  With r table entries on a
// page and g of them in this call's ranges, that is: all copy when r > g, all
// but the last when r = g.  Found in time linear in the shared entries by
// lending the page's own count: g is taken off it, then where nothing is left
// the lowest -(item + 1) names the last, then the count is put back.
__device__ void mark_copies(int* refs, const ReserveScratch& s, int shared, int slots, int* needs)
{
    const int t = threadIdx.x;
    const auto copy = [&](int item)
    {
        s.flags[item] = 1;
        atomicAdd(&needs[item / slots], 1);
    };
    for (int a = t; a < shared; a += PLAN_THREADS)
        atomicSub(&refs[s.shared[a].x], 1);
    __syncthreads();
    for (int a = t; a < shared; a += PLAN_THREADS)
    {
        const int2 mine = s.shared[a];
        if (__ldcg(&refs[mine.x]) > 0)
            copy(mine.y);
        else
            atomicMin(&refs[mine.x], -(mine.y + 1));
    }
    __syncthreads();
    for (int a = t; a < shared; a += PLAN_THREADS)
    {
        const int2 mine = s.shared[a];
        const int left = __ldcg(&refs[mine.x]);
        if (left <= 0 && left != -(mine.y + 1))
            copy(mine.y);
    }
    __syncthreads();
    for (int a = t; a < shared; a += PLAN_THREADS)
    {
        const int2 mine = s.shared[a];
        if (__ldcg(&refs[mine.x]) == -(mine.y + 1))
            atomicExch(&refs[mine.x], 0);
    }
    __syncthreads();
    for (int a = t; a < shared; a += PLAN_THREADS)
        atomicAdd(&refs[s.shared[a].x], 1);
    __syncthreads();
}

// One CTA plans the whole call.  It is bound by a few dependent round trips to
// L2 (lengths, tables, reference counts, then the free pages), not by bytes.
__global__ void __launch_bounds__(PLAN_THREADS)
    cache_reserve_kernel(CacheView c, const int* sequences, const int* positions, int count,
                         int slots, ReserveScratch s, unsigned* error_word)
{
    pdl_prologue();
    __shared__ unsigned seen[CACHE_MAX_SEQUENCES / 32];
    __shared__ int needs[CACHE_MAX_LIST];
    __shared__ int warp_sums[32];
    __shared__ int shared_count, copies, bad;
    const int t = threadIdx.x;
    for (int k = t; k < (c.sequences + 31) / 32; k += PLAN_THREADS)
        seen[k] = 0;
    if (t == 0)
    {
        shared_count = copies = bad = 0;
        *s.copies_count = 0;
    }
    __syncthreads();
    for (int i = t; i < count; i += PLAN_THREADS)
    {
        WriteRange w;
        needs[i] = 0;
        if (!write_range(c, sequences, positions, i, slots, w) ||
            (atomicOr(&seen[w.sequence >> 5], 1u << (w.sequence & 31)) >> (w.sequence & 31) & 1u))
        {
            bad = 1;
            continue;
        }
        for (int j = w.first; j <= w.last && j < w.held; ++j)
        {
            const int item = i * slots + j - w.first;
            const int page = cache_page(c, w.sequence, w.held, j);
            const int refs = page < 0 ? 0 : c.refs[page];
            if (refs < 1)
                bad = 1;
            else if (refs > 1)
                s.shared[atomicAdd(&shared_count, 1)] = make_int2(page, item);
            s.flags[item] = 0;
        }
        const int fresh = w.first > w.held ? w.first : w.held;
        needs[i] = w.last >= fresh ? w.last - fresh + 1 : 0;
    }
    __syncthreads();
    if (bad)
    {
        if (t == 0)
            raise(error_word, error_cache);
        return;
    }
    if (shared_count)
        mark_copies(c.refs, s, shared_count, slots, needs);
    // Exclusive sums of the needs, four consecutive list entries per thread.
    int four[4], sum = 0, total;
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        four[k] = 4 * t + k < count ? needs[4 * t + k] : 0;
        sum += four[k];
    }
    int offset = block_exclusive(sum, warp_sums, total);
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        if (4 * t + k < count)
            needs[4 * t + k] = offset;
        offset += four[k];
    }
    if (total == 0)
        return;
    if (select_pages(c.refs, 0, c.pages, total, s.free_pages, warp_sums, [](int refs) { return refs == 0; }) < total)
    {
        if (t == 0)
            raise(error_word, error_pages);
        return;
    }
    // The pages behind the held ones, one thread per page whichever sequence
    // takes it: a prompt's thousands must not wait for one thread (one sequence
    // of 2,048 pages, the whole call: 18 us, by one thread 157 us).
    for (int k = t; k < total; k += PLAN_THREADS)
    {
        int i = 0, behind = count; // the entry whose pages hold the k-th
        while (behind - i > 1)
        {
            const int middle = (i + behind) >> 1;
            (needs[middle] <= k ? i : behind) = middle;
        }
        WriteRange w;
        write_range(c, sequences, positions, i, slots, w);
        const int end = i + 1 < count ? needs[i + 1] : total; // the entry's copies come first
        const int j = w.last - (end - 1 - k);
        if (j < w.first || j < w.held)
            continue;
        const int page = s.free_pages[k];
        c.refs[page] = 1;
        c.tables[static_cast<size_t>(w.sequence) * c.max_pages + j] = page;
    }
    __syncthreads(); // the counts have been read
    for (int i = t; i < count; i += PLAN_THREADS)
    {
        WriteRange w;
        write_range(c, sequences, positions, i, slots, w);
        int next = needs[i];
        int* table = c.tables + static_cast<size_t>(w.sequence) * c.max_pages;
        for (int j = w.first; j <= w.last && j < w.held; ++j)
        {
            if (!s.flags[i * slots + j - w.first])
                continue;
            const int page = s.free_pages[next++], old = table[j];
            s.copies[atomicAdd(&copies, 1)] = make_int2(old, page);
            atomicSub(&c.refs[old], 1);
            c.refs[page] = 1;
            table[j] = page;
        }
        if (w.last >= w.held)
            c.counts[w.sequence] = w.last + 1;
    }
    __syncthreads();
    if (t == 0)
        *s.copies_count = copies;
}

// Copies whole pages of every plane, HBM-bound: one unit is 32 KiB of one
// page of one plane, eight 16-byte loads in flight per thread.  Sources and
// destinations are distinct pages, so units are independent.
__device__ __forceinline__ void copy_pages(const CacheView& c, const int2* pairs, long long count)
{
    const int page_chunks = static_cast<int>(c.page_bytes() >> 4);
    const int parts = (page_chunks + COPY_CHUNKS - 1) / COPY_CHUNKS;
    const long long units = count * c.planes * parts;
    const bool small = units <= 0x7fffffff; // 32-bit division serves
    for (long long u = blockIdx.x; u < units; u += gridDim.x)
    {
        const long long rest = small ? static_cast<unsigned>(u) / static_cast<unsigned>(parts) : u / parts;
        const int part = static_cast<int>(u - rest * parts);
        const long long index = small ? static_cast<unsigned>(rest) / static_cast<unsigned>(c.planes) : rest / c.planes;
        const int2 pair = pairs[index];
        unsigned char* plane = c.pool + (rest - index * c.planes) * c.plane_bytes;
        const auto* from = reinterpret_cast<const uint4*>(plane + pair.x * c.page_bytes());
        auto* to = reinterpret_cast<uint4*>(plane + pair.y * c.page_bytes());
        uint4 v[COPY_AHEAD];
#pragma unroll
        for (int k = 0; k < COPY_AHEAD; ++k)
        {
            const int at = part * COPY_CHUNKS + k * COPY_THREADS + threadIdx.x;
            if (at < page_chunks)
                v[k] = __ldcs(from + at);
        }
#pragma unroll
        for (int k = 0; k < COPY_AHEAD; ++k)
        {
            const int at = part * COPY_CHUNKS + k * COPY_THREADS + threadIdx.x;
            if (at < page_chunks)
                __stcs(to + at, v[k]);
        }
    }
}

__global__ void __launch_bounds__(COPY_THREADS)
    cache_copy_kernel(CacheView c, const int* count, const int2* pairs)
{
    pdl_prologue();
    copy_pages(c, pairs, *count);
}

// --------------------------------------------------------- fork and release --
// One CTA per (parent, child).  A pair is skipped, and reported, when either
// is no sequence, when the child holds pages, when an earlier pair names the
// same child, or when its parent is some pair's child (whose table this call
// is writing).
__global__ void __launch_bounds__(256)
    cache_fork_kernel(CacheView c, const int* parents, const int* children, int count,
                      unsigned* error_word)
{
    pdl_prologue();
    const int i = blockIdx.x;
    const int parent = cache_sequence(c, parents, i), child = cache_sequence(c, children, i);
    const bool named = parent >= 0 && child >= 0;
    // Read before the list is: one round trip for both.
    const int length = named ? c.lengths[parent] : 0, held = named ? cache_held(c, parent) : 0;
    const bool empty = named && c.counts[child] == 0;
    bool clash = false;
    for (int k = threadIdx.x; k < count; k += 256)
        clash |= (k < i && children[k] == child) || children[k] == parent;
    const int share = length > 0 ? (length - 1 >> c.page_shift) + 1 : 0;
    bool bad = __syncthreads_or(clash) || !empty || length < 0 || share > held;
    if (!bad)
    {
        bool broken = false;
        for (int j = threadIdx.x; j < share; j += 256)
        {
            const int page = cache_page(c, parent, share, j);
            broken |= page < 0 || c.refs[page] < 1; // counts only rise in this launch, from 1 at least
        }
        bad = __syncthreads_or(broken);
    }
    if (bad)
    {
        if (threadIdx.x == 0)
            raise(error_word, error_cache);
        return;
    }
    const int* from = c.tables + static_cast<size_t>(parent) * c.max_pages;
    int* to = c.tables + static_cast<size_t>(child) * c.max_pages;
    for (int j = threadIdx.x; j < share; j += 256)
    {
        const int page = from[j];
        atomicAdd(&c.refs[page], 1);
        to[j] = page;
    }
    if (threadIdx.x == 0)
    {
        c.counts[child] = share;
        c.lengths[child] = length;
    }
}

__global__ void __launch_bounds__(256)
    cache_release_kernel(CacheView c, const int* sequences, const int* positions,
                         unsigned* error_word)
{
    pdl_prologue();
    const int i = blockIdx.x;
    const int sequence = cache_sequence(c, sequences, i);
    const int keep = positions ? positions[i] : 0;
    bool again = false;
    if (sequences)
        for (int k = threadIdx.x; k < i; k += 256)
            again |= sequences[k] == sequence;
    if (__syncthreads_or(again) || sequence < 0 || keep < 0)
    {
        if (threadIdx.x == 0)
            raise(error_word, error_cache);
        return;
    }
    const int held = cache_held(c, sequence);
    const int stay = keep > 0 ? (keep - 1 >> c.page_shift) + 1 : 0;
    int* table = c.tables + static_cast<size_t>(sequence) * c.max_pages;
    bool broken = false;
    for (int j = stay + threadIdx.x; j < held; j += 256)
    {
        const int page = table[j];
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.pages))
        {
            broken = true;
        }
        else if (atomicSub(&c.refs[page], 1) < 1)
        {
            atomicAdd(&c.refs[page], 1); // more entries than the count says: it stays as it was
            broken = true;
        }
        table[j] = -1;
    }
    if (broken)
        raise(error_word, error_cache);
    __syncthreads(); // every thread has read the count
    if (threadIdx.x == 0)
    {
        if (stay < held)
            c.counts[sequence] = stay;
        if (keep < c.lengths[sequence])
            c.lengths[sequence] = keep;
    }
}

// ------------------------------------------------------------------- append --
// One warp per row (its keys and its values), a lane per 16-byte chunk.  The
// row's chunks are loaded before its page is looked up (length, count, table,
// reference count: four dependent reads of L2), so that the two latencies
// overlap.  A row is written only into a page that its sequence holds alone.
constexpr int APPEND_WARPS = 4, APPEND_CHUNKS = 4; // chunks of keys and of values in flight per lane

__global__ void __launch_bounds__(APPEND_WARPS * 32)
    cache_append_kernel(CacheView c, int layer, AppendRows rows, const int* sequences, const int* nodes,
                        const int* starts, int max_nodes, long long row_count, unsigned* error_word)
{
    pdl_prologue();
    const int lane = threadIdx.x & 31;
    const int row_chunks = rows.heads * rows.head_chunks;
    for (long long row = blockIdx.x * static_cast<long long>(APPEND_WARPS) + (threadIdx.x >> 5); row < row_count;
         row += static_cast<long long>(gridDim.x) * APPEND_WARPS)
    {
        // 32-bit division where it serves: the 64-bit one is a long routine.
        const int i = row <= 0x7fffffff ? static_cast<int>(static_cast<unsigned>(row) / static_cast<unsigned>(max_nodes))
                                        : static_cast<int>(row / max_nodes);
        const int n = static_cast<int>(row - static_cast<long long>(i) * max_nodes);
        if (nodes && n >= nodes[i])
            continue;
        const auto load = [&](int value, int chunk)
        {
            const int head = chunk / rows.head_chunks, part = chunk - head * rows.head_chunks;
            return __ldcs(reinterpret_cast<const uint4*>(rows.source[value] + i * rows.batch_bytes[value] +
                                                         n * rows.node_bytes[value] + head * rows.head_bytes[value]) +
                          part);
        };
        uint4* place[2] = {nullptr, nullptr};
        for (int first = lane; first - lane < row_chunks; first += 32 * APPEND_CHUNKS)
        {
            uint4 v[2][APPEND_CHUNKS];
#pragma unroll
            for (int k = 0; k < APPEND_CHUNKS; ++k)
                if (first + 32 * k < row_chunks)
                {
                    v[0][k] = load(0, first + 32 * k);
                    v[1][k] = load(1, first + 32 * k);
                }
            if (first == lane)
            {
                const int sequence = cache_sequence(c, sequences, i);
                int page = -1;
                long long position = -1;
                if (sequence >= 0)
                {
                    const int start = starts ? starts[i] : c.lengths[sequence];
                    position = static_cast<long long>(start) + n;
                    if (start >= 0)
                        page = cache_page(c, sequence, cache_held(c, sequence),
                                          static_cast<int>(position >> c.page_shift));
                }
                if (page < 0 || c.refs[page] != 1)
                {
                    if (lane == 0)
                        raise(error_word, error_cache);
                    break;
                }
                unsigned char* to = c.pool + 2ll * layer * c.plane_bytes + page * c.page_bytes() +
                                    (position & (c.page_size() - 1)) * c.row_bytes;
                place[0] = reinterpret_cast<uint4*>(to);
                place[1] = reinterpret_cast<uint4*>(to + c.plane_bytes);
            }
#pragma unroll
            for (int k = 0; k < APPEND_CHUNKS; ++k)
                if (first + 32 * k < row_chunks)
                {
                    place[0][first + 32 * k] = v[0][k];
                    place[1][first + 32 * k] = v[1][k];
                }
        }
    }
}

// --------------------------------------------------------------------- keep --
// Whether list entry i may move its rows: the path ascends, its rows and
// places lie in held pages, and the places' pages are the sequence's alone.
// Called by a whole CTA; every thread returns the same answer.
__device__ __forceinline__ bool keep_valid(const CacheView& c, const int* sequences, const int* path, const int* accepted,
                           const int* starts, int i, int width, int& sequence, int& start, int& n)
{
    sequence = cache_sequence(c, sequences, i);
    n = accepted[i];
    bool bad = sequence < 0 || n < 0 || n > width;
    start = bad ? 0 : (starts ? starts[i] : c.lengths[sequence]);
    const int held = bad ? 0 : cache_held(c, sequence);
    bad |= start < 0 || static_cast<long long>(start) + n > static_cast<long long>(held) << c.page_shift;
    bool wrong = false;
    if (!bad)
    {
        const int* mine = path + static_cast<size_t>(i) * width;
        for (int j = threadIdx.x; j < n; j += blockDim.x)
        {
            const int from = mine[j];
            wrong |= from < 0 || (j > 0 && mine[j - 1] >= from);
            const long long at = static_cast<long long>(start) + from;
            wrong |= at >= static_cast<long long>(held) << c.page_shift ||
                     cache_page(c, sequence, held, static_cast<int>(at >> c.page_shift)) < 0;
            const int to = cache_page(c, sequence, held, start + j >> c.page_shift);
            wrong |= to < 0 || (from != j && c.refs[to] != 1);
        }
        if (sequences)
            for (int k = threadIdx.x; k < i; k += blockDim.x)
                wrong |= sequences[k] == sequence;
    }
    return !(__syncthreads_or(wrong) || bad);
}

// One CTA per (list entry, plane) moves row path[j] to place j, ascending.  A
// batch is loaded whole before it is stored (one barrier), and since path[j]
// >= j, no batch reads a row that an earlier one has overwritten.
__global__ void __launch_bounds__(COPY_THREADS)
    cache_keep_kernel(CacheView c, const int* sequences, const int* path,
                      const int* accepted, const int* starts, int* lengths_out, int width,
                      unsigned* error_word)
{
    pdl_prologue();
    const int i = blockIdx.x, plane_index = blockIdx.y;
    int sequence, start, n;
    if (!keep_valid(c, sequences, path, accepted, starts, i, width, sequence, start, n))
    {
        if (threadIdx.x == 0 && plane_index == 0)
            raise(error_word, error_cache);
        return;
    }
    const int* mine = path + static_cast<size_t>(i) * width;
    const int* table = c.tables + static_cast<size_t>(sequence) * c.max_pages;
    unsigned char* plane = c.pool + plane_index * c.plane_bytes;
    const int row_chunks = c.row_bytes >> 4;
    const int in_page = c.page_size() - 1;
    auto row_at = [&](int position)
    {
        return reinterpret_cast<uint4*>(plane + table[position >> c.page_shift] * c.page_bytes() +
                                        static_cast<long long>(position & in_page) * c.row_bytes);
    };
    const long long chunks = static_cast<long long>(n) * row_chunks;
    for (long long base = 0; base < chunks; base += 4 * COPY_THREADS)
    {
        uint4 v[4];
        uint4* to[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const long long at = base + k * COPY_THREADS + threadIdx.x;
            to[k] = nullptr;
            if (at < chunks)
            {
                const int j = static_cast<int>(at / row_chunks), chunk = static_cast<int>(at - static_cast<long long>(j) * row_chunks);
                const int from = mine[j];
                if (from != j)
                {
                    to[k] = row_at(start + j) + chunk;
                    v[k] = row_at(start + from)[chunk];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (to[k])
                *to[k] = v[k];
    }
    if (lengths_out && plane_index == 0 && threadIdx.x == 0)
        lengths_out[sequences ? sequence : i] = start + n;
}

// New lengths of the kept sequences where they replace the starts that every
// plane's CTA has read: a launch of its own behind the moves.
__global__ void __launch_bounds__(128)
    cache_keep_lengths_kernel(CacheView c, const int* sequences, const int* path,
                              const int* accepted, int width)
{
    pdl_prologue();
    int sequence, start, n;
    const int i = blockIdx.x;
    const bool ok = keep_valid(c, sequences, path, accepted, nullptr, i, width, sequence, start, n);
    if (ok && threadIdx.x == 0)
        c.lengths[sequence] = start + n;
}

// ------------------------------------------------------------------ compact --
struct CompactScratch
{
    int* copies_count;
    int2* copies;  // (from, to)
    int* map;      // [pages] a page's place after the call, -1: not in use
    int* selected; // [2][pages] live pages above the live count; holes below it
};

CompactScratch compact_layout(void* scratch, size_t pages)
{
    auto* base = static_cast<unsigned char*>(scratch);
    CompactScratch s;
    s.copies_count = reinterpret_cast<int*>(base);
    s.copies = reinterpret_cast<int2*>(base + 16);
    s.map = reinterpret_cast<int*>(s.copies + pages);
    s.selected = s.map + pages;
    return s;
}

// With L pages live, the k-th live page at or above L moves into the k-th
// hole below L: the fewest moves that leave the live pages at [0, L).  Live is
// a positive count and a hole anything else, so that there is a hole for every
// move whatever the counts are; a negative one is reported and becomes 0.
__global__ void __launch_bounds__(PLAN_THREADS)
    cache_compact_plan_kernel(CacheView c, int* refs_out, int* live_out, CompactScratch s, unsigned* error_word)
{
    pdl_prologue();
    __shared__ int warp_sums[32];
    const int t = threadIdx.x;
    int mine = 0, live;
    bool negative = false;
#pragma unroll 4
    for (int page = t; page < c.pages; page += PLAN_THREADS)
    {
        mine += c.refs[page] > 0;
        negative |= c.refs[page] < 0;
    }
    if (negative)
        raise(error_word, error_cache);
    block_exclusive(mine, warp_sums, live);
    const int moves = select_pages(c.refs, live, c.pages, c.pages, s.selected, warp_sums, [](int refs) { return refs > 0; });
    select_pages(c.refs, 0, live, c.pages, s.selected + c.pages, warp_sums, [](int refs) { return refs <= 0; });
    for (int page = t; page < c.pages; page += PLAN_THREADS)
    {
        const int refs = c.refs[page];
        s.map[page] = refs > 0 ? page : -1;
        refs_out[page] = refs > 0 ? refs : 0;
    }
    __syncthreads();
    for (int k = t; k < moves; k += PLAN_THREADS)
    {
        const int from = s.selected[k], to = s.selected[c.pages + k];
        s.copies[k] = make_int2(from, to);
        s.map[from] = to;
        refs_out[to] = c.refs[from];
    }
    __syncthreads(); // the counts of moved pages have been read
    for (int k = t; k < moves; k += PLAN_THREADS)
        refs_out[s.selected[k]] = 0;
    if (t == 0)
    {
        *s.copies_count = moves;
        *live_out = live;
    }
}

__global__ void __launch_bounds__(COPY_THREADS)
    cache_compact_kernel(CacheView c, int* tables_out, CompactScratch s, unsigned* error_word)
{
    pdl_prologue();
    const long long entries = static_cast<long long>(c.sequences) * c.max_pages;
    for (long long at = blockIdx.x * static_cast<long long>(COPY_THREADS) + threadIdx.x; at < entries;
         at += static_cast<long long>(gridDim.x) * COPY_THREADS)
    {
        const int sequence = static_cast<int>(at / c.max_pages), entry = static_cast<int>(at - static_cast<long long>(sequence) * c.max_pages);
        const int held = cache_held(c, sequence);
        const int page = cache_page(c, sequence, held, entry);
        const int place = page < 0 ? -1 : s.map[page];
        if (place < 0 && entry < held)
            raise(error_word, error_cache);
        tables_out[at] = place;
    }
    copy_pages(c, s.copies, *s.copies_count);
}

// Copy grids: eight CTAs of 256 threads fill an SM, and units are strided over them.
int copy_grid()
{
    int device = 0, sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess)
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return sms * 8;
}
} // namespace

size_t cache_reserve_scratch(size_t count, size_t slots)
{
    return 16 + count * slots * (2 * sizeof(int2) + sizeof(int) + 1);
}

void cache_reserve(const CacheView& c, const int* sequences, const int* positions, int count, int slots,
                   void* scratch, unsigned* error_word, cudaStream_t stream)
{
    const ReserveScratch s = reserve_layout(scratch, static_cast<size_t>(count) * slots);
    launch_pdl(cache_reserve_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, c, sequences, positions, count, slots, s,
               error_word);
    note_launch();
    launch_pdl(cache_copy_kernel, dim3(copy_grid()), dim3(COPY_THREADS), 0, stream, c,
               static_cast<const int*>(s.copies_count), static_cast<const int2*>(s.copies));
    note_launch();
}

void cache_fork(const CacheView& c, const int* parents, const int* children, int count, unsigned* error_word,
                cudaStream_t stream)
{
    launch_pdl(cache_fork_kernel, dim3(count), dim3(256), 0, stream, c, parents, children, count, error_word);
    note_launch();
}

void cache_release(const CacheView& c, const int* sequences, const int* positions, int count, unsigned* error_word,
                   cudaStream_t stream)
{
    launch_pdl(cache_release_kernel, dim3(count), dim3(256), 0, stream, c, sequences, positions, error_word);
    note_launch();
}

void cache_append(const CacheView& c, int layer, const AppendRows& rows, const int* sequences, const int* nodes,
                  const int* starts, int count, int max_nodes, unsigned* error_word, cudaStream_t stream)
{
    const long long row_count = static_cast<long long>(count) * max_nodes;
    const long long blocks = (row_count + APPEND_WARPS - 1) / APPEND_WARPS;
    const int grid = static_cast<int>(blocks < 2 * copy_grid() ? blocks : 2 * copy_grid());
    launch_pdl(cache_append_kernel, dim3(grid), dim3(APPEND_WARPS * 32), 0, stream, c, layer, rows, sequences, nodes,
               starts, max_nodes, row_count, error_word);
    note_launch();
}

void cache_keep(const CacheView& c, const int* sequences, const int* path, const int* accepted, const int* starts,
                int* lengths_out, int count, int width, unsigned* error_word, cudaStream_t stream)
{
    const bool in_place = !starts && lengths_out == c.lengths;
    launch_pdl(cache_keep_kernel, dim3(count, c.planes), dim3(COPY_THREADS), 0, stream, c, sequences, path, accepted,
               starts, in_place ? static_cast<int*>(nullptr) : lengths_out, width, error_word);
    note_launch();
    if (in_place)
    {
        launch_pdl(cache_keep_lengths_kernel, dim3(count), dim3(128), 0, stream, c, sequences, path, accepted, width);
        note_launch();
    }
}

size_t cache_compact_scratch(size_t pages)
{
    return 16 + pages * (sizeof(int2) + 3 * sizeof(int));
}

void cache_compact(const CacheView& c, int* tables_out, int* refs_out, int* live, void* scratch,
                   unsigned* error_word, cudaStream_t stream)
{
    const CompactScratch s = compact_layout(scratch, static_cast<size_t>(c.pages));
    launch_pdl(cache_compact_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, c, refs_out, live, s, error_word);
    note_launch();
    launch_pdl(cache_compact_kernel, dim3(copy_grid()), dim3(COPY_THREADS), 0, stream, c, tables_out, s, error_word);
    note_launch();
}
} // namespace tsacb::dev
