// Attention of trees of drafted tokens over a paged key/value cache, for few
// query rows per key head.
//
//   o = sum_k p_k v_k / sum_k p_k,  p_k = exp2(z_k - max z),  z = q.k scale log2(e)
// over the committed positions and the row's own ancestors.  One pass: each
// warp keeps a running maximum, sum and output of its rows over its share of
// the keys, and the shares are joined at the end (warps in shared memory, CTAs
// in a second small launch).  Sums and outputs are 32-bit; p is rounded to the
// input type for the second product, as its operand must be.  For fp16 the
// reference is 15 below the running maximum (Half2::weight_powers): a p then
// keeps all its bits down to 2^-29 of the row's largest, and is nothing from
// 2^-40 on.
//
// Bound: the keys and values cross HBM once per key head, M / 2 multiply-adds
// per byte for M query rows; up to 32 rows that is below what mma.sync
// sustains, so the layout is chosen for bytes in flight: each warp streams its
// own keys of a tile (16 of 64 at 128 columns, 32 of 128 at 64) through a
// private three-stage ring (16-byte asynchronous copies, any page size), so no
// barrier couples the warps before the end of an item, and two CTAs of four
// warps keep up to 128 KiB in flight per SM.  (16 keys of 64 columns a stage,
// half of that, took 133 us for 96 single tokens over up to 8,191 positions;
// 32 take 112.)
#include "kernels/half_types.cuh"
#include "kernels/launch_count.hpp"
#include "kernels/pdl.cuh"
#include "kernels/tree_attention.cuh"

#include <algorithm>
#include <mutex>

namespace tsacb::dev
{
namespace
{
constexpr int WARPS = 4, THREADS = WARPS * 32, STAGES = 3;

__device__ __forceinline__ void load_matrices(std::uint32_t address, std::uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(std::uint32_t address, std::uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D> struct Layout
{
    static constexpr int ROWS = 16; // of an item: the rows of an mma.sync tile
    static constexpr int WARP_KEYS = D == 128 ? 16 : 32, KEYS = WARPS * WARP_KEYS;
    static constexpr int row_bytes = 2 * D, chunks = D / 8;
    static constexpr int stage_bytes = 2 * WARP_KEYS * row_bytes; // keys, then values
    static constexpr int ring_bytes = WARPS * STAGES * stage_bytes;
    static constexpr int merge_bytes = WARPS * ROWS * D * 4;
    static constexpr int smem = ring_bytes > merge_bytes ? ring_bytes : merge_bytes;
};

template <class T, int D>
__global__ void __launch_bounds__(THREADS, 2)
    tree_attention_kernel(const TreeArgs a, float* pieces, TreeShared* shared_items)
{
    pdl_prologue();
    using L = Layout<D>;
    using Work = TreeWork<L::KEYS, L::ROWS, 1>;
    constexpr int WARP_KEYS = L::WARP_KEYS, NT = WARP_KEYS / 8; // keys of a warp, and their groups of 8
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long masks[DRAFT_MAX_NODES];
    __shared__ long long warp_sums[WARPS];
    __shared__ typename Work::Start found;
    __shared__ float row_max[WARPS][L::ROWS], row_sum[WARPS][L::ROWS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int cta = blockIdx.x;
    const auto start = Work::template find<THREADS>(a, cta, gridDim.x, warp_sums, &found);
    if (t == 0)
        shared_items[cta].pieces = 0;
    if (cta >= start.ctas)
        return;
    const std::uint32_t ring = static_cast<std::uint32_t>(__cvta_generic_to_shared(smem)) + warp * STAGES * L::stage_bytes;
    const unsigned char* plane = a.cache.pool + 2ll * a.layer * a.cache.plane_bytes;

    typename Work::Cursor cursor(start);
    typename Work::Segment g;
    while (cursor.next(a, g))
    {
        const auto& e = g.e;
        const int head = g.head, first_row = g.first_row, rows = g.rows;
        const int tile_begin = g.tile_begin, tile_end = g.tile_end;
        // Each lane follows one of the warp's keys.
        const auto key_row = [&](int tile)
        { return Work::key_row(a, g, tile, warp * WARP_KEYS + (lane & (WARP_KEYS - 1))); };
        // Rows of L::chunks 16-byte chunks, chunk c of row r at place c ^ (r & 7): conflict-free for ldmatrix.
        const auto fetch = [&](int stage, long long row_offset)
        {
            constexpr int rows_at_once = 32 / L::chunks;
            const std::uint32_t base = ring + stage * L::stage_bytes;
#pragma unroll
            for (int i = 0; i < WARP_KEYS / rows_at_once; ++i)
            {
                const int row = i * rows_at_once + lane / L::chunks, chunk = lane % L::chunks;
                const long long offset = __shfl_sync(0xffffffffu, row_offset, row);
                const unsigned bytes = offset >= 0 ? 16u : 0u;
                const unsigned char* from = plane + (offset >= 0 ? offset + 16 * chunk : 0);
                const std::uint32_t to = base + row * L::row_bytes + ((chunk ^ (row & 7)) << 4);
                copy_16(to, from, bytes);
                copy_16(to + WARP_KEYS * L::row_bytes, from + a.cache.plane_bytes, bytes);
            }
        };
        __syncwarp();
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s)
        {
            fetch(s, key_row(tile_begin + s));
            copies_commit();
        }
        long long next_row = key_row(tile_begin + STAGES - 1);
        // While the first keys and values are on their way: the tree's masks and the query.
        if (tile_end == e.tiles)
        {
            if (warp == 0)
                ancestor_masks(a.parents + static_cast<long long>(g.list_entry) * a.max_nodes, e.nodes, masks,
                               a.error_word, lane);
            __syncthreads();
        }

        // Query fragments: row lane / 4 (+ 8), columns 2 (lane % 4) (+ 8) of each 16.
        std::uint32_t q[D / 16][4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
        {
            const int row = first_row + 8 * r + (lane >> 2);
            const int node = row / a.group, in_group = row - node * a.group;
            const std::uint16_t* from = a.query + g.list_entry * a.query_batch + node * a.query_node +
                                        (head * a.group + in_group) * a.query_head + 2 * (lane & 3);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
            {
                q[k][r] = row < rows ? *reinterpret_cast<const std::uint32_t*>(from + 16 * k) : 0u;
                q[k][r + 2] = row < rows ? *reinterpret_cast<const std::uint32_t*>(from + 16 * k + 8) : 0u;
            }
        }
        float o[D / 8][4] = {};
        // The running maximum less Half2::weight_powers: what p is a power of two from.
        float reference[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

        int stage = 0;
        for (int tile = tile_begin; tile < tile_end; ++tile)
        {
            // The stage refilled here was consumed in the previous step by this warp alone.
            fetch(stage == 0 ? STAGES - 1 : stage - 1, next_row);
            copies_commit();
            next_row = key_row(tile + STAGES);
            copies_wait<STAGES - 1>();
            __syncwarp();
            const std::uint32_t keys = ring + stage * L::stage_bytes, values = keys + WARP_KEYS * L::row_bytes;
            stage = stage + 1 == STAGES ? 0 : stage + 1;

            float s[NT][4] = {};
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int half = 0; half < NT / 2; ++half) // 16 keys each
                {
                    // Matrices: keys 0-7 and 8-15 by the two halves of the 16 columns.
                    const int row = 16 * half + (lane & 7) + ((lane >> 4) << 3), chunk = 2 * k + ((lane >> 3) & 1);
                    std::uint32_t b[4];
                    load_matrices(keys + row * L::row_bytes + ((chunk ^ (row & 7)) << 4), b);
                    Half2<T>::mma(s[2 * half], q[k], b[0], b[1]);
                    Half2<T>::mma(s[2 * half + 1], q[k], b[2], b[3]);
                }
            const bool last = Work::is_last(g, tile);
            const bool masked = Work::is_masked(g, tile);
            // The warp's keys are bits `first_bit` and on of the 32 that `visible` gives.
            const int first_bit = (warp * WARP_KEYS) & 31;
            const int first_node = Work::base(g, tile) + warp * WARP_KEYS - e.length; // of the warp's first key, if drafted
            unsigned tainted = 0; // drafted rows with a value that is not finite
            if (last && first_node > -WARP_KEYS && first_node < e.nodes)
            {
                for (int row = max(0, -first_node); row < WARP_KEYS; ++row)
                {
                    bool odd = false;
                    if (lane < L::chunks)
                    {
                        const uint4 v = *reinterpret_cast<const uint4*>(
                            smem + (values - static_cast<std::uint32_t>(__cvta_generic_to_shared(smem))) +
                            row * L::row_bytes + (lane << 4));
                        const std::uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            odd |= nonfinite_mask<T>(words[w]) != 0;
                    }
                    tainted |= __any_sync(0xffffffffu, odd) ? 1u << row : 0u;
                }
            }
            std::uint32_t p[NT / 2][4];
            float exact_p[2][2 * NT];
#pragma unroll
            for (int r = 0; r < 2; ++r)
            {
                std::uint32_t sees = ~0u;
                if (masked)
                {
                    const int row = first_row + 8 * r + (lane >> 2);
                    sees = Work::visible(g, tile, warp * WARP_KEYS / 32, last && row < rows ? masks[row / a.group] : 0ull) >>
                           (first_bit + 2 * (lane & 3)); // this lane's keys: bits 0 and 1 of each 8
                }
                float z[2 * NT], best = -INFINITY;
#pragma unroll
                for (int k = 0; k < 2 * NT; ++k)
                {
                    z[k] = s[k >> 1][2 * r + (k & 1)] * a.scale_log2;
                    if (!(sees >> ((k & 1) + 8 * (k >> 1)) & 1u))
                        z[k] = -INFINITY;
                    best = fmaxf(best, z[k]);
                }
                best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
                best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
                best = fmaxf(reference[r], __fadd_ru(best, -Half2<T>::weight_powers)); // p is 2^weight_powers at most
                const float shift = best == -INFINITY ? 0.0f : best; // rows that have seen nothing yet
                const float scale = power_of_two(reference[r] - shift);
                reference[r] = best;
                float partial = 0.0f;
#pragma unroll
                for (int k = 0; k < 2 * NT; ++k)
                {
                    z[k] = power_of_two(z[k] - shift);
                    partial += z[k];
                    exact_p[r][k] = z[k];
                }
                sum[r] = fmaf(sum[r], scale, partial);
#pragma unroll
                for (int half = 0; half < NT / 2; ++half)
                {
                    p[half][r] = Half2<T>::pack(z[4 * half], z[4 * half + 1]);
                    p[half][r + 2] = Half2<T>::pack(z[4 * half + 2], z[4 * half + 3]);
                }
                if (__any_sync(0xffffffffu, scale != 1.0f))
                {
#pragma unroll
                    for (int n = 0; n < D / 8; ++n)
                    {
                        o[n][2 * r] *= scale;
                        o[n][2 * r + 1] *= scale;
                    }
                }
            }
            if (tainted)
            {
                // 0 x NaN would reach rows that do not see the node: take such
                // rows out of the product and add them where they are seen.
                const auto base = values - static_cast<std::uint32_t>(__cvta_generic_to_shared(smem));
                for (int key = 0; key < WARP_KEYS; ++key)
                {
                    if (!(tainted >> key & 1u))
                        continue;
                    const int k = (key & 1) + 2 * (key >> 3), from = (lane & ~3) | ((key & 7) >> 1);
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                    {
                        const int row = first_row + 8 * r + (lane >> 2);
                        const bool seen = row < rows && (masks[row / a.group] >> (first_node + key) & 1ull);
                        float weight = 0.0f;
#pragma unroll
                        for (int kk = 0; kk < 2 * NT; ++kk)
                        {
                            const float w = __shfl_sync(0xffffffffu, exact_p[r][kk], from);
                            weight = kk == k ? w : weight;
                        }
#pragma unroll
                        for (int n = 0; n < D / 8; ++n)
                        {
                            const std::uint32_t v = *reinterpret_cast<const std::uint32_t*>(
                                smem + base + key * L::row_bytes + ((n ^ (key & 7)) << 4) + 4 * (lane & 3));
                            if (seen)
                            {
                                o[n][2 * r] = fmaf(weight, Half2<T>::value(v & 0xffffu), o[n][2 * r]);
                                o[n][2 * r + 1] = fmaf(weight, Half2<T>::value(v >> 16), o[n][2 * r + 1]);
                            }
                        }
                    }
                }
                __syncwarp();
                for (int key = 0; key < WARP_KEYS; ++key)
                    if ((tainted >> key & 1u) && lane < L::chunks)
                        *reinterpret_cast<uint4*>(smem + base + key * L::row_bytes + (lane << 4)) = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
#pragma unroll
            for (int half = 0; half < NT / 2; ++half)
#pragma unroll
                for (int n = 0; n < D / 16; ++n)
                {
                    // Matrices: keys 0-7 and 8-15 by the two halves of 16 output columns.
                    const int row = 16 * half + (lane & 7) + (((lane >> 3) & 1) << 3), chunk = 2 * n + (lane >> 4);
                    std::uint32_t b[4];
                    load_matrices_transposed(values + row * L::row_bytes + ((chunk ^ (row & 7)) << 4), b);
                    Half2<T>::mma(o[2 * n], p[half], b[0], b[1]);
                    Half2<T>::mma(o[2 * n + 1], p[half], b[2], b[3]);
                }
            __syncwarp(); // the stage may be refilled
        }
        copies_wait<0>();
        // Join the warps: common maximum, scaled outputs through shared memory.
#pragma unroll
        for (int r = 0; r < 2; ++r)
        {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
            if ((lane & 3) == 0)
            {
                row_max[warp][8 * r + (lane >> 2)] = reference[r];
                row_sum[warp][8 * r + (lane >> 2)] = sum[r];
            }
        }
        __syncthreads();
        float* merge = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int r = 0; r < 2; ++r)
        {
            const int row = 8 * r + (lane >> 2);
            float best = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                best = fmaxf(best, row_max[w][row]);
            const float scale = best == -INFINITY ? 0.0f : power_of_two(reference[r] - best);
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float2*>(merge + (warp * L::ROWS + row) * D + 8 * n + 2 * (lane & 3)) =
                    make_float2(o[n][2 * r] * scale, o[n][2 * r + 1] * scale);
        }
        __syncthreads();
        const bool whole = tile_begin == 0 && tile_end == e.tiles;
        // A piece that begins its item goes to the CTA's second place, any other to its first.
        float* piece = pieces + (2ll * cta + (tile_begin == 0)) * tree_piece_floats(L::ROWS, D);
        for (int at = t; at < L::ROWS * (D / 4); at += THREADS)
        {
            const int row = at / (D / 4), column = 4 * (at - row * (D / 4));
            if (first_row + row >= rows)
                continue;
            float best = -INFINITY, total = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                best = fmaxf(best, row_max[w][row]);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
            {
                // A row of undefined scores has no maximum, but an undefined sum.
                total += best == -INFINITY ? row_sum[w][row] : row_sum[w][row] * power_of_two(row_max[w][row] - best);
                const float4 x = *reinterpret_cast<const float4*>(merge + (w * L::ROWS + row) * D + column);
                v.x += x.x;
                v.y += x.y;
                v.z += x.z;
                v.w += x.w;
            }
            if (!whole)
            {
                float* to = piece + row * (D + TREE_PIECE_HEAD);
                *reinterpret_cast<float4*>(to + TREE_PIECE_HEAD + column) = v;
                if (column == 0)
                {
                    to[0] = best;
                    to[1] = total;
                }
                continue;
            }
            const int node = (first_row + row) / a.group, in_group = first_row + row - node * a.group;
            const float inverse = total == 0.0f ? 0.0f : 1.0f / total; // a row that sees nothing gives zeros
            std::uint16_t* to = a.out + g.list_entry * a.out_batch + node * a.out_node +
                                (head * a.group + in_group) * a.out_head + column;
            *reinterpret_cast<uint2*>(to) =
                make_uint2(Half2<T>::pack(v.x * inverse, v.y * inverse), Half2<T>::pack(v.z * inverse, v.w * inverse));
            if (a.lse && column == 0)
                a.lse[(static_cast<long long>(g.list_entry) * a.max_nodes + node) * a.heads * a.group + head * a.group +
                      in_group] = total == 0.0f ? -INFINITY : (best + log2f(total)) * 0.6931471805599453f;
        }
        if (tile_begin == 0 && !whole && t == 0)
            shared_items[cta] = TreeShared{g.list_entry, head, first_row,
                                           Work::owner(start.units, g.item_start + e.tiles - 1, start.ctas) - cta + 1, e.nodes};
        __syncthreads(); // the ring and the row statistics are free again
    }
}

// Joins the pieces of an item that several CTAs share.  Piece 0 is in the first
// CTA's second place, the others in their CTAs' first places.  Each CTA lists
// the shared items, so that the rows spread over the whole grid, and gives each
// row up to 16 warps, one for four pieces as far as the grid has warps for all
// rows at once: the warps take the pieces in turn, four in flight, and are
// joined in shared memory in a fixed order.  Bound by the latency of two
// dependent reads, so a thread has the registers for four pieces in flight (3
// lanes x 12 nodes, the whole call: 13.4 us; 15.8 us at three CTAs per SM) and
// the grid is one CTA per SM (13.7 us with two, the second behind the first).
constexpr int COMBINE_WARPS = 16, COMBINE_THREADS = COMBINE_WARPS * 32;

template <class T, int D>
__global__ void __launch_bounds__(COMBINE_THREADS, 1)
    tree_combine_kernel(const TreeArgs a, int rows_per_item, int ctas, const float* pieces, const TreeShared* shared_items)
{
    pdl_prologue();
    constexpr int PER = D / 32; // columns of one lane
    __shared__ float part[COMBINE_WARPS][D + 2];
    __shared__ int rows_until[COMBINE_THREADS], warp_sums[COMBINE_WARPS], most_pieces;
    __shared__ TreeShared items[COMBINE_THREADS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int until = 0; // rows of the shared items up to the thread's
    if (t == 0)
        most_pieces = 0;
    __syncthreads();
    if (t < ctas)
    {
        const TreeShared s = shared_items[t];
        items[t] = s;
        until = s.pieces ? min(s.nodes * a.group - s.first_row, rows_per_item) : 0;
        if (s.pieces)
            atomicMax(&most_pieces, s.pieces);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
    {
        const int up = __shfl_up_sync(0xffffffffu, until, d);
        until += lane >= d ? up : 0;
    }
    if (lane == 31)
        warp_sums[warp] = until;
    __syncthreads();
    for (int w = 0; w < warp; ++w)
        until += warp_sums[w];
    rows_until[t] = until;
    __syncthreads();
    const int rows = rows_until[COMBINE_THREADS - 1];
    const int warps = static_cast<int>(gridDim.x) * COMBINE_WARPS;
    int shares = 1; // warps of one row, a power of two
    while (shares < COMBINE_WARPS && 4 * shares < most_pieces && 2 * shares * rows <= warps)
        shares *= 2;
    const int at_once = COMBINE_WARPS / shares, share = warp & (shares - 1);
    for (int first = blockIdx.x * at_once; first < rows; first += gridDim.x * at_once)
    {
        const int index = first + warp / shares;
        const bool live = index < rows;
        int cta = 0; // the first whose running count exceeds the row's
        for (int step = COMBINE_THREADS / 2; step; step >>= 1)
            cta += rows_until[cta + step - 1] <= (live ? index : 0) ? step : 0;
        const TreeShared item = items[cta];
        const int row = index - (cta ? rows_until[cta - 1] : 0);
        const long long stride = 2 * tree_piece_floats(rows_per_item, D);
        const auto piece = [&](int k)
        { return pieces + (cta + k) * stride + (k == 0 ? stride / 2 : 0) + row * (D + TREE_PIECE_HEAD); };
        float best = -INFINITY, total = 0.0f, v[PER] = {};
        constexpr int AHEAD = 4;
        for (int k0 = share; live && k0 < item.pieces; k0 += AHEAD * shares)
        {
            float2 head[AHEAD]; // maximum and sum
            float x[AHEAD][PER];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
            {
                const int k = k0 + j * shares;
                head[j] = make_float2(-INFINITY, 0.0f);
                if (k < item.pieces)
                {
                    const float* from = piece(k);
                    head[j] = *reinterpret_cast<const float2*>(from);
                    if constexpr (PER == 4)
                        *reinterpret_cast<float4*>(x[j]) = *reinterpret_cast<const float4*>(from + TREE_PIECE_HEAD + 4 * lane);
                    else
                        *reinterpret_cast<float2*>(x[j]) = *reinterpret_cast<const float2*>(from + TREE_PIECE_HEAD + 2 * lane);
                }
                else
                {
#pragma unroll
                    for (int c = 0; c < PER; ++c)
                        x[j][c] = 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
            {
                const float raised = fmaxf(best, head[j].x), zero = raised == -INFINITY ? 0.0f : raised;
                const float old_scale = power_of_two(best - zero), new_scale = power_of_two(head[j].x - zero);
                best = raised;
                total = fmaf(total, old_scale, head[j].y * new_scale);
#pragma unroll
                for (int c = 0; c < PER; ++c)
                    v[c] = fmaf(v[c], old_scale, x[j][c] * new_scale);
            }
        }
        if (shares > 1)
        {
            __syncthreads(); // the last rows have been read
#pragma unroll
            for (int c = 0; c < PER; ++c)
                part[warp][lane * PER + c] = v[c];
            if (lane == 0)
            {
                part[warp][D] = best;
                part[warp][D + 1] = total;
            }
            __syncthreads();
            if (share == 0)
                for (int w = warp + 1; w < warp + shares; ++w)
                {
                    const float raised = fmaxf(best, part[w][D]), zero = raised == -INFINITY ? 0.0f : raised;
                    const float old_scale = power_of_two(best - zero), new_scale = power_of_two(part[w][D] - zero);
                    best = raised;
                    total = fmaf(total, old_scale, part[w][D + 1] * new_scale);
#pragma unroll
                    for (int c = 0; c < PER; ++c)
                        v[c] = fmaf(v[c], old_scale, part[w][lane * PER + c] * new_scale);
                }
        }
        if (!live || share != 0)
            continue;
        const int node = (item.first_row + row) / a.group, in_group = item.first_row + row - node * a.group;
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        std::uint16_t* to = a.out + item.entry * a.out_batch + node * a.out_node + (item.head * a.group + in_group) * a.out_head;
#pragma unroll
        for (int c = 0; c < PER; c += 2)
            *reinterpret_cast<std::uint32_t*>(to + lane * PER + c) = Half2<T>::pack(v[c] * inverse, v[c + 1] * inverse);
        if (a.lse && lane == 0)
            a.lse[(static_cast<long long>(item.entry) * a.max_nodes + node) * a.heads * a.group + item.head * a.group + in_group] =
                total == 0.0f ? -INFINITY : (best + log2f(total)) * 0.6931471805599453f;
    }
}

int sms()
{
    int device = 0, count = 148;
    if (cudaGetDevice(&device) == cudaSuccess)
        cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
    return count;
}

// CTAs of the launch and rows of one item, by rows per key head.
struct Shape
{
    int ctas, rows;
    explicit Shape(int rows_per_head)
        : ctas(std::min(COMBINE_THREADS, tree_attention_many(rows_per_head) ? sms() : 2 * sms())),
          rows(tree_attention_many(rows_per_head) ? tree_attention_tc_rows(rows_per_head) : 16)
    {
    }
};

template <class T, int D>
void launch_few(const TreeArgs& a, const Shape& shape, float* pieces, TreeShared* items, cudaStream_t stream)
{
    using L = Layout<D>;
    static std::once_flag once[64];
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64)
        std::call_once(once[device],
                       []
                       {
                           cudaFuncSetAttribute(tree_attention_kernel<T, D>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem);
                       });
    launch_pdl(tree_attention_kernel<T, D>, dim3(shape.ctas), dim3(THREADS), L::smem, stream, a, pieces, items);
    note_launch();
}

template <class T, int D> cudaError_t launch(const TreeArgs& a, ValueType type, void* scratch, cudaStream_t stream)
{
    const int rows = a.max_nodes * a.group;
    const Shape shape(rows);
    auto* pieces = static_cast<float*>(scratch);
    auto* items = reinterpret_cast<TreeShared*>(pieces + 2ll * shape.ctas * tree_piece_floats(shape.rows, D));
    if (tree_attention_many(rows))
    {
        const cudaError_t status = tree_attention_tc(a, type, shape.ctas, pieces, items, stream);
        if (status != cudaSuccess)
            return status;
    }
    else
    {
        launch_few<T, D>(a, shape, pieces, items, stream);
    }
    launch_pdl(tree_combine_kernel<T, D>, dim3(sms()), dim3(COMBINE_THREADS), 0, stream, a, shape.rows, shape.ctas,
               static_cast<const float*>(pieces), static_cast<const TreeShared*>(items));
    note_launch();
    return cudaGetLastError();
}

template <class T> cudaError_t launch_type(const TreeArgs& a, ValueType type, void* scratch, cudaStream_t stream)
{
    return a.head_dim == 64 ? launch<T, 64>(a, type, scratch, stream) : launch<T, 128>(a, type, scratch, stream);
}
} // namespace

// 16 rows are one mma.sync tile of each warp.  Two tiles would spill at 128
// columns, and at 64 took 188 us for 96 sequences of up to 8,191 positions with
// 32 rows, the tensor cores 158.
bool tree_attention_many(int rows)
{
    return rows > 16;
}

size_t tree_attention_scratch(int head_dim, int rows)
{
    const Shape shape(rows);
    return static_cast<size_t>(shape.ctas) *
           (2 * sizeof(float) * static_cast<size_t>(tree_piece_floats(shape.rows, head_dim)) + sizeof(TreeShared));
}

cudaError_t tree_attention(const TreeArgs& a, ValueType type, void* scratch, cudaStream_t stream)
{
    return type == ValueType::bf16 ? launch_type<__nv_bfloat16>(a, type, scratch, stream)
                                   : launch_type<__half>(a, type, scratch, stream);
}
} // namespace tsacb::dev
