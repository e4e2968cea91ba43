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
// of one list entry and key head.  The committed positions of a sequence make
// ceil(length / KEYS) tiles and its drafted nodes one tile of their own, so
// only that last tile needs the tree's mask.  CTA c of the first g = min(grid, U)
// takes the units [U c / g, U (c + 1) / g): equal shares, none of them empty,
// whatever the lengths, with at most two items of each CTA shared with its
// neighbours.
template <int KEYS, int ROWS> struct TreeWork
{
    static constexpr int keys_per_tile = KEYS, rows_per_item = ROWS;

    struct Entry
    {
        int sequence, held, length, nodes, tiles, row_items;
        long long units;
    };

    // Tiles and items of list entry i; one that is invalid (reported) or empty has none.
    static __device__ __forceinline__ Entry entry(const TreeArgs& a, int i)
    {
        Entry e;
        e.sequence = cache_sequence(a.cache, a.sequences, i);
        e.nodes = a.nodes ? a.nodes[i] : a.max_nodes;
        e.nodes = e.nodes < a.max_nodes ? e.nodes : a.max_nodes;
        e.units = e.tiles = e.row_items = e.length = e.held = 0;
        if (e.nodes <= 0)
            return e;
        bool valid = e.sequence >= 0;
        if (valid)
        {
            e.held = cache_held(a.cache, e.sequence);
            e.length = a.cache.lengths[e.sequence];
            valid = e.length >= 0 &&
                    static_cast<long long>(e.length) + e.nodes <= static_cast<long long>(e.held) << a.cache.page_shift;
        }
        if (!valid)
        {
            if (a.error_word)
                atomicOr(a.error_word, error_cache);
            return e;
        }
        e.tiles = (e.length + KEYS - 1) / KEYS + 1;
        e.row_items = (e.nodes * a.group + ROWS - 1) / ROWS;
        e.units = static_cast<long long>(e.tiles) * e.row_items * a.heads;
        return e;
    }

    static __device__ __forceinline__ long long first_unit(long long units, int cta, int ctas)
    {
        return units * cta / ctas;
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
    };

    // The CTA's first list entry, by the whole CTA (THREADS threads, a multiple of 32).
    template <int THREADS>
    static __device__ Start find(const TreeArgs& a, int cta, int ctas, long long* warp_sums, Start* found)
    {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int each = (a.count + THREADS - 1) / THREADS;
        const int begin = min(a.count, static_cast<int>(threadIdx.x) * each), end = min(a.count, begin + each);
        long long mine = 0;
        for (int i = begin; i < end; ++i)
            mine += entry(a, i).units;
        long long inclusive = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1)
        {
            const long long up = __shfl_up_sync(0xffffffffu, inclusive, d);
            inclusive += lane >= d ? up : 0;
        }
        if (lane == 31)
            warp_sums[warp] = inclusive;
        if (threadIdx.x == 0)
            *found = Start{0, 0, a.count, 0};
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
        if (u >= before && u < before + mine)
        {
            for (int i = begin; i < end; ++i)
            {
                const long long n = entry(a, i).units;
                if (u < before + n)
                {
                    *found = Start{units, before, i, sharing};
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
};

// What a CTA leaves for the combining launch: the item it began and did not finish.
struct TreeShared
{
    int entry, head, first_row, pieces; // pieces of the item, the first by this CTA; 0 = none
    int nodes;
};

// A piece's row: running maximum (of scores x log2(e)), sum, and the unscaled output.
constexpr int TREE_PIECE_HEAD = 4; // floats before a row's outputs, 16-byte aligned: maximum, sum
inline __host__ __device__ long long tree_piece_floats(int rows, int head_dim)
{
    return static_cast<long long>(rows) * (head_dim + TREE_PIECE_HEAD);
}

size_t tree_attention_scratch(int head_dim);
cudaError_t tree_attention(const TreeArgs& a, ValueType type, void* scratch, cudaStream_t stream);
} // namespace tsacb::dev
