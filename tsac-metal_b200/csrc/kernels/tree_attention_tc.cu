// Attention of trees of drafted tokens over a paged key/value cache, for many
// query rows per key head, on the tensor cores (tcgen05).
//
// The formula and the division of the work are those of tree_attention.cu and
// tree_attention.cuh, with tiles of 128 keys and items of 128 or 256 rows.  A
// tile of 128 keys is two products of 128 x 128 x D per 128 rows: at 128 rows
// the tensor cores need about a third of the time that the tile's bytes take
// to arrive, at 256 rows two thirds, and the exponentials (16 per clock and
// SM) about as much.  So a CTA takes up to 256 rows of a key head at once, the
// keys and values cross HBM once, and the kernel is bound by HBM as long as
// products, exponentials and loads overlap.
//
// One CTA per SM, 12 warps:
//   warps 0-3, 4-7  two softmax groups, one query row per thread.  Each has its
//                   own scores S and output O in TMEM.  With 256 rows each
//                   group has 128 of them and sees every tile; with 128 rows
//                   the groups take alternate tiles of the same rows, and their
//                   outputs are joined at the end of the item.
//   warp 8          TMEM owner and MMA issuer: S = Q K^T from shared memory,
//                   then O += P V with P in TMEM over the columns of S.  The
//                   two groups' products alternate, so that one group's
//                   exponentials overlap the other's products.
//   warps 9, 10     producers, half of each key or value tile each, into a ring
//                   of shared-memory slots in the 128-byte swizzle that the MMA
//                   reads, by TMA: one box per page (or 64 rows), a lane each.
//                   Value tiles with rows behind the last position come by
//                   16-byte asynchronous copies that make those rows zeros, as
//                   does everything where TMA does not serve: pages of fewer
//                   than 8 rows (a swizzle atom), or 2^31 rows in a plane.
//                   Copies of every tile by the two warps bound the kernel by
//                   their address arithmetic (290 against 209 us for 64 x 16
//                   nodes over up to 4,096 positions).
//   warp 11         the query rows of the next segment, as soon as the last
//                   scores of this one are made, and its tree's masks.
// The reference that p is a power of two from is a whole number and moves only
// when a row's scores exceed it by more than LIMIT: scores are read once, and
// what has been computed with the old reference, p of the same tile included, is
// rescaled rarely and by powers of two.  For bf16 it is the running maximum with
// a slack of 8: p stays below 2^8, which bf16 and the 32-bit sums hold as well
// as 1.  For fp16 it is 11 below the maximum with a slack of 4: p stays below
// 2^15 and the row's largest is 2^10 at least, so that a p keeps all its bits
// down to 2^-24 of it and is nothing from 2^-35 on.  (A slack of 2 costs
// rescaling: 2 x 64 nodes over 131,072 positions 267 us, 253 with 4 and with 8.)
// The loop over a tile's scores is kept small: unrolled over the whole tile it
// delayed the MMA warp (64 x 16 nodes 172 against 162 us), and exponentials of
// some pairs by a polynomial on the FMA pipes gained nothing over the special
// function units' 16 per clock.
//
// What bounds it now.  128 rows: the loads (64 x 16 nodes 154 us, the same with
// products and softmax left out).  256 rows: products and exponentials, which
// overlap little.  A tile needs 2,048 clocks of each (32 MMAs of 128 x 128 x 16
// at 64, 32,768 exponentials at 16 per clock); 2 x 64 nodes over up to 131,072
// positions, 94 tiles per SM, take 4,500 (253 us at 1.68 GHz) to 4,900 clocks a
// tile (293 us at 1.56 GHz, after seconds at the 1,000 W limit, which sets the
// clock).  Loads alone take 160 us, products and loads 168 to 193, softmax and
// loads 184 to 200; issuing a group's next scores without waiting for its
// product, or handing P on in two parts, gained 7 to 16 us in those and nothing
// in the whole.
//
// Every wait is bounded (tc_common.cuh).  One that gives up raises
// error_timeout and the CTA's abort flag; softmax threads then run through
// their loops without waiting, so that no thread waits at a barrier that
// others have left, and give NaN for the rows that they could not finish.
#include "kernels/half_types.cuh"
#include "kernels/launch_count.hpp"
#include "kernels/pdl.cuh"
#include "kernels/tc_common.cuh"
#include "kernels/tree_attention.cuh"

namespace tsacb::dev
{
namespace
{
using namespace tc;

constexpr int KEYS = 128;
constexpr int GROUP_THREADS = 128, SOFTMAX_THREADS = 2 * GROUP_THREADS;
// Twelve warps leave each thread 168 registers; a 13th would leave 128, and the
// softmax threads would spill.
constexpr int MMA_WARP = 8, PRODUCER_WARP = 9, PRODUCERS = 64, PRODUCER_ROWS = KEYS / 2;
constexpr int QUERY_WARP = PRODUCER_WARP + PRODUCERS / 32;
constexpr int THREADS = (QUERY_WARP + 1) * 32;
constexpr int TMEM_COLUMNS = 512, OUTPUT_COLUMN = 256; // S of the groups at 0 and 128, O at 256 and 384
constexpr int TAINT_SLOTS = 16; // segments that the producers can be ahead of the epilogue, and more

template <int D, bool TWO> struct Tiles
{
    static constexpr int ROWS = TWO ? 256 : 128;
    static constexpr int panels = D / 64;
    static constexpr int operand_bytes = KEYS * 2 * D;
    static constexpr int panel_bytes = KEYS * 128; // queries: 64 columns of 128 rows
    static constexpr int group_bytes = 1024 * panels; // keys and values: 8 rows, the panels' atoms side by side
    static constexpr int query_bytes = operand_bytes * (ROWS / 128);
    static constexpr int SLOTS = (TWO ? 160 : 192) * 1024 / operand_bytes;
    static constexpr int chunks = D / 8;
    // Byte of a 16-byte chunk of a key or value row within its slot.
    static __device__ __forceinline__ int place(int row, int chunk)
    {
        return (row >> 3) * group_bytes + (chunk >> 3) * 1024 + (row & 7) * 128 + (((chunk & 7) ^ (row & 7)) << 4);
    }
    static constexpr int ring_offset = query_bytes;
    static constexpr int tail_offset = ring_offset + SLOTS * operand_bytes;
    static constexpr int tail_bytes = D == 128 ? 2048 : 4096; // barriers and small arrays
    static constexpr int smem = tail_offset + tail_bytes + 1024; // the rest: alignment
    static_assert(smem <= 227 * 1024, "shared memory of one SM");
};

template <int SLOTS> struct Tail
{
    uint64_t full[SLOTS], empty[SLOTS];
    uint64_t scores[2], weights[2], products[2], query, query_free, done, drain;
    // The softmax threads read the masks of a segment at its start; the query warp may be two ahead.
    unsigned long long masks[3][DRAFT_MAX_NODES];
    unsigned long long tainted[TAINT_SLOTS];
    long long warp_sums[THREADS / 32];
    long long start[6]; // TreeWork::Start
    uint32_t tmem;
    int abort;
};
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32"
                 " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
                 " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(address)
                 : "memory");
}

__device__ __forceinline__ uint32_t tmem_load1(uint32_t address)
{
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r)
                 : "r"(address)
                 : "memory");
    return r;
}

// Waits for this thread's TMEM loads; r is named so that no use of it moves before the wait.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
                 " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(address),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

__device__ __forceinline__ void tmem_store2(uint32_t address, uint32_t a, uint32_t b)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(address), "r"(a), "r"(b) : "memory");
}

__device__ __forceinline__ void tmem_wait_stores()
{
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void fence_async_proxy()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void tma_5d(uint32_t to, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4,
                                       uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(to),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
                 : "memory");
}

// Barrier of the softmax threads.
__device__ __forceinline__ void softmax_sync()
{
    asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_THREADS) : "memory");
}

// Key and value tiles are atoms of 8 rows x 64 columns (1,024 bytes, 128-byte
// swizzle), the atoms of the same 8 rows side by side, so that one box brings
// whole rows of a page.  Keys, K-major: the next 8 rows are group_bytes further
// (the columns' atoms are stepped over by the start address).
__device__ __forceinline__ uint64_t key_desc(uint32_t address, uint32_t group_bytes)
{
    uint64_t d = static_cast<uint64_t>((address & 0x3ffffu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(group_bytes >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Values, MN-major: the next 64 columns one atom, the next 8 rows group_bytes further.
__device__ __forceinline__ uint64_t value_desc(uint32_t address, uint32_t group_bytes)
{
    uint64_t d = static_cast<uint64_t>((address & 0x3ffffu) >> 4);
    d |= static_cast<uint64_t>(1024 >> 4) << 16;
    d |= static_cast<uint64_t>(group_bytes >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// kind::f16 with 32-bit accumulation, M = 128.
template <class T> __device__ __forceinline__ constexpr uint32_t instruction(int n, bool b_mn_major)
{
    return (1u << 4) | (Half2<T>::mma_format << 7) | (Half2<T>::mma_format << 10) | (b_mn_major ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

// The MMA warp runs converged, and only the instruction itself is predicated on
// one lane: descriptors, which the instruction takes from uniform registers,
// then need no transfer for each MMA (in a branch of one lane an issue took
// about 100 cycles, the product itself 64).
__device__ __forceinline__ bool elect_one()
{
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "elect.sync _|p, 0xffffffff;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(chosen));
    return chosen != 0;
}

__device__ __forceinline__ void mma_shared(bool leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                           bool accumulate)
{
    asm volatile("{\n\t.reg .pred p, q;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(static_cast<uint32_t>(leader))
                 : "memory");
}

__device__ __forceinline__ void mma_tmem(bool leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                         bool accumulate)
{
    asm volatile("{\n\t.reg .pred p, q;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(static_cast<uint32_t>(leader))
                 : "memory");
}

__device__ __forceinline__ void commit_if(bool leader, uint32_t bar)
{
    asm volatile("{\n\t.reg .pred q;\n\t"
                 "setp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
                 "r"(static_cast<uint32_t>(leader))
                 : "memory");
}

// A value that is the same in every lane, in a form that the compiler knows to be.
__device__ __forceinline__ int uniform(int v)
{
    return __shfl_sync(0xffffffffu, v, 0);
}

// Operand `op` of a segment of `tiles` tiles, in the order in which the MMA
// warp first needs them: whether it is a value tile, and of which tile.
template <bool TWO> __device__ __forceinline__ void operand(int op, int tiles, bool& value, int& tile)
{
    if (TWO || tiles == 1)
    {
        value = op & 1;
        tile = op >> 1;
        return;
    }
    // K0 K1, then V(j) K(j + 2), then the last two V.
    const int k = op - 2, steady = 2 * (tiles - 2);
    value = k >= steady || (k >= 0 && !(k & 1));
    tile = k < 0 ? op : (k >= steady ? tiles - 2 + (k - steady) : (k & 1 ? (k >> 1) + 2 : k >> 1));
}

// ------------------------------------------------- pairs of 32-bit numbers --
using Pair = unsigned long long;

__device__ __forceinline__ Pair make_pair(float a, float b)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c)
{
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair add_pair(Pair a, Pair b)
{
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul_pair(Pair a, Pair b)
{
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// One number for each softmax group, selected without an array in memory.
template <class N> struct Both
{
    N first, second;
    __device__ __forceinline__ N operator()(int group) const { return group ? second : first; }
    __device__ __forceinline__ void add(int group, N n)
    {
        first += group ? N(0) : n;
        second += group ? n : N(0);
    }
};

template <class T, int D, bool TWO>
__global__ void __launch_bounds__(THREADS, 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map, const TreeArgs a, const int box_rows,
                             float* pieces, TreeShared* shared_items)
{
    pdl_prologue();
    using L = Tiles<D, TWO>;
    using Work = TreeWork<KEYS, L::ROWS, 3>;
    // Powers of two: how far a score may exceed the reference, and how far the one that moves it does.
    constexpr bool narrow = Half2<T>::weight_powers > 0.0f;
    constexpr float LIMIT = narrow ? Half2<T>::weight_powers : 8.0f, PLACE = narrow ? LIMIT - 4.0f : 0.0f;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                           ~static_cast<uintptr_t>(1023));
    using TailOf = Tail<L::SLOTS>;
    static_assert(sizeof(TailOf) <= L::tail_bytes, "tail of the shared memory");
    TailOf& tail = *reinterpret_cast<TailOf*>(smem + L::tail_offset);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int cta = blockIdx.x;
    static_assert(sizeof(typename Work::Start) <= sizeof(tail.start));
    const auto start = Work::template find<THREADS>(a, cta, gridDim.x, tail.warp_sums,
                                                    reinterpret_cast<typename Work::Start*>(tail.start));
    if (t == 0)
        shared_items[cta].pieces = 0;
    if (cta >= start.ctas)
        return;
    if (t == 0)
    {
        for (int s = 0; s < L::SLOTS; ++s)
        {
            bar_init(smem_u32(&tail.full[s]), PRODUCERS / 32);
            bar_init(smem_u32(&tail.empty[s]), 1);
        }
        for (int g = 0; g < 2; ++g)
        {
            bar_init(smem_u32(&tail.scores[g]), 1);
            bar_init(smem_u32(&tail.weights[g]), GROUP_THREADS);
            bar_init(smem_u32(&tail.products[g]), 1);
        }
        bar_init(smem_u32(&tail.query), 1);
        bar_init(smem_u32(&tail.query_free), SOFTMAX_THREADS + 1);
        bar_init(smem_u32(&tail.done), SOFTMAX_THREADS);
        bar_init(smem_u32(&tail.drain), 1);
        for (int k = 0; k < TAINT_SLOTS; ++k)
            tail.tainted[k] = 0;
        tail.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail.tmem)),
                     "r"(TMEM_COLUMNS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tail.tmem;
    volatile int* abort_flag = &tail.abort;
    const unsigned char* plane = a.cache.pool + 2ll * a.layer * a.cache.plane_bytes;
    bool ok = true;
    const auto wait = [&](uint64_t& bar, int phase)
    {
        if (ok && !bar_wait(smem_u32(&bar), static_cast<uint32_t>(phase & 1), abort_flag))
        {
            ok = false;
            *abort_flag = 1;
            if (a.error_word)
                atomicOr(a.error_word, error_timeout);
        }
        return ok;
    };
    typename Work::Cursor cursor(start);
    typename Work::Segment g;

    if (warp >= PRODUCER_WARP && warp < QUERY_WARP)
    {
        // ------------------------------------------------------------ producers --
        const int first_row = (warp - PRODUCER_WARP) * PRODUCER_ROWS; // this warp's rows of each tile
        constexpr int rows_at_once = 32 / L::chunks;
        const int boxes = box_rows ? PRODUCER_ROWS / box_rows : 0; // of this warp's half tile
        int slot = 0, round = 0; // uses of the slot so far
        int copied = -1, copied_segment = 0; // a slot whose copies have been issued and not yet announced
        int copied_draft = -1, copied_nodes = 0; // its first drafted row, -1: none; drafted rows
        // Announces the copied slot, once its copies have landed: all but the newest `behind` group.
        const auto announce = [&](bool behind)
        {
            if (copied < 0)
                return;
            if (behind)
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            else
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (copied_draft >= 0)
            {
                __syncwarp(); // a wait covers a lane's own copies, and the rows below are other lanes'
                // 0 x NaN would reach rows that do not see the node: values that are not
                // finite leave the product and are added where they are seen.
                const int chunk = lane % L::chunks;
                const int end = min(first_row + PRODUCER_ROWS, copied_draft + copied_nodes);
#pragma unroll 2
                for (int row = max(first_row, copied_draft) + lane / L::chunks; row < end; row += rows_at_once)
                {
                    auto* at = reinterpret_cast<uint4*>(smem + L::ring_offset + copied * L::operand_bytes + L::place(row, chunk));
                    const uint4 v = *at;
                    const uint32_t odd[4] = {nonfinite_mask<T>(v.x), nonfinite_mask<T>(v.y), nonfinite_mask<T>(v.z),
                                             nonfinite_mask<T>(v.w)};
                    if (odd[0] | odd[1] | odd[2] | odd[3])
                    {
                        *at = make_uint4(v.x & ~odd[0], v.y & ~odd[1], v.z & ~odd[2], v.w & ~odd[3]);
                        atomicOr(&tail.tainted[copied_segment % TAINT_SLOTS], 1ull << ((row - copied_draft) & 63));
                    }
                }
            }
            fence_async_proxy(); // the copies are generic writes, the MMA reads through the async proxy
            __syncwarp();
            if (lane == 0)
                bar_arrive(smem_u32(&tail.full[copied]));
            copied = -1;
        };
        for (int segment = 0; ok && cursor.next(a, g); ++segment)
        {
            const int tiles = g.tile_end - g.tile_begin;
            for (int op = 0; op < 2 * tiles; ++op)
            {
                bool value;
                int tile;
                operand<TWO>(op, tiles, value, tile);
                tile += g.tile_begin;
                const uint32_t base = smem_u32(smem + L::ring_offset + slot * L::operand_bytes);
                const uint32_t bar = smem_u32(&tail.full[slot]);
                // Scores of keys behind the last are masked whatever they are; values have to be zeros.
                const bool boxed = boxes && (!value || !Work::is_masked(g, tile));
                // The tile's table entries are on their way while the slot is awaited.
                int eight_rows = 0; // of the layer's two planes, in units of 8
                long long low_rows = -1, high_rows = -1;
                if (boxed)
                {
                    if (lane < boxes)
                    {
                        const int position = Work::base(g, tile) + first_row + lane * box_rows;
                        const int page = position < Work::limit(g, tile)
                                             ? cache_page(a.cache, g.e.sequence, g.e.held, position >> a.cache.page_shift)
                                             : -1;
                        if (page < 0 && position < Work::limit(g, tile) && a.error_word)
                            atomicOr(a.error_word, error_cache);
                        const int plane_groups = a.cache.pages << a.cache.page_shift >> 3;
                        eight_rows = page < 0 ? 2 * plane_groups // outside: zeros
                                              : (value ? plane_groups : 0) +
                                                    ((page << a.cache.page_shift) + (position & (a.cache.page_size() - 1)) >> 3);
                    }
                }
                else
                {
                    low_rows = Work::key_row(a, g, tile, first_row + lane);
                    high_rows = Work::key_row(a, g, tile, first_row + 32 + lane);
                }
                wait(tail.empty[slot], round + 1);
                ok = __all_sync(0xffffffffu, ok); // the warp goes on or leaves together
                if (!ok)
                    break;
                if (boxed)
                {
                    if (lane == 0)
                        bar_expect_tx(bar, L::operand_bytes / 2);
                    __syncwarp();
                    if (lane < boxes)
                        tma_5d(base + (first_row + lane * box_rows >> 3) * L::group_bytes, &map, 0, 0, 0, g.head, eight_rows, bar);
                    announce(false);
                }
                else
                {
                    const unsigned char* from = plane + (value ? a.cache.plane_bytes : 0);
                    const int chunk = lane % L::chunks;
#pragma unroll 8
                    for (int i = 0; i < PRODUCER_ROWS / rows_at_once; ++i)
                    {
                        const int row = i * rows_at_once + lane / L::chunks;
                        const long long offset =
                            __shfl_sync(0xffffffffu, i * rows_at_once < 32 ? low_rows : high_rows, row & 31);
                        copy_16(base + L::place(first_row + row, chunk),
                                from + (offset >= 0 ? offset + 16 * chunk : 0), offset >= 0 ? 16u : 0u);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    announce(true);
                    copied = slot;
                    copied_draft = Work::is_last(g, tile) && value ? g.e.length - g.e.last_base : -1;
                    copied_nodes = g.e.nodes;
                    copied_segment = segment;
                }
                if (++slot == L::SLOTS)
                {
                    slot = 0;
                    ++round;
                }
            }
            announce(false);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!ok) // this warp's TMA boxes land before the CTA ends
        {
            volatile int never = 0;
            const int used = round * L::SLOTS + slot; // operands issued; every earlier use of a slot was waited for
            for (int n = used > L::SLOTS ? used - L::SLOTS : 0; n < used; ++n)
                bar_wait(smem_u32(&tail.full[n % L::SLOTS]), static_cast<uint32_t>(n / L::SLOTS & 1), &never);
        }
    }
    else if (warp == QUERY_WARP)
    {
        // -------------------------------------------------------------- queries --
        // A negative scale turns the query's signs and a zero one clears it (to NaN where it is not
        // finite, as the product with zero is), so that the softmax's factor is positive: the largest
        // product is the largest score.
        const bool zero = a.scale_log2 == 0.0f;
        const auto turned = [&](uint32_t v) { return zero ? nonfinite_mask<T>(v) : v ^ 0x80008000u; };
        constexpr int rows_at_once = 32 / L::chunks;
        const int chunk = lane % L::chunks;
        for (int segment = 0; ok && cursor.next(a, g); ++segment)
        {
            const bool has_draft = g.tile_end == g.e.tiles;
            if (has_draft)
                ancestor_masks(a.parents + static_cast<long long>(g.list_entry) * a.max_nodes, g.e.nodes,
                               tail.masks[segment % 3], a.error_word, lane);
            wait(tail.query_free, segment + 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            const auto place = [&](int row) // of the item
            {
                return (chunk >> 3) * L::panel_bytes + (row >> 7) * L::operand_bytes + (row & 127) * 128 +
                       (((chunk & 7) ^ (row & 7)) << 4);
            };
            // A lane finds the place of one row in 32; the copies take it by shuffle.
            const std::uint16_t* from = a.query + g.list_entry * a.query_batch + 8 * chunk;
            for (int block = 0; block < L::ROWS; block += 32)
            {
                const int mine = g.first_row + block + lane, node = mine / a.group;
                const long long offset = node * a.query_node + (g.head * a.group + mine - node * a.group) * a.query_head;
                if (g.first_row + block >= g.rows) // nothing but zeros from here on
                {
                    for (int row = block + lane / L::chunks; row < L::ROWS; row += rows_at_once)
                        *reinterpret_cast<uint4*>(smem + place(row)) = make_uint4(0, 0, 0, 0);
                    break;
                }
#pragma unroll
                for (int i = 0; i < 32; i += rows_at_once)
                {
                    const int in_block = i + lane / L::chunks;
                    const bool live = g.first_row + block + in_block < g.rows;
                    const long long at = __shfl_sync(0xffffffffu, offset, in_block);
                    copy_16(smem_u32(smem) + place(block + in_block), live ? from + at : a.query, live ? 16u : 0u);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (a.scale_log2 <= 0.0f)
                for (int row = lane / L::chunks; row < L::ROWS; row += rows_at_once)
                {
                    auto* at = reinterpret_cast<uint4*>(smem + place(row));
                    const uint4 v = *at;
                    *at = make_uint4(turned(v.x), turned(v.y), turned(v.z), turned(v.w));
                }
            fence_async_proxy();
            __syncwarp();
            if (lane == 0)
                bar_arrive(smem_u32(&tail.query));
        }
    }
    else if (warp == MMA_WARP)
    {
        // ------------------------------------------------------------------ MMA --
        constexpr uint32_t score_idesc = instruction<T>(KEYS, false), value_idesc = instruction<T>(D, true);
        const bool leader = elect_one();
        const uint32_t tm = static_cast<uint32_t>(uniform(static_cast<int>(tmem)));
        const uint32_t query = smem_u32(smem), ring = query + L::ring_offset;
        int slot = 0, round = 0;
        Both<int> made{0, 0}; // products issued
        bool any = false;
        const auto wait_all = [&](uint64_t& bar, int phase)
        {
            wait(bar, phase);
            ok = __all_sync(0xffffffffu, ok);
            return ok;
        };
        const auto take = [&]() -> int // the next operand's slot, once it has landed
        {
            const int s = slot;
            wait_all(tail.full[s], round);
            if (++slot == L::SLOTS)
            {
                slot = 0;
                ++round;
            }
            return s;
        };
        const auto score = [&](int group, int s)
        {
            if (!ok)
                return;
            const uint64_t q = sw128_desc(query + (TWO ? group * L::operand_bytes : 0));
            const uint64_t k = key_desc(ring + s * L::operand_bytes, L::group_bytes);
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
            {
                constexpr int unit = 16; // of a descriptor's address
                mma_shared(leader, tm + group * KEYS, q + ((kk >> 2) * L::panel_bytes + (kk & 3) * 32) / unit,
                           k + ((kk >> 2) * 1024 + (kk & 3) * 32) / unit, score_idesc, kk != 0);
            }
            commit_if(leader, smem_u32(&tail.scores[group]));
            any = true;
        };
        const auto product = [&](int group, int s, bool accumulate)
        {
            if (!ok || !wait_all(tail.weights[group], made(group)))
                return;
            const uint64_t v = value_desc(ring + s * L::operand_bytes, L::group_bytes);
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < KEYS / 16; ++kk)
                mma_tmem(leader, tm + OUTPUT_COLUMN + group * 128, tm + group * KEYS + 8 * kk, v + kk * 2 * L::group_bytes / 16,
                         value_idesc, accumulate || kk != 0);
            commit_if(leader, smem_u32(&tail.products[group]));
            made.add(group, 1);
        };
        // P lies over S: the next scores of a group wait for its product.
        const auto after_product = [&](int group) { wait_all(tail.products[group], made(group) - 1); };
        const auto free_slot = [&](int s)
        {
            if (ok)
                commit_if(leader, smem_u32(&tail.empty[s]));
        };
        const auto free_query = [&]
        {
            if (ok)
                commit_if(leader, smem_u32(&tail.query_free));
        };
        for (int segment = 0; ok && uniform(cursor.next(a, g)); ++segment)
        {
            const int tiles = uniform(g.tile_end - g.tile_begin);
            wait_all(tail.query, segment);
            if (segment) // the softmax threads have read the last segment's P and O
                wait_all(tail.done, segment - 1);
            if constexpr (TWO)
            {
                int k = take();
                score(0, k);
                score(1, k);
                free_slot(k);
                if (tiles == 1)
                    free_query();
                for (int j = 0; j < tiles && ok; ++j)
                {
                    const int v = take();
                    const bool more = j + 1 < tiles;
                    product(0, v, j > 0);
                    if (more)
                    {
                        k = take();
                        after_product(0);
                        score(0, k);
                    }
                    product(1, v, j > 0);
                    free_slot(v);
                    if (more)
                    {
                        after_product(1);
                        score(1, k);
                        free_slot(k);
                        if (j + 2 == tiles)
                            free_query();
                    }
                }
            }
            else
            {
                for (int j = 0; j < 2 && j < tiles; ++j)
                {
                    const int k = take();
                    score(j, k);
                    free_slot(k);
                }
                if (tiles <= 2)
                    free_query();
                for (int j = 0; j < tiles && ok; ++j)
                {
                    const int v = take();
                    product(j & 1, v, j > 1);
                    free_slot(v);
                    if (j + 2 < tiles)
                    {
                        const int k = take();
                        after_product(j & 1);
                        score(j & 1, k);
                        free_slot(k);
                        if (j + 3 == tiles)
                            free_query();
                    }
                }
            }
        }
        if (any)
        {
            commit_if(leader, smem_u32(&tail.drain));
            volatile int never = 0;
            bar_wait(smem_u32(&tail.drain), 0, &never);
        }
    }
    else
    {
        // -------------------------------------------------------------- softmax --
        const int group = warp >> 2, row = t & (GROUP_THREADS - 1);
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t my_scores = lanes + group * KEYS, my_output = lanes + OUTPUT_COLUMN + group * 128;
        const float scale = a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2); // the query has its sign
        int scores_seen = 0;
        Both<int> products_seen{0, 0};
        for (int segment = 0; cursor.next(a, g); ++segment)
        {
            const int tiles = g.tile_end - g.tile_begin;
            const bool has_draft = g.tile_end == g.e.tiles;
            const int item_row = TWO ? t : row; // this thread's row of the item
            const bool live = g.first_row + item_row < g.rows;
            const int node = live ? (g.first_row + item_row) / a.group : 0;
            const int query_head = g.head * a.group + (g.first_row + item_row - node * a.group);
            wait(tail.query, segment); // the masks are there
            const unsigned long long sees = has_draft && live ? tail.masks[segment % 3][node] : 0ull;
            bar_arrive(smem_u32(&tail.query_free)); // the masks are read; the MMA warp adds that the rows are

            // A warp without a live row has nothing to compute: whatever its lanes of TMEM hold stays there.
            const bool busy = __any_sync(0xffffffffu, live);
            // Scores above `threshold` move the reference; -infinity: every tile takes that way.
            float reference = -INFINITY, threshold = -INFINITY, sum = 0.0f;
            for (int j = TWO ? 0 : group; j < tiles; j += TWO ? 1 : 2)
            {
                const int tile = g.tile_begin + j;
                const bool masked = Work::is_masked(g, tile);
                wait(tail.scores[group], scores_seen++);
                __syncwarp();
                tc_fence_after();
                if (busy)
                {
                    Pair part = make_pair(0.0f, 0.0f);
#pragma unroll 1
                    for (int c = 0; c < KEYS / 32; ++c)
                    {
                        uint32_t s[32];
                        tmem_load32(my_scores + 32 * c, s);
                        if (masked)
                        {
                            const uint32_t bits = Work::visible(g, tile, c, sees);
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                s[k] = bits >> k & 1u ? s[k] : 0xff800000u; // -infinity
                        }
                        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int k = 0; k < 32; k += 2)
                            best[k >> 1 & 3] = max3(best[k >> 1 & 3], __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
                        const float highest = max3(best[0], best[1], fmaxf(best[2], best[3]));
                        const float top = highest == -INFINITY ? -INFINITY : highest * scale;
                        float factor = scale;
                        if (__any_sync(0xffffffffu, top > threshold))
                        {
                            // From 2^23 on (and below infinity) a product's rounding moves a weight by powers of
                            // two: the scores are then rounded like the maximum that the reference comes from.
                            const bool coarse = fabsf(top) >= 0x1p23f && fabsf(top) < INFINITY;
                            if (__any_sync(0xffffffffu, coarse))
                            {
                                const float early = coarse ? scale : 1.0f;
                                factor = coarse ? 1.0f : scale;
#pragma unroll
                                for (int k = 0; k < 32; ++k)
                                    s[k] = __float_as_uint(__uint_as_float(s[k]) * early);
                            }
                            const float raised = fmaxf(reference, __fadd_ru(ceilf(top), -PLACE));
                            const float shrink = reference == -INFINITY ? 0.0f : power_of_two(reference - raised);
                            reference = raised;
                            threshold = fabsf(raised) >= 0x1p22f && fabsf(raised) < INFINITY ? -INFINITY : raised + LIMIT;
                            sum *= shrink;
                            part = mul_pair(part, make_pair(shrink, shrink));
                            // P of this tile's earlier scores, then the output; its last product is
                            // complete, these scores were issued after it.
                            tmem_wait_stores();
#pragma unroll 1
                            for (int b = 0; b < c; ++b)
                            {
                                uint32_t w[16];
                                tmem_load16(my_scores + 16 * b, w);
                                tmem_wait16(w);
#pragma unroll
                                for (int k = 0; k < 16; ++k)
                                    w[k] = Half2<T>::pack(Half2<T>::value(static_cast<std::uint16_t>(w[k])) * shrink,
                                                          Half2<T>::value(static_cast<std::uint16_t>(w[k] >> 16)) * shrink);
                                tmem_store16(my_scores + 16 * b, w);
                            }
#pragma unroll 1
                            for (int b = 0; b < D / 16 && (TWO ? j > 0 : j > 1); ++b)
                            {
                                uint32_t w[16];
                                tmem_load16(my_output + 16 * b, w);
                                tmem_wait16(w);
#pragma unroll
                                for (int k = 0; k < 16; ++k)
                                    w[k] = __float_as_uint(__uint_as_float(w[k]) * shrink);
                                tmem_store16(my_output + 16 * b, w);
                            }
                        }
                        const float shift = reference == -INFINITY ? 0.0f : -reference;
                        uint32_t p[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2)
                        {
                            float x, y;
                            split(fma_pair(make_pair(__uint_as_float(s[k]), __uint_as_float(s[k + 1])),
                                           make_pair(factor, factor), make_pair(shift, shift)),
                                  x, y);
                            x = power_of_two(x);
                            y = power_of_two(y);
                            part = add_pair(part, make_pair(x, y));
                            p[k / 2] = Half2<T>::pack(x, y);
                        }
                        tmem_store16(my_scores + 16 * c, p); // over scores that have been read
                    }
                    float even, odd;
                    split(part, even, odd);
                    sum += even + odd;
                    tmem_wait_stores();
                }
                tc_fence_before();
                bar_arrive(smem_u32(&tail.weights[group]));
            }
            // ------------------------------------------------------- epilogue --
            const Both<int> made{TWO ? tiles : (tiles + 1) / 2, TWO ? tiles : tiles / 2};
            if (made(group))
                wait(tail.products[group], products_seen(group) + made(group) - 1);
            sum = ok ? sum : NAN;
            Both<float> part{1.0f, 1.0f}; // factors of the groups' outputs
            if constexpr (!TWO)
            {
                // The groups exchange their statistics in TMEM, in columns of S that P leaves free.
                tmem_store2(my_scores + KEYS / 2, __float_as_uint(reference), __float_as_uint(sum));
                tmem_wait_stores();
                tc_fence_before();
                softmax_sync();
                // The other group has seen its product complete; this makes it visible here.
                if (made(1 - group))
                    wait(tail.products[1 - group], products_seen(1 - group) + made(1 - group) - 1);
                __syncwarp();
                tc_fence_after();
                const float m0 = __uint_as_float(tmem_load1(lanes + KEYS / 2)), m1 = __uint_as_float(tmem_load1(lanes + KEYS + KEYS / 2));
                const float sum0 = __uint_as_float(tmem_load1(lanes + KEYS / 2 + 1)), sum1 = __uint_as_float(tmem_load1(lanes + KEYS + KEYS / 2 + 1));
                reference = fmaxf(m0, m1);
                part.first = m0 == -INFINITY ? 0.0f : power_of_two(m0 - reference);
                part.second = m1 == -INFINITY ? 0.0f : power_of_two(m1 - reference);
                sum = ok ? sum0 * part.first + sum1 * part.second : NAN;
            }
            __syncwarp();
            tc_fence_after();
            products_seen.first += made.first;
            products_seen.second += made.second;
            // One lane's answer for the warp, whose threads load TMEM together for each of the nodes.
            const unsigned long long tainted =
                __shfl_sync(0xffffffffu, has_draft ? tail.tainted[segment % TAINT_SLOTS] : 0ull, 0);
            const int draft_group = TWO ? group : (tiles - 1) & 1; // whose P is the drafted tile's
            const bool whole = g.tile_begin == 0 && has_draft;
            // A piece that begins its item goes to the CTA's second place, any other to its first.
            float* piece = pieces + (2ll * cta + (g.tile_begin == 0)) * tree_piece_floats(L::ROWS, D) +
                           item_row * (D + TREE_PIECE_HEAD);
            std::uint16_t* out = a.out + g.list_entry * a.out_batch + node * a.out_node + query_head * a.out_head;
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum; // a row that sees nothing gives zeros
            constexpr int columns = TWO ? D : D / 2;                  // of this thread
            const int first_column = TWO ? 0 : group * columns;
            constexpr int step = 16;
#pragma unroll 1
            for (int c = 0; busy && c < columns; c += step)
            {
                const int column = first_column + c;
                uint32_t o[step];
                if constexpr (TWO)
                {
                    tmem_load16(my_output + column, o);
                    tmem_wait16(o);
                }
                else
                {
                    uint32_t other[step];
                    tmem_load16(lanes + OUTPUT_COLUMN + column, o); // the first group always has a tile
                    if (made.second)
                        tmem_load16(lanes + OUTPUT_COLUMN + 128 + column, other);
                    tmem_wait16(o);
                    if (made.second)
                        tmem_wait16(other);
#pragma unroll
                    for (int k = 0; k < step; ++k)
                    {
                        float x = __uint_as_float(o[k]) * part.first;
                        if (made.second)
                            x = fmaf(__uint_as_float(other[k]), part.second, x);
                        o[k] = __float_as_uint(x);
                    }
                }
                for (unsigned long long rest = tainted; rest; rest &= rest - 1)
                {
                    const int key = __ffsll(static_cast<long long>(rest)) - 1;
                    const int in_tile = g.e.length - g.e.last_base + key;
                    const uint32_t pair = tmem_load1(lanes + draft_group * KEYS + in_tile / 2);
                    const long long offset = sees >> key & 1ull ? Work::key_row(a, g, g.e.tiles - 1, in_tile) : -1;
                    if (offset >= 0)
                    {
                        const float weight = Half2<T>::value(static_cast<std::uint16_t>(in_tile & 1 ? pair >> 16 : pair)) *
                                             part(TWO ? 0 : draft_group);
                        const auto* values = reinterpret_cast<const std::uint16_t*>(plane + a.cache.plane_bytes + offset) + column;
#pragma unroll
                        for (int k = 0; k < step; ++k)
                            if (nonfinite_mask<T>(values[k]) & 0xffffu)
                                o[k] = __float_as_uint(fmaf(weight, Half2<T>::value(values[k]), __uint_as_float(o[k])));
                    }
                    __syncwarp();
                }
                if (live && whole)
                {
#pragma unroll
                    for (int k = 0; k < step; k += 8)
                    {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            w[j] = Half2<T>::pack(__uint_as_float(o[k + 2 * j]) * inverse,
                                                  __uint_as_float(o[k + 2 * j + 1]) * inverse);
                        *reinterpret_cast<uint4*>(out + column + k) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                else if (live)
                {
#pragma unroll
                    for (int k = 0; k < step; k += 4)
                        *reinterpret_cast<uint4*>(piece + TREE_PIECE_HEAD + column + k) =
                            make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
                __syncwarp();
            }
            if (live && first_column == 0)
            {
                if (!whole)
                {
                    piece[0] = reference;
                    piece[1] = sum;
                }
                else if (a.lse)
                {
                    a.lse[(static_cast<long long>(g.list_entry) * a.max_nodes + node) * a.heads * a.group + query_head] =
                        sum == 0.0f ? -INFINITY : (reference + log2f(sum)) * 0.6931471805599453f;
                }
            }
            if (g.tile_begin == 0 && !whole && t == 0)
                shared_items[cta] = TreeShared{g.list_entry, g.head, g.first_row,
                                               Work::owner(start.units, g.item_start + g.e.tiles - 1, start.ctas) - cta + 1,
                                               g.e.nodes};
            // The groups' statistics and the tainted nodes have been read.  Whether to wait must not depend on
            // the nodes: after a wait that gave up, the threads may have read them at different times.
            if (!TWO || has_draft)
                softmax_sync();
            if (t == 0 && has_draft)
                tail.tainted[segment % TAINT_SLOTS] = 0;
            tc_fence_before();
            bar_arrive(smem_u32(&tail.done));
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLUMNS));
}

// The layer's two planes as [8 rows][head][64 columns][row of 8][column], in
// boxes of `rows` whole rows of one head.  A box per 64 columns is twice as many:
// 64 x 16 nodes over pages of 16 took 159 us with them, 154 us with these.
bool make_map(CUtensorMap* map, const TreeArgs& a, int rows)
{
    const auto fn = encode_fn();
    const CacheView& c = a.cache;
    const cuuint64_t plane_rows = static_cast<cuuint64_t>(c.pages) << c.page_shift;
    if (!fn || plane_rows >= 0x7fffffffull)
        return false;
    const cuuint64_t panels = static_cast<cuuint64_t>(a.head_dim / 64);
    const cuuint64_t dims[5] = {64, 8, panels, static_cast<cuuint64_t>(a.heads), 2 * plane_rows / 8};
    const cuuint64_t strides[4] = {static_cast<cuuint64_t>(c.row_bytes), 128, static_cast<cuuint64_t>(2 * a.head_dim),
                                   8 * static_cast<cuuint64_t>(c.row_bytes)};
    const cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(panels), 1, static_cast<cuuint32_t>(rows / 8)};
    const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, c.pool + 2ll * a.layer * c.plane_bytes, dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, bool TWO>
void launch(const TreeArgs& a, int ctas, float* pieces, TreeShared* shared_items, cudaStream_t stream)
{
    using L = Tiles<D, TWO>;
    static std::once_flag once[64];
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64)
        std::call_once(once[device],
                       []
                       {
                           cudaFuncSetAttribute(tree_attention_tc_kernel<T, D, TWO>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem);
                       });
    // Boxes of a page, or of the 64 rows that a producer warp fills.
    CUtensorMap map{};
    int box_rows = a.cache.page_size() < PRODUCER_ROWS ? a.cache.page_size() : PRODUCER_ROWS;
    if (box_rows < 8 || !make_map(&map, a, box_rows))
        box_rows = 0;
    launch_pdl(tree_attention_tc_kernel<T, D, TWO>, dim3(ctas), dim3(THREADS), L::smem, stream, map, a, box_rows,
               pieces, shared_items);
    note_launch();
}

template <class T>
void launch_shape(const TreeArgs& a, int ctas, float* pieces, TreeShared* shared_items, cudaStream_t stream)
{
    const bool two = tree_attention_tc_rows(a.max_nodes * a.group) == 256;
    if (a.head_dim == 64)
        two ? launch<T, 64, true>(a, ctas, pieces, shared_items, stream) : launch<T, 64, false>(a, ctas, pieces, shared_items, stream);
    else
        two ? launch<T, 128, true>(a, ctas, pieces, shared_items, stream) : launch<T, 128, false>(a, ctas, pieces, shared_items, stream);
}
} // namespace

int tree_attention_tc_rows(int rows)
{
    return rows > 128 ? 256 : 128;
}

cudaError_t tree_attention_tc(const TreeArgs& a, ValueType type, int ctas, float* pieces, TreeShared* shared_items,
                              cudaStream_t stream)
{
    if (type == ValueType::bf16)
        launch_shape<__nv_bfloat16>(a, ctas, pieces, shared_items, stream);
    else
        launch_shape<__half>(a, ctas, pieces, shared_items, stream);
    return cudaGetLastError();
}
} // namespace tsacb::dev
