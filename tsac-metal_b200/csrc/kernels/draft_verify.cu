// Verification of drafted tokens against the target's probabilities from given
// random numbers.
//
// The walk starts at node 0 and tries the children of the node it stands on in
// ascending order.  With w the target's distribution there, child c with token
// x and coin u is accepted when
//   without a draft distribution:  u * (1 - sum of the rejected siblings' p) < p(x)
//   with the draft's q:            u * q(x) < w(x)
// and a rejection leaves w = p without the rejected tokens, or
// w = max(w - q, 0) / Z with Z its sum.  Where no child is accepted the next
// token is the first whose cumulative weight exceeds draw * total.  Accepting
// x with probability min(1, w / q) and else drawing from the normalised excess
// of w over q leaves the target's distribution, whatever the draft's.
//
// B200 mapping.  Only the last node's rows are read whole, so a call is bound
// by one row of p (and one of q) per sequence: latency for small vocabularies,
// HBM for large ones.  The gathers p(x), q(x) of every node are loaded at once
// before the walk.  Each warp then walks for itself: its lanes hold two nodes
// each, a ballot finds the children of the current node, and nothing waits for
// another warp.  A whole-row pass is spread over a cluster of CTAs: each warp
// owns a contiguous range of the row and sums it with 16-byte loads, the
// ranges' sums are exchanged through distributed shared memory (one cluster
// barrier per pass), and the CTA that owns the crossing range reads it once
// more, from cache, to find the token.
//
// All sums and the excess are in 64 bits: the token is an integer that one
// rounding near a border would change, and 32-bit partial sums over 10^5
// probabilities are off by up to 10^5 * 2^-24.  They are not what bounds a
// call: with 32-bit sums 160 rows of 131,072 fp32 values took 27.7 us in place
// of 28.2, 148 rows, one per SM, 24.9 in place of 25.1 (48 rows of 50,001 bf16
// values with a draft, short as they are, 11.4 in place of 12.8).
#include "kernels/draft_verify.cuh"
#include "kernels/error_bits.hpp"
#include "kernels/launch_count.hpp"
#include "kernels/pdl.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace tsacb::dev
{
namespace
{
namespace cg = cooperative_groups;

constexpr int MAX_RANGES = 128; // warps of a cluster, at most: 8 CTAs of 512 threads

__device__ __forceinline__ double to_double(float v) { return v; }
__device__ __forceinline__ double to_double(__half v) { return __half2float(v); }
__device__ __forceinline__ double to_double(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T> struct alignas(16) Vector
{
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    T v[N];
};

// The same 16 bytes as words.
struct Words
{
    std::uint32_t w[4];
    __device__ __forceinline__ Words() : w{0, 0, 0, 0} {}
    __device__ __forceinline__ explicit Words(const uint4& v) : w{v.x, v.y, v.z, v.w} {}
    template <class T> __device__ __forceinline__ double value(int j) const
    {
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(w[j]);
        else if constexpr (std::is_same_v<T, __half>)
            return to_double(__ushort_as_half(static_cast<unsigned short>(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu)));
        else // a bf16 value is the upper half of a 32-bit one
            return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    }
};

struct Shared
{
    int parents[DRAFT_MAX_NODES], tokens[DRAFT_MAX_NODES], path[DRAFT_MAX_NODES];
    float coins[DRAFT_MAX_NODES];
    double p[DRAFT_MAX_NODES], q[DRAFT_MAX_NODES];
    double scale[DRAFT_MAX_NODES]; // 1 / Z of each round of rejections
    double sums[2][MAX_RANGES];    // sums of the warps' ranges, by pass parity
    double scan[16];               // of a CTA's warps
    int first;
};

// The weights at the current node.  With a draft: the target's row after
// `rounds` applications of max(w / Z - q, 0); else: without the tokens of the
// rejected nodes, of which a warp keeps those that lie in its range.
template <class T, bool DRAFT> struct Weights
{
    const T* p;
    const T* q;
    int rounds;
    const double* scale;
    unsigned long long rejected; // nodes
    const int* tokens;           // of the nodes

    __device__ __forceinline__ void keep(int first, int last)
    {
        if constexpr (!DRAFT)
        {
            const int lane = threadIdx.x & 31;
            const auto inside = [&](int n)
            { return (rejected >> n & 1ull) && tokens[n] >= first && tokens[n] < last; };
            const unsigned low = __ballot_sync(0xffffffffu, inside(lane)), high = __ballot_sync(0xffffffffu, inside(lane + 32));
            rejected = static_cast<unsigned long long>(high) << 32 | low;
        }
    }
    __device__ __forceinline__ double excess(double w, double q_value) const
    {
        if (rounds > 0)
            w = above(w - q_value);
#pragma unroll 1
        for (int i = 1; i < rounds; ++i)
            w = above(w * scale[i] - q_value);
        return w;
    }
    __device__ __forceinline__ double at(int token, double p_value, double q_value) const
    {
        if constexpr (DRAFT)
        {
            return excess(p_value, q_value);
        }
        else
        {
#pragma unroll 1
            for (unsigned long long rest = rejected; rest; rest &= rest - 1)
                p_value = tokens[__ffsll(static_cast<long long>(rest)) - 1] == token ? 0.0 : p_value;
            return p_value;
        }
    }
    static __device__ __forceinline__ double above(double d)
    {
        return d > 0.0 ? d : (d <= 0.0 ? 0.0 : d); // keeps a NaN
    }
};

// A row in 16-byte blocks: block b holds tokens [b N - skew, b N - skew + N),
// with the row's first element `skew` elements into block 0.  Rows of p and q
// with different skews are read element by element.
template <class T, bool DRAFT> struct Row
{
    static constexpr int N = Vector<T>::N;
    int skew, blocks, vocab;
    bool vectors;

    __device__ __forceinline__ Row(const T* p, const T* q, int vocab_) : vocab(vocab_)
    {
        const auto skew_of = [](const T* x) { return static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T) % N); };
        skew = skew_of(p);
        vectors = !DRAFT || skew_of(q) == skew;
        blocks = (vocab + skew + N - 1) / N;
    }
    __device__ __forceinline__ int first_token(int block) const { return block * N - skew; }
    // Blocks [whole_begin, whole_end) lie in the row and may be read at once.
    __device__ __forceinline__ int whole_begin() const { return vectors ? (skew ? 1 : 0) : blocks; }
    __device__ __forceinline__ int whole_end() const { return vectors ? (vocab + skew) / N : blocks; }
    __device__ __forceinline__ void load(const T* x, int block, Vector<T>& out) const
    {
        const int token = block * N - skew;
        if (vectors && token >= 0 && token + N <= vocab)
        {
            *reinterpret_cast<uint4*>(&out) = *reinterpret_cast<const uint4*>(x + token);
            return;
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
            out.v[k] = token + k >= 0 && token + k < vocab ? x[token + k] : T(0.0f);
    }
};

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// The sum of a block's weights, token by token compared with the rejected ones.
template <class T, bool DRAFT>
__device__ __forceinline__ double block_weight(const Weights<T, DRAFT>& w, const Row<T, DRAFT>& row, int block,
                                               const Vector<T>& p, const Vector<T>& q)
{
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < Row<T, DRAFT>::N; ++k)
        sum += w.at(row.first_token(block) + k, to_double(p.v[k]), DRAFT ? to_double(q.v[k]) : 0.0);
    return sum;
}

// Running sums of the warps' ranges, by each warp for itself: lane l gets those
// of ranges l, l + 32, ..., by the same additions everywhere.
template <int RANGES> struct RangeSums
{
    static constexpr int EACH = (RANGES + 31) / 32;
    double own[EACH], until[EACH], total;

    __device__ __forceinline__ explicit RangeSums(const double* sums)
    {
        const int lane = threadIdx.x & 31;
        double before = 0.0;
#pragma unroll
        for (int k = 0; k < EACH; ++k)
        {
            own[k] = 32 * k + lane < RANGES ? sums[32 * k + lane] : 0.0;
            double v = own[k];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1)
            {
                const double up = __shfl_up_sync(0xffffffffu, v, d);
                v = lane >= d ? v + up : v;
            }
            until[k] = before + v;
            before = __shfl_sync(0xffffffffu, until[k], 31);
        }
        total = before;
    }
};

template <int CLUSTER> __device__ __forceinline__ int cluster_rank()
{
    return CLUSTER > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
}

// Sums the weights of the whole row; every thread of the cluster returns the
// total, and sums holds each warp range's sum.
template <class T, bool DRAFT, int CLUSTER, int THREADS>
__device__ double whole_row(Weights<T, DRAFT> w, const Row<T, DRAFT>& row, int per, double* sums)
{
    constexpr int WARPS = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int mine = cluster_rank<CLUSTER>() * WARPS + warp;
    const int end = min(row.blocks, (mine + 1) * per);
    w.keep(row.first_token(mine * per), row.first_token(end));
    constexpr int UNROLL = DRAFT ? 4 : 8; // 16-byte loads in flight per row and lane
    constexpr int N = Row<T, DRAFT>::N;
    double sum = 0.0;
    // Blocks that are not whole, and all of rows that cannot be read in vectors.
    const int low = min(end, max(mine * per, row.whole_begin())), high = max(low, min(end, row.whole_end()));
    for (int b = mine * per + lane; b < end; b += 32)
    {
        if (b >= low && b < high)
        {
            b += (high - b + 31) / 32 * 32 - 32; // to the first of this lane's blocks from `high` on
            continue;
        }
        Vector<T> p, q;
        row.load(w.p, b, p);
        if constexpr (DRAFT)
            row.load(w.q, b, q);
        sum += block_weight<T, DRAFT>(w, row, b, p, q);
    }
    // Whole blocks, with nothing in the loop but loads, conversions and sums by a tree (a
    // chain of 64-bit additions would wait for each).
    double parts[4] = {};
    bool undefined = false;
    const auto* from_p = reinterpret_cast<const uint4*>(w.p - row.skew);
    const auto* from_q = reinterpret_cast<const uint4*>(DRAFT ? w.q - row.skew : w.p);
    const bool subtract = w.rounds > 0;
    for (int first = low; first < high; first += 32 * UNROLL)
    {
        Words p[UNROLL], q[DRAFT ? UNROLL : 1];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
        {
            const int b = first + lane + 32 * k;
            p[k] = b < high ? Words(from_p[b]) : Words();
            if constexpr (DRAFT)
                q[k] = b < high && subtract ? Words(from_q[b]) : Words();
        }
        if constexpr (!DRAFT)
        {
            // A rejected token of these blocks is cleared where it was loaded.
            for (unsigned long long rest = w.rejected; rest; rest &= rest - 1)
            {
                const int token = w.tokens[__ffsll(static_cast<long long>(rest)) - 1] + row.skew;
                const int away = token / N - first, byte = token % N * static_cast<int>(sizeof(T));
                if (away >= 0 && away < 32 * UNROLL && (away & 31) == lane)
                {
                    const std::uint32_t stays = sizeof(T) == 4 ? 0u : (byte & 2 ? 0x0000ffffu : 0xffff0000u);
#pragma unroll
                    for (int k = 0; k < UNROLL; ++k)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            p[k].w[j] &= k == away / 32 && j == byte / 4 ? stays : ~0u;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
        {
            double sums[N];
#pragma unroll
            for (int j = 0; j < N; ++j)
            {
                sums[j] = p[k].template value<T>(j);
                if constexpr (DRAFT)
                {
                    sums[j] -= q[k].template value<T>(j);
                    undefined |= sums[j] != sums[j];
                    sums[j] = sums[j] > 0.0 ? sums[j] : 0.0;
                }
            }
            if (DRAFT && w.rounds > 1)
            {
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll 1
                    for (int i = 1; i < w.rounds; ++i)
                        sums[j] = Weights<T, DRAFT>::above(sums[j] * w.scale[i] - q[DRAFT ? k : 0].template value<T>(j));
            }
#pragma unroll
            for (int n = N / 2; n; n /= 2)
#pragma unroll
                for (int j = 0; j < n; ++j)
                    sums[j] += sums[j + n];
            parts[k & 3] += sums[0];
        }
    }
    sum += (parts[0] + parts[1]) + (parts[2] + parts[3]);
    if (undefined)
        sum = NAN;
    sum = warp_sum(sum);
    if constexpr (CLUSTER > 1)
    {
        auto cluster = cg::this_cluster();
        if (lane < CLUSTER)
            cluster.map_shared_rank(sums, lane)[mine] = sum;
        cluster.sync();
    }
    else
    {
        if (lane == 0)
            sums[mine] = sum;
        __syncthreads();
    }
    return RangeSums<CLUSTER * WARPS>(sums).total;
}

// The first token whose cumulative weight exceeds `threshold`, by the CTA that
// owns its range; the last token of positive weight if rounding leaves none.
template <class T, bool DRAFT, int CLUSTER, int THREADS>
__device__ void pick(Weights<T, DRAFT> w, const Row<T, DRAFT>& row, int per, const double* sums, double threshold,
                     Shared& sh, int* token)
{
    constexpr int WARPS = THREADS / 32;
    // The last range with weight that starts at or below the threshold.
    const RangeSums<CLUSTER * WARPS> scan(sums);
    int range = -1;
    double before = 0.0;
#pragma unroll
    for (int k = 0; k < RangeSums<CLUSTER * WARPS>::EACH; ++k)
    {
        const double start = scan.until[k] - scan.own[k];
        const unsigned found = __ballot_sync(0xffffffffu, scan.own[k] > 0.0 && !(start > threshold));
        const int last = 31 - __clz(found);
        const double there = __shfl_sync(0xffffffffu, start, found ? last : 0);
        range = found ? 32 * k + last : range;
        before = found ? there : before;
    }
    if (range < 0 || range / WARPS != cluster_rank<CLUSTER>())
        return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int begin = range * per, end = min(row.blocks, begin + per);
    w.keep(row.first_token(begin), row.first_token(end));
    const int each = (per + THREADS - 1) / THREADS;
    const int b0 = min(end, begin + static_cast<int>(threadIdx.x) * each), b1 = min(end, b0 + each);
    double sum = 0.0;
    for (int b = b0; b < b1; ++b)
    {
        Vector<T> p, q;
        row.load(w.p, b, p);
        if constexpr (DRAFT)
            row.load(w.q, b, q);
        sum += block_weight<T, DRAFT>(w, row, b, p, q);
    }
    double inclusive = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
    {
        const double up = __shfl_up_sync(0xffffffffu, inclusive, d);
        inclusive = lane >= d ? inclusive + up : inclusive;
    }
    double exclusive = __shfl_up_sync(0xffffffffu, inclusive, 1);
    exclusive = lane ? exclusive : 0.0;
    if (lane == 31)
        sh.scan[warp] = inclusive;
    if (threadIdx.x == 0)
        sh.first = -1;
    __syncthreads();
    for (int k = 0; k < warp; ++k)
        before += sh.scan[k];
    // The last thread with weight that starts at or below the threshold holds the crossing.
    if (sum > 0.0 && !(before + exclusive > threshold))
        atomicMax(&sh.first, static_cast<int>(threadIdx.x));
    __syncthreads();
    if (sh.first != static_cast<int>(threadIdx.x))
        return;
    double cumulative = before + exclusive;
    int found = -1;
    bool crossed = false;
    for (int b = b0; b < b1 && !crossed; ++b)
    {
        Vector<T> p, q;
        row.load(w.p, b, p);
        if constexpr (DRAFT)
            row.load(w.q, b, q);
#pragma unroll
        for (int k = 0; k < Row<T, DRAFT>::N; ++k)
        {
            const int candidate = row.first_token(b) + k;
            const double weight = w.at(candidate, to_double(p.v[k]), DRAFT ? to_double(q.v[k]) : 0.0);
            cumulative += weight;
            if (!crossed && weight > 0.0)
            {
                found = candidate;
                crossed = cumulative > threshold;
            }
        }
    }
    *token = found;
}

template <class T, bool DRAFT, int CLUSTER, int THREADS>
__global__ void __launch_bounds__(THREADS, (DRAFT ? 512 : 1024) / THREADS) draft_verify_kernel(const VerifyArgs a)
{
    if constexpr (CLUSTER > 1)
        cg::this_cluster().barrier_arrive();
    pdl_prologue();
    __shared__ Shared sh;
    constexpr int RANGES = CLUSTER * THREADS / 32;
    const int sequence = blockIdx.x / CLUSTER;
    const int t = threadIdx.x, lane = t & 31;
    const long long list = static_cast<long long>(sequence) * a.max_nodes;
    int nodes = a.nodes ? a.nodes[sequence] : a.max_nodes;
    nodes = nodes < 0 ? 0 : (nodes < a.max_nodes ? nodes : a.max_nodes);
    const T* target = static_cast<const T*>(a.target) + sequence * a.target_batch;
    const T* draft = DRAFT ? static_cast<const T*>(a.draft) + sequence * a.draft_batch : nullptr;
    const float draw = fmaxf(a.draws[sequence], 0.0f); // outside [0, 1): the first or the last token of positive weight
    if (t < DRAFT_MAX_NODES)
    {
        const bool there = t < nodes;
        const int parent = there ? a.parents[list + t] : -1, token = there ? a.tokens[list + t] : -1;
        const bool real = t > 0 && parent >= 0 && parent < t;
        const bool known = static_cast<unsigned>(token) < static_cast<unsigned>(a.vocab);
        sh.parents[t] = real ? parent : -1;
        sh.tokens[t] = token;
        sh.coins[t] = there ? a.coins[list + t] : 0.0f;
        // A token outside the vocabulary has probability 0 and is never accepted.
        sh.p[t] = real && known ? to_double(target[parent * a.target_node + token]) : 0.0;
        if constexpr (DRAFT)
            sh.q[t] = real && known ? to_double(draft[parent * a.draft_node + token]) : 0.0;
    }
    if constexpr (CLUSTER > 1)
        cg::this_cluster().barrier_wait(); // every CTA runs before its shared memory is written to
    __syncthreads();
    int accepted = 0, passes = 0;
    bool failed = false;
    if (nodes > 0)
    {
        const int parents[2] = {sh.parents[lane], sh.parents[lane + 32]};
        const auto children_of = [&](int node)
        {
            const unsigned low = __ballot_sync(0xffffffffu, parents[0] == node), high = __ballot_sync(0xffffffffu, parents[1] == node);
            return static_cast<unsigned long long>(high) << 32 | low;
        };
        int node = 0, rounds = 0;
        bool summed = false; // the last pass summed the current weights
        double total = 0.0, left = 1.0;
        unsigned long long rejected = 0;
        accepted = 1;
        if (t == 0)
            sh.path[0] = 0;
        const auto weights = [&](int n, unsigned long long without)
        {
            return Weights<T, DRAFT>{target + node * a.target_node, DRAFT ? draft + node * a.draft_node : nullptr, n,
                                     sh.scale, without, sh.tokens};
        };
        unsigned long long children = children_of(0);
        while (children && !failed)
        {
            const int n = __ffsll(static_cast<long long>(children)) - 1;
            children &= children - 1;
            double p = sh.p[n];
            bool pass;
            if constexpr (DRAFT)
            {
                p = weights(rounds, 0).excess(p, sh.q[n]);
                p = rounds ? p * sh.scale[rounds] : p;
                pass = sh.coins[n] * sh.q[n] < p;
            }
            else
            {
                for (unsigned long long rest = rejected; rest; rest &= rest - 1)
                    p = sh.tokens[__ffsll(static_cast<long long>(rest)) - 1] == sh.tokens[n] ? 0.0 : p;
                pass = sh.coins[n] * left < p;
            }
            if (pass)
            {
                if (t == 0)
                    sh.path[accepted] = n;
                ++accepted;
                node = n;
                rounds = 0;
                summed = false;
                left = 1.0;
                rejected = 0;
                children = children_of(n);
                continue;
            }
            if constexpr (DRAFT)
            {
                const Weights<T, DRAFT> w = weights(rounds + 1, 0);
                const Row<T, DRAFT> row(w.p, w.q, a.vocab);
                const double z = whole_row<T, DRAFT, CLUSTER, THREADS>(w, row, (row.blocks + RANGES - 1) / RANGES,
                                                                      sh.sums[passes & 1]);
                ++passes;
                summed = z > 0.0 && z < INFINITY;
                if (summed)
                {
                    total = z;
                    ++rounds;
                    if (t == 0)
                        sh.scale[rounds] = 1.0 / z;
                    __syncthreads();
                }
                else // no excess: the weights stay; a NaN or an infinity ends the walk
                {
                    failed = !(z == 0.0);
                }
            }
            else
            {
                rejected |= 1ull << n;
                left -= p;
            }
        }
        const auto finish = [&](unsigned long long without)
        {
            const Weights<T, DRAFT> w = weights(rounds, without);
            const Row<T, DRAFT> row(w.p, w.q, a.vocab);
            const int per = (row.blocks + RANGES - 1) / RANGES;
            if (!summed)
                total = whole_row<T, DRAFT, CLUSTER, THREADS>(w, row, per, sh.sums[passes++ & 1]);
            if (!(total > 0.0 && total < INFINITY))
                return false;
            pick<T, DRAFT, CLUSTER, THREADS>(w, row, per, sh.sums[(passes - 1) & 1], static_cast<double>(draw) * total, sh,
                                             a.token + sequence);
            return true;
        };
        if (!failed)
        {
            bool done = finish(rejected);
            if constexpr (!DRAFT)
                if (!done && rejected && total == 0.0) // nothing left beside the rejected tokens
                    done = finish(0);
            failed = !done;
        }
    }
    if (blockIdx.x % CLUSTER == 0)
    {
        __syncthreads();
        for (int n = t; n < a.max_nodes; n += THREADS)
            a.path[list + n] = n < accepted ? sh.path[n] : -1;
        if (t == 0)
        {
            a.accepted[sequence] = accepted;
            if (failed || nodes == 0)
                a.token[sequence] = -1;
            if (failed && a.error_word)
                atomicOr(a.error_word, error_nonfinite);
        }
    }
}

template <class T, bool DRAFT, int CLUSTER, int THREADS> cudaError_t launch(const VerifyArgs& a, int batch, cudaStream_t stream)
{
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(batch * CLUSTER);
    config.blockDim = dim3(THREADS);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = CLUSTER;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    cudaLaunchKernelEx(&config, draft_verify_kernel<T, DRAFT, CLUSTER, THREADS>, a);
    note_launch();
    return cudaGetLastError();
}

// CTAs for one sequence.  Small vocabularies are latency alone: one CTA of 128
// threads.  Others: CTAs of 512 threads (256 with a draft, whose pass needs
// twice the registers), two per SM; of 1, 2, 4 or 8 the number that costs
// least, where a wave of CTAs costs its start (about 6 us, in which a CTA reads
// 240 KB, or 72 KB with a draft) and its part of the rows.  Measured in us:
// 160 x 131,072 fp32, 1 CTA 24.6, 4 in three waves 71; 48 x 50,001 bf16 with a
// draft, 4 CTAs 10.3, 8 in two waves 14.4.
template <class T, bool DRAFT> cudaError_t launch_cluster(const VerifyArgs& a, int batch, cudaStream_t stream)
{
    constexpr int THREADS = DRAFT ? 256 : 512;
    constexpr long long start_bytes = DRAFT ? 72 << 10 : 240 << 10;
    if (a.vocab <= 8192)
        return launch<T, DRAFT, 1, 128>(a, batch, stream);
    int device = 0, sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess)
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    const long long row_bytes = static_cast<long long>(a.vocab) * sizeof(T) * (DRAFT ? 2 : 1);
    const auto cost = [&](int cluster)
    {
        const long long waves = (static_cast<long long>(batch) * cluster + 2 * sms - 1) / (2 * sms);
        return waves * (start_bytes + row_bytes / cluster);
    };
    int best = 1;
    for (int cluster = 2; cluster <= 8; cluster *= 2)
        best = cost(cluster) < cost(best) ? cluster : best;
    switch (best)
    {
    case 8:
        return launch<T, DRAFT, 8, THREADS>(a, batch, stream);
    case 4:
        return launch<T, DRAFT, 4, THREADS>(a, batch, stream);
    case 2:
        return launch<T, DRAFT, 2, THREADS>(a, batch, stream);
    default:
        return launch<T, DRAFT, 1, THREADS>(a, batch, stream);
    }
}

template <class T> cudaError_t launch_type(const VerifyArgs& a, int batch, cudaStream_t stream)
{
    return a.draft ? launch_cluster<T, true>(a, batch, stream) : launch_cluster<T, false>(a, batch, stream);
}
} // namespace

cudaError_t draft_verify(const VerifyArgs& a, ValueType type, int batch, cudaStream_t stream)
{
    switch (type)
    {
    case ValueType::bf16:
        return launch_type<__nv_bfloat16>(a, batch, stream);
    case ValueType::fp16:
        return launch_type<__half>(a, batch, stream);
    default:
        return launch_type<float>(a, batch, stream);
    }
}
} // namespace tsacb::dev
