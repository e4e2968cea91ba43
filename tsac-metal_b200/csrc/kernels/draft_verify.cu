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
// before the walk, which then runs redundantly in every thread from shared
// memory.  A whole-row pass is spread over a cluster of CTAs: each warp owns a
// contiguous range of the row and sums it with 16-byte loads, the ranges' sums
// are exchanged through distributed shared memory (one cluster barrier per
// pass), and the CTA that owns the crossing range reads it once more, from
// cache, to find the token.
//
// All sums and the excess are in 64 bits: the token is an integer that one
// rounding near a border would change, and 32-bit partial sums over 10^5
// probabilities are off by up to 10^5 * 2^-24.  The conversions and additions
// take a few percent of the time the loads take.
#include "kernels/draft_verify.cuh"
#include "kernels/error_bits.hpp"
#include "kernels/launch_count.hpp"
#include "kernels/pdl.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tsacb::dev
{
namespace
{
namespace cg = cooperative_groups;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int WIDE = 8; // CTAs of a cluster for a large vocabulary

__device__ __forceinline__ double to_double(float v) { return v; }
__device__ __forceinline__ double to_double(__half v) { return __half2float(v); }
__device__ __forceinline__ double to_double(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T> struct alignas(16) Vector
{
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    T v[N];
};

struct Shared
{
    int parents[DRAFT_MAX_NODES], tokens[DRAFT_MAX_NODES], path[DRAFT_MAX_NODES];
    float coins[DRAFT_MAX_NODES];
    double p[DRAFT_MAX_NODES], q[DRAFT_MAX_NODES];
    double scale[DRAFT_MAX_NODES];           // 1 / Z of each round of rejections
    int rejected[DRAFT_MAX_NODES];           // tokens rejected at the current node
    double sums[2][WIDE * WARPS];            // sums of the warps' ranges, by pass parity
    double scan[WARPS];
    int first;
};

// The weights at the current node: the target's row, reduced once per round.
template <class T, bool DRAFT> struct Weights
{
    const T* p;
    const T* q;
    int rounds; // with a draft: applications of max(w / Z - q, 0); else: rejected tokens
    const double* scale;
    const int* rejected;

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
            for (int i = 0; i < rounds; ++i)
                p_value = rejected[i] == token ? 0.0 : p_value;
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

template <class T, bool DRAFT>
__device__ __forceinline__ double block_weight(const Weights<T, DRAFT>& w, const Row<T, DRAFT>& row, int block,
                                               const Vector<T>& p, const Vector<T>& q)
{
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < Row<T, DRAFT>::N; ++k)
        sum += w.at(block * Row<T, DRAFT>::N - row.skew + k, to_double(p.v[k]), DRAFT ? to_double(q.v[k]) : 0.0);
    return sum;
}

// Sums the weights of the whole row; every thread of the cluster returns the
// total, and sums holds each warp range's sum.
template <class T, bool DRAFT, int CLUSTER>
__device__ double whole_row(const Weights<T, DRAFT>& w, const Row<T, DRAFT>& row, int per, double* sums)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = CLUSTER > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
    const int mine = rank * WARPS + warp;
    const int end = min(row.blocks, (mine + 1) * per);
    double sum = 0.0;
    constexpr int UNROLL = 4;
    for (int b = mine * per + lane; b < end; b += 32 * UNROLL)
    {
        Vector<T> p[UNROLL], q[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
            if (b + 32 * k < end)
            {
                row.load(w.p, b + 32 * k, p[k]);
                if constexpr (DRAFT)
                    row.load(w.q, b + 32 * k, q[k]);
            }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k)
            if (b + 32 * k < end)
                sum += block_weight<T, DRAFT>(w, row, b + 32 * k, p[k], q[k]);
    }
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
    double total = 0.0;
#pragma unroll 8
    for (int k = 0; k < CLUSTER * WARPS; ++k)
        total += sums[k];
    return total;
}

// The first token whose cumulative weight exceeds `threshold`, by the CTA that
// owns its range; the last token of positive weight if rounding leaves none.
template <class T, bool DRAFT, int CLUSTER>
__device__ void pick(const Weights<T, DRAFT>& w, const Row<T, DRAFT>& row, int per, const double* sums,
                     double threshold, Shared& sh, int* token)
{
    int range = -1;
    double before = 0.0, running = 0.0;
#pragma unroll 8
    for (int k = 0; k < CLUSTER * WARPS; ++k)
    {
        const double next = running + sums[k];
        if (sums[k] > 0.0 && !(running > threshold))
        {
            range = k;
            before = running;
        }
        running = next;
    }
    const int rank = CLUSTER > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
    if (range / WARPS != rank || range < 0)
        return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int begin = range * per, end = min(row.blocks, begin + per);
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
            const int candidate = b * Row<T, DRAFT>::N - row.skew + k;
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

template <class T, bool DRAFT, int CLUSTER>
__global__ void __launch_bounds__(THREADS, 2) draft_verify_kernel(const VerifyArgs a)
{
    pdl_prologue();
    __shared__ Shared sh;
    const int sequence = blockIdx.x / CLUSTER;
    const bool leader = blockIdx.x % CLUSTER == 0;
    const int t = threadIdx.x;
    const long long list = static_cast<long long>(sequence) * a.max_nodes;
    int nodes = a.nodes ? a.nodes[sequence] : a.max_nodes;
    nodes = nodes < 0 ? 0 : (nodes < a.max_nodes ? nodes : a.max_nodes);
    const T* target = static_cast<const T*>(a.target) + sequence * a.target_batch;
    const T* draft = DRAFT ? static_cast<const T*>(a.draft) + sequence * a.draft_batch : nullptr;
    if (t < nodes)
    {
        const int parent = a.parents[list + t], token = a.tokens[list + t];
        const bool real = t > 0 && parent >= 0 && parent < t;
        const bool known = static_cast<unsigned>(token) < static_cast<unsigned>(a.vocab);
        sh.parents[t] = real ? parent : -1;
        sh.tokens[t] = token;
        sh.coins[t] = a.coins[list + t];
        // A token outside the vocabulary has probability 0 and is never accepted.
        sh.p[t] = real && known ? to_double(target[parent * a.target_node + token]) : 0.0;
        if constexpr (DRAFT)
            sh.q[t] = real && known ? to_double(draft[parent * a.draft_node + token]) : 0.0;
    }
    if constexpr (CLUSTER > 1)
        cg::this_cluster().sync(); // every CTA runs before its shared memory is written to
    else
        __syncthreads();
    int accepted = 0, passes = 0;
    bool failed = false;
    if (nodes > 0)
    {
        int node = 0, rounds = 0;
        bool summed = false; // the last pass summed the current weights
        double total = 0.0, left = 1.0;
        accepted = 1;
        if (t == 0)
            sh.path[0] = 0;
        const auto weights = [&](int at, int n)
        {
            return Weights<T, DRAFT>{target + at * a.target_node, DRAFT ? draft + at * a.draft_node : nullptr, n, sh.scale,
                                     sh.rejected};
        };
        const int ranges = CLUSTER * WARPS;
        for (int n = 1; n < nodes && !failed; ++n)
        {
            if (sh.parents[n] != node)
                continue;
            double p = sh.p[n];
            bool pass;
            if constexpr (DRAFT)
            {
                const Weights<T, DRAFT> w = weights(node, rounds);
                p = w.excess(p, sh.q[n]);
                p = rounds ? p * sh.scale[rounds] : p;
                pass = sh.coins[n] * sh.q[n] < p;
            }
            else
            {
                for (int i = 0; i < rounds; ++i)
                    p = sh.rejected[i] == sh.tokens[n] ? 0.0 : p;
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
                __syncthreads(); // the rejected tokens have been read
                continue;
            }
            if constexpr (DRAFT)
            {
                const Weights<T, DRAFT> w = weights(node, rounds + 1);
                const Row<T, DRAFT> row(w.p, w.q, a.vocab);
                const double z = whole_row<T, DRAFT, CLUSTER>(w, row, (row.blocks + ranges - 1) / ranges, sh.sums[passes & 1]);
                if (z > 0.0 && z < INFINITY)
                {
                    total = z;
                    summed = true;
                    ++rounds;
                    ++passes;
                    if (t == 0)
                        sh.scale[rounds] = 1.0 / z;
                    __syncthreads();
                }
                else // no excess: the weights stay; a NaN or an infinity ends the walk
                {
                    failed = !(z == 0.0);
                    summed = false;
                    ++passes;
                }
            }
            else
            {
                if (t == 0)
                    sh.rejected[rounds] = sh.tokens[n];
                left -= p;
                ++rounds;
                __syncthreads();
            }
        }
        const auto finish = [&](int n)
        {
            const Weights<T, DRAFT> w = weights(node, n);
            const Row<T, DRAFT> row(w.p, w.q, a.vocab);
            const int per = (row.blocks + ranges - 1) / ranges;
            if (!summed)
                total = whole_row<T, DRAFT, CLUSTER>(w, row, per, sh.sums[passes++ & 1]);
            if (!(total > 0.0 && total < INFINITY))
                return false;
            pick<T, DRAFT, CLUSTER>(w, row, per, sh.sums[(passes - 1) & 1],
                                    static_cast<double>(a.draws[sequence]) * total, sh, a.token + sequence);
            return true;
        };
        if (!failed)
        {
            bool done = finish(rounds);
            if constexpr (!DRAFT)
                if (!done && rounds && total == 0.0) // nothing left beside the rejected tokens
                    done = finish(0);
            failed = !done;
        }
    }
    if (leader)
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

template <class T, bool DRAFT, int CLUSTER> cudaError_t launch(const VerifyArgs& a, int batch, cudaStream_t stream)
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
    const cudaError_t status = cudaLaunchKernelEx(&config, draft_verify_kernel<T, DRAFT, CLUSTER>, a);
    note_launch();
    return status;
}

template <class T> cudaError_t launch_type(const VerifyArgs& a, int batch, cudaStream_t stream)
{
    if (a.vocab >= 16384)
        return a.draft ? launch<T, true, WIDE>(a, batch, stream) : launch<T, false, WIDE>(a, batch, stream);
    return a.draft ? launch<T, true, 1>(a, batch, stream) : launch<T, false, 1>(a, batch, stream);
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
