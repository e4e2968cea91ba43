// The two 16-bit element types of the drafted-decoding kernels.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tsacb::dev
{
template <class T> struct Half2;
template <> struct Half2<__nv_bfloat16>
{
    static __device__ __forceinline__ std::uint32_t pack(float lo, float hi)
    {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const std::uint32_t*>(&v);
    }
    static __device__ __forceinline__ float value(std::uint16_t x)
    {
        return __bfloat162float(__ushort_as_bfloat16(x));
    }
    static constexpr std::uint32_t exponents = 0x7f807f80u;
    // Softmax weights p are kept as 2^(z - reference) with the largest of a row near 2^weight_powers.
    // The exponents of bf16 reach as far down as those of the 32-bit sums.
    static constexpr float weight_powers = 0.0f;
    static constexpr std::uint32_t mma_format = 1; // kind::f16 operand format: bf16
    static __device__ __forceinline__ void mma(float (&d)[4], const std::uint32_t (&a)[4], std::uint32_t b0,
                                               std::uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
                     " {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Half2<__half>
{
    static __device__ __forceinline__ std::uint32_t pack(float lo, float hi)
    {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const std::uint32_t*>(&v);
    }
    static __device__ __forceinline__ float value(std::uint16_t x) { return __half2float(__ushort_as_half(x)); }
    static constexpr std::uint32_t exponents = 0x7c007c00u;
    // fp16 ends at 65,504 above and loses bits below 2^-14: with the largest weight at 1, one of 2^-25 is
    // nothing, and 10^5 of those beside a dominant key are 0.3 % of the row.
    static constexpr float weight_powers = 15.0f;
    static constexpr std::uint32_t mma_format = 0; // kind::f16 operand format: fp16
    static __device__ __forceinline__ void mma(float (&d)[4], const std::uint32_t (&a)[4], std::uint32_t b0,
                                               std::uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
                     " {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// Which of a word's two elements are infinite or NaN, as masks of their bits.
template <class T> __device__ __forceinline__ std::uint32_t nonfinite_mask(std::uint32_t word)
{
    const std::uint32_t x = word & Half2<T>::exponents;
    return ((x & 0xffffu) == (Half2<T>::exponents & 0xffffu) ? 0xffffu : 0u) |
           ((x >> 16) == (Half2<T>::exponents >> 16) ? 0xffff0000u : 0u);
}

__device__ __forceinline__ float power_of_two(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16-byte asynchronous copy into shared memory, or 16 zero bytes when `bytes` is 0.
__device__ __forceinline__ void copy_16(std::uint32_t to, const void* from, unsigned bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
} // namespace tsacb::dev
