// What the attention kernels share: element types, warp-level matrix products on 16-bit operands, asynchronous 16-byte copies into
// shared memory, and the argument checks that their launchers have in common.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mf {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
struct Bf16 {
    static constexpr bool value = false;
};
template <>
struct Bf16<__nv_bfloat16> {
    static constexpr bool value = true;
};

__device__ __forceinline__ uint32_t SmemAddr32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes global -> shared, asynchronously; with `bytes` 0 nothing is read and the place is filled with zeros.
__device__ __forceinline__ void CpAsync16(uint32_t dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void CpCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void CpWait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void LdMatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void LdMatrix4T(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Two matrices of 16 rows of 16 bytes, transposed: r[0], r[1] hold columns lane / 4 and lane / 4 + 8 of the first, rows 4 (lane % 4) and the next three.
__device__ __forceinline__ void LdMatrix2T8(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// The 8 x 8 matrix of 16-bit values that a warp holds (row lane / 4, columns 2 (lane % 4) and the next), transposed.
__device__ __forceinline__ uint32_t Transposed8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// c[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums.
template <typename T>
__device__ __forceinline__ void Mma16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void Mma16x8x16<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void Mma16x8x16<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two floats rounded to a pair of T, `lo` in the low half.
template <typename T>
__device__ __forceinline__ uint32_t Pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t Pack2<__nv_bfloat16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t Pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ float2 Unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 Unpack2<__nv_bfloat16>(uint32_t v)
{
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 Unpack2<__half>(uint32_t v)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// Where the reference of a row's weights lies, in powers of two: kLift below its maximum when it is set, and set anew when a weight would pass 2^kSlack.
// fp16 weights are lifted so that those of a thousandth and less of the largest are not subnormal.
template <typename T>
struct Weights {
    static constexpr float kLift = Bf16<T>::value ? 0.0f : 6.0f, kSlack = Bf16<T>::value ? 8.0f : 14.0f;
};

// Two e4m3 values (low 16 bits) as a pair of fp16, which holds all of them exactly.
__device__ __forceinline__ uint32_t E4m3ToHalf2(uint32_t v)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)v));
    return r;
}

// 2^x to about two units in the last place of fp32; -inf gives 0.
__device__ __forceinline__ float Exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

}  // namespace attn
}  // namespace mf
