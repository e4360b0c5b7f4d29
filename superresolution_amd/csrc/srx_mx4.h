// Device-side helpers of the normalisation and 4-bit block layers (internal header).
//
// The 4-bit block form (OCP microscaling, MXFP4): the values of a row are taken in blocks of 32, the last one filled
// up with zeros.  A block is held as one scale byte s (e8m0: the factor 2^(s - 127), 255 = NaN) and 32 codes of 4 bits
// (e2m1: sign, then the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6), element 2i in the low half of byte i.
#pragma once

#include "srx_device.h"

namespace srx {
namespace dev {

// Division of numbers below 2^31 by a constant d: (mulhi(n, mul) + n) >> shift, division by an invariant integer through
// multiplication (Granlund and Montgomery, 1994).
struct Divider
{
    unsigned mul = 0, shift = 0, d = 1;
    Divider() = default;
    explicit Divider(unsigned by) : d(by)
    {
        while ((uint64_t(1) << shift) < by) ++shift;
        mul = unsigned((uint64_t(1) << 32) * ((uint64_t(1) << shift) - by) / by + 1);
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// Grids of up to 2^31 - 1 workgroups: one dimension has to stay below 2^32 threads, so they come in rows of 2^21.
constexpr unsigned kGridRow = 1u << 21;
inline dim3 gridOf(int64_t blocks)
{
    return blocks <= int64_t(kGridRow) ? dim3(unsigned(blocks)) : dim3(kGridRow, unsigned((blocks + kGridRow - 1) / kGridRow));
}
// Number of this workgroup; a kernel has nothing to do for those behind the last one of the grid asked for.
__device__ __forceinline__ unsigned blockNumber() { return blockIdx.y * kGridRow + blockIdx.x; }

constexpr int kMxBlock = 32;                          // values that share a scale
constexpr int kMxBytes = kMxBlock / 2;                // bytes of a block's codes

__host__ __device__ inline int64_t mxBlocks(int64_t columns) { return (columns + kMxBlock - 1) / kMxBlock; }

// Scale byte of a block whose largest magnitude is `most` (of its bits, sign clear): 2^(floor(log2 most) - 2) puts the
// largest value into [4, 8), where 6 is the largest code; below 2^-125 the smallest scale is taken.  An infinity or a
// NaN in the block makes the scale NaN.  `most` may have lost its low bits, never its exponent.
__device__ __forceinline__ unsigned mxScale(unsigned mostBits)
{
    const unsigned e = mostBits >> 23;
    return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}

// 2^(127 - s) for a scale byte 0 .. 252: exact, and normal (a product with it is rounded only below 2^-126).
__device__ __forceinline__ float mxInverse(unsigned s) { return __uint_as_float((254u - s) << 23); }

// 2^(s - 127): 2^-127 is subnormal, 255 stands for NaN.
__device__ __forceinline__ float mxFactor(unsigned s)
{
    return __uint_as_float(s == 0u ? 0x00400000u : (s == 255u ? 0x7fc00000u : s << 23));
}

// Eight values, already divided by their block's factor, as eight codes.  The conversion rounds to nearest, ties to the
// even code, and saturates at 6.
__device__ __forceinline__ unsigned mxCodes8(const float (&v)[8])
{
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
    return r;
}

// What eight codes stand for before the block's factor.
__device__ __forceinline__ void mxValues8(unsigned codes, float (&v)[8])
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}

// Four neighbouring lanes hold one block, eight values each: the largest of their four values.
__device__ __forceinline__ unsigned quadMax(unsigned v)
{
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));    // lanes 1, 0, 3, 2
    return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true)); // lanes 2, 3, 0, 1
}

// Quantise a lane's eight values of a block shared by four neighbouring lanes (all four active): returns the lane's
// codes and the block's scale.  Magnitudes are compared as integers: the order of the bits of positive floats, with
// NaN above infinity.
__device__ __forceinline__ unsigned mxQuantise(float (&v)[8], unsigned& scale)
{
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    scale = mxScale(quadMax(most));
    if (scale == 255u) return 0u;
    const float inv = mxInverse(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
    return mxCodes8(v);
}

// Eight consecutive values from any element-aligned address (the hardware reads vectors from any byte address).
__device__ __forceinline__ void load8(const f16* p, float (&v)[8])
{
    f16x8 h;
    __builtin_memcpy(&h, p, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8])
{
    f32x4 a, b;
    __builtin_memcpy(&a, p, 16);
    __builtin_memcpy(&b, p + 4, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void store8(f16* p, const float (&v)[8])
{
    f16x8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (f16)v[i];
    __builtin_memcpy(p, &h, 16);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8])
{
    f32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
    __builtin_memcpy(p, &a, 16);
    __builtin_memcpy(p + 4, &b, 16);
}
// Tensors over this size pass by the last-level cache (256 MB): what an operator reads again, or the next one reads, stays
// there.  Normalising 265 MB: 143 instead of 184 us, as the input is still cached when it is read again.
constexpr int64_t kStreamBytes = int64_t(96) << 20;

// The same past the caches.
__device__ __forceinline__ void streamIn8(const f16* p, float (&v)[8])
{
    typedef f16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));
    const f16x8u h = __builtin_nontemporal_load(reinterpret_cast<const f16x8u*>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
__device__ __forceinline__ void streamIn8(const float* p, float (&v)[8])
{
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const f32x4u a = __builtin_nontemporal_load(reinterpret_cast<const f32x4u*>(p)), b = __builtin_nontemporal_load(reinterpret_cast<const f32x4u*>(p + 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void streamOut8(f16* p, const float (&v)[8])
{
    typedef f16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));
    f16x8u h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (f16)v[i];
    __builtin_nontemporal_store(h, reinterpret_cast<f16x8u*>(p));
}
__device__ __forceinline__ void streamOut8(float* p, const float (&v)[8])
{
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    __builtin_nontemporal_store(f32x4u{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4u*>(p));
    __builtin_nontemporal_store(f32x4u{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4u*>(p + 4));
}
// The first `count` (0 .. 8) of eight values.  Where eight are in the tensor (which ends at `end`) all are read, and the
// others are somebody else's; only at the tensor's end are they read one by one, and the others are zeros.
template <typename T>
__device__ __forceinline__ void loadUpTo8(const T* p, int count, const T* end, float (&v)[8])
{
    if (count >= 8 || p + 8 <= end) { load8(p, v); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? (float)p[i] : 0.0f;
}
// Stores the first `count` of eight values: eight, or four, two and one.
template <typename T>
__device__ __forceinline__ void storeUpTo8(T* p, int count, const float (&v)[8])
{
    if (count >= 8) { store8(p, v); return; }
    typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    typedef T T2 __attribute__((ext_vector_type(2), aligned(sizeof(T))));
    const T v0 = (T)v[0], v1 = (T)v[1], v2 = (T)v[2], v3 = (T)v[3], v4 = (T)v[4], v5 = (T)v[5], v6 = (T)v[6];
    const bool four = count & 4, two = count & 2;
    if (four) *reinterpret_cast<T4*>(p) = T4{v0, v1, v2, v3};
    const T a = four ? v4 : v0, b = four ? v5 : v1, c = four ? v6 : v2;
    T* q = four ? p + 4 : p;
    if (two) *reinterpret_cast<T2*>(q) = T2{a, b};
    if (count & 1) q[two ? 2 : 0] = two ? c : a;
}

// 0 none, 1 ReLU, 2 SiLU: y / (1 + exp(-y)), with the exponential and the reciprocal of the special function unit
// (one part in 2^22 each; the product of y and log2(e) adds |y| parts in 2^24 where y is negative, and results below 1e-36
// in magnitude may become zero).  ReLU is the maximum that passes a NaN on.
__device__ __forceinline__ float activate(float y, int activation)
{
    if (activation == 1) return __builtin_elementwise_maximum(y, 0.0f);
    if (activation == 2) return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.44269504088896340736f));
    return y;
}

}  // namespace dev
}  // namespace srx
