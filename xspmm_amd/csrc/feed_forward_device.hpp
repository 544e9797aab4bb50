// feed_forward_device.hpp -- device code that the feed-forward kernels share:
// value types, loads, matrix instructions, activations.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "feed_forward.hpp"

namespace xspmm {
namespace detail {
namespace ff {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// Offset of what is not there: past the end of every buffer, and still so with
// the offset of a row within a block added (operands of kernels that use it have
// less than 2^31 bytes, rows past the last included).
constexpr uint32_t kNone = 0x80000000u;

constexpr int kXcds = 8;  // accelerator dies of an MI355X, each with its own L2

template <typename T>
constexpr bool is_f32 = sizeof(T) == 4;

// VEC consecutive elements at any element's address (the GPU reads and writes
// vectors off their alignment; aligned ones are no slower for this type).
template <typename T, int VEC>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[VEC];
};

// The same as dwords, for the operands of matrix instructions; one 16-bit
// element takes a dword of its own.
template <typename T, int VEC>
constexpr int kDwords = VEC * (int)sizeof(T) < 4 ? 1 : VEC * (int)sizeof(T) / 4;

template <int D>
struct Dwords {
    uint32_t d[D];
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_buffer(const void* base, uint32_t bytes)
{
    // raw dword access; a load past `bytes` gives zeros and touches no memory
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}

template <typename T, int VEC>
__device__ __forceinline__ Dwords<kDwords<T, VEC>> buffer_load(__amdgpu_buffer_rsrc_t r, uint32_t off)
{
    Dwords<kDwords<T, VEC>> o;
    constexpr int bytes = VEC * (int)sizeof(T);
    if constexpr (bytes == 2) {
        o.d[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, 0);
    } else if constexpr (bytes == 4) {
        o.d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
    } else if constexpr (bytes == 8) {
        const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0);
        o.d[0] = v.x;
        o.d[1] = v.y;
    } else {
        static_assert(bytes == 16);
        const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) o.d[i] = v[i];
    }
    return o;
}

template <typename T, int VEC>
__device__ __forceinline__ Dwords<kDwords<T, VEC>> global_load(const T* p)
{
    Dwords<kDwords<T, VEC>> o;
    if constexpr (VEC * sizeof(T) == 2) {
        o.d[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
        struct __attribute__((packed, aligned(sizeof(T)))) P {
            uint32_t d[kDwords<T, VEC>];
        };
        const P v = *reinterpret_cast<const P*>(p);
#pragma unroll
        for (int i = 0; i < kDwords<T, VEC>; ++i) o.d[i] = v.d[i];
    }
    return o;
}

__device__ __forceinline__ uint32_t lds_address(const void* p)
{
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// A load straight into LDS: lane l's 16 bytes at byte `off` of the buffer land at
// LDS address lds + 16 l (zeros past its end).  The compiler does not see it:
// dma_wait() before the barrier that lets the others read, and the wait state that
// the load wants after a scalar write of M0.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4_t dma_buffer(const void* base, uint32_t bytes)
{
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return i32x4_t{(int)(uint32_t)a, (int)(uint32_t)((a >> 32) & 0xffffu), (int)bytes, 0x00020000};
}
__device__ __forceinline__ void dma_to_lds(uint32_t lds, uint32_t off, i32x4_t buffer)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(off), "s"(buffer)
                 : "memory", "m0");
}
// Until at most LEFT of this wave's loads, the latest ones, are under way.
template <int LEFT>
__device__ __forceinline__ void dma_wait()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

// D += A B of 16x16x32 16-bit values: lane l holds row (column) l % 16 of A
// (B) at k = 8 (l / 16) .. + 7, and column l % 16 of D at rows 4 (l / 16) .. + 3.
template <typename T>
__device__ __forceinline__ float4_t mfma16(u32x4_t a, u32x4_t b, float4_t c)
{
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b),
                                                      c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// D += A B of 16x16x16 16-bit values: as above, at k = 4 (l / 16) .. + 3.
template <typename T>
__device__ __forceinline__ float4_t mfma16_half(u32x2_t a, u32x2_t b, float4_t c)
{
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4_t, a), __builtin_bit_cast(half4_t, b), c,
                                                     0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a),
                                                         __builtin_bit_cast(short4_t, b), c, 0, 0, 0);
}

// D += A B of 16x16x4 fp32 values: lane l holds row (column) l % 16 at k = l / 16.
__device__ __forceinline__ float4_t mfma32(uint32_t a, uint32_t b, float4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b), c, 0, 0,
                                                0);
}

// ---------------------------------------------------------------------------
// activations, in fp32.  Sums are taken to where an activation and its slope have
// reached their limits, so that infinite ones give these, too (a NaN stays).
// ---------------------------------------------------------------------------

__device__ __forceinline__ float at_least(float z, float low) { return z < low ? low : z; }
__device__ __forceinline__ float within(float z, float most) { return z < -most ? -most : z > most ? most : z; }

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }

// The normal distribution's density (times sqrt(2 pi)) and integral P(z), which is
// (1 + erf(z / sqrt 2)) / 2 but keeps its digits where it vanishes: 1 + erf cancels, at
// z = -5 to a hundredth of the value.  P(-|z|) = exp(-z^2 / 2) t Q(t), t = 1 / (1 + 0.35
// |z|); Q has degree 8, with the smallest largest relative error (half of 2^-24) on
// |z| <= 16.5.  All in all (6 + 0.6 z^2) 2^-24 of P, most of it exp's argument.  One exp
// and no branch: an erfc costs a product of 14336 x 4096 and 2048 tokens 14 us of 277.
__device__ __forceinline__ float normal_density(float z) { return expf(-0.5f * z * z); }
__device__ __forceinline__ float normal_integral(float z, float density)
{
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(z), 1.f));
    float q = -0.0291653033f;
    q = fmaf(q, t, 0.144067645f);
    q = fmaf(q, t, -0.255916327f);
    q = fmaf(q, t, 0.159409836f);
    q = fmaf(q, t, -0.0232758019f);
    q = fmaf(q, t, 0.105580017f);
    q = fmaf(q, t, 0.119814134f);
    q = fmaf(q, t, 0.139864534f);
    q = fmaf(q, t, 0.139621243f);
    q *= t * density;
    return z < 0.f ? q : 1.f - q;
}

constexpr float kGeluA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;
// where the sigmoid, and the two gelus' share of z, are 0 and 1 in fp32
constexpr float kSiluEnd = 128.f, kGeluEnd = 16.f;

template <int ACT>
__device__ __forceinline__ float act_value(float z)
{
    if constexpr (ACT == kActRelu) return at_least(z, 0.f);
    if constexpr (ACT == kActSilu) {
        const float c = at_least(z, -kSiluEnd);
        return c / (1.f + expf(-c));
    }
    if constexpr (ACT == kActGelu) {
        const float c = at_least(z, -kGeluEnd);
        return c * normal_integral(c, normal_density(c));
    }
    // 0.5 (1 + tanh u) = sigmoid(2u)
    if constexpr (ACT == kActGeluTanh) {
        const float c = at_least(z, -kGeluEnd);
        return c / (1.f + expf(-kGeluA * (c + kGeluB * c * c * c)));
    }
    return z;
}

// value and slope
template <int ACT>
__device__ __forceinline__ float act_slope(float z, float* value)
{
    if constexpr (ACT == kActRelu) {
        *value = at_least(z, 0.f);
        return z > 0.f ? 1.f : z == z ? 0.f : z;
    }
    if constexpr (ACT == kActSilu) {
        const float c = within(z, kSiluEnd), p = sigmoid(c);
        *value = at_least(z, -kSiluEnd) * p;
        return p * (1.f + c * (1.f - p));
    }
    if constexpr (ACT == kActGelu) {
        const float c = within(z, kGeluEnd), e = normal_density(c), p = normal_integral(c, e);
        *value = at_least(z, -kGeluEnd) * p;
        return p + 0.3989422804014327f * c * e;
    }
    if constexpr (ACT == kActGeluTanh) {
        const float c = within(z, kGeluEnd), p = sigmoid(kGeluA * (c + kGeluB * c * c * c));
        *value = at_least(z, -kGeluEnd) * p;
        return p + c * p * (1.f - p) * kGeluA * (1.f + 3.f * kGeluB * c * c);
    }
    *value = z;
    return 1.f;
}

// f(constant activation)
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f)
{
    switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
    }
}

// Work item of workgroup w in a grid of 8 * xcd_chunk(total): each XCD takes a
// contiguous range of items, so that neighbours share its L2.  -1: padding.
__host__ __device__ __forceinline__ int64_t xcd_chunk(int64_t total) { return (total + kXcds - 1) / kXcds; }
__device__ __forceinline__ int64_t xcd_item(int64_t w, int64_t total)
{
    const int64_t i = (w % kXcds) * xcd_chunk(total) + w / kXcds;
    return i < total ? i : -1;
}

// The same in 32 bits (a launch has less than 2^32 threads): divisions of 64 bits take a
// wave more than half a microsecond each.
__device__ __forceinline__ uint32_t xcd_item32(uint32_t w, uint32_t total)
{
    const uint32_t i = w % kXcds * ((total + kXcds - 1) / kXcds) + w / kXcds;
    return i < total ? i : ~0u;
}

}  // namespace ff
}  // namespace detail
}  // namespace xspmm
