// int8_device.hpp -- device code that the 8-bit kernels share: rounding to whole
// numbers, what finishes a product.
#pragma once

#include "feed_forward_device.hpp"
#include "int8.hpp"

namespace xspmm {
namespace detail {
namespace ff {

typedef int int4_t __attribute__((ext_vector_type(4)));

// The largest of |v|, as bits: whole numbers order them with the infinities and
// the NaNs, of which one stays, on top.
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
constexpr uint32_t kInfinite = 0x7f800000u;

struct Rounding {
    float by;      // 127 / most
    float most;    // its fraction, 0.5 <= most < 1, and exponent
    int exponent;
    bool none;     // nothing to round: zeros, or no finite maximum
    bool far;      // 127 / most is no normal number, or nearly none

    Rounding() = default;
    __device__ __forceinline__ explicit Rounding(uint32_t bits)
    {
        const float v = __builtin_bit_cast(float, bits);
        none = bits == 0u || bits >= kInfinite;
        most = __builtin_amdgcn_frexp_mantf(v);
        exponent = __builtin_amdgcn_frexp_expf(v);
        far = exponent < -100 || exponent > 100;
        by = 127.f / v;
        scale = bits == 0u ? 0.f : none ? __builtin_nanf("") : v / 127.f;
        if (none) {
            by = 0.f;
            far = bits != 0u;  // an infinity or a NaN times 0 is none
        }
    }
    float scale;
};

// Rounds to whole numbers, in the low 8 bits, by the addition of a large number;
// `off` is the largest distance of a quotient from its whole number.  A quotient is
// off by at most two roundings, 127 * 2^-23 < 2^-16: where `off` is that near to 1/2
// (never, where no `off` is) the quotients are looked at once more.
constexpr float kLarge = 12582912.f;  // 1.5 * 2^23
constexpr float kNear = 0.5f - 0x1p-15f;

__device__ __forceinline__ uint32_t round_quickly(float v, float by, float& off)
{
    const float t = v * by, k = t + kLarge;
    off = fmaxf(off, fabsf(t - (k - kLarge)));
    return __builtin_bit_cast(uint32_t, k);
}
// 127 v - k most is exact in two parts, of which the upper one is next to most / 2
// where it matters, so that its difference from that is exact, too.
__device__ __forceinline__ uint32_t round_exactly(float v, const Rounding& r)
{
    if (r.none) return 0u;
    v = ldexpf(v, -r.exponent);
    float k = rintf(v * (127.f / r.most));
    const float hi = 127.f * v, lo = fmaf(127.f, v, -hi), left = fmaf(-k, r.most, hi), half = 0.5f * r.most;
    const float above = (left - half) + lo, below = (left + half) + lo;
    const bool odd = (int)k & 1;
    if (above > 0.f || (above == 0.f && odd))
        k += 1.f;
    else if (below < 0.f || (below == 0.f && odd))
        k -= 1.f;
    return (uint32_t)(int)k;
}

// The low bytes of four numbers.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                 0x05040100u);
}

// Sixteen features of a token.
__device__ __forceinline__ u32x4_t round_features(const float (&v)[16], const Rounding& r)
{
    u32x4_t w;
    float off = r.far ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = pack4(round_quickly(v[4 * i], r.by, off), round_quickly(v[4 * i + 1], r.by, off),
                     round_quickly(v[4 * i + 2], r.by, off), round_quickly(v[4 * i + 3], r.by, off));
    if (off > kNear)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = pack4(round_exactly(v[4 * i], r), round_exactly(v[4 * i + 1], r), round_exactly(v[4 * i + 2], r),
                         round_exactly(v[4 * i + 3], r));
    return w;
}

// The 16 features of block kb of token n, zeros past the last.
template <typename T>
__device__ __forceinline__ void load_features(const T* x, int64_t K, int64_t N, int64_t kb, int64_t n, float (&v)[16])
{
    if (16 * kb + 16 <= K) {
        T p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = x[(16 * kb + i) * N + n];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = (float)p[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = 16 * kb + i < K;
            const T p = x[(in ? 16 * kb + i : K - 1) * N + n];
            v[i] = in ? (float)p : 0.f;
        }
    }
}

__device__ __forceinline__ void store_features(int8_t* q, int64_t N, int64_t kb, int64_t n, const float (&v)[16],
                                               const Rounding& round)
{
    *reinterpret_cast<u32x4_t*>(q + (kb * N + n) * 16) = round_features(v, round);
}

// The largest of `m` over the threads of a column tile that have the same token.
template <int THREADS, int LT>
__device__ __forceinline__ void join(uint32_t& m, uint32_t* red)
{
    const int t = threadIdx.x;
#pragma unroll
    for (int d = LT; d < 64; d *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    constexpr int kWaves = THREADS / 64;
    const int lane = t & 63, wave = t >> 6;
    if (lane < LT) red[wave * LT + lane] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = max(m, red[w * LT + (t % LT)]);
}

// Between what lanes of a wave leave in LDS and what others of it read or write there.  LDS
// takes a wave's operations in their order, so nothing waits; the compiler has to keep it.
__device__ __forceinline__ void lanes_in_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

struct Int8Side {
    const int32_t* ptr;
    const int32_t* col;
    const int32_t* map;
    const int8_t* vals;
    const float* scale;
    const void* bias;
};

template <typename T>
struct Int8Product {
    Int8Side side[2];
    const T* raw;  // activations that the kernel rounds itself
    const int8_t* x;
    const float* x_scale;
    const T* residual;
    T* y;
    int32_t rows, block_rows;
    int32_t in_rows, in_blocks;  // of x
    int64_t N;
    uint32_t vals_bytes[2];  // 0 where they pass 2^31
    int act;
};

// D += A B of 16 x 64 and 64 x 16 whole numbers: lane l holds row (column) l % 16 of A
// (B) at k = 16 (l / 16) .. + 15, and column l % 16 of D at rows 4 (l / 16) .. + 3.
__device__ __forceinline__ int4_t mfma8(u32x4_t a, u32x4_t b, int4_t c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4_t, a), __builtin_bit_cast(int4_t, b), c, 0, 0,
                                                 0);
}

// An activation of a result in 16 bits: exponentials by the hardware's exp2, off by the
// rounding of its argument (2^-24 of up to 185, 1e-5 of the value), and quotients by its
// reciprocal: 2^-16 in all where the result's own rounding is 2^-11 at least.  With expf
// and a division the epilogue of 14336 x 2048 gelus takes 10 us longer.
__device__ __forceinline__ float exp_quick(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
template <typename T, int ACT>
__device__ __forceinline__ float finish_act(float z)
{
    if constexpr (is_f32<T> || ACT == kActNone || ACT == kActRelu) return act_value<ACT>(z);
    if constexpr (ACT == kActSilu) {
        const float c = at_least(z, -kSiluEnd);
        return c * __builtin_amdgcn_rcpf(1.f + exp_quick(-c));
    }
    if constexpr (ACT == kActGelu) {
        const float c = at_least(z, -kGeluEnd);
        return c * normal_integral(c, exp_quick(-0.5f * c * c));
    }
    const float c = at_least(z, -kGeluEnd);
    return c * __builtin_amdgcn_rcpf(1.f + exp_quick(-kGeluA * (c + kGeluB * c * c * c)));
}

template <typename T, int NACC>
__device__ __forceinline__ float int8_finish(const Int8Product<T>& a, const int (&sum)[NACC], int64_t row, int64_t n,
                                             float x_scale)
{
    float z[NACC];
#pragma unroll
    for (int l = 0; l < NACC; ++l) {
        z[l] = (float)sum[l] * a.side[l].scale[row] * x_scale;
        if (a.side[l].bias) z[l] += (float)static_cast<const T*>(a.side[l].bias)[row];
    }
    with_act(a.act, [&](auto act) { z[0] = finish_act<T, decltype(act)::value>(z[0]); });
    if constexpr (NACC == 2) z[0] *= z[1];
    if (a.residual) z[0] += (float)a.residual[row * a.N + n];
    return z[0];
}

// Sixteen rows of a product and WIDE tokens, whose sums a wave has left in O (rows of
// WIDE + 4 floats, SIDES times 16 of them): eight tokens of a row a thread.  xs: the scales
// of the thread's tokens; lane `shift` + r has row r's scale and bias.
template <typename T, int SIDES, int WIDE>
__device__ __forceinline__ void int8_rows(const Int8Product<T>& a, const float* O, int64_t row0, int64_t n0,
                                          const float (&xs)[8], const float (&rs)[SIDES], const float (&bias)[SIDES],
                                          int shift)
{
    constexpr int kLanes = WIDE / 8, kAtOnce = 64 / kLanes, kRow = WIDE + 4;
    const int lane = threadIdx.x & 63, c = lane % kLanes * 8;
    const int64_t n = n0 + c;
#pragma unroll 1
    for (int v = 0; v < 16 / kAtOnce; ++v) {
        const int r = kAtOnce * v + lane / kLanes;
        const int64_t row = row0 + r;
        float z[SIDES][8];
#pragma unroll
        for (int l = 0; l < SIDES; ++l) {
            const float4_t lo = *reinterpret_cast<const float4_t*>(O + (l * 16 + r) * kRow + c);
            const float4_t hi = *reinterpret_cast<const float4_t*>(O + (l * 16 + r) * kRow + c + 4);
            const float scale = __shfl(rs[l], shift + r), add = __shfl(bias[l], shift + r);
#pragma unroll
            for (int q = 0; q < 8; ++q) z[l][q] = (q < 4 ? lo[q] : hi[q - 4]) * scale * xs[q] + add;
        }
        if (row >= a.rows || n >= a.N) continue;
        with_act(a.act, [&](auto act) {
#pragma unroll
            for (int q = 0; q < 8; ++q) z[0][q] = finish_act<T, decltype(act)::value>(z[0][q]);
        });
        if constexpr (SIDES == 2)
#pragma unroll
            for (int q = 0; q < 8; ++q) z[0][q] *= z[1][q];
        const int64_t at = row * a.N + n;
        if (n + 8 <= a.N) {
            if (a.residual) {
                const Pack<T, 8> k = *reinterpret_cast<const Pack<T, 8>*>(a.residual + at);
#pragma unroll
                for (int q = 0; q < 8; ++q) z[0][q] += (float)k.v[q];
            }
            Pack<T, 8> k;
#pragma unroll
            for (int q = 0; q < 8; ++q) k.v[q] = (T)z[0][q];
            *reinterpret_cast<Pack<T, 8>*>(a.y + at) = k;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (n + q < a.N) a.y[at + q] = (T)(z[0][q] + (a.residual ? (float)a.residual[at + q] : 0.f));
        }
    }
}

}  // namespace ff

// The products by lists of blocks (the first `fours` of a row fetched ahead) and by tiles,
// both with x in LDS.
template <typename T>
void int8_lists(const ff::Int8Product<T>& a, int weights, int fours, hipStream_t s);
template <typename T>
void int8_tiles(const ff::Int8Product<T>& a, int weights, hipStream_t s);

}  // namespace detail
}  // namespace xspmm
