// ff_grad.hip -- the backward pass through the activation, with the sums over
// the tokens.
#include "feed_forward_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// ---------------------------------------------------------------------------
// dz = dy [up] act'(z), dup = dy act(z), and their sums over the tokens.
// One wave per row, so that the sums need no other wave's; they are fp32, of the
// values before they are rounded.  dz is rounded to its type once, as the products
// with it want 16-bit operands (in fp16 past 65504 to an infinity).  Bound by memory:
// gated, 14336 rows of 2048 tokens in bf16, 294 MB in 48 us, 6.1 TB/s.
// ---------------------------------------------------------------------------

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

template <typename T, int ACT, bool GATED>
__global__ __launch_bounds__(256) void ff_act_backward_kernel(const T* __restrict__ z, const T* __restrict__ up,
                                                              const T* __restrict__ dy, T* __restrict__ dz,
                                                              T* __restrict__ dup, T* __restrict__ dbias,
                                                              T* __restrict__ dbias_up, int64_t M, int64_t N)
{
    constexpr int V = 16 / sizeof(T);
    constexpr bool kReads = GATED || ACT != kActNone;  // z
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (row >= M) return;
    const int64_t at = row * N;
    float sum = 0.f, sum_up = 0.f;
    auto one = [&](float zv, float uv, float g, bool own, float& o, float& ou) {
        float value = zv;
        const float slope = act_slope<ACT>(zv, &value);
        o = GATED ? g * uv * slope : g * slope;
        ou = GATED ? g * value : 0.f;
        sum += own ? o : 0.f;
        sum_up += own ? ou : 0.f;
    };
    if (N >= V) {
        for (int64_t n = V * lane; n < N; n += 64 * V) {
            // the last pack moves back into the row: what it does again gives the
            // same, and counts once
            const int64_t m = n + V <= N ? n : N - V;
            const auto g = *reinterpret_cast<const Pack<T, V>*>(dy + at + m);
            Pack<T, V> zz, uu, o, ou;
            if (kReads) zz = *reinterpret_cast<const Pack<T, V>*>(z + at + m);
            if (GATED) uu = *reinterpret_cast<const Pack<T, V>*>(up + at + m);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float a, b;
                one(kReads ? (float)zz.v[i] : 0.f, GATED ? (float)uu.v[i] : 0.f, (float)g.v[i], m + i >= n, a, b);
                o.v[i] = (T)a;
                ou.v[i] = (T)b;
            }
            if (dz) *reinterpret_cast<Pack<T, V>*>(dz + at + m) = o;
            if (GATED) *reinterpret_cast<Pack<T, V>*>(dup + at + m) = ou;
        }
    } else if (lane < N) {
        float a, b;
        one(kReads ? (float)z[at + lane] : 0.f, GATED ? (float)up[at + lane] : 0.f, (float)dy[at + lane], true, a, b);
        if (dz) dz[at + lane] = (T)a;
        if (GATED) dup[at + lane] = (T)b;
    }
    if (dbias) {
        sum = wave_sum(sum);
        if (lane == 0) dbias[row] = (T)sum;
    }
    if (GATED && dbias_up) {
        sum_up = wave_sum(sum_up);
        if (lane == 0) dbias_up[row] = (T)sum_up;
    }
}

template <typename T, bool GATED>
void launch_act_backward(const T* z, const T* up, const T* dy, T* dz, T* dup, T* db, T* dbu, int act, int64_t M,
                         int64_t N, hipStream_t s)
{
    const dim3 grid((unsigned)((M + 3) / 4)), block(256);
    auto go = [&](auto a) {
        hipLaunchKernelGGL((ff_act_backward_kernel<T, decltype(a)::value, GATED>), grid, block, 0, s, z, up, dy, dz,
                           dup, db, dbu, M, N);
    };
    switch (act) {
    case kActRelu: go(std::integral_constant<int, kActRelu>{}); break;
    case kActSilu: go(std::integral_constant<int, kActSilu>{}); break;
    case kActGelu: go(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: go(std::integral_constant<int, kActGeluTanh>{}); break;
    default: go(std::integral_constant<int, kActNone>{}); break;
    }
    XSPMM_LAUNCH_CHECK();
}

}  // namespace ff

template <typename T>
void activation_backward(const T* z, const T* up, const T* dy, T* dz, T* dup, T* dbias, T* dbias_up, int act,
                         int64_t M, int64_t N, hipStream_t s)
{
    if (M == 0) return;
    if (up)
        ff::launch_act_backward<T, true>(z, up, dy, dz, dup, dbias, dbias_up, act, M, N, s);
    else
        ff::launch_act_backward<T, false>(z, up, dy, dz, dup, dbias, dbias_up, act, M, N, s);
}

#define XSPMM_FF_GRAD(T)                                                                                            \
    template void activation_backward<T>(const T*, const T*, const T*, T*, T*, T*, T*, int, int64_t, int64_t,       \
                                         hipStream_t);
XSPMM_FF_GRAD(float)
XSPMM_FF_GRAD(_Float16)
XSPMM_FF_GRAD(__bf16)
#undef XSPMM_FF_GRAD

}  // namespace detail
}  // namespace xspmm
