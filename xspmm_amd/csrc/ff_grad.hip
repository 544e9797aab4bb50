// ff_grad.hip -- the backward pass around the products: the gradient through
// the activation with the sums over the tokens, and the gradient of a weight's
// stored blocks (a product sampled at their positions).
#include "feed_forward_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// ---------------------------------------------------------------------------
// dz = dy [up] act'(z), dup = dy act(z), and their sums over the tokens.
// One wave per row; sums in fp32, of the values before they are rounded.
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
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (row >= M) return;
    const int64_t at = row * N;
    float sum = 0.f, sum_up = 0.f;
    auto one = [&](float zv, float uv, float g, float& o, float& ou) {
        float value = zv;
        const float slope = act_slope<ACT>(zv, &value);
        o = GATED ? g * uv * slope : g * slope;
        ou = GATED ? g * value : 0.f;
        sum += o;
        sum_up += ou;
    };
    for (int64_t n = V * lane; n < N; n += 64 * V) {
        if (n + V <= N) {
            const auto g = *reinterpret_cast<const Pack<T, V>*>(dy + at + n);
            Pack<T, V> zz, uu, o, ou;
            if (ACT != kActNone) zz = *reinterpret_cast<const Pack<T, V>*>(z + at + n);
            if (GATED) uu = *reinterpret_cast<const Pack<T, V>*>(up + at + n);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float a, b;
                one(ACT != kActNone ? (float)zz.v[i] : 0.f, GATED ? (float)uu.v[i] : 0.f, (float)g.v[i], a, b);
                o.v[i] = (T)a;
                ou.v[i] = (T)b;
            }
            if (dz) *reinterpret_cast<Pack<T, V>*>(dz + at + n) = o;
            if (GATED) *reinterpret_cast<Pack<T, V>*>(dup + at + n) = ou;
        } else {
            for (int64_t m = n; m < N; ++m) {
                float a, b;
                one(ACT != kActNone ? (float)z[at + m] : 0.f, GATED ? (float)up[at + m] : 0.f, (float)dy[at + m], a, b);
                if (dz) dz[at + m] = (T)a;
                if (GATED) dup[at + m] = (T)b;
            }
        }
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

// ---------------------------------------------------------------------------
// dvals[b] = dz[16 row(b) ..][:] x[16 col(b) ..][:]^T: the sum runs along the
// tokens, which are contiguous in both operands, so every lane's operands are
// plain loads of 16 bytes.  x is the left operand: a lane then holds four
// consecutive columns of one row of the block.
// ---------------------------------------------------------------------------

template <typename T>
struct Eight {
    u32x4_t v[is_f32<T> ? 2 : 1];
};

template <typename T, int SPLIT>
__global__ __launch_bounds__(256) void ff_sampled_kernel(const int32_t* __restrict__ row, const int32_t* __restrict__ col,
                                                         const T* __restrict__ dz, const T* __restrict__ x,
                                                         T* __restrict__ dvals, int64_t nnzb, int32_t M, int32_t K,
                                                         int64_t N)
{
    constexpr int V = 16 / sizeof(T);  // tokens a lane takes per step
    constexpr int kStep = 4 * V;
    constexpr int kPer = 4 / SPLIT;
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int li = lane & 15, g = lane >> 4;
    const int64_t b = (int64_t)blockIdx.x * kPer + wave / SPLIT;
    const int part = wave % SPLIT;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    int32_t r0 = 0, c0 = 0;
    if (b < nnzb) {
        r0 = 16 * row[b];
        c0 = 16 * col[b];
        // rows past the edge read the last one; their results are not kept
        const T* pd = dz + (int64_t)min(r0 + li, M - 1) * N;
        const T* px = x + (int64_t)min(c0 + li, K - 1) * N;
        const int64_t steps = (N + kStep - 1) / kStep;
        const int64_t lo = steps * part / SPLIT, hi = steps * (part + 1) / SPLIT;
        for (int64_t st = lo; st < hi; ++st) {
            const int64_t n = st * kStep + V * g;
            uint32_t a[4] = {0, 0, 0, 0}, d[4] = {0, 0, 0, 0};
            if (n + V <= N) {
                const auto va = global_load<T, V>(px + n), vd = global_load<T, V>(pd + n);
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = va.d[i], d[i] = vd.d[i];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (n + i < N) {
                        const uint32_t ua = global_load<T, 1>(px + n + i).d[0], ud = global_load<T, 1>(pd + n + i).d[0];
                        if constexpr (is_f32<T>) {
                            a[i] = ua, d[i] = ud;
                        } else {
                            a[i / 2] |= ua << (16 * (i % 2)), d[i / 2] |= ud << (16 * (i % 2));
                        }
                    }
            }
            if constexpr (is_f32<T>) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc = mfma32(a[i], d[i], acc);
            } else {
                acc = mfma16<T>(u32x4_t{a[0], a[1], a[2], a[3]}, u32x4_t{d[0], d[1], d[2], d[3]}, acc);
            }
        }
    }
    if constexpr (SPLIT > 1) {
        __shared__ float4_t red[kPer][SPLIT][64];
        red[wave / SPLIT][part][lane] = acc;
        __syncthreads();
        if (part > 0) return;
        for (int p = 1; p < SPLIT; ++p) acc += red[wave / SPLIT][p][lane];
    }
    if (b >= nnzb) return;
    // lane: row li of the block, columns 4 g .. + 3
    Pack<T, 4> o;
#pragma unroll
    for (int q = 0; q < 4; ++q) o.v[q] = (T)(r0 + li < M && c0 + 4 * g + q < K ? acc[q] : 0.f);
    *reinterpret_cast<Pack<T, 4>*>(dvals + b * 256 + li * 16 + 4 * g) = o;
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

template <typename T>
void sampled_product(const BlockIndex& w, const T* dz, const T* x, T* dvals, int64_t N, hipStream_t s)
{
    if (w.nnzb == 0) return;
    if (w.nnzb < 4096 && N >= 512)
        hipLaunchKernelGGL((ff::ff_sampled_kernel<T, 4>), dim3((unsigned)w.nnzb), dim3(256), 0, s, w.row, w.col, dz, x,
                           dvals, w.nnzb, (int32_t)w.M, (int32_t)w.K, N);
    else
        hipLaunchKernelGGL((ff::ff_sampled_kernel<T, 1>), dim3((unsigned)((w.nnzb + 3) / 4)), dim3(256), 0, s, w.row,
                           w.col, dz, x, dvals, w.nnzb, (int32_t)w.M, (int32_t)w.K, N);
    XSPMM_LAUNCH_CHECK();
}

#define XSPMM_FF_GRAD(T)                                                                                            \
    template void activation_backward<T>(const T*, const T*, const T*, T*, T*, T*, T*, int, int64_t, int64_t,       \
                                         hipStream_t);                                                              \
    template void sampled_product<T>(const BlockIndex&, const T*, const T*, T*, int64_t, hipStream_t);
XSPMM_FF_GRAD(float)
XSPMM_FF_GRAD(_Float16)
XSPMM_FF_GRAD(__bf16)
#undef XSPMM_FF_GRAD

}  // namespace detail
}  // namespace xspmm
