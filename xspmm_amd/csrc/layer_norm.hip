// layer_norm.hip -- layer norm over the features of every token, forward and
// backward, on activations of features x tokens (row-major, K x N):
//
//   y = (x - mean) rstd w + b           mean, rstd of each column
//   g = dy w, h = (x - mean) rstd
//   dx = rstd (g - mean(g) - h mean(g h)),  dw = sum_n dy h,  db = sum_n dy
//
// The sums over the features run down the columns, so a workgroup takes a slice
// of the rows for a tile of columns, and the slices' results are joined.  The
// forward variance is joined from the mean and the squared deviations of parts
// (n, m, M2): n = na + nb, d = mb - ma, m = ma + d nb / n,
// M2 = M2a + M2b + d^2 na nb / n, which loses nothing where a feature is far
// off the others.  All sums are fp32, in a fixed order.
#include "feed_forward_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// How a wave covers a tile: np lanes along the tokens, V tokens each, and
// 64 / np rows at a time.
struct NormShape {
    int np;           // power of two, at most 64
    int v;            // tokens per lane
    int64_t tiles;    // of np * v columns
    int64_t slices;   // of the rows
    int64_t len;      // rows per slice
};

constexpr int kNormWaves = 4;

struct Moments {
    float n, m, s;  // count, mean, sum of squared deviations
};

__device__ __forceinline__ Moments join(Moments a, Moments b)
{
    const float n = a.n + b.n;
    if (n == 0.f) return a;
    const float d = b.m - a.m, share = b.n / n;
    return {n, a.m + d * share, a.s + b.s + d * d * a.n * share};
}

template <typename T, int V>
__device__ __forceinline__ void load_tokens(float (&v)[V], const T* p, int64_t n, int64_t N)
{
    if (n + V <= N) {
        const auto q = *reinterpret_cast<const Pack<T, V>*>(p + n);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)q.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = n + i < N ? (float)p[n + i] : 0.f;
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_tokens(T* p, const float (&v)[V], int64_t n, int64_t N)
{
    if (n + V <= N) {
        Pack<T, V> q;
#pragma unroll
        for (int i = 0; i < V; ++i) q.v[i] = (T)v[i];
        *reinterpret_cast<Pack<T, V>*>(p + n) = q;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (n + i < N) p[n + i] = (T)v[i];
    }
}

// Moments of rows [k0 + sub, k1) step `step` of the lane's columns, kU rows at
// a time: mean and deviations of those first, then joined.
template <typename T, int V>
__device__ __forceinline__ void column_moments(Moments (&mo)[V], const T* x, int64_t k0, int64_t k1, int64_t step,
                                               int64_t n, int64_t N)
{
    constexpr int kU = 8;
#pragma unroll
    for (int i = 0; i < V; ++i) mo[i] = {0.f, 0.f, 0.f};
    if (n >= N) return;
    for (int64_t k = k0; k < k1; k += kU * step) {
        float v[kU][V];
        float count = 0.f;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int64_t r = k + u * step;
            if (r < k1) {
                load_tokens<T, V>(v[u], x + r * N, n, N);
                count += 1.f;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[u][i] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < kU; ++u) sum += v[u][i];
            const float m = sum / count;
            float s = 0.f;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const float d = k + u * step < k1 ? v[u][i] - m : 0.f;
                s += d * d;
            }
            mo[i] = join(mo[i], {count, m, s});
        }
    }
}

// Joins the lanes of a wave that hold the same columns, then the waves (LDS:
// [waves][np * V]); the first wave's first np lanes have the result.
template <int V, int WAVES>
__device__ __forceinline__ void join_workgroup(Moments (&mo)[V], int np, Moments* red)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = np; d < 64; d <<= 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const Moments o = {__shfl_down(mo[i].n, d, 64), __shfl_down(mo[i].m, d, 64), __shfl_down(mo[i].s, d, 64)};
            mo[i] = join(mo[i], o);
        }
    }
    if (lane < np)
#pragma unroll
        for (int i = 0; i < V; ++i) red[(wave * np + lane) * V + i] = mo[i];
    __syncthreads();
    if (wave == 0 && lane < np)
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int i = 0; i < V; ++i) mo[i] = join(mo[i], red[(w * np + lane) * V + i]);
}

template <typename T, int V>
__global__ __launch_bounds__(64 * kNormWaves) void ln_stats_kernel(const T* __restrict__ x, float2* __restrict__ part,
                                                                   int64_t K, int64_t N, NormShape h)
{
    __shared__ Moments red[kNormWaves * 64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x % h.tiles, slice = blockIdx.x / h.tiles;
    const int64_t n = (tile * h.np + lane % h.np) * V;
    const int64_t k0 = slice * h.len, k1 = min(K, k0 + h.len);
    const int per = 64 / h.np;
    Moments mo[V];
    column_moments<T, V>(mo, x, k0 + wave * per + lane / h.np, k1, kNormWaves * per, n, N);
    join_workgroup<V, kNormWaves>(mo, h.np, red);
    if (wave == 0 && lane < h.np)
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (n + i < N) part[slice * N + n + i] = float2{mo[i].m, mo[i].s};
}

__device__ __forceinline__ float rstd_of(float s, float K, float eps) { return 1.f / sqrtf(s / K + eps); }

__global__ __launch_bounds__(256) void ln_join_kernel(const float2* __restrict__ part, float* __restrict__ mean,
                                                      float* __restrict__ rstd, int64_t K, int64_t N, NormShape h,
                                                      float eps)
{
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    Moments mo = {0.f, 0.f, 0.f};
    for (int64_t s = 0; s < h.slices; ++s) {
        const float2 p = part[s * N + n];
        mo = join(mo, {(float)(min(K, (s + 1) * h.len) - s * h.len), p.x, p.y});
    }
    mean[n] = mo.m;
    rstd[n] = rstd_of(mo.s, (float)K, eps);
}

template <typename T, int V>
__device__ __forceinline__ void normalize(const T* x, const T* w, const T* b, T* y, const float (&m)[V],
                                          const float (&r)[V], int64_t k0, int64_t k1, int64_t step, int64_t n,
                                          int64_t N)
{
    if (n >= N) return;
#pragma unroll 4
    for (int64_t k = k0; k < k1; k += step) {
        float v[V];
        load_tokens<T, V>(v, x + k * N, n, N);
        const float wk = w ? (float)w[k] : 1.f, bk = b ? (float)b[k] : 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (v[i] - m[i]) * r[i] * wk + bk;
        store_tokens<T, V>(y + k * N, v, n, N);
    }
}

template <typename T, int V>
__global__ __launch_bounds__(64 * kNormWaves) void ln_apply_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                   const T* __restrict__ b,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, T* __restrict__ y,
                                                                   int64_t K, int64_t N, NormShape h)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x % h.tiles, slice = blockIdx.x / h.tiles;
    const int64_t n = (tile * h.np + lane % h.np) * V;
    const int64_t k0 = slice * h.len, k1 = min(K, k0 + h.len);
    const int per = 64 / h.np;
    float m[V], r[V];
    load_tokens<float, V>(m, mean, n, N);
    load_tokens<float, V>(r, rstd, n, N);
    normalize<T, V>(x, w, b, y, m, r, k0 + wave * per + lane / h.np, k1, kNormWaves * per, n, N);
}

// Few tokens: a workgroup takes all rows of a tile, twice.
constexpr int kSmallWaves = 16;
template <typename T, int V>
__global__ __launch_bounds__(64 * kSmallWaves) void ln_small_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                    const T* __restrict__ b, float eps,
                                                                    T* __restrict__ y, float* __restrict__ mean,
                                                                    float* __restrict__ rstd, int64_t K, int64_t N,
                                                                    int np)
{
    __shared__ Moments red[kSmallWaves * 64 * V];
    __shared__ float2 stats[64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = ((int64_t)blockIdx.x * np + lane % np) * V;
    const int per = 64 / np;
    const int64_t k0 = wave * per + lane / np, step = kSmallWaves * per;
    Moments mo[V];
    column_moments<T, V>(mo, x, k0, K, step, n, N);
    join_workgroup<V, kSmallWaves>(mo, np, red);
    if (wave == 0 && lane < np)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float r = rstd_of(mo[i].s, (float)K, eps);
            stats[lane * V + i] = float2{mo[i].m, r};
            if (mean && n + i < N) {
                mean[n + i] = mo[i].m;
                rstd[n + i] = r;
            }
        }
    __syncthreads();
    float m[V], r[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 q = stats[(lane % np) * V + i];
        m[i] = q.x;
        r[i] = q.y;
    }
    normalize<T, V>(x, w, b, y, m, r, k0, K, step, n, N);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// Sums of a slice and a tile: down the columns of g and g h (colpart
// [slices][N]), along the rows of dy h and dy (rowpart [tiles][K]).
template <typename T, int V>
__global__ __launch_bounds__(64 * kNormWaves) void ln_backward_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, float2* __restrict__ colpart, float2* __restrict__ rowpart, int64_t K, int64_t N,
    NormShape h)
{
    __shared__ float2 red[kNormWaves * 64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x % h.tiles, slice = blockIdx.x / h.tiles;
    const int64_t n = (tile * h.np + lane % h.np) * V;
    const int64_t k1 = min(K, (slice + 1) * h.len);
    const int per = 64 / h.np;
    float m[V], r[V], c1[V], c2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) c1[i] = c2[i] = m[i] = r[i] = 0.f;
    if (n < N) {
        load_tokens<float, V>(m, mean, n, N);
        load_tokens<float, V>(r, rstd, n, N);
    }
    // every lane of a wave makes the same rounds: rows are reduced across lanes
    const int64_t first = slice * h.len + wave * per;
    for (int64_t kb = first; kb < k1; kb += kNormWaves * per) {
        const int64_t k = kb + lane / h.np;
        float a = 0.f, b = 0.f;
        if (k < k1 && n < N) {
            float g[V], v[V];
            load_tokens<T, V>(g, dy + k * N, n, N);
            load_tokens<T, V>(v, x + k * N, n, N);
            const float wk = w ? (float)w[k] : 1.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hv = (v[i] - m[i]) * r[i];  // a token past the last has rstd 0 and dy 0
                const float gh = g[i] * hv;
                a += gh;
                b += g[i];
                c1[i] += g[i] * wk;
                c2[i] += gh * wk;
            }
        }
        for (int d = h.np / 2; d > 0; d >>= 1) {
            a += __shfl_down(a, d, 64);
            b += __shfl_down(b, d, 64);
        }
        if (k < k1 && lane % h.np == 0) rowpart[tile * K + k] = float2{a, b};
    }
    for (int d = h.np; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c1[i] += __shfl_down(c1[i], d, 64);
            c2[i] += __shfl_down(c2[i], d, 64);
        }
    if (lane < h.np)
#pragma unroll
        for (int i = 0; i < V; ++i) red[(wave * h.np + lane) * V + i] = float2{c1[i], c2[i]};
    __syncthreads();
    if (wave == 0 && lane < h.np)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            for (int q = 1; q < kNormWaves; ++q) {
                const float2 o = red[(q * h.np + lane) * V + i];
                c1[i] += o.x;
                c2[i] += o.y;
            }
            if (n + i < N) colpart[slice * N + n + i] = float2{c1[i], c2[i]};
        }
}

// workgroups [0, ceil(N / 256)): a column's means; the rest: a row's sums
template <typename T>
__global__ __launch_bounds__(256) void ln_backward_join_kernel(const float2* __restrict__ colpart,
                                                               const float2* __restrict__ rowpart,
                                                               float2* __restrict__ means, T* __restrict__ dw,
                                                               T* __restrict__ db, int64_t K, int64_t N, NormShape h)
{
    const int64_t cols = (N + 255) / 256;
    if (blockIdx.x < cols) {
        const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (n >= N) return;
        float a = 0.f, b = 0.f;
        for (int64_t s = 0; s < h.slices; ++s) {
            const float2 p = colpart[s * N + n];
            a += p.x;
            b += p.y;
        }
        means[n] = float2{a / (float)K, b / (float)K};
    } else {
        const int64_t k = ((int64_t)blockIdx.x - cols) * 256 + threadIdx.x;
        if (k >= K) return;
        float a = 0.f, b = 0.f;
        for (int64_t t = 0; t < h.tiles; ++t) {
            const float2 p = rowpart[t * K + k];
            a += p.x;
            b += p.y;
        }
        if (dw) dw[k] = (T)a;
        if (db) db[k] = (T)b;
    }
}

template <typename T, int V>
__global__ __launch_bounds__(64 * kNormWaves) void ln_backward_apply_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float2* __restrict__ means, T* __restrict__ dx, int64_t K, int64_t N,
    NormShape h)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x % h.tiles, slice = blockIdx.x / h.tiles;
    const int64_t n = (tile * h.np + lane % h.np) * V;
    if (n >= N) return;
    const int64_t k1 = min(K, (slice + 1) * h.len);
    const int per = 64 / h.np;
    float m[V], r[V], c1[V], c2[V];
    load_tokens<float, V>(m, mean, n, N);
    load_tokens<float, V>(r, rstd, n, N);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 p = n + i < N ? means[n + i] : float2{0.f, 0.f};
        c1[i] = p.x;
        c2[i] = p.y;
    }
#pragma unroll 2
    for (int64_t k = slice * h.len + wave * per + lane / h.np; k < k1; k += kNormWaves * per) {
        float g[V], v[V];
        load_tokens<T, V>(g, dy + k * N, n, N);
        load_tokens<T, V>(v, x + k * N, n, N);
        const float wk = w ? (float)w[k] : 1.f;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (g[i] * wk - c1[i] - (v[i] - m[i]) * r[i] * c2[i]) * r[i];
        store_tokens<T, V>(dx + k * N, v, n, N);
    }
}

int pow2_at_least(int64_t n, int most)
{
    int p = 1;
    while (p < most && p < n) p *= 2;
    return p;
}

// size: bytes of an element
NormShape norm_shape(int64_t K, int64_t N, int v)
{
    NormShape h{1, v, 0, 0, 0};
    if (N == 0) return h;
    h.np = pow2_at_least((N + v - 1) / v, 64);
    h.tiles = (N + h.np * v - 1) / (h.np * v);
    const int64_t rows = kNormWaves * (64 / h.np);  // a workgroup's rows at a time
    // about 1024 workgroups of at least 8 rounds
    int64_t slices = (1024 + h.tiles - 1) / h.tiles;
    const int64_t most = (K + 8 * rows - 1) / (8 * rows);
    if (slices > most) slices = most;
    if (slices < 1) slices = 1;
    h.len = (K + slices - 1) / slices;
    h.slices = (K + h.len - 1) / h.len;
    return h;
}

int forward_v(int64_t N) { return N >= 128 ? 2 : 1; }
int backward_v(int64_t N) { return N >= 256 ? 4 : 1; }
bool small_norm(int64_t K, int64_t N) { return K * N <= 65536 || N <= 16; }

dim3 norm_grid(const NormShape& h)
{
    const int64_t g = h.tiles * h.slices;
    if (g > 0x7fffffffLL) throw std::invalid_argument("xSpMM: too many tokens for one launch.");
    return dim3((unsigned)g);
}

}  // namespace ff

int64_t layer_norm_scratch(int64_t K, int64_t N, int backward)
{
    using namespace ff;
    if (K <= 0 || N <= 0) return 0;
    Carve c;
    if (backward) {
        const NormShape h = norm_shape(K, N, backward_v(N));
        c.take((size_t)(h.slices * N) * 8);
        c.take((size_t)(h.tiles * K) * 8);
        c.take((size_t)N * 8);
    } else {
        if (small_norm(K, N)) return 0;
        const NormShape h = norm_shape(K, N, forward_v(N));
        c.take((size_t)(h.slices * N) * 8);
        c.take((size_t)N * 4);
        c.take((size_t)N * 4);
    }
    return (int64_t)c.end;
}

template <typename T>
void layer_norm(const T* x, const T* weight, const T* bias, float eps, T* y, float* mean, float* rstd, int64_t K,
                int64_t N, void* scratch, hipStream_t s)
{
    using namespace ff;
    if (K == 0 || N == 0) return;
    if (small_norm(K, N)) {
        const int np = pow2_at_least(N, 8);
        hipLaunchKernelGGL((ln_small_kernel<T, 1>), dim3((unsigned)((N + np - 1) / np)), dim3(64 * kSmallWaves), 0, s,
                           x, weight, bias, eps, y, mean, rstd, K, N, np);
        XSPMM_LAUNCH_CHECK();
        return;
    }
    const NormShape h = norm_shape(K, N, forward_v(N));
    char* p = static_cast<char*>(scratch);
    Carve c;
    float2* part = reinterpret_cast<float2*>(p + c.take((size_t)(h.slices * N) * 8));
    float* m = reinterpret_cast<float*>(p + c.take((size_t)N * 4));
    float* r = reinterpret_cast<float*>(p + c.take((size_t)N * 4));
    if (mean) m = mean;
    if (rstd) r = rstd;
    auto go = [&](auto v) {
        constexpr int V = decltype(v)::value;
        hipLaunchKernelGGL((ln_stats_kernel<T, V>), norm_grid(h), dim3(64 * kNormWaves), 0, s, x, part, K, N, h);
        hipLaunchKernelGGL(ln_join_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s, part, m, r, K, N, h,
                           eps);
        hipLaunchKernelGGL((ln_apply_kernel<T, V>), norm_grid(h), dim3(64 * kNormWaves), 0, s, x, weight, bias, m, r,
                           y, K, N, h);
    };
    if (h.v == 2)
        go(std::integral_constant<int, 2>{});
    else
        go(std::integral_constant<int, 1>{});
    XSPMM_LAUNCH_CHECK();
}

template <typename T>
void layer_norm_backward(const T* dy, const T* x, const T* weight, const float* mean, const float* rstd, T* dx,
                         T* dweight, T* dbias, int64_t K, int64_t N, void* scratch, hipStream_t s)
{
    using namespace ff;
    if (K == 0) return;
    const NormShape h = norm_shape(K, N, backward_v(N));
    char* p = static_cast<char*>(scratch);
    Carve c;
    float2* colpart = reinterpret_cast<float2*>(p + c.take((size_t)(h.slices * N) * 8));
    float2* rowpart = reinterpret_cast<float2*>(p + c.take((size_t)(h.tiles * K) * 8));
    float2* means = reinterpret_cast<float2*>(p + c.take((size_t)N * 8));
    auto go = [&](auto v) {
        constexpr int V = decltype(v)::value;
        if (N > 0)
            hipLaunchKernelGGL((ln_backward_sums_kernel<T, V>), norm_grid(h), dim3(64 * kNormWaves), 0, s, dy, x,
                               weight, mean, rstd, colpart, rowpart, K, N, h);
        hipLaunchKernelGGL((ln_backward_join_kernel<T>), dim3((unsigned)((N + 255) / 256 + (K + 255) / 256)),
                           dim3(256), 0, s, colpart, rowpart, means, dweight, dbias, K, N, h);
        if (N > 0 && dx)
            hipLaunchKernelGGL((ln_backward_apply_kernel<T, V>), norm_grid(h), dim3(64 * kNormWaves), 0, s, dy, x,
                               weight, mean, rstd, means, dx, K, N, h);
    };
    if (h.v == 4)
        go(std::integral_constant<int, 4>{});
    else
        go(std::integral_constant<int, 1>{});
    XSPMM_LAUNCH_CHECK();
}

#define XSPMM_LAYER_NORM(T)                                                                                          \
    template void layer_norm<T>(const T*, const T*, const T*, float, T*, float*, float*, int64_t, int64_t, void*,    \
                                hipStream_t);                                                                        \
    template void layer_norm_backward<T>(const T*, const T*, const T*, const float*, const float*, T*, T*, T*,       \
                                         int64_t, int64_t, void*, hipStream_t);
XSPMM_LAYER_NORM(float)
XSPMM_LAYER_NORM(_Float16)
XSPMM_LAYER_NORM(__bf16)
#undef XSPMM_LAYER_NORM

}  // namespace detail
}  // namespace xspmm
