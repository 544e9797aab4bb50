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
//
// Both passes are bound by memory: x (backward: x and dy) is read twice, as no
// workgroup can hold a column tile wide enough for whole lines of memory, the second
// time from the cache that sits before HBM where it fits.  Forward, fp16 4096 x
// 2048: 7.2 + 9.2 us, 2.3 and 3.6 TB/s, of which launch and first latency are about 5
// (columns held in registers, 16 tokens a workgroup: 20).  Backward, bf16 4096 x
// 8001: 30 + 31 us, 4.4 and 6.3 TB/s.
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

constexpr int kForwardWaves = 8, kBackwardWaves = 8;

// count (the same for all V columns), means, sums of squared deviations
template <int V>
struct Moments {
    float n, m[V], s[V];
};

// d * weight first: where a part is empty that is zero, and d * d may be past fp32's range.
template <int V>
__device__ __forceinline__ void join(Moments<V>& a, const Moments<V>& b)
{
    const float n = a.n + b.n;
    const float share = n > 0.f ? b.n / n : 0.f, weight = a.n * share;
    a.n = n;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float d = b.m[i] - a.m[i];
        a.m[i] += d * share;
        a.s[i] += b.s[i] + d * (d * weight);
    }
}

// A lane's V tokens start at min(n, N - V): no load or store needs a condition
// (one on a load makes the wave wait for it before the next), and the lanes at
// the end do the same work for the same tokens.  Where they would count twice,
// own() leaves a lane its tokens from n on.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_tokens(const T* p)
{
    return *reinterpret_cast<const Pack<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void store_tokens(T* p, const float (&v)[V])
{
    Pack<T, V> q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = (T)v[i];
    *reinterpret_cast<Pack<T, V>*>(p) = q;
}

__device__ __forceinline__ bool own(int64_t n, int64_t at, int64_t N, int i) { return at + i >= n && at + i < N; }

// Moments of rows [k0, k1) step `step` of the lane's columns, kU rows at a
// time: mean and deviations of those first, then joined.  x is at the lane's
// first token.
template <typename T, int V>
__device__ __forceinline__ Moments<V> column_moments(const T* x, int64_t k0, int64_t k1, int64_t step, int64_t N)
{
    constexpr int kU = V >= 4 ? 8 : 16;
    Moments<V> all;
    all.n = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) all.m[i] = all.s[i] = 0.f;
    for (int64_t k = k0; k < k1; k += kU * step) {
        Pack<T, V> raw[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) raw[u] = load_tokens<T, V>(x + min(k + u * step, k1 - 1) * N);
        const int64_t left = (k1 - k + step - 1) / step;
        Moments<V> mo;
        mo.n = left < kU ? (float)left : (float)kU;
        const float inv = 1.f / mo.n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < kU; ++u) sum += u < left ? (float)raw[u].v[i] : 0.f;
            mo.m[i] = sum * inv;
            mo.s[i] = 0.f;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const float d = u < left ? (float)raw[u].v[i] - mo.m[i] : 0.f;
                mo.s[i] += d * d;
            }
        }
        join(all, mo);
    }
    return all;
}

// Joins the lanes of a wave that hold the same columns, then the waves (LDS:
// [waves][np]); the first wave's first np lanes have the result.
template <int V, int WAVES>
__device__ __forceinline__ void join_workgroup(Moments<V>& mo, int np, Moments<V>* red)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = np; d < 64; d <<= 1) {
        Moments<V> o;
        o.n = __shfl_down(mo.n, d, 64);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            o.m[i] = __shfl_down(mo.m[i], d, 64);
            o.s[i] = __shfl_down(mo.s[i], d, 64);
        }
        join(mo, o);
    }
    if (lane < np) red[wave * np + lane] = mo;
    __syncthreads();
    if (wave == 0 && lane < np)
#pragma unroll
        for (int w = 1; w < WAVES; ++w) join(mo, red[w * np + lane]);
}

__device__ __forceinline__ float rstd_of(float s, float K, float eps) { return 1.f / sqrtf(s / K + eps); }

template <typename T, int V>
__global__ __launch_bounds__(64 * kForwardWaves) void ln_stats_kernel(const T* __restrict__ x, float2* __restrict__ part,
                                                                   int64_t K, int64_t N, NormShape h)
{
    __shared__ Moments<V> red[kForwardWaves * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x / h.slices, slice = blockIdx.x % h.slices;
    const int64_t at = min((tile * h.np + lane % h.np) * V, N - V);
    const int64_t k0 = slice * h.len, k1 = min(K, k0 + h.len);
    const int per = 64 / h.np;
    Moments<V> mo = column_moments<T, V>(x + at, k0 + wave * per + lane / h.np, k1, kForwardWaves * per, N);
    join_workgroup<V, kForwardWaves>(mo, h.np, red);
    if (wave == 0 && lane < h.np)
#pragma unroll
        for (int i = 0; i < V; ++i) part[slice * N + at + i] = float2{mo.m[i], mo.s[i]};
}

// U rows of a lane on their way: its tokens, weight and bias
template <typename T, int V, int U>
struct Rows {
    Pack<T, V> raw[U];
    T w[U], b[U];

    // x at the lane's first token
    __device__ __forceinline__ void load(const T* x, const T* wp, const T* bp, int64_t k, int64_t k1, int64_t step,
                                         int64_t N)
    {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = min(k + u * step, k1 - 1);
            raw[u] = load_tokens<T, V>(x + q * N);
            w[u] = wp ? wp[q] : (T)1.f;
            b[u] = bp ? bp[q] : (T)0.f;
        }
    }
    __device__ __forceinline__ void store(T* y, const float (&m)[V], const float (&r)[V], int64_t k, int64_t k1,
                                          int64_t step, int64_t N) const
    {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + u * step >= k1) break;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = ((float)raw[u].v[i] - m[i]) * r[i] * (float)w[u] + (float)b[u];
            store_tokens<T, V>(y + (k + u * step) * N, v);
        }
    }
};

// Every workgroup joins the slices' moments of its columns (a few KB that its
// XCD's L2 holds) rather than waiting for a launch of its own to do it.
template <typename T, int V>
__global__ __launch_bounds__(64 * kForwardWaves) void ln_apply_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                   const T* __restrict__ b,
                                                                   const float2* __restrict__ part, float eps,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   T* __restrict__ y, int64_t K, int64_t N, NormShape h)
{
    constexpr int kThreads = 64 * kForwardWaves;
    __shared__ Moments<1> red[kThreads];
    __shared__ float2 stats[64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x / h.slices, slice = blockIdx.x % h.slices;
    const int per = 64 / h.np;
    const int64_t at = min((tile * h.np + lane % h.np) * V, N - V);
    const int64_t k1 = min(K, (slice + 1) * h.len), step = kForwardWaves * per;
    int64_t k = slice * h.len + wave * per + lane / h.np;
    constexpr int U = V >= 4 ? 8 : 16;
    Rows<T, V, U> rows;
    if (k < k1) rows.load(x + at, w, b, k, k1, step, N);  // under way while the moments are joined
    const int cols = h.np * V, shares = kThreads / cols;
    const int64_t base = max(min(tile * cols, N - cols), (int64_t)0);  // the last tile moves back
    {
        const int c = threadIdx.x % cols, share = threadIdx.x / cols;
        const int64_t col = base + c;
        Moments<1> mo = {0.f, {0.f}, {0.f}};
        if (col < N) {
            for (int64_t s0 = share; s0 < h.slices; s0 += 4 * shares) {
                float2 p[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) p[u] = part[min(s0 + u * shares, h.slices - 1) * N + col];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t s = s0 + u * shares;
                    if (s < h.slices)
                        join(mo, Moments<1>{(float)(min(K, (s + 1) * h.len) - s * h.len), {p[u].x}, {p[u].y}});
                }
            }
        }
        red[threadIdx.x] = mo;
        __syncthreads();
        if (share == 0) {
            for (int q = 1; q < shares; ++q) join(mo, red[q * cols + c]);
            const float r = rstd_of(mo.s[0], (float)K, eps);
            stats[c] = float2{mo.m[0], r};
            if (slice == 0 && mean && col < N) {
                mean[col] = mo.m[0];
                rstd[col] = r;
            }
        }
        __syncthreads();
    }
    float m[V], r[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 q = stats[at - base + i];
        m[i] = q.x;
        r[i] = q.y;
    }
    while (k < k1) {
        rows.store(y + at, m, r, k, k1, step, N);
        k += U * step;
        if (k < k1) rows.load(x + at, w, b, k, k1, step, N);
    }
}

// Few tokens: a workgroup takes all rows of np columns.  Up to kHeld values a
// thread stay in registers between the mean, the deviations and the result;
// beyond that the rows are read again.  One launch, and that is its time: fp16 4096
// features of one token 6.0 us.
constexpr int kSmallWaves = 16;
constexpr int kHeld = 16;

// sums of v over the lanes and waves with the same lane % np, for all of them
__device__ __forceinline__ float sum_workgroup(float v, int np, float* red)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 32; d >= np; d >>= 1) v += __shfl_xor(v, d, 64);
    if (lane < np) red[wave * np + lane] = v;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < kSmallWaves; ++w) all += red[w * np + lane % np];
    __syncthreads();
    return all;
}

template <typename T>
__global__ __launch_bounds__(64 * kSmallWaves) void ln_small_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                    const T* __restrict__ b, float eps,
                                                                    T* __restrict__ y, float* __restrict__ mean,
                                                                    float* __restrict__ rstd, int32_t K, int64_t N,
                                                                    int np)
{
    __shared__ float red[kSmallWaves * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = (int64_t)blockIdx.x * np + lane % np;
    const int32_t per = 64 / np, k0 = wave * per + lane / np, step = kSmallWaves * per;
    const bool there = n < N;
    float v[kHeld];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int64_t k = k0 + (int64_t)u * step;
        v[u] = there && k < K ? (float)x[k * N + n] : 0.f;
        sum += v[u];
    }
    const int64_t rest = k0 + (int64_t)kHeld * step;
    if (there)
        for (int64_t k = rest; k < K; k += step) sum += (float)x[k * N + n];
    const float m = sum_workgroup(sum, np, red) / (float)K;
    sum = 0.f;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const float d = k0 + (int64_t)u * step < K ? v[u] - m : 0.f;
        sum += d * d;
    }
    if (there)
        for (int64_t k = rest; k < K; k += step) {
            const float d = (float)x[k * N + n] - m;
            sum += d * d;
        }
    const float r = rstd_of(sum_workgroup(sum, np, red), (float)K, eps);
    if (!there) return;
    if (mean && threadIdx.x < np) {
        mean[n] = m;
        rstd[n] = r;
    }
    auto put = [&](int64_t k, float xv) {
        const float wk = w ? (float)w[k] : 1.f, bk = b ? (float)b[k] : 0.f;
        y[k * N + n] = (T)((xv - m) * r * wk + bk);
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int64_t k = k0 + (int64_t)u * step;
        if (k < K) put(k, v[u]);
    }
    for (int64_t k = rest; k < K; k += step) put(k, (float)x[k * N + n]);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// The sums over a wave of eight values a lane: lane l returns sum l / 8.
__device__ __forceinline__ float reduce_eight(const float (&q)[8], int lane)
{
    float h4[4], h2[2];
    const bool b5 = lane & 32, b4 = lane & 16, b3 = lane & 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float mine = b5 ? q[4 + i] : q[i], give = b5 ? q[i] : q[4 + i];
        h4[i] = mine + __shfl_xor(give, 32, 64);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float mine = b4 ? h4[2 + i] : h4[i], give = b4 ? h4[i] : h4[2 + i];
        h2[i] = mine + __shfl_xor(give, 16, 64);
    }
    float v = (b3 ? h2[1] : h2[0]) + __shfl_xor(b3 ? h2[0] : h2[1], 8, 64);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// Sums of a slice and a tile: down the columns of g and g h (colpart
// [slices][N]), along the rows of dy h and dy (rowpart [tiles][K]).
template <typename T, int V>
__global__ __launch_bounds__(64 * kBackwardWaves) void ln_backward_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, float2* __restrict__ colpart, float2* __restrict__ rowpart, int64_t K, int64_t N,
    NormShape h)
{
    __shared__ float2 red[kBackwardWaves * 64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x / h.slices, slice = blockIdx.x % h.slices;
    const int64_t n = (tile * h.np + lane % h.np) * V, at = min(n, N - V);
    const int64_t k1 = min(K, (slice + 1) * h.len);
    const int per = 64 / h.np;
    const auto m = load_tokens<float, V>(mean + at), r = load_tokens<float, V>(rstd + at);
    float c1[V], c2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) c1[i] = c2[i] = 0.f;
    // whether every lane of the wave owns all its tokens
    const bool whole = (tile + 1) * h.np * V <= N;
    // Four rows at a time: their eight row sums are reduced across the np lanes
    // together, lanes taking half of the remaining sums each (10 exchanges for
    // np = 64 rather than 48).  Every lane of a wave makes the same rounds.
    const int64_t first = slice * h.len + wave * per;
    const int64_t step = kBackwardWaves * per;
    for (int64_t kb = first; kb < k1; kb += 4 * step) {
        float q[8];  // sums of dy h of the four rows, then of dy
        Pack<T, V> g[4], v[4];
        T wt[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t k = min(kb + lane / h.np + u * step, k1 - 1);
            g[u] = load_tokens<T, V>(dy + k * N + at);
            v[u] = load_tokens<T, V>(x + k * N + at);
            if (w) wt[u] = w[k];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = kb + lane / h.np + u * step < k1;
            const float wk = !in ? 0.f : w ? (float)wt[u] : 1.f;
            float a = 0.f, b = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float gv = (float)g[u].v[i], gh = gv * ((float)v[u].v[i] - m.v[i]) * r.v[i];
                if (!whole && !own(n, at, N, i)) gv = gh = 0.f;
                a += gh;
                b += gv;
                c1[i] += in ? gv * wk : 0.f;
                c2[i] += in ? gh * wk : 0.f;
            }
            q[u] = a;
            q[4 + u] = b;
        }
        if (h.np == 64) {
            const float total = reduce_eight(q, lane);
            // lane 8 i (bits 5, 4, 3 of the lane choose the sum) holds sum i
            const int which = lane >> 3, u = which & 3;
            const int64_t k = kb + u * step;
            if ((lane & 7) == 0 && k < k1) {
                float* o = reinterpret_cast<float*>(rowpart + tile * K + k);
                o[which >> 2] = total;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float a = q[u], b = q[4 + u];
                for (int d = h.np / 2; d > 0; d >>= 1) {
                    a += __shfl_down(a, d, 64);
                    b += __shfl_down(b, d, 64);
                }
                const int64_t k = kb + lane / h.np + u * step;
                if (k < k1 && lane % h.np == 0) rowpart[tile * K + k] = float2{a, b};
            }
        }
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
            for (int q = 1; q < kBackwardWaves; ++q) {
                const float2 o = red[(q * h.np + lane) * V + i];
                c1[i] += o.x;
                c2[i] += o.y;
            }
            if (own(n, at, N, i)) colpart[slice * N + at + i] = float2{c1[i], c2[i]};
        }
}

// sum of p[i * ld], i < n, in order, eight loads at a time
__device__ __forceinline__ float2 sum_strided(const float2* p, int64_t n, int64_t ld)
{
    float a = 0.f, b = 0.f;
    for (int64_t i = 0; i < n; i += 8) {
        float2 q[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) q[u] = p[min(i + u, n - 1) * ld];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            a += i + u < n ? q[u].x : 0.f;
            b += i + u < n ? q[u].y : 0.f;
        }
    }
    return {a, b};
}

// dweight and dbias of row k
template <typename T>
__device__ __forceinline__ void join_row(const float2* __restrict__ rowpart, T* __restrict__ dw, T* __restrict__ db,
                                         int64_t k, int64_t K, int64_t tiles)
{
    const float2 p = sum_strided(rowpart + k, tiles, K);
    if (dw) dw[k] = (T)p.x;
    if (db) db[k] = (T)p.y;
}

// where dx is not wanted
template <typename T>
__global__ __launch_bounds__(64) void ln_backward_rows_kernel(const float2* __restrict__ rowpart, T* __restrict__ dw,
                                                               T* __restrict__ db, int64_t K, int64_t tiles)
{
    const int64_t k = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (k < K) join_row(rowpart, dw, db, k, K, tiles);
}

// As in the forward pass, every workgroup joins the slices' sums of its columns
// itself, and those of its share of the rows (in a launch of its own between the two,
// fp16 16384 x 100 took 33 us and bf16 4096 x 2048 30; so it is 17 and 25).
template <typename T, int V>
__global__ __launch_bounds__(64 * kBackwardWaves) void ln_backward_apply_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float2* __restrict__ colpart, const float2* __restrict__ rowpart,
    T* __restrict__ dx, T* __restrict__ dw, T* __restrict__ db, int64_t K, int64_t N, NormShape h)
{
    constexpr int kThreads = 64 * kBackwardWaves;
    __shared__ float2 red[kThreads];
    __shared__ float2 means[64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x / h.slices, slice = blockIdx.x % h.slices;
    const int64_t at = min((tile * h.np + lane % h.np) * V, N - V);
    const int64_t k1 = min(K, (slice + 1) * h.len);
    const int per = 64 / h.np;
    constexpr int U = 4;
    const int64_t step = kBackwardWaves * per;
    int64_t k = slice * h.len + wave * per + lane / h.np;
    Pack<T, V> g[U], v[U];
    T wt[U];
    auto load = [&] {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = min(k + u * step, k1 - 1);
            g[u] = load_tokens<T, V>(dy + q * N + at);
            v[u] = load_tokens<T, V>(x + q * N + at);
            if (w) wt[u] = w[q];
        }
    };
    if (k < k1) load();  // under way while the sums are joined
    const auto m = load_tokens<float, V>(mean + at), r = load_tokens<float, V>(rstd + at);
    static_assert(64 * V <= kThreads);
    const int cols = h.np * V, shares = kThreads / cols;
    const int64_t base = max(min(tile * cols, N - cols), (int64_t)0);  // the last tile moves back
    {
        const int c = threadIdx.x % cols, share = threadIdx.x / cols;
        const int64_t col = base + c;
        float2 sum = {0.f, 0.f};
        if (col < N && share < h.slices)
            sum = sum_strided(colpart + share * N + col, (h.slices - share + shares - 1) / shares, shares * N);
        red[threadIdx.x] = sum;
        __syncthreads();
        if (share == 0) {
            for (int q = 1; q < shares; ++q) {
                const float2 o = red[q * cols + c];
                sum.x += o.x;
                sum.y += o.y;
            }
            means[c] = float2{sum.x / (float)K, sum.y / (float)K};
        }
        __syncthreads();
    }
    {
        const int64_t rows = (K + gridDim.x - 1) / gridDim.x, end = min(K, (blockIdx.x + 1) * rows);
        for (int64_t q = blockIdx.x * rows + threadIdx.x; q < end; q += kThreads) join_row(rowpart, dw, db, q, K, h.tiles);
    }
    float c1[V], c2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 q = means[at - base + i];
        c1[i] = q.x;
        c2[i] = q.y;
    }
    while (k < k1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + u * step >= k1) break;
            const float wk = w ? (float)wt[u] : 1.f;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i)
                o[i] = ((float)g[u].v[i] * wk - c1[i] - ((float)v[u].v[i] - m.v[i]) * r.v[i] * c2[i]) * r.v[i];
            store_tokens<T, V>(dx + (k + u * step) * N + at, o);
        }
        k += U * step;
        if (k < k1) load();
    }
}

// Few values of at most 64 tokens: one workgroup has every row, np lanes to each,
// and reads dy and x again for dx.  What it saves is a launch, until its one CU takes
// longer than the host (us a call in one launch and in two: fp32 4096 x 2 11.5 and
// 15.1, bf16 16384 x 1 12.0 and 21.1, fp16 4096 x 8 25.8 and 15.0).
constexpr int64_t kSmallBackward = 8192, kOneBackward = 32768;  // values; of a single token
template <typename T>
__global__ __launch_bounds__(64 * kSmallWaves) void ln_small_backward_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ dx, T* __restrict__ dw, T* __restrict__ db, int32_t K, int32_t N,
    int np)
{
    __shared__ float red[kSmallWaves * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t per = 64 / np, step = kSmallWaves * per, col = lane % np;
    const bool own = col < N;
    const int32_t n = own ? col : N - 1;
    const float m = mean[n], r = rstd[n];
    constexpr int U = 8;
    float c1 = 0.f, c2 = 0.f;
    // every lane of a wave makes the same rounds
    for (int32_t first = wave * per; first < K; first += U * step) {
        float g[U], h[U], wk[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int32_t k = min(first + lane / np + u * step, K - 1);
            g[u] = (float)dy[k * N + n];
            h[u] = (float)x[k * N + n];
            wk[u] = w ? (float)w[k] : 1.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int32_t k = first + lane / np + u * step;
            float b = own && k < K ? g[u] : 0.f, a = own && k < K ? g[u] * ((h[u] - m) * r) : 0.f;
            c1 += own && k < K ? g[u] * wk[u] : 0.f;
            c2 += own && k < K ? a * wk[u] : 0.f;
            if (dw || db) {
                for (int d = np / 2; d > 0; d >>= 1) {
                    a += __shfl_down(a, d, 64);
                    b += __shfl_down(b, d, 64);
                }
                if (col == 0 && k < K) {
                    if (dw) dw[k] = (T)a;
                    if (db) db[k] = (T)b;
                }
            }
        }
    }
    if (!dx) return;
    c1 = sum_workgroup(c1, np, red) / (float)K;
    c2 = sum_workgroup(c2, np, red) / (float)K;
    if (!own) return;
    for (int32_t k0 = wave * per + lane / np; k0 < K; k0 += U * step) {
        float g[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int32_t k = min(k0 + u * step, K - 1);
            g[u] = (float)dy[k * N + n] * (w ? (float)w[k] : 1.f);
            v[u] = (float)x[k * N + n];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u * step < K) dx[(k0 + u * step) * N + n] = (T)((g[u] - c1 - (v[u] - m) * r * c2) * r);
    }
}

int pow2_at_least(int64_t n, int most)
{
    int p = 1;
    while (p < most && p < n) p *= 2;
    return p;
}

// size: bytes of an element
NormShape norm_shape(int64_t K, int64_t N, int v, int np, int waves, int64_t groups)
{
    NormShape h{1, v, 0, 0, 0};
    if (N == 0) return h;
    h.np = pow2_at_least((N + v - 1) / v, np);
    h.tiles = (N + h.np * v - 1) / (h.np * v);
    const int64_t rows = waves * (64 / h.np);  // a workgroup's rows at a time
    // about `groups` workgroups of at least 8 rounds
    int64_t slices = (groups + h.tiles - 1) / h.tiles;
    const int64_t most = (K + 8 * rows - 1) / (8 * rows);
    if (slices > most) slices = most;
    if (slices < 1) slices = 1;
    h.len = (K + slices - 1) / slices;
    h.slices = (K + h.len - 1) / h.len;
    return h;
}

// Lanes along the tokens: as many as leave 16 tiles, from 8 to 32 (us with 8, 16 and
// 32: fp16 16384 x 100 14, 16, 16; 4096 x 2048 -, 17, 20; bf16 4096 x 8001, whose rows
// start anywhere in a line, 63, 59, 37).
NormShape forward_shape(int64_t K, int64_t N, int64_t size)
{
    if (N < 64) return norm_shape(K, N, 1, 64, kForwardWaves, 256);
    const int v = (int)(16 / size), np = pow2_at_least(N / (16 * v), 32);
    return norm_shape(K, N, v, np < 8 ? 8 : np, kForwardWaves, 256);
}
// Here from 16 to 64 (us with 16, 32 and 64: f16 4096 x 512 17, 19, 21; 16384 x 1000
// 38, 41, 44; bf16 4096 x 8001 117, 81, 73), and a workgroup a CU (with two 16384 x
// 1000 42 us, 4096 x 8001 76).
NormShape backward_shape(int64_t K, int64_t N, int64_t size)
{
    if (N < 256) return norm_shape(K, N, 1, 64, kBackwardWaves, 256);
    const int v = (int)(16 / size), np = pow2_at_least(N / (16 * v), 64);
    return norm_shape(K, N, v, np < 16 ? 16 : np, kBackwardWaves, 256);
}
// One launch where a workgroup holds its columns, and up to 16 tokens.  us of a
// captured call in one launch and in slices, fp16: 4096 features of 1 token 6.6 and 38,
// of 4 10.9 and 17; but of 8 19 and 13, 16384 features of 4 36 and 17, of 16 71 and 12
// (rows beyond kHeld are read three times, one load at a time).
bool small_norm(int64_t K, int64_t N) { return K * N <= 65536 || N <= 16; }

static_assert(kForwardWaves == kBackwardWaves);
dim3 norm_grid(const NormShape& h) { return launch_grid(h.tiles * h.slices, 64 * kForwardWaves); }

}  // namespace ff

int64_t layer_norm_scratch(int64_t K, int64_t N, int64_t size, int backward)
{
    using namespace ff;
    if (K <= 0 || N <= 0) return 0;
    Carve c;
    if (backward) {
        const NormShape h = backward_shape(K, N, size);
        c.take((size_t)(h.slices * N) * 8);
        c.take((size_t)(h.tiles * K) * 8);
    } else {
        if (small_norm(K, N)) return 0;
        const NormShape h = forward_shape(K, N, size);
        c.take((size_t)(h.slices * N) * 8);
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
        hipLaunchKernelGGL((ln_small_kernel<T>), dim3((unsigned)((N + np - 1) / np)), dim3(64 * kSmallWaves), 0, s, x,
                           weight, bias, eps, y, mean, rstd, (int32_t)K, N, np);
        XSPMM_LAUNCH_CHECK();
        return;
    }
    const NormShape h = forward_shape(K, N, sizeof(T));
    float2* part = static_cast<float2*>(scratch);
    auto go = [&](auto v) {
        constexpr int V = decltype(v)::value;
        hipLaunchKernelGGL((ln_stats_kernel<T, V>), norm_grid(h), dim3(64 * kForwardWaves), 0, s, x, part, K, N, h);
        hipLaunchKernelGGL((ln_apply_kernel<T, V>), norm_grid(h), dim3(64 * kForwardWaves), 0, s, x, weight, bias, part,
                           eps, mean, rstd, y, K, N, h);
    };
    constexpr int most = 16 / sizeof(T);
    if (h.v == most)
        go(std::integral_constant<int, most>{});
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
    if (N > 0 && N <= 64 && K <= (N == 1 ? kOneBackward : kSmallBackward / N)) {
        hipLaunchKernelGGL((ln_small_backward_kernel<T>), dim3(1), dim3(64 * kSmallWaves), 0, s, dy, x, weight, mean,
                           rstd, dx, dweight, dbias, (int32_t)K, (int32_t)N, pow2_at_least(N, 64));
        XSPMM_LAUNCH_CHECK();
        return;
    }
    const NormShape h = backward_shape(K, N, sizeof(T));
    char* p = static_cast<char*>(scratch);
    Carve c;
    float2* colpart = reinterpret_cast<float2*>(p + c.take((size_t)(h.slices * N) * 8));
    float2* rowpart = reinterpret_cast<float2*>(p + c.take((size_t)(h.tiles * K) * 8));
    auto go = [&](auto v) {
        constexpr int V = decltype(v)::value;
        if (N > 0)
            hipLaunchKernelGGL((ln_backward_sums_kernel<T, V>), norm_grid(h), dim3(64 * kBackwardWaves), 0, s, dy, x,
                               weight, mean, rstd, colpart, rowpart, K, N, h);
        if (N > 0 && dx)
            hipLaunchKernelGGL((ln_backward_apply_kernel<T, V>), norm_grid(h), dim3(64 * kBackwardWaves), 0, s, dy, x,
                               weight, mean, rstd, colpart, rowpart, dx, dweight, dbias, K, N, h);
        else if (dweight || dbias)
            hipLaunchKernelGGL((ln_backward_rows_kernel<T>), dim3((unsigned)((K + 63) / 64)), dim3(64), 0, s, rowpart,
                               dweight, dbias, K, h.tiles);
    };
    constexpr int most = 16 / sizeof(T);
    if (h.v == most)
        go(std::integral_constant<int, most>{});
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
