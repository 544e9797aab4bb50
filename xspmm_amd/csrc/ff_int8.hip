// ff_int8.hip -- values to whole numbers of 8 bits:
//
//   weight   q = round(127 v / m), scale = m / 127, m the largest |v| of a row's
//            stored values
//   tokens   the same of every token's features (columns of x)
//
// Rounding is half to even of the quotient itself, whatever a division in 32 bits
// would make of it; 127 m / m is exact, so |q| <= 127.  A row or token that holds an
// infinity or a NaN has the scale NaN and zeros; one of zeros has the scale 0.
//
// Tokens are bound by memory: x is read for the maxima and once more for the
// quotients, where it fits in the caches behind the first pass.
#include "feed_forward_device.hpp"
#include "int8.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// The largest of |v|, as bits: whole numbers order them with the infinities and
// the NaNs, of which one stays, on top.
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
constexpr uint32_t kInfinite = 0x7f800000u;

struct Rounding {
    float most, by;  // 127 / most
    bool none;       // nothing to round: zeros, or no finite maximum

    Rounding() = default;
    __device__ __forceinline__ explicit Rounding(uint32_t bits)
        : most(__builtin_bit_cast(float, bits)), none(bits == 0u || bits >= kInfinite)
    {
        by = 127.f / most;
    }
    __device__ __forceinline__ float scale() const
    {
        return most == 0.f ? 0.f : none ? __builtin_nanf("") : most / 127.f;
    }
    // v / most is off by at most 2 * 2^-24 relative, |q| * 2^-23 < 2^-16; nearer than
    // that to a border (or where 127 / most is infinite) 64 bits decide: the quotient of
    // two 24-bit numbers, times 127, is a border itself or farther from one than 2^-33.
    __device__ __forceinline__ int operator()(float v) const
    {
        if (none) return 0;
        const float t = v * by, k = rintf(t);
        if (!(fabsf(fabsf(t - k) - 0.5f) > 0x1p-15f && fabsf(t) < 128.f)) {
            return (int)rint((double)v * 127.0 / (double)most);
        }
        return (int)k;
    }
};

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d)
{
    return ((uint32_t)a & 0xffu) | (((uint32_t)b & 0xffu) << 8) | (((uint32_t)c & 0xffu) << 16) | ((uint32_t)d << 24);
}

// A workgroup per block-row, a thread per four values of a block, sixteen waves'
// worth of blocks at a time.
template <typename T>
__global__ __launch_bounds__(256) void ff_int8_weight_kernel(const int32_t* __restrict__ ptr,
                                                             const int32_t* __restrict__ col,
                                                             const T* __restrict__ vals, int8_t* __restrict__ q,
                                                             float* __restrict__ scale, int32_t M, int32_t K)
{
    __shared__ uint32_t most[4][16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int r = lane >> 2, c = 4 * (lane & 3);  // a wave's lanes cover one block
    const int32_t br = (int32_t)blockIdx.x, b0 = ptr[br], b1 = ptr[br + 1];
    const bool row_in = 16 * br + r < M;
    auto load = [&](int32_t b, float(&v)[4]) {
        const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4>*>(vals + (int64_t)b * 256 + 4 * lane);
        const int32_t k = 16 * col[b] + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = row_in && k + i < K ? (float)p.v[i] : 0.f;
    };
    uint32_t m = 0;
    for (int32_t b = b0 + wave; b < b1; b += 4) {
        float v[4];
        load(b, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, magnitude(v[i]));
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    if ((lane & 3) == 0) most[wave][r] = m;
    __syncthreads();
    m = max(max(most[0][r], most[1][r]), max(most[2][r], most[3][r]));
    const Rounding round(m);
    if (wave == 0 && (lane & 3) == 0 && row_in) scale[16 * br + r] = round.scale();
    for (int32_t b = b0 + wave; b < b1; b += 4) {
        float v[4];
        load(b, v);
        *reinterpret_cast<uint32_t*>(q + (int64_t)b * 256 + 4 * lane) =
            pack4(round(v[0]), round(v[1]), round(v[2]), round(v[3]));
    }
}

// Tiles of LT * VEC tokens, LT threads along them; the others take blocks of 16
// features in turn.
template <typename T, int VEC>
__device__ __forceinline__ void load_features(const T* x, int64_t K, int64_t N, int64_t kb, int64_t n,
                                              float (&v)[16][VEC])
{
    using P = Pack<T, VEC>;
    if (16 * kb + 16 <= K) {
        P p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = *reinterpret_cast<const P*>(x + (16 * kb + i) * N + n);
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int c = 0; c < VEC; ++c) v[i][c] = (float)p[i].v[c];
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = 16 * kb + i < K;
            const P p = *reinterpret_cast<const P*>(x + (in ? 16 * kb + i : K - 1) * N + n);
#pragma unroll
            for (int c = 0; c < VEC; ++c) v[i][c] = in ? (float)p.v[c] : 0.f;
        }
    }
}

template <int VEC>
__device__ __forceinline__ void store_features(int8_t* q, int64_t N, int64_t kb, int64_t n, const float (&v)[16][VEC],
                                               const Rounding* round)
{
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = pack4(round[c](v[4 * i][c]), round[c](v[4 * i + 1][c]), round[c](v[4 * i + 2][c]),
                         round[c](v[4 * i + 3][c]));
        *reinterpret_cast<u32x4_t*>(q + ((int64_t)kb * N + n + c) * 16) = w;
    }
}

// The largest of `m` over the threads of a column tile that have the same tokens.
template <int THREADS, int LT, int VEC>
__device__ __forceinline__ void join(uint32_t (&m)[VEC], uint32_t* red)
{
    const int t = threadIdx.x;
#pragma unroll
    for (int c = 0; c < VEC; ++c)
#pragma unroll
        for (int d = LT; d < 64; d *= 2) m[c] = max(m[c], (uint32_t)__shfl_xor((int)m[c], d));
    constexpr int kWaves = THREADS / 64;
    const int lane = t & 63, wave = t >> 6;
    if (lane < LT)
#pragma unroll
        for (int c = 0; c < VEC; ++c) red[(wave * LT + lane) * VEC + c] = m[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
        m[c] = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m[c] = max(m[c], red[(w * LT + (t % LT)) * VEC + c]);
    }
}

// The first token of a thread; the last tile moves back into the matrix.
template <int LT, int VEC>
__device__ __forceinline__ int64_t first_token(int64_t tile, int64_t N)
{
    const int64_t n = (tile * LT + threadIdx.x % LT) * VEC;
    return n + VEC <= N ? n : N - VEC;
}

template <typename T, int VEC, int LT>
__global__ __launch_bounds__(1024) void ff_tokens_whole_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                               float* __restrict__ scale, int64_t K, int64_t N)
{
    __shared__ uint32_t red[16 * LT * VEC];
    const int64_t n = first_token<LT, VEC>(blockIdx.x, N), Kb = (K + 15) / 16;
    float v[16][VEC];
    uint32_t m[VEC] = {};
    for (int64_t kb = threadIdx.x / LT; kb < Kb; kb += 1024 / LT) {
        load_features<T, VEC>(x, K, N, kb, n, v);
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int c = 0; c < VEC; ++c) m[c] = max(m[c], magnitude(v[i][c]));
    }
    join<1024, LT, VEC>(m, red);
    const Rounding round[1] = {Rounding(m[0])};
    static_assert(VEC == 1);
    if (threadIdx.x < LT) scale[n] = round[0].scale();
    for (int64_t kb = threadIdx.x / LT; kb < Kb; kb += 1024 / LT) {
        load_features<T, VEC>(x, K, N, kb, n, v);
        store_features<VEC>(q, N, kb, n, v, round);
    }
}

// part[slice][n]: bits of the largest magnitude of a slice of the features
template <typename T, int VEC, int LT>
__global__ __launch_bounds__(256) void ff_tokens_most_kernel(const T* __restrict__ x, uint32_t* __restrict__ part,
                                                             int64_t K, int64_t N, int32_t slices)
{
    __shared__ uint32_t red[4 * LT * VEC];
    const int64_t tile = blockIdx.x / slices, s = blockIdx.x % slices, Kb = (K + 15) / 16;
    const int64_t n = first_token<LT, VEC>(tile, N);
    float v[16][VEC];
    uint32_t m[VEC] = {};
    const int64_t end = Kb * (s + 1) / slices;
    for (int64_t kb = Kb * s / slices + threadIdx.x / LT; kb < end; kb += 256 / LT) {
        load_features<T, VEC>(x, K, N, kb, n, v);
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int c = 0; c < VEC; ++c) m[c] = max(m[c], magnitude(v[i][c]));
    }
    join<256, LT, VEC>(m, red);
    if (threadIdx.x < LT)
#pragma unroll
        for (int c = 0; c < VEC; ++c) part[s * N + n + c] = m[c];
}

template <typename T, int VEC, int LT>
__global__ __launch_bounds__(256) void ff_tokens_round_kernel(const T* __restrict__ x,
                                                              const uint32_t* __restrict__ part,
                                                              int8_t* __restrict__ q, float* __restrict__ scale,
                                                              int64_t K, int64_t N, int32_t slices)
{
    __shared__ uint32_t red[4 * LT * VEC];
    const int64_t tile = blockIdx.x / slices, s = blockIdx.x % slices, Kb = (K + 15) / 16;
    const int64_t n = first_token<LT, VEC>(tile, N);
    uint32_t m[VEC] = {};
    for (int32_t p = threadIdx.x / LT; p < slices; p += 256 / LT)
#pragma unroll
        for (int c = 0; c < VEC; ++c) m[c] = max(m[c], part[p * N + n + c]);
    join<256, LT, VEC>(m, red);
    Rounding round[VEC] = {};
#pragma unroll
    for (int c = 0; c < VEC; ++c) round[c] = Rounding(m[c]);
    if (s == 0 && threadIdx.x < LT)
#pragma unroll
        for (int c = 0; c < VEC; ++c) scale[n + c] = round[c].scale();
    const int64_t end = Kb * (s + 1) / slices;
    float v[16][VEC];
    for (int64_t kb = Kb * s / slices + threadIdx.x / LT; kb < end; kb += 256 / LT) {
        load_features<T, VEC>(x, K, N, kb, n, v);
        store_features<VEC>(q, N, kb, n, v, round);
    }
}

struct TokenPlan {
    bool whole;  // one launch, a workgroup to a tile
    int vec, lanes;
    int64_t tiles;
    int32_t slices;
};

TokenPlan token_plan(int64_t K, int64_t N)
{
    TokenPlan p{};
    const int64_t Kb = (K + 15) / 16;
    p.lanes = N == 1 ? 1 : N < 64 ? 16 : 64;
    p.vec = 1;
    auto tiles = [&](int lanes, int vec) { return (N + lanes * vec - 1) / (lanes * vec); };
    p.whole = N < 64 ? Kb * p.lanes <= 8 * 1024 : N <= 1024 && Kb <= 64;
    if (p.whole) {
        if (N >= 64) p.lanes = 16;
        p.tiles = tiles(p.lanes, 1);
        return p;
    }
    if (N >= 512) p.vec = 4;
    p.tiles = tiles(p.lanes, p.vec);
    const int64_t want = (1024 + p.tiles - 1) / p.tiles, most = (Kb + 256 / p.lanes - 1) / (256 / p.lanes);
    p.slices = (int32_t)(want < most ? want : most);
    return p;
}

template <typename T, int VEC, int LT>
void launch_tokens(const T* x, int8_t* q, float* scale, int64_t K, int64_t N, void* scratch, const TokenPlan& p,
                   hipStream_t s)
{
    uint32_t* part = static_cast<uint32_t*>(scratch);
    const dim3 grid = launch_grid(p.tiles * p.slices, 256);
    hipLaunchKernelGGL((ff_tokens_most_kernel<T, VEC, LT>), grid, dim3(256), 0, s, x, part, K, N, p.slices);
    hipLaunchKernelGGL((ff_tokens_round_kernel<T, VEC, LT>), grid, dim3(256), 0, s, x, part, q, scale, K, N, p.slices);
    XSPMM_LAUNCH_CHECK();
}

}  // namespace ff

template <typename T>
void int8_weight(const BlockIndex& w, const T* vals, int8_t* q, float* scale, hipStream_t s)
{
    if (w.Mb == 0) return;
    hipLaunchKernelGGL((ff::ff_int8_weight_kernel<T>), launch_grid(w.Mb, 256), dim3(256), 0, s, w.ptr, w.col, vals, q,
                       scale, (int32_t)w.M, (int32_t)w.K);
    XSPMM_LAUNCH_CHECK();
}

int64_t quantize_tokens_scratch(int64_t K, int64_t N)
{
    if (K == 0 || N == 0) return 0;
    const ff::TokenPlan p = ff::token_plan(K, N);
    return p.whole ? 0 : (int64_t)p.slices * N * 4;
}

namespace ff {
__global__ __launch_bounds__(256) void ff_zero_scale_kernel(float* __restrict__ scale, int64_t N)
{
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n < N) scale[n] = 0.f;
}
}  // namespace ff

template <typename T>
void quantize_tokens(const T* x, int8_t* q, float* scale, int64_t K, int64_t N, void* scratch, hipStream_t s)
{
    if (N == 0) return;
    if (K == 0) {  // tokens without features: nothing but zeros
        hipLaunchKernelGGL(ff::ff_zero_scale_kernel, launch_grid((N + 255) / 256, 256), dim3(256), 0, s, scale, N);
        XSPMM_LAUNCH_CHECK();
        return;
    }
    const ff::TokenPlan p = ff::token_plan(K, N);
    if (p.whole) {
        const dim3 grid = launch_grid(p.tiles, 1024);
        if (p.lanes == 1)
            hipLaunchKernelGGL((ff::ff_tokens_whole_kernel<T, 1, 1>), grid, dim3(1024), 0, s, x, q, scale, K, N);
        else
            hipLaunchKernelGGL((ff::ff_tokens_whole_kernel<T, 1, 16>), grid, dim3(1024), 0, s, x, q, scale, K, N);
        XSPMM_LAUNCH_CHECK();
        return;
    }
    if (p.vec == 4)
        ff::launch_tokens<T, 4, 64>(x, q, scale, K, N, scratch, p, s);
    else if (p.lanes == 64)
        ff::launch_tokens<T, 1, 64>(x, q, scale, K, N, scratch, p, s);
    else if (p.lanes == 16)
        ff::launch_tokens<T, 1, 16>(x, q, scale, K, N, scratch, p, s);
    else
        ff::launch_tokens<T, 1, 1>(x, q, scale, K, N, scratch, p, s);
}

#define XSPMM_INT8(T)                                                                            \
    template void int8_weight<T>(const BlockIndex&, const T*, int8_t*, float*, hipStream_t);       \
    template void quantize_tokens<T>(const T*, int8_t*, float*, int64_t, int64_t, void*, hipStream_t);
XSPMM_INT8(float)
XSPMM_INT8(_Float16)
XSPMM_INT8(__bf16)
#undef XSPMM_INT8

}  // namespace detail
}  // namespace xspmm
