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
// quotients, where it fits in the caches behind the first pass: bf16 14336 x 2048 (59 MB)
// 10.9 us (5.4 TB/s) for the maxima and 27 (3.3 TB/s with what it writes) for the
// rounding.  One token of 14336 takes 2.6 us; a weight of 14336 x 4096, 25 % stored, 21.
#include "int8_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// A workgroup per block-row, a wave per block, a thread per four of its values.
constexpr int kWeightWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kWeightWaves) void ff_int8_weight_kernel(const int32_t* __restrict__ ptr,
                                                             const int32_t* __restrict__ col,
                                                             const T* __restrict__ vals, int8_t* __restrict__ q,
                                                             float* __restrict__ scale, int32_t M, int32_t K)
{
    __shared__ uint32_t most[kWeightWaves][16];
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
    for (int32_t b = b0 + wave; b < b1; b += kWeightWaves) {
        float v[4];
        load(b, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, magnitude(v[i]));
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    if ((lane & 3) == 0) most[wave][r] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWeightWaves; ++w) m = max(m, most[w][r]);
    const Rounding round(m);
    if (wave == 0 && (lane & 3) == 0 && row_in) scale[16 * br + r] = round.scale;
    for (int32_t b = b0 + wave; b < b1; b += kWeightWaves) {
        float v[4];
        load(b, v);
        *reinterpret_cast<uint32_t*>(q + (int64_t)b * 256 + 4 * lane) =
            pack4(round_exactly(v[0], round), round_exactly(v[1], round), round_exactly(v[2], round),
                  round_exactly(v[3], round));
    }
}

// Tiles of LT tokens, LT threads along them; the others take blocks of 16 features in
// turn.

// The token of a thread; past the last one that again.
template <int LT>
__device__ __forceinline__ int64_t token_of(int64_t tile, int64_t N)
{
    return min(tile * LT + threadIdx.x % LT, N - 1);
}

// Few tokens: a workgroup to a tile, whose features stay in registers.
constexpr int kKept = 2;  // blocks of features of a thread
template <typename T, int LT>
__global__ __launch_bounds__(1024) void ff_tokens_whole_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                               float* __restrict__ scale, int64_t K, int64_t N)
{
    __shared__ uint32_t red[16 * LT];
    const int64_t n = token_of<LT>(blockIdx.x, N), Kb = (K + 15) / 16;
    float v[kKept][16];
#pragma unroll
    for (int u = 0; u < kKept; ++u) {
        const int64_t kb = threadIdx.x / LT + u * (1024 / LT);
        if (kb < Kb)
            load_features<T>(x, K, N, kb, n, v[u]);
        else
#pragma unroll
            for (int i = 0; i < 16; ++i) v[u][i] = 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < kKept; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, magnitude(v[u][i]));
    join<1024, LT>(m, red);
    const Rounding round(m);
    if (threadIdx.x < LT) scale[n] = round.scale;
#pragma unroll
    for (int u = 0; u < kKept; ++u) {
        const int64_t kb = threadIdx.x / LT + u * (1024 / LT);
        if (kb < Kb) store_features(q, N, kb, n, v[u], round);
    }
}

// A single token: its features are consecutive, and a thread's stay in registers.
constexpr int64_t kOneMost = 16 * 1024;
template <typename T>
__global__ __launch_bounds__(1024) void ff_token_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                        float* __restrict__ scale, int32_t K)
{
    __shared__ uint32_t red[16];
    const int32_t k = 16 * threadIdx.x;
    float v[16] = {};
    if (k + 16 <= K) {
        const Pack<T, 16> p = *reinterpret_cast<const Pack<T, 16>*>(x + k);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = (float)p.v[i];
    } else if (k < K) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = k + i < K ? (float)x[k + i] : 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, magnitude(v[i]));
    join<1024, 1>(m, red);
    const Rounding round(m);
    if (threadIdx.x == 0) scale[0] = round.scale;
    if (k < K) *reinterpret_cast<u32x4_t*>(q + k) = round_features(v, round);
}

// part[slice][n]: bits of the largest magnitude of a slice of the features, of VEC tokens a
// thread (the last of them move back into the matrix)
constexpr int kSliceThreads = 1024;
template <typename T, int VEC, int LT>
__global__ __launch_bounds__(kSliceThreads) void ff_tokens_most_kernel(const T* __restrict__ x, uint32_t* __restrict__ part,
                                                             int64_t K, int64_t N, int32_t slices)
{
    __shared__ uint32_t red[VEC][kSliceThreads / 64 * LT];
    const int64_t tile = blockIdx.x / slices, s = blockIdx.x % slices, Kb = (K + 15) / 16;
    const int64_t n = min((tile * LT + threadIdx.x % LT) * VEC, N - VEC);
    uint32_t m[VEC] = {};
    const int64_t end = Kb * (s + 1) / slices;
    for (int64_t kb = Kb * s / slices + threadIdx.x / LT; kb < end; kb += kSliceThreads / LT) {
        Pack<T, VEC> p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = *reinterpret_cast<const Pack<T, VEC>*>(x + min(16 * kb + i, K - 1) * N + n);
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int c = 0; c < VEC; ++c) m[c] = max(m[c], magnitude((float)p[i].v[c]));
    }
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
        join<kSliceThreads, LT>(m[c], red[c]);
        if (threadIdx.x < LT) part[s * N + n + c] = m[c];
    }
}

// A thread takes one token at a time: 64 of them store 1 KB side by side (with four
// tokens a thread, 64 bytes apart, 31 us instead of 26 at bf16 14336 x 2048).
template <typename T, int LT>
__global__ __launch_bounds__(kSliceThreads) void ff_tokens_round_kernel(const T* __restrict__ x,
                                                                        const uint32_t* __restrict__ part,
                                                                        int8_t* __restrict__ q,
                                                                        float* __restrict__ scale, int64_t K,
                                                                        int64_t N, int32_t slices)
{
    __shared__ uint32_t red[kSliceThreads / 64 * LT];
    const int64_t tile = blockIdx.x / slices, s = blockIdx.x % slices, Kb = (K + 15) / 16;
    const int64_t n = token_of<LT>(tile, N);
    uint32_t m = 0;
    for (int32_t p = threadIdx.x / LT; p < slices; p += kSliceThreads / LT) m = max(m, part[p * N + n]);
    join<kSliceThreads, LT>(m, red);
    const Rounding round(m);
    if (s == 0 && threadIdx.x < LT) scale[n] = round.scale;
    const int64_t end = Kb * (s + 1) / slices;
    for (int64_t kb = Kb * s / slices + threadIdx.x / LT; kb < end; kb += kSliceThreads / LT) {
        float v[16];
        load_features<T>(x, K, N, kb, n, v);
        store_features(q, N, kb, n, v, round);
    }
}

struct TokenPlan {
    bool whole;  // one launch, a workgroup to a tile
    int lanes, vec;   // a tile's threads along the tokens, and a thread's tokens (for the maxima)
    int64_t tiles;
    int32_t slices;
};

// size: bytes of a value.  us of whole tokens by four lanes (4) and sixteen (16), and in slices by
// sixteen (s16) and by 64 (s64), of x that has left L2:
//   bf16   1000 x 2288   15.3 (4), 8.5 (16), 13.9 (s16), 11.7 (s64)
//          1695 x 936     8.7,    13.6,      15.3,       14.7
//          3453 x 414    10.8,                15.2,       14.6
//          5163 x 791    17.7,                21.3,       15.3
//          4705 x 96     12.0,                12.3,       11.1
//          1298 x 5245   31.6,    21.9,      34.0,       17.0
//          862 x 11664   46.5,    23.4,      47.8,       25.8
//   fp32   1936 x 163     7.0 (4), 8.1 (16),  9.5 (s16),   8.5 (s64)
//          788 x 675      8.0,     7.7,      11.8,        9.7
//          1733 x 994    13.5,    10.3,      13.6,       11.0
//          5007 x 89     14.1,               13.6,       12.6
//          6706 x 33     13.9,               10.0
// and of x that stays there: bf16 4999 x 31 8.6 (4), 12.3 (s16), 4096 x 512 13.5 (4), 11.0 (s64).
// Whole tokens read x once; a workgroup then reads every row, of which four lanes use 8 or 16
// bytes, in a time that goes by the features.  Over 862 drawn sizes the rule is 1.5 % slower
// than the fastest way in the mean, 1.1 % where x stays in L2.  Four 16-bit tokens a thread read
// the maxima of more than 48 MB faster (us of one and four: 14336 x 2048 38.2 and 35.7, 10958 x
// 4237 80.4 and 76.1, 15936 x 3067 74.1 and 72.4), of less slower (6991 x 3663 49.8 and 49.9, 5783 x
// 3598 37.9 and 40.9, 9174 x 1943 27.2 and 34.9).
TokenPlan token_plan(int64_t K, int64_t N, int size)
{
    TokenPlan p{};
    const int64_t Kb = (K + 15) / 16;
    if (N == 1) {
        p.lanes = 1;
        p.whole = K <= kOneMost;
    } else if (Kb * 4 <= kKept * 1024 && N <= 1024 && (K * N * size <= 3 << 18 || (size == 2 && Kb <= 220))) {
        p.lanes = 4;
        p.whole = true;
    } else if (Kb <= (size == 4 ? 128 : 96) && N <= 8192) {
        static_assert(128 * 16 <= kKept * 1024);
        p.lanes = 16;
        p.whole = true;
    } else {
        p.lanes = N < 64 ? 16 : 64;
    }
    p.vec = p.lanes == 64 && size == 2 && N >= 256 && K * N > 3 << 23 ? 4 : 1;
    p.tiles = (N + p.lanes * p.vec - 1) / (p.lanes * p.vec);
    if (p.whole) return p;
    // Rounds of a workgroup a CU, filled as far as they can be, in the time of 16 features of a
    // tile, of which a workgroup costs some 24 beside its own (us, bf16): at 5350 x 1385 22
    // tiles by twelve slices, eight workgroups more than CUs, 26.0, by eleven 21.0; at 6661 x
    // 8893 139 tiles by one slice 125, by three 95; at 537 x 9362 147 by one 18.9, by three 21.7.
    const int each = kSliceThreads / p.lanes;
    const int64_t most = (Kb + each - 1) / each;
    double least = 0.0;
    for (int64_t rounds = 1; rounds <= 4; ++rounds) {
        int64_t s = 256 * rounds / p.tiles;
        s = s < 1 ? 1 : s < most ? s : most;
        const double time = (double)((p.tiles * s + 255) / 256) * ((double)Kb / (double)s + 24.0);
        if (rounds == 1 || time < least) {
            least = time;
            p.slices = (int32_t)s;
        }
    }
    return p;
}

template <typename T, int VEC, int LT>
void launch_tokens(const T* x, int8_t* q, float* scale, int64_t K, int64_t N, void* scratch, const TokenPlan& p,
                   hipStream_t s)
{
    uint32_t* part = static_cast<uint32_t*>(scratch);
    const dim3 grid = launch_grid(p.tiles * p.slices, kSliceThreads), threads(kSliceThreads);
    const dim3 narrow = launch_grid((N + LT - 1) / LT * p.slices, kSliceThreads);
    hipLaunchKernelGGL((ff_tokens_most_kernel<T, VEC, LT>), grid, threads, 0, s, x, part, K, N, p.slices);
    hipLaunchKernelGGL((ff_tokens_round_kernel<T, LT>), narrow, threads, 0, s, x, part, q, scale, K, N, p.slices);
    XSPMM_LAUNCH_CHECK();
}

}  // namespace ff

template <typename T>
void int8_weight(const BlockIndex& w, const T* vals, int8_t* q, float* scale, hipStream_t s)
{
    if (w.Mb == 0) return;
    hipLaunchKernelGGL((ff::ff_int8_weight_kernel<T>), launch_grid(w.Mb, 64 * ff::kWeightWaves), dim3(64 * ff::kWeightWaves), 0, s,
                       w.ptr, w.col, vals, q, scale, (int32_t)w.M, (int32_t)w.K);
    XSPMM_LAUNCH_CHECK();
}

int64_t quantize_tokens_scratch(int64_t K, int64_t N)
{
    if (K == 0 || N == 0) return 0;
    int64_t most = 0;  // of any type
    for (int size : {2, 4}) {
        const ff::TokenPlan p = ff::token_plan(K, N, size);
        if (!p.whole && p.slices * N * 4 > most) most = p.slices * N * 4;
    }
    return most;
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
    const ff::TokenPlan p = ff::token_plan(K, N, (int)sizeof(T));
    if (p.whole) {
        const dim3 grid = launch_grid(p.tiles, 1024);
        if (N == 1)
            hipLaunchKernelGGL((ff::ff_token_kernel<T>), dim3(1), dim3(1024), 0, s, x, q, scale, (int32_t)K);
        else if (p.lanes == 4)
            hipLaunchKernelGGL((ff::ff_tokens_whole_kernel<T, 4>), grid, dim3(1024), 0, s, x, q, scale, K, N);
        else
            hipLaunchKernelGGL((ff::ff_tokens_whole_kernel<T, 16>), grid, dim3(1024), 0, s, x, q, scale, K, N);
        XSPMM_LAUNCH_CHECK();
        return;
    }
    if (p.lanes == 64) {
        if constexpr (sizeof(T) == 2)
            if (p.vec == 4) {
                ff::launch_tokens<T, 4, 64>(x, q, scale, K, N, scratch, p, s);
                return;
            }
        ff::launch_tokens<T, 1, 64>(x, q, scale, K, N, scratch, p, s);
    } else if (p.lanes == 16) {
        ff::launch_tokens<T, 1, 16>(x, q, scale, K, N, scratch, p, s);
    } else {
        ff::launch_tokens<T, 1, 1>(x, q, scale, K, N, scratch, p, s);
    }
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
