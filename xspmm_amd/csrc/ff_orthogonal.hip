// ff_orthogonal.hip -- an update U of a block-sparse weight, orthogonalised:
//
//   X = U / (|U| + eps), then `steps` times  S = X X^T,  X <- a X + (b S + c S S) X
//
// at the stored blocks.  An odd polynomial of X acts on its singular values alone; with
// the usual coefficients five steps bring all but the smallest ones near 1.  X has the
// weight's smaller side as its rows (U^T is X where U has fewer columns).
//
// Products are of fp16 operands with fp32 sums.  16-bit updates: X is held as two halves,
// of which products take the upper one and a X both, so that X loses nothing from step
// to step.  (A rounding E of X that went through a X would grow with the
// singular values that grow, 3.4 times a step; through S and the product it does not:
// what b S + c S S multiplies by E vanishes where the singular values do.)  The
// diagonal of b S + c S S stays in fp32 and multiplies X itself.  Together 3e-4 to 1e-3
// of the result's rms, rank 32 to full, where a bf16 result's rounding is 1.7e-3; with
// X in one half 2e-2 at rank 32.  fp32 updates: every operand in two halves, three
// products each (the fourth is below 2^-22): 1e-5 and less.
// Halves hold 2^12 times their values: an element of X is between 1 / sqrt(elements),
// far below fp16's normal numbers in a large matrix, and 1.2.
#include "feed_forward_device.hpp"
#include "orthogonal.hpp"

namespace xspmm {
namespace detail {
namespace ff {

constexpr float kHeld = 4096.f;  // times what a half stands for

struct Halves {
    _Float16* hi;
    _Float16* lo;  // null where products take the upper half alone and nothing else reads it
};

constexpr int kDeepK = 64;  // of a product's step

template <int TILE>
struct Shape {
    static constexpr int kWaves = TILE == 256 ? 8 : 4;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int kWaveI = TILE / 2, kWaveJ = TILE / (kWaves / 2);  // a wave's rows and columns
    static constexpr int FI = kWaveI / 16, FJ = kWaveJ / 16;
    static constexpr int kSide = TILE * kDeepK * 2;  // bytes of one operand's stage
    static constexpr int kStage = 2 * kSide;
    static constexpr int kLds = 2 * kStage;
};

// What becomes of a product's sums.
enum Purpose {
    kPart,    // a share of the sum, to be joined
    kGram,    // S
    kSquare,  // b S + c S S
    kApply,   // X
    kLast     // X at the stored blocks
};

struct Product {
    const _Float16* p[3];  // rows i, k along them
    const _Float16* q[3];  // rows j, k along them; or rows k, j along them
    int64_t p_ld, q_ld;
    int32_t tiles_i, tiles_j;
    int32_t steps;   // of kDeepK
    int32_t splits;  // of the steps
    float* part;
    bool lower;      // tiles on and below the diagonal, and their mirror images
};

template <typename T>
struct Finish {
    float a, b, c;
    Halves s, out;
    float* diagonal;     // of b S + c S S
    Halves x;
    int64_t ld;          // of what is written
    // kLast
    T* blocks;
    const int32_t *ptr, *col, *map;
    int32_t M, K, Mb, Kb;
    bool transposed;
};

// position of block (r, c), or -1
template <typename T>
__device__ __forceinline__ int32_t block_at(const Finish<T>& f, int32_t r, int32_t c)
{
    if (r >= f.Mb || c >= f.Kb) return -1;
    if (f.map) return f.map[(int64_t)r * f.Kb + c];
    int32_t lo = f.ptr[r], hi = f.ptr[r + 1];
    const int32_t end = hi;
    while (lo < hi) {
        const int32_t mid = lo + (hi - lo) / 2;
        if (f.col[mid] < c)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo < end && f.col[lo] == c ? lo : -1;
}

__device__ __forceinline__ void halves(float v, _Float16& hi, _Float16& lo)
{
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// Element i, j .. + 3 of a product's sums (i0, j0: of its 16 x 16 tile).
template <typename T, int PURPOSE>
__device__ __forceinline__ void finish_four(const Finish<T>& f, const float4_t v, int64_t i, int64_t j, int64_t i0,
                                            int64_t j0, bool mirror)
{
    typedef Pack<_Float16, 4> P;
    const int64_t at = i * f.ld + j;
    if constexpr (PURPOSE == kGram || PURPOSE == kSquare) {
        P hi, lo;
        float w[4];
        if constexpr (PURPOSE == kGram) {
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = v[q] * (1.f / kHeld);
        } else {
            const P sh = *reinterpret_cast<const P*>(f.s.hi + at);
            P sl{};
            if (f.s.lo) sl = *reinterpret_cast<const P*>(f.s.lo + at);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                w[q] = f.b * ((float)sh.v[q] + (float)sl.v[q]) + f.c * (v[q] * (1.f / kHeld));
                if (i == j + q) {
                    f.diagonal[i] = w[q] * (1.f / kHeld);
                    w[q] = 0.f;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) halves(w[q], hi.v[q], lo.v[q]);
        *reinterpret_cast<P*>(f.out.hi + at) = hi;
        if (f.out.lo) *reinterpret_cast<P*>(f.out.lo + at) = lo;
        if (mirror) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f.out.hi[(j + q) * f.ld + i] = hi.v[q];
                if (f.out.lo) f.out.lo[(j + q) * f.ld + i] = lo.v[q];
            }
        }
    }
    if constexpr (PURPOSE == kApply || PURPOSE == kLast) {
        const P xh = *reinterpret_cast<const P*>(f.x.hi + at), xl = *reinterpret_cast<const P*>(f.x.lo + at);
        const float d = f.a + f.diagonal[i];
        float w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = fmaf(d, (float)xh.v[q] + (float)xl.v[q], v[q] * (1.f / kHeld));
        if constexpr (PURPOSE == kApply) {
            P hi, lo;
#pragma unroll
            for (int q = 0; q < 4; ++q) halves(w[q], hi.v[q], lo.v[q]);
            *reinterpret_cast<P*>(f.out.hi + at) = hi;
            *reinterpret_cast<P*>(f.out.lo + at) = lo;
        } else {
            const int64_t r = f.transposed ? j : i, c = f.transposed ? i : j;
            const int32_t b = block_at(f, (int32_t)((f.transposed ? j0 : i0) / 16), (int32_t)((f.transposed ? i0 : j0) / 16));
            if (b < 0) return;
            T* o = f.blocks + (int64_t)b * 256 + (r % 16) * 16 + c % 16;
            if (f.transposed) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    o[16 * q] = r + q < f.M && c < f.K ? (T)(w[q] * (1.f / kHeld)) : (T)0.f;
            } else {
                Pack<T, 4> k;
#pragma unroll
                for (int q = 0; q < 4; ++q) k.v[q] = r < f.M && c + q < f.K ? (T)(w[q] * (1.f / kHeld)) : (T)0.f;
                *reinterpret_cast<Pack<T, 4>*>(o) = k;
            }
        }
    }
}

// tile t of the lower triangle: row i, column j <= i
__device__ __forceinline__ void triangle(int64_t t, int32_t& i, int32_t& j)
{
    int32_t r = (int32_t)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((int64_t)r * (r + 1) / 2 > t) --r;
    while ((int64_t)(r + 1) * (r + 2) / 2 <= t) ++r;
    i = r;
    j = (int32_t)(t - (int64_t)r * (r + 1) / 2);
}

__host__ __device__ __forceinline__ int64_t product_tiles(const Product& a)
{
    return a.lower ? (int64_t)a.tiles_i * (a.tiles_i + 1) / 2 : (int64_t)a.tiles_i * a.tiles_j;
}

__device__ __forceinline__ void tile_place(const Product& a, int64_t t, int32_t& ti, int32_t& tj)
{
    if (a.lower) {
        triangle(t, ti, tj);
    } else {
        // bands of 8 rows of tiles, column by column
        const int64_t band = t / (8 * (int64_t)a.tiles_j) * 8;
        const int64_t h = min((int64_t)8, a.tiles_i - band), in = t - band * a.tiles_j;
        ti = (int32_t)(band + in % h);
        tj = (int32_t)(in / h);
    }
}

typedef __attribute__((address_space(3))) short4_t lds_short4_t;
__device__ __forceinline__ u32x2_t read_across(const unsigned char* p)
{
    return __builtin_bit_cast(u32x2_t,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)const_cast<unsigned char*>(p)));
}

// Rows of 128 bytes, chunk c (16 bytes) of row r at c ^ (r & 7); rows of TILE values,
// chunk c of row k at c ^ 2 (k & 7): what one read touches is in different banks.
template <typename T, int TILE, bool ACROSS, int PASSES, int PURPOSE>
__global__ __launch_bounds__(Shape<TILE>::kThreads, 2) void ff_orthogonal_product_kernel(const Product a, const Finish<T> f)
{
    using S = Shape<TILE>;
    constexpr int FI = S::FI, FJ = S::FJ;
    __shared__ __align__(16) unsigned char smem[S::kLds];
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wi = wave & 1, wj = wave >> 1;
    const int64_t tiles = product_tiles(a), item = xcd_item(blockIdx.x, tiles * a.splits);
    if (item < 0) return;
    const int64_t tile = item / a.splits;
    const int32_t split = (int32_t)(item % a.splits);
    int32_t ti, tj;
    tile_place(a, tile, ti, tj);
    const int64_t i0 = (int64_t)ti * TILE, j0 = (int64_t)tj * TILE;
    const int32_t from = (int32_t)((int64_t)a.steps * split / a.splits);
    const int32_t count = (int32_t)((int64_t)a.steps * (split + 1) / a.splits) - from;
    const uint32_t lds0 = lds_address(smem);

    // this lane's bytes of what the wave loads, a KB at a time
    constexpr int kPer = S::kSide / 1024 / S::kWaves;
    uint32_t p_lane[kPer], q_lane[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
        const int r = 8 * (wave * kPer + u) + (lane >> 3);
        p_lane[u] = (uint32_t)(r * a.p_ld * 2) + 16u * (uint32_t)((lane & 7) ^ (r & 7));
        if constexpr (ACROSS) {
            constexpr int kChunks = TILE / 8;
            const int at = (wave * kPer + u) * 64 + lane, k = at / kChunks, c = at % kChunks;
            q_lane[u] = (uint32_t)(k * a.q_ld * 2) + 16u * (uint32_t)(c ^ (2 * (k & 7)));
        } else {
            q_lane[u] = (uint32_t)(r * a.q_ld * 2) + 16u * (uint32_t)((lane & 7) ^ (r & 7));
        }
    }
    const uint32_t p_bytes = (uint32_t)(TILE * a.p_ld * 2);
    const uint32_t q_bytes = (uint32_t)((ACROSS ? kDeepK : TILE) * a.q_ld * 2);

    auto issue = [&](int pass, int32_t step, int stage) {
        const _Float16* p = a.p[pass] + i0 * a.p_ld + (int64_t)step * kDeepK;
        const _Float16* q = ACROSS ? a.q[pass] + (int64_t)step * kDeepK * a.q_ld + j0
                                   : a.q[pass] + j0 * a.q_ld + (int64_t)step * kDeepK;
        const i32x4_t pb = dma_buffer(p, p_bytes), qb = dma_buffer(q, q_bytes);
        const uint32_t to = lds0 + (uint32_t)(stage * S::kStage);
#pragma unroll
        for (int u = 0; u < kPer; ++u) dma_to_lds(to + (uint32_t)(wave * kPer + u) * 1024u, p_lane[u], pb);
#pragma unroll
        for (int u = 0; u < kPer; ++u) dma_to_lds(to + S::kSide + (uint32_t)(wave * kPer + u) * 1024u, q_lane[u], qb);
    };

    float4_t acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

    auto multiply = [&](int stage) {
        const unsigned char* P = smem + stage * S::kStage;
        const unsigned char* Q = P + S::kSide;
#pragma unroll
        for (int h = 0; h < kDeepK / 32; ++h) {
            u32x4_t x[FI], y[FJ];
#pragma unroll
            for (int j = 0; j < FJ; ++j) {
                if constexpr (ACROSS) {
                    const int k = 32 * h + 8 * g + (li >> 2), c = 2 * (wj * FJ + j) + ((li & 3) >> 1);
                    const u32x2_t lo = read_across(Q + k * (TILE * 2) + ((c ^ (2 * (k & 7))) * 16) + 8 * (li & 1));
                    const u32x2_t hi =
                        read_across(Q + (k + 4) * (TILE * 2) + ((c ^ (2 * ((k + 4) & 7))) * 16) + 8 * (li & 1));
                    y[j] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
                } else {
                    const int r = wj * S::kWaveJ + 16 * j + li;
                    y[j] = *reinterpret_cast<const u32x4_t*>(Q + r * 128 + (((4 * h + g) ^ (r & 7)) * 16));
                }
            }
#pragma unroll
            for (int i = 0; i < FI; ++i) {
                const int r = wi * S::kWaveI + 16 * i + li;
                x[i] = *reinterpret_cast<const u32x4_t*>(P + r * 128 + (((4 * h + g) ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = mfma16<_Float16>(y[j], x[i], acc[i][j]);
        }
    };

    // the steps of all passes one after the other
    const int32_t all = PASSES * count;
    if (all > 0) issue(0, from, 0);
    for (int32_t st = 0; st < all; ++st) {
        dma_wait<0>();
        __syncthreads();
        if (st + 1 < all) {
            const int32_t n = st + 1;
            issue(PASSES == 1 ? 0 : n / count, from + (PASSES == 1 ? n : n % count), n & 1);
        }
        multiply(st & 1);
    }

    if constexpr (PURPOSE == kPart) {
        float* part = a.part + item * (int64_t)(TILE * TILE);
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
                *reinterpret_cast<float4_t*>(part + (wi * S::kWaveI + 16 * i + li) * TILE + wj * S::kWaveJ + 16 * j + 4 * g) =
                    acc[i][j];
    } else {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) {
                const int64_t it = i0 + wi * S::kWaveI + 16 * i, jt = j0 + wj * S::kWaveJ + 16 * j;
                finish_four<T, PURPOSE>(f, acc[i][j], it + li, jt + 4 * g, it, jt, a.lower && ti != tj);
            }
    }
}

// The shares of a tile's sums, in their order.
template <typename T, int TILE, int PURPOSE>
__global__ __launch_bounds__(256) void ff_orthogonal_join_kernel(const Product a, const Finish<T> f)
{
    constexpr int kPieces = TILE * TILE / 1024;  // of a tile: 256 threads, four values each
    const int64_t tile = blockIdx.x / kPieces;
    const int piece = (int)(blockIdx.x % kPieces);
    int32_t ti, tj;
    tile_place(a, tile, ti, tj);
    // pieces are 16 x 64: four rows of 16 x 16 tiles' lanes as the sums have them
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
    const int i = piece / (TILE / 64) * 16 + li, j = piece % (TILE / 64) * 64 + (t >> 6) * 16 + 4 * g;
    const float* part = a.part + tile * a.splits * (int64_t)(TILE * TILE) + i * TILE + j;
    float4_t v = *reinterpret_cast<const float4_t*>(part);
    for (int32_t s = 1; s < a.splits; ++s) v += *reinterpret_cast<const float4_t*>(part + s * (int64_t)(TILE * TILE));
    const int64_t it = (int64_t)ti * TILE + i - li, jt = (int64_t)tj * TILE + j - 4 * g;
    finish_four<T, PURPOSE>(f, v, it + li, jt + 4 * g, it, jt, a.lower && ti != tj);
}

// Sums of squares of the stored values inside the weight, a share of the blocks each.
constexpr int kNormShares = 512;
template <typename T>
__global__ __launch_bounds__(256) void ff_square_sum_kernel(const T* __restrict__ u, const int32_t* __restrict__ row,
                                                            const int32_t* __restrict__ col, int64_t nnzb, int32_t M,
                                                            int32_t K, double* __restrict__ part)
{
    __shared__ double red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum = 0.0;
    for (int64_t b = blockIdx.x * 4 + wave; b < nnzb; b += 4 * kNormShares) {
        const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4>*>(u + b * 256 + 4 * lane);
        const int32_t r = 16 * row[b] + lane / 4, c = 16 * col[b] + 4 * (lane & 3);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const double v = r < M && c + q < K ? (double)(float)p.v[q] : 0.0;
            sum += v * v;
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// X = U / (|U| + eps), zeros where no block is stored and past the edges; a thread
// per eight values.
template <typename T>
__global__ __launch_bounds__(256) void ff_orthogonal_start_kernel(const Finish<T> f, const T* __restrict__ u,
                                                                  const double* __restrict__ part, double eps,
                                                                  int64_t rows)
{
    __shared__ double red[4];
    const int t = threadIdx.x;
    double sum = part[t] + part[t + 256];
#pragma unroll
    for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    if ((t & 63) == 0) red[t >> 6] = sum;
    __syncthreads();
    const double norm = sqrt(red[0] + red[1] + red[2] + red[3]) + eps;
    // an update of zeros stays one
    const double by = norm == 0.0 ? 0.0 : (double)kHeld / norm;
    const int64_t per = f.ld / 8;
    for (int64_t e = (int64_t)blockIdx.x * 256 + t; e < rows * per; e += (int64_t)gridDim.x * 256) {
        const int64_t i = e / per, j = e % per * 8;
        const int64_t r = f.transposed ? j : i, c = f.transposed ? i : j;
        const int32_t b = block_at(f, (int32_t)(r / 16), (int32_t)(c / 16));
        Pack<_Float16, 8> hi{}, lo{};
        if (b >= 0) {
            const T* v = u + (int64_t)b * 256 + r % 16 * 16 + c % 16;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const bool in = f.transposed ? r + q < f.M && c < f.K : r < f.M && c + q < f.K;
                const float w = in ? (float)((double)(float)v[f.transposed ? 16 * q : q] * by) : 0.f;
                halves(w, hi.v[q], lo.v[q]);
            }
        }
        *reinterpret_cast<Pack<_Float16, 8>*>(f.out.hi + i * f.ld + j) = hi;
        *reinterpret_cast<Pack<_Float16, 8>*>(f.out.lo + i * f.ld + j) = lo;
    }
}

// Sizes and memory of one orthogonalised update.
struct OrthogonalPlan {
    bool transposed, split;
    int tile;
    int64_t m, k;  // rows and columns of X, to whole tiles
    int gram_splits, square_splits;
    size_t x_hi[2], x_lo[2], s_hi, s_lo, b_hi, b_lo, diagonal, norm, part, end;
};

OrthogonalPlan orthogonal_plan(const BlockIndex& w, int64_t size)
{
    OrthogonalPlan p{};
    p.transposed = w.M > w.K;
    p.split = size == 4;
    const int64_t rows = p.transposed ? w.K : w.M, columns = p.transposed ? w.M : w.K;
    p.tile = rows <= 1024 ? 128 : 256;
    p.m = (rows + p.tile - 1) / p.tile * p.tile;
    p.k = (columns + p.tile - 1) / p.tile * p.tile;
    const int64_t n = p.m / p.tile, tiles = n * (n + 1) / 2;
    // shares of a sum: rounds of 256 workgroups, a share each
    auto splits = [&](int64_t steps) {
        int best = 1;
        double least = 1e30;
        for (int s = 1; s <= 8 && steps / s >= 4; ++s) {
            const double time = (double)((tiles * s + 255) / 256) * ((double)steps / s + 2.0) + (s > 1 ? 4.0 + 0.02 * s * tiles : 0.0);
            if (time < least) {
                least = time;
                best = s;
            }
        }
        return best;
    };
    p.gram_splits = splits(p.k / kDeepK);
    p.square_splits = splits(p.m / kDeepK);
    Carve c;
    const size_t x = (size_t)(p.m * p.k) * 2, s = (size_t)(p.m * p.m) * 2;
    p.x_hi[0] = c.take(x);
    p.x_hi[1] = c.take(x);
    p.x_lo[0] = c.take(x);
    p.x_lo[1] = p.split ? c.take(x) : p.x_lo[0];
    p.s_hi = c.take(s);
    p.b_hi = c.take(s);
    p.s_lo = p.split ? c.take(s) : 0;
    p.b_lo = p.split ? c.take(s) : 0;
    p.diagonal = c.take((size_t)p.m * 4);
    p.norm = c.take(kNormShares * 8);
    const int most = p.gram_splits > p.square_splits ? p.gram_splits : p.square_splits;
    p.part = c.take(most > 1 ? (size_t)(tiles * most) * p.tile * p.tile * 4 : 0);
    p.end = c.end;
    return p;
}

template <typename T, int TILE, bool ACROSS, int PASSES, int PURPOSE>
void launch_orthogonal(const Product& a, const Finish<T>& f, hipStream_t s)
{
    const int64_t tiles = product_tiles(a);
    constexpr int threads = Shape<TILE>::kThreads;
    const dim3 grid = launch_grid(kXcds * xcd_chunk(tiles * a.splits), threads);
    if (a.splits > 1) {
        if constexpr (!ACROSS) {
            hipLaunchKernelGGL((ff_orthogonal_product_kernel<T, TILE, ACROSS, PASSES, kPart>), grid, dim3(threads), 0, s, a, f);
            hipLaunchKernelGGL((ff_orthogonal_join_kernel<T, TILE, PURPOSE>), launch_grid(tiles * (TILE * TILE / 1024), 256),
                               dim3(256), 0, s, a, f);
        }
    } else {
        hipLaunchKernelGGL((ff_orthogonal_product_kernel<T, TILE, ACROSS, PASSES, PURPOSE>), grid, dim3(threads), 0, s, a, f);
    }
    XSPMM_LAUNCH_CHECK();
}

template <typename T, int TILE>
void orthogonal_steps(const BlockIndex& w, const T* update, T* out, const OrthogonalArgs& o, const OrthogonalPlan& p,
                      char* at, hipStream_t s)
{
    constexpr int PASSES = is_f32<T> ? 3 : 1;
    auto half = [&](size_t offset) { return reinterpret_cast<_Float16*>(at + offset); };
    const Halves x[2] = {{half(p.x_hi[0]), half(p.x_lo[0])}, {half(p.x_hi[1]), half(p.x_lo[1])}};
    const Halves S = {half(p.s_hi), p.split ? half(p.s_lo) : nullptr};
    const Halves B = {half(p.b_hi), p.split ? half(p.b_lo) : nullptr};
    Finish<T> f{};
    f.a = o.a;
    f.b = o.b;
    f.c = o.c;
    f.diagonal = reinterpret_cast<float*>(at + p.diagonal);
    f.blocks = out;
    f.ptr = w.ptr;
    f.col = w.col;
    f.map = w.map;
    f.M = (int32_t)w.M;
    f.K = (int32_t)w.K;
    f.Mb = (int32_t)w.Mb;
    f.Kb = (int32_t)w.Kb;
    f.transposed = p.transposed;
    double* norm = reinterpret_cast<double*>(at + p.norm);
    hipLaunchKernelGGL((ff_square_sum_kernel<T>), dim3(kNormShares), dim3(256), 0, s, update, w.row, w.col, w.nnzb,
                       (int32_t)w.M, (int32_t)w.K, norm);
    f.out = x[0];
    f.ld = p.k;
    hipLaunchKernelGGL((ff_orthogonal_start_kernel<T>), dim3(4096), dim3(256), 0, s, f, update, norm, (double)o.eps, p.m);
    XSPMM_LAUNCH_CHECK();
    // upper times upper half, upper times lower, lower times upper
    auto operands = [&](Product& a, const Halves& l, const Halves& r) {
        a.p[0] = a.p[1] = l.hi;
        a.q[0] = a.q[2] = r.hi;
        a.p[2] = l.lo;
        a.q[1] = r.lo;
    };
    for (int step = 0; step < o.steps; ++step) {
        const Halves &from = x[step % 2], &to = x[(step + 1) % 2];
        Product a{};
        a.part = reinterpret_cast<float*>(at + p.part);
        operands(a, from, from);
        a.p_ld = a.q_ld = p.k;
        a.tiles_i = a.tiles_j = (int32_t)(p.m / TILE);
        a.steps = (int32_t)(p.k / kDeepK);
        a.splits = p.gram_splits;
        a.lower = true;
        f.out = S;
        f.ld = p.m;
        launch_orthogonal<T, TILE, false, PASSES, kGram>(a, f, s);
        operands(a, S, S);
        a.p_ld = a.q_ld = p.m;
        a.steps = (int32_t)(p.m / kDeepK);
        a.splits = p.square_splits;
        f.s = S;
        f.out = B;
        launch_orthogonal<T, TILE, false, PASSES, kSquare>(a, f, s);
        operands(a, B, from);
        a.q_ld = p.k;
        a.tiles_j = (int32_t)(p.k / TILE);
        a.splits = 1;
        a.lower = false;
        f.x = from;
        f.out = to;
        f.ld = p.k;
        if (step + 1 < o.steps)
            launch_orthogonal<T, TILE, true, PASSES, kApply>(a, f, s);
        else
            launch_orthogonal<T, TILE, true, PASSES, kLast>(a, f, s);
    }
}

}  // namespace ff

int64_t orthogonal_scratch(const BlockIndex& w, int64_t size)
{
    if (w.nnzb == 0) return 0;
    return (int64_t)ff::orthogonal_plan(w, size).end;
}

template <typename T>
void orthogonalize(const BlockIndex& w, const T* update, T* out, const OrthogonalArgs& o, void* scratch, hipStream_t s)
{
    if (w.nnzb == 0) return;
    const ff::OrthogonalPlan p = ff::orthogonal_plan(w, sizeof(T));
    if (p.tile == 256)
        ff::orthogonal_steps<T, 256>(w, update, out, o, p, static_cast<char*>(scratch), s);
    else
        ff::orthogonal_steps<T, 128>(w, update, out, o, p, static_cast<char*>(scratch), s);
}

#define XSPMM_ORTHOGONAL(T) \
    template void orthogonalize<T>(const BlockIndex&, const T*, T*, const OrthogonalArgs&, void*, hipStream_t);
XSPMM_ORTHOGONAL(float)
XSPMM_ORTHOGONAL(_Float16)
XSPMM_ORTHOGONAL(__bf16)
#undef XSPMM_ORTHOGONAL

}  // namespace detail
}  // namespace xspmm
