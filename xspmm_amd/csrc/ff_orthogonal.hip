// ff_orthogonal.hip -- an update U of a block-sparse weight, orthogonalised:
//
//   X = U / (|U| + eps), then `steps` times  S = X X^T,  X <- a X + (b S + c S S) X
//
// at the stored blocks.  An odd polynomial of X acts on its singular values alone; with
// the usual coefficients five steps bring all but the smallest ones near 1.  X has the
// weight's smaller side as its rows (U^T is X where U has fewer columns).
//
// Products are of fp16 operands with fp32 sums.  bf16 updates: X is held as two halves, of
// which products take the upper one and a X both, so that X loses nothing from step
// to step.  (A rounding E of X that went through a X would grow with the
// singular values that grow, 3.4 times a step; through S and the product it does not:
// what b S + c S S multiplies by E vanishes where the singular values do.)  The
// diagonal of b S + c S S stays in fp32 and multiplies X itself.  Together 3e-4 to 1e-3
// of the result's rms, rank 32 to full, where a bf16 result's rounding is 1.7e-3 (at 512 x
// 1792 4.4e-4: one element in six is rounded to its other neighbour, 1.3e-3 of the norm in
// all); with X in one half 2e-2 at rank 32.  fp16 and fp32 updates: every operand in two
// halves, three products each (the fourth is below 2^-22): 1e-5 and less, beside a
// rounding of 2e-4 in fp16.  (Of fp16 updates the last four of five steps would have to be
// so.)  At 4096 x 14336 that takes 11.2 ms and one half 4.0, at 1792 x 512 169 us and 137:
// bf16 updates, rounded as they are, do without.
// Halves hold 2^12 times their values: an element of X is between 1 / sqrt(elements),
// far below fp16's normal numbers in a large matrix, and 1.2.
#include "feed_forward_device.hpp"
#include "orthogonal.hpp"

namespace xspmm {
namespace detail {
namespace ff {

constexpr float kHeld = 4096.f;  // times what a half stands for

// whether products take both halves
template <typename T>
constexpr bool is_split = !__is_same(T, __bf16);

struct Halves {
    _Float16* hi;
    _Float16* lo;  // null where products take the upper half alone and nothing else reads it
};

// X, S and b S + c S S lie as blocks of 16 x 32 halves, 1 KB each, that follow each other
// along the rows: one load into LDS, of an operand's rows or of a step's columns, is one
// block, and so is one store of a result.  (From rows of whole matrices a step takes 64
// bytes each, half a line, and gets half of L2's rate: 538 us instead of 460 for a X + Y X
// at 4096 x 14336.)
constexpr int kBlock = 512;
__device__ __forceinline__ int64_t block_place(int64_t r, int64_t c, int64_t ld)
{
    return (r / 16 * (ld / 32) + c / 32) * kBlock;
}

constexpr int kDeepK = 32;  // of a product's step

// A workgroup of four waves takes TI rows and 128 columns (of 64 rows, 64), a wave half of
// either.  Two
// workgroups share a CU and are not in step: while one multiplies, the other reads its
// operands, or reads and writes X at a tile's end (512 KB of 256 x 256 elements, which
// with one workgroup of eight waves a CU took 157 of 545 us at 4096 x 14336).  Operands
// in two halves (SPLIT) take twice the LDS, and three products of each step's: one
// workgroup a CU has as much to multiply as two have without.
constexpr int tile_columns(int rows) { return rows == 64 ? 64 : 128; }
constexpr int kProductWaves = 4, kProductThreads = 64 * kProductWaves;
template <int TI, bool SPLIT>
struct Shape {
    static constexpr int TJ = tile_columns(TI);
    static constexpr int kWaveI = TI / 2, kWaveJ = TJ / 2;  // a wave's rows and columns
    static constexpr int FI = kWaveI / 16, FJ = kWaveJ / 16;
    static constexpr int kHalves = SPLIT ? 2 : 1;
    static constexpr int kSideI = TI * kDeepK * 2, kSideJ = TJ * kDeepK * 2;  // bytes of an operand's step
    static constexpr int kStage = kHalves * (kSideI + kSideJ);
    static constexpr int kStages = TI == 256 ? 3 : 4;  // steps in LDS
    static constexpr int kLds = kStages * kStage;
    static_assert(kLds <= (SPLIT ? 160 : 80) * 1024);
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
    Halves p;  // rows i, k along them
    Halves q;  // rows j, k along them; or rows k, j along them
    int64_t p_ld, q_ld;
    int32_t tiles_i, tiles_j;
    int32_t steps;   // of kDeepK
    int32_t splits;  // of the steps
    uint32_t items;  // tiles times splits
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

// N values as halves, side by side.
template <int N>
__device__ __forceinline__ void store_halves(const Halves& to, int64_t at, const float (&v)[N])
{
    Pack<_Float16, N> hi, lo;
#pragma unroll
    for (int q = 0; q < N; ++q) halves(v[q], hi.v[q], lo.v[q]);
    *reinterpret_cast<Pack<_Float16, N>*>(to.hi + at) = hi;
    if (to.lo) *reinterpret_cast<Pack<_Float16, N>*>(to.lo + at) = lo;
}

// Two tiles of 16 x 16 side by side, of which a lane has row li and columns 4 g .. + 3
// each: lanes of even g take the first one's columns 4 g .. + 7 (with the next lanes'),
// those of odd g the second one's, 16 + 4 (g - 1) .. + 7.
__device__ __forceinline__ void pair_up(const float4_t a, const float4_t b, float (&v)[8])
{
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[q]), __float_as_uint(b[q]), false, false);
        v[q] = __uint_as_float(r[0]);
        v[4 + q] = __uint_as_float(r[1]);
    }
}
// which of the four eights of 32 columns that is
__device__ __forceinline__ int paired_chunk(int g) { return 2 * (g & 1) + (g >> 1); }

// A product's sums of 32 x 32 elements at (i, j), two pairs of tiles: S, or b S + c S S, and
// its mirror image.  turn: 2 (4 with lower halves) KB of LDS of this wave's.
template <typename T, int PURPOSE>
__device__ __forceinline__ void finish_symmetric(const Finish<T>& f, float (&v)[2][8], int64_t i, int64_t j, int li,
                                                 int g, bool mirror, _Float16* turn)
{
    typedef Pack<_Float16, 8> P;
    const int chunk = paired_chunk(g), lane = 16 * g + li;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t at = block_place(i + 16 * u, j, f.ld) + li * 32 + 8 * chunk;
        if constexpr (PURPOSE == kGram) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[u][q] *= 1.f / kHeld;
        } else {
            const P sh = *reinterpret_cast<const P*>(f.s.hi + at);
            P sl{};
            if (f.s.lo) sl = *reinterpret_cast<const P*>(f.s.lo + at);
            const int64_t row = i + 16 * u + li, column = j + 8 * chunk;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                v[u][q] = f.b * ((float)sh.v[q] + (float)sl.v[q]) + f.c * (v[u][q] * (1.f / kHeld));
                if (row == column + q) {
                    f.diagonal[row] = v[u][q] * (1.f / kHeld);
                    v[u][q] = 0.f;
                }
            }
        }
        store_halves<8>(f.out, at, v[u]);
    }
    if (!mirror) return;
    // through LDS: column by column, 64 bytes of 32 rows each
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            _Float16 hi, lo;
            halves(v[u][q], hi, lo);
            const int at = (8 * chunk + q) * 32 + 16 * u + li;
            turn[at] = hi;
            if (f.out.lo) turn[1024 + at] = lo;
        }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int64_t at = block_place(j + 16 * u, i, f.ld) + lane * 8;
        *reinterpret_cast<P*>(f.out.hi + at) = *reinterpret_cast<const P*>(turn + u * 512 + lane * 8);
        if (f.out.lo) *reinterpret_cast<P*>(f.out.lo + at) = *reinterpret_cast<const P*>(turn + 1024 + u * 512 + lane * 8);
    }
    __builtin_amdgcn_wave_barrier();
}

// a X + Y X of 16 x 32 elements at (i, j): X, or (kLast) what of it is stored.
template <typename T, int PURPOSE>
__device__ __forceinline__ void finish_product(const Finish<T>& f, float (&v)[8], int64_t i, int64_t j, int li, int g)
{
    typedef Pack<_Float16, 8> P;
    const int chunk = paired_chunk(g);
    const int64_t at = block_place(i, j, f.ld) + li * 32 + 8 * chunk;
    const P xh = *reinterpret_cast<const P*>(f.x.hi + at), xl = *reinterpret_cast<const P*>(f.x.lo + at);
    const float d = f.a + f.diagonal[i + li];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = fmaf(d, (float)xh.v[q] + (float)xl.v[q], v[q] * (1.f / kHeld));
    if constexpr (PURPOSE == kApply) {
        store_halves<8>(f.out, at, v);
    } else {
        const int64_t column = j + 8 * chunk;
        const int64_t r = f.transposed ? column : i + li, c = f.transposed ? i + li : column;
        const int32_t b = block_at(f, (int32_t)(r / 16), (int32_t)(c / 16));
        if (b < 0) return;
        T* o = f.blocks + (int64_t)b * 256 + r % 16 * 16 + c % 16;
        if (f.transposed) {
#pragma unroll
            for (int q = 0; q < 8; ++q) o[16 * q] = r + q < f.M && c < f.K ? (T)(v[q] * (1.f / kHeld)) : (T)0.f;
        } else {
            Pack<T, 8> k;
#pragma unroll
            for (int q = 0; q < 8; ++q) k.v[q] = r < f.M && c + q < f.K ? (T)(v[q] * (1.f / kHeld)) : (T)0.f;
            *reinterpret_cast<Pack<T, 8>*>(o) = k;
        }
    }
}

// Tiles, of a symmetric result those that have an element on or below the diagonal: TI / TJ
// * (i + 1) of them in row i.
__host__ __device__ __forceinline__ int64_t product_tiles(const Product& a)
{
    return a.lower ? (int64_t)a.tiles_i * (a.tiles_i + 1) / 2 * (a.tiles_j / a.tiles_i)
                   : (int64_t)a.tiles_i * a.tiles_j;
}

template <int TI>
__device__ __forceinline__ void tile_place(const Product& a, uint32_t t, int32_t& ti, int32_t& tj)
{
    if (a.lower) {
        constexpr uint32_t per = TI / tile_columns(TI);
        const uint32_t pair = t / per;
        uint32_t r = (uint32_t)((sqrtf(8.f * (float)pair + 1.f) - 1.f) * 0.5f);
        while ((uint64_t)r * (r + 1) / 2 > pair) --r;
        while ((uint64_t)(r + 1) * (r + 2) / 2 <= pair) ++r;
        ti = (int32_t)r;
        tj = (int32_t)(t - (uint32_t)((uint64_t)r * (r + 1) / 2) * per);
    } else {
        // bands of 8 rows of tiles, column by column
        const uint32_t wide = (uint32_t)a.tiles_j, band = t / (8 * wide) * 8;
        const uint32_t h = min(8u, (uint32_t)a.tiles_i - band), in = t - band * wide;
        ti = (int32_t)(band + in % h);
        tj = (int32_t)(in / h);
    }
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
}

typedef __attribute__((address_space(3))) short4_t lds_short4_t;
__device__ __forceinline__ u32x2_t read_across(const unsigned char* p)
{
    return __builtin_bit_cast(u32x2_t,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)const_cast<unsigned char*>(p)));
}

// Chunk c (16 bytes) of row r of a block lies in LDS at c ^ row_swizzle(r), of one that is
// read across its rows at c ^ across_swizzle(r), so that what is read at once is in
// different banks.  A read of 16 bytes a lane takes sixteen lanes at once, lanes 0-3, 12-15,
// 20-27 first and 4-11, 16-19, 28-31 next: eight rows of one g and the other eight of the
// next; a transposed read of 8 bytes takes 32.
__device__ __forceinline__ int row_swizzle(int r)
{
    const int x = (r >> 2) & 3;  // 0, 2, 3, 1
    return ((x ^ (x >> 1)) & 1) << 1 | x >> 1;
}
__device__ __forceinline__ int across_swizzle(int r) { return (r >> 3) << 1; }

template <typename T, int TI, bool ACROSS, int PURPOSE>
__global__ __launch_bounds__(kProductThreads, is_split<T> ? 1 : 2) void ff_orthogonal_product_kernel(const Product a, const Finish<T> f)
{
    constexpr bool SPLIT = is_split<T>;
    using S = Shape<TI, SPLIT>;
    constexpr int FI = S::FI, FJ = S::FJ, TJ = S::TJ, kStages = S::kStages, kHalves = S::kHalves;
    __shared__ __align__(16) unsigned char smem[S::kLds];
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wi = wave & 1, wj = wave >> 1;
    const uint32_t item = xcd_item32(blockIdx.x, a.items);
    if (item == ~0u) return;
    const uint32_t tile = a.splits == 1 ? item : item / (uint32_t)a.splits;
    const int32_t split = __builtin_amdgcn_readfirstlane((int32_t)(item - tile * (uint32_t)a.splits));
    int32_t ti, tj;
    tile_place<TI>(a, tile, ti, tj);
    const int64_t i0 = (int64_t)ti * TI, j0 = (int64_t)tj * TJ;
    // (at most 2^15 steps and 8 shares)
    const int32_t from = a.steps * split / a.splits, all = a.steps * (split + 1) / a.splits - from;
    const uint32_t lds0 = lds_address(smem);

    // This lane's bytes of the blocks that the wave loads.
    constexpr int kPerI = S::kSideI / 1024 / kProductWaves, kPerJ = S::kSideJ / 1024 / kProductWaves;
    const int row = lane >> 2;
    const uint32_t across_p = (uint32_t)(a.p_ld / 32) * 1024u, across_q = (uint32_t)(a.q_ld / 32) * 1024u;
    const uint32_t in_row = (uint32_t)(row * 64 + (((lane & 3) ^ row_swizzle(row)) * 16));
    const uint32_t in_across = (uint32_t)(row * 64 + (((lane & 3) ^ across_swizzle(row)) * 16));
    uint32_t p_lane[kPerI], q_lane[kPerJ];
#pragma unroll
    for (int u = 0; u < kPerI; ++u) p_lane[u] = (uint32_t)(wave * kPerI + u) * across_p + in_row;
#pragma unroll
    for (int u = 0; u < kPerJ; ++u) {
        const int b = wave * kPerJ + u;
        q_lane[u] = ACROSS ? (uint32_t)(b / (TJ / 32)) * across_q + (uint32_t)(b % (TJ / 32)) * 1024u + in_across
                           : (uint32_t)b * across_q + in_row;
    }
    const uint32_t p_bytes = (uint32_t)(TI / 16) * across_p;
    const uint32_t q_bytes = (uint32_t)((ACROSS ? kDeepK : TJ) / 16) * across_q;

    // the loads of step n into stage `stage`: of either half p's and q's
    constexpr int kLoads = kHalves * (kPerI + kPerJ);
    auto issue = [&](int32_t n, int stage) {
        const int64_t k = (int64_t)(from + n) * kDeepK;
        const int64_t at_p = block_place(i0, k, a.p_ld), at_q = ACROSS ? block_place(k, j0, a.q_ld) : block_place(j0, k, a.q_ld);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const i32x4_t pb = dma_buffer((h ? a.p.lo : a.p.hi) + at_p, p_bytes);
            const i32x4_t qb = dma_buffer((h ? a.q.lo : a.q.hi) + at_q, q_bytes);
            const uint32_t to = lds0 + (uint32_t)(stage * S::kStage + h * (S::kSideI + S::kSideJ));
#pragma unroll
            for (int u = 0; u < kPerI; ++u) dma_to_lds(to + (uint32_t)(wave * kPerI + u) * 1024u, p_lane[u], pb);
#pragma unroll
            for (int u = 0; u < kPerJ; ++u)
                dma_to_lds(to + S::kSideI + (uint32_t)(wave * kPerJ + u) * 1024u, q_lane[u], qb);
        }
    };

    float4_t acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

    struct Operands {
        u32x4_t x[FI], y[FJ];
    };
    auto read = [&](int stage, int h, Operands& o) {
        auto& [x, y] = o;
        const unsigned char* P = smem + stage * S::kStage + h * (S::kSideI + S::kSideJ);
        const unsigned char* Q = P + S::kSideI;
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
            if constexpr (ACROSS) {
                // rows 8 g .. + 7 of the step, 8 bytes (four columns) a lane
                const int r = 8 * (g & 1) + (li >> 2), c = (2 * (j & 1) + ((li & 3) >> 1)) ^ across_swizzle(r);
                const unsigned char* q = Q + ((g >> 1) * (TJ / 32) + wj * (FJ / 2) + j / 2) * 1024 + r * 64 + c * 16 + 8 * (li & 1);
                const u32x2_t lo = read_across(q), hi = read_across(q + 4 * 64);
                y[j] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
            } else {
                const int r = wj * S::kWaveJ + 16 * j + li;
                y[j] = *reinterpret_cast<const u32x4_t*>(Q + r * 64 + ((g ^ row_swizzle(li)) * 16));
            }
        }
#pragma unroll
        for (int i = 0; i < FI; ++i) {
            const int r = wi * S::kWaveI + 16 * i + li;
            x[i] = *reinterpret_cast<const u32x4_t*>(P + r * 64 + ((g ^ row_swizzle(li)) * 16));
        }
    };
    auto multiply = [&](const u32x4_t (&x)[FI], const u32x4_t (&y)[FJ]) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) acc[i][j] = mfma16<_Float16>(y[j], x[i], acc[i][j]);
    };

    // Step n goes to stage n % kStages; kStages - 1 steps are under way at most, the latest
    // kStages - 2 of them past the wait for one.
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n)
        if (n < all) issue(n, n);
    for (int32_t n = 0, stage = 0; n < all; ++n) {
        if (n + kStages - 2 < all)
            dma_wait<(kStages - 2) * kLoads>();
        else
            dma_wait<0>();
        // all have in registers what stood where the next loads go
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (n + kStages - 1 < all) issue(n + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
        Operands hi, lo;
        read(stage, 0, hi);
        if constexpr (SPLIT) read(stage, 1, lo);
        __builtin_amdgcn_s_setprio(1);
        multiply(hi.x, hi.y);
        if constexpr (SPLIT) {
            multiply(hi.x, lo.y);
            multiply(lo.x, hi.y);
        }
        __builtin_amdgcn_s_setprio(0);
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }

    // a lane has columns 4 g .. + 3 of row li of every tile of 16 x 16
    static_assert(FJ % 2 == 0 && FI % 2 == 0);
    const int64_t iw = i0 + wi * S::kWaveI, jw = j0 + wj * S::kWaveJ;
    if constexpr (PURPOSE == kPart) {
        float4_t* part = reinterpret_cast<float4_t*>(a.part) + ((int64_t)item * (TI * TJ / 256) + wave * (FI * FJ)) * 64 + lane;
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) part[(i * FJ + j) * 64] = acc[i][j];
    } else if constexpr (PURPOSE == kGram || PURPOSE == kSquare) {
        __syncthreads();
        _Float16* turn = reinterpret_cast<_Float16*>(smem) + wave * 2048;
#pragma unroll
        for (int i = 0; i < FI; i += 2)
#pragma unroll
            for (int j = 0; j < FJ; j += 2) {
                float v[2][8];
                pair_up(acc[i][j], acc[i][j + 1], v[0]);
                pair_up(acc[i + 1][j], acc[i + 1][j + 1], v[1]);
                finish_symmetric<T, PURPOSE>(f, v, iw + 16 * i, jw + 16 * j, li, g, j0 + TJ <= i0, turn);
            }
    } else {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; j += 2) {
                float v[8];
                pair_up(acc[i][j], acc[i][j + 1], v);
                finish_product<T, PURPOSE>(f, v, iw + 16 * i, jw + 16 * j, li, g);
            }
    }
}

// The shares of a tile's sums, in their order; a wave to 32 x 32 of them.
template <typename T, int TI, int PURPOSE>
__global__ __launch_bounds__(256) void ff_orthogonal_join_kernel(const Product a, const Finish<T> f)
{
    using S = Shape<TI, is_split<T>>;
    constexpr int FI = S::FI, FJ = S::FJ, TJ = S::TJ, kPieces = TI * TJ / 4096;  // workgroups of a tile
    __shared__ __align__(16) _Float16 turn[4][2048];
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x / kPieces;
    // the product's wave, and its tiles (i, j) to (i + 1, j + 1)
    const int piece = (int)(blockIdx.x % kPieces) * 4 + wave, of = piece / (FI * FJ / 4);
    const int i = piece % (FI * FJ / 4) / (FJ / 2) * 2, j = piece % (FJ / 2) * 2;
    int32_t ti, tj;
    tile_place<TI>(a, tile, ti, tj);
    const int64_t i0 = (int64_t)ti * TI, j0 = (int64_t)tj * TJ;
    const float4_t* part =
        reinterpret_cast<const float4_t*>(a.part) + ((int64_t)tile * a.splits * (TI * TJ / 256) + of * (FI * FJ)) * 64 + lane;
    float4_t v[2][2] = {};
    for (int32_t s = 0; s < a.splits; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < 2; ++w)
                v[u][w] += part[(s * (int64_t)(TI * TJ / 256) + (i + u) * FJ + j + w) * 64];
    float e[2][8];
    pair_up(v[0][0], v[0][1], e[0]);
    pair_up(v[1][0], v[1][1], e[1]);
    finish_symmetric<T, PURPOSE>(f, e, i0 + (of & 1) * S::kWaveI + 16 * i, j0 + (of >> 1) * S::kWaveJ + 16 * j, li, g,
                                 j0 + TJ <= i0, turn[wave]);
}

// Sums of squares of the stored values inside the weight, a share of the blocks each.
constexpr int kNormShares = 512, kNormWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kNormWaves) void ff_square_sum_kernel(const T* __restrict__ u, const int32_t* __restrict__ row,
                                                            const int32_t* __restrict__ col, int64_t nnzb, int32_t M,
                                                            int32_t K, double* __restrict__ part)
{
    __shared__ double red[kNormWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum = 0.0;
    for (int64_t b = blockIdx.x * kNormWaves + wave; b < nnzb; b += kNormWaves * kNormShares) {
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
    if (threadIdx.x == 0) {
        double all = red[0];
        for (int w = 1; w < kNormWaves; ++w) all += red[w];
        part[blockIdx.x] = all;
    }
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
    // a wave per block (less than 2^31 of them: they have 1 KB each)
    const int lane = t & 63;
    const uint32_t per = (uint32_t)(f.ld / 32), blocks = (uint32_t)(rows / 16) * per;
    for (uint32_t block = blockIdx.x * 4 + (uint32_t)(t >> 6); block < blocks; block += gridDim.x * 4) {
        const uint32_t br = block / per;
        const int64_t e = (int64_t)block * 64 + lane, i = (int64_t)br * 16 + lane / 4, j = (int64_t)(block - br * per) * 32 + lane % 4 * 8;
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
        *reinterpret_cast<Pack<_Float16, 8>*>(f.out.hi + e * 8) = hi;
        *reinterpret_cast<Pack<_Float16, 8>*>(f.out.lo + e * 8) = lo;
    }
}

// Sizes and memory of one orthogonalised update.
struct OrthogonalPlan {
    bool transposed, split;
    int tile;      // rows of one
    int64_t m, k;  // rows and columns of X, to whole tiles
    int gram_splits, square_splits;
    size_t x_hi[2], x_lo[2], s_hi, s_lo, b_hi, b_lo, diagonal, norm, part, end;
};

OrthogonalPlan orthogonal_plan(const BlockIndex& w, bool split)
{
    OrthogonalPlan p{};
    p.transposed = w.M > w.K;
    p.split = split;
    const int64_t rows = p.transposed ? w.K : w.M, columns = p.transposed ? w.M : w.K;
    // The largest tiles of which there are enough: a CU gets no more than 25 GB/s of what
    // other dies have just written, and few workgroups wait for that, while small tiles read
    // their operands more often.  us by 64 and 128 rows: bf16 512 x 1792 137 and 195, 1000 x
    // 2500 227 and 275, 2048 x 2048 434 and 452, fp32 1000 x 2500 334 and 362; by 128 and
    // 256: bf16 1536 x 4096 410 and 440, 2048 x 5632 706 and 661.  With operands in two halves
    // there is no size for 128 (fp32 1536 x 4096 757, by 256 726).
    auto count = [&](int64_t side) { return (rows + side - 1) / side * ((columns + side - 1) / side); };
    p.tile = count(64) <= 1024 ? 64 : !p.split && count(128) <= 512 ? 128 : 256;
    const int64_t tj = tile_columns(p.tile);
    p.m = (rows + p.tile - 1) / p.tile * p.tile;
    p.k = (columns + tj - 1) / tj * tj;
    const int64_t n = p.m / p.tile, tiles = n * (n + 1) / 2 * (p.tile / tj);
    // Shares of a sum: rounds of workgroups, two a CU (one where operands are split, whose
    // steps take three times as long), and what a launch and joining cost, in steps' time.
    const int64_t at_once = p.split ? 256 : 512;
    const double step = p.split ? 3.0 : 1.0;
    auto splits = [&](int64_t steps) {
        int best = 1;
        double least = 1e30;
        for (int s = 1; s <= 8 && steps / s >= 8; ++s) {
            const double join = s == 1 ? 0.0 : 19.0 + 0.08 * (double)(s * tiles);
            const double time = (double)((tiles * s + at_once - 1) / at_once) * ((double)steps / s * step + 28.0) + join;
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
    p.part = c.take(most > 1 ? (size_t)(tiles * most * p.tile * tj) * 4 : 0);
    p.end = c.end;
    return p;
}

template <typename T, int TI, bool ACROSS, int PURPOSE>
void launch_orthogonal(Product a, const Finish<T>& f, hipStream_t s)
{
    const int64_t tiles = product_tiles(a);
    constexpr int threads = kProductThreads;
    const dim3 grid = launch_grid(kXcds * xcd_chunk(tiles * a.splits), threads);
    a.items = (uint32_t)(tiles * a.splits);
    if (a.splits > 1) {
        if constexpr (!ACROSS) {
            hipLaunchKernelGGL((ff_orthogonal_product_kernel<T, TI, ACROSS, kPart>), grid, dim3(threads), 0, s, a, f);
            hipLaunchKernelGGL((ff_orthogonal_join_kernel<T, TI, PURPOSE>), launch_grid(tiles * (TI * tile_columns(TI) / 4096), 256),
                               dim3(256), 0, s, a, f);
        }
    } else {
        hipLaunchKernelGGL((ff_orthogonal_product_kernel<T, TI, ACROSS, PURPOSE>), grid, dim3(threads), 0, s, a, f);
    }
    XSPMM_LAUNCH_CHECK();
}

template <typename T, int TI>
void orthogonal_steps(const BlockIndex& w, const T* update, T* out, const OrthogonalArgs& o, const OrthogonalPlan& p,
                      char* at, hipStream_t s)
{
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
    hipLaunchKernelGGL((ff_square_sum_kernel<T>), dim3(kNormShares), dim3(64 * kNormWaves), 0, s, update, w.row, w.col, w.nnzb,
                       (int32_t)w.M, (int32_t)w.K, norm);
    f.out = x[0];
    f.ld = p.k;
    hipLaunchKernelGGL((ff_orthogonal_start_kernel<T>), dim3(4096), dim3(256), 0, s, f, update, norm, (double)o.eps, p.m);
    XSPMM_LAUNCH_CHECK();
    for (int step = 0; step < o.steps; ++step) {
        const Halves &from = x[step % 2], &to = x[(step + 1) % 2];
        Product a{};
        a.part = reinterpret_cast<float*>(at + p.part);
        a.p = a.q = from;
        a.p_ld = a.q_ld = p.k;
        a.tiles_i = (int32_t)(p.m / TI);
        a.tiles_j = (int32_t)(p.m / tile_columns(TI));
        a.steps = (int32_t)(p.k / kDeepK);
        a.splits = p.gram_splits;
        a.lower = true;
        f.out = S;
        f.ld = p.m;
        launch_orthogonal<T, TI, false, kGram>(a, f, s);
        a.p = a.q = S;
        a.p_ld = a.q_ld = p.m;
        a.steps = (int32_t)(p.m / kDeepK);
        a.splits = p.square_splits;
        f.s = S;
        f.out = B;
        launch_orthogonal<T, TI, false, kSquare>(a, f, s);
        a.p = B;
        a.q = from;
        a.q_ld = p.k;
        a.tiles_j = (int32_t)(p.k / tile_columns(TI));
        a.splits = 1;
        a.lower = false;
        f.x = from;
        f.out = to;
        f.ld = p.k;
        if (step + 1 < o.steps)
            launch_orthogonal<T, TI, true, kApply>(a, f, s);
        else
            launch_orthogonal<T, TI, true, kLast>(a, f, s);
    }
}

}  // namespace ff

template <typename T>
int64_t orthogonal_scratch(const BlockIndex& w)
{
    if (w.nnzb == 0) return 0;
    return (int64_t)ff::orthogonal_plan(w, ff::is_split<T>).end;
}

template <typename T>
void orthogonalize(const BlockIndex& w, const T* update, T* out, const OrthogonalArgs& o, void* scratch, hipStream_t s)
{
    if (w.nnzb == 0) return;
    const ff::OrthogonalPlan p = ff::orthogonal_plan(w, ff::is_split<T>);
    char* at = static_cast<char*>(scratch);
    if (p.tile == 64)
        ff::orthogonal_steps<T, 64>(w, update, out, o, p, at, s);
    else if (p.tile == 256)
        ff::orthogonal_steps<T, 256>(w, update, out, o, p, at, s);
    else if constexpr (!ff::is_split<T>)
        ff::orthogonal_steps<T, 128>(w, update, out, o, p, at, s);
}

#define XSPMM_ORTHOGONAL(T)                                     \
    template int64_t orthogonal_scratch<T>(const BlockIndex&); \
    template void orthogonalize<T>(const BlockIndex&, const T*, T*, const OrthogonalArgs&, void*, hipStream_t);
XSPMM_ORTHOGONAL(float)
XSPMM_ORTHOGONAL(_Float16)
XSPMM_ORTHOGONAL(__bf16)
#undef XSPMM_ORTHOGONAL

}  // namespace detail
}  // namespace xspmm
