// ff_sampled.hip -- the gradient of a weight's stored blocks: the product
// dz x^T, 16 x 16 tokens-long dot products at each block's position.
//
// The sum runs along the tokens, which are contiguous in both operands, so the
// matrix instructions' operands are plain pieces of rows.  x is the left
// operand: a lane's four results are consecutive columns of one row of the
// block and leave as one store.
#include "feed_forward_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// ---------------------------------------------------------------------------
// One wave per stored block (SPLIT waves share its tokens), operands straight
// from memory: for 32-bit values, few blocks, and operands of any size.
// ---------------------------------------------------------------------------

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

// ---------------------------------------------------------------------------
// 16-bit tiles: a workgroup takes 128 rows of dz and 128 rows of x, 64 tokens at
// a time through LDS, and multiplies where the tile holds a block.  A wave owns
// 4 x 4 of its positions, with an accumulator for each.
//
// Every row of the tile is read once for all its blocks, where the kernel above
// reads both rows anew for each block; what is not stored costs its share of the
// reads but no matrix instruction.
// ---------------------------------------------------------------------------

template <typename T>
struct SampledSide {
    const int32_t* map;
    const T* dz;
    T* dvals;
};

template <typename T>
struct SampledTile {
    SampledSide<T> side[2];
    const T* x;
    int32_t M, K, Mb, Kb;
    int64_t N;
    uint32_t dz_bytes, x_bytes;
    int64_t items;  // tiles of one side
    int32_t sides;
};

constexpr int kWR = 2, kWC = 2, kB = 4;   // a grid of 2 x 2 waves with 4 x 4 positions each
constexpr int kEdge = kWR * kB;           // blocks along either edge of a tile
constexpr int kSide = 16 * kEdge;         // its rows of dz, and of x
constexpr int kThreads = 64 * kWR * kWC;
constexpr int kTokens = 64;               // per step: a row's piece is 8 chunks of 16 bytes, a line of memory
constexpr int kPieces = kTokens / 8;
constexpr int kStage = 2 * kSide * 2 * kTokens;
constexpr int kLoads = 2 * kSide * kPieces / kThreads;  // chunks a thread moves per step
constexpr int kBand = 8;
static_assert(kWR == kWC && kEdge * kEdge <= kThreads && kB * kB <= 32);

template <typename T, bool DMA>
__global__ __launch_bounds__(kThreads) void ff_sampled_tile_kernel(const SampledTile<T> a)
{
    __shared__ __align__(16) unsigned char smem[2 * kStage];
    __shared__ int32_t place[kEdge * kEdge];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int wr = wave / kWC, wc = wave % kWC;

    int64_t item = xcd_item(blockIdx.x, a.items * a.sides);
    if (item < 0) return;
    const int which = item >= a.items;
    const SampledSide<T> s = a.side[which];
    item -= which * a.items;
    const int32_t panels = (a.Kb + kEdge - 1) / kEdge;
    // bands of kBand row panels, column panel by column panel: what an XCD works
    // on at a time is about square, so that its L2 sees each row the most often
    const int32_t tall = (a.Mb + kEdge - 1) / kEdge;
    const int32_t band = (int32_t)(item / ((int64_t)kBand * panels)) * kBand;
    const int32_t h = min(kBand, tall - band), in = (int32_t)(item - (int64_t)band * panels);
    const int32_t br0 = (band + in % h) * kEdge, bc0 = in / h * kEdge;

    // which blocks of the tile are stored, and where
    if (t < kEdge * kEdge) {
        const int32_t r = br0 + t / kEdge, c = bc0 + t % kEdge;
        place[t] = r < a.Mb && c < a.Kb ? s.map[(int64_t)r * a.Kb + c] : -1;
    }
    __syncthreads();
    uint32_t mask;  // bit r kB + c: this wave's block (r, c) is stored
    {
        const int r = lane / kB, c = lane % kB;
        const bool there = lane < kB * kB && place[(wr * kB + r) * kEdge + wc * kB + c] >= 0;
        mask = (uint32_t)__ballot(there);
    }
    if (!__syncthreads_or(mask != 0)) return;

    // Thread t moves, for each j, what lies at chunk t % 8 of tile row
    // t / 8 + j kThreads / 8 (rows of dz, then of x): chunk (t % 8) ^ (row % 8) of
    // the row's piece, so that the rows that an operand read touches lie in
    // different banks.
    auto swizzle = [](int row) { return row % 8; };
    uint32_t base[kLoads];
    const uint32_t ld = (uint32_t)a.N * 2u;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int row = t / kPieces + j * (kThreads / kPieces);
        const bool is_dz = row < kSide;
        const int32_t at = is_dz ? 16 * br0 + row : 16 * bc0 + row - kSide;
        base[j] = at < (is_dz ? a.M : a.K) ? (uint32_t)at * ld : kNone;
    }
    const int chunk = (t % kPieces) ^ swizzle(t / kPieces);  // kThreads / kPieces is a multiple of 8
    const int32_t steps = (int32_t)((a.N + kTokens - 1) / kTokens);
    const uint32_t lds0 = lds_address(smem);
    const i32x4_t dma_dz = dma_buffer(s.dz, a.dz_bytes), dma_x = dma_buffer(a.x, a.x_bytes);
    u32x4_t held[DMA ? 1 : kLoads];
    auto issue = [&](int32_t st) {
        const int32_t n = st * kTokens + 8 * chunk;
        if constexpr (DMA) {
            const uint32_t to = lds0 + (uint32_t)(st % 2) * kStage + (uint32_t)wave * 1024u;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const uint32_t off = n < a.N && base[j] != kNone ? base[j] + (uint32_t)n * 2u : kNone;
                dma_to_lds(to + (uint32_t)j * (kThreads * 16u), off, j < kSide * kPieces / kThreads ? dma_dz : dma_x);
            }
        } else {
            const auto bd = make_buffer(s.dz, a.dz_bytes), bx = make_buffer(a.x, a.x_bytes);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const auto& b = j < kSide * kPieces / kThreads ? bd : bx;
                if (st + 1 < steps || n + 8 <= a.N) {
                    const auto v = buffer_load<T, 8>(b, base[j] != kNone ? base[j] + (uint32_t)n * 2u : kNone);
                    held[j] = u32x4_t{v.d[0], v.d[1], v.d[2], v.d[3]};
                } else {  // the row ends within the chunk
                    held[j] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n + i < a.N && base[j] != kNone)
                            held[j][i / 2] |= buffer_load<T, 1>(b, base[j] + (uint32_t)(n + i) * 2u).d[0] << (16 * (i % 2));
                }
            }
        }
    };

    float4_t acc[kB][kB];
#pragma unroll
    for (int r = 0; r < kB; ++r)
#pragma unroll
        for (int c = 0; c < kB; ++c) acc[r][c] = float4_t{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int32_t st) {
#pragma unroll
        for (int h = 0; h < kTokens / 32; ++h) {
            const unsigned char* S =
                smem + (st % 2) * kStage + li * (2 * kTokens) + (((4 * h + g) ^ swizzle(li)) * 16);
            u32x4_t xo[kB];
#pragma unroll
            for (int c = 0; c < kB; ++c)
                xo[c] = *reinterpret_cast<const u32x4_t*>(S + (kSide + 16 * (wc * kB + c)) * (2 * kTokens));
#pragma unroll
            for (int r = 0; r < kB; ++r) {
                if (!((mask >> (r * kB)) & ((1u << kB) - 1u))) continue;
                const u32x4_t d = *reinterpret_cast<const u32x4_t*>(S + 16 * (wr * kB + r) * (2 * kTokens));
#pragma unroll
                for (int c = 0; c < kB; ++c)
                    if (mask & (1u << (r * kB + c))) acc[r][c] = mfma16<T>(xo[c], d, acc[r][c]);
            }
        }
    };

    // Step st is computed while the loads of the next are under way, which go
    // where step st - 1 was read before this step's barrier.
    if (steps > 0) issue(0);
    for (int32_t st = 0; st < steps; ++st) {
        if constexpr (DMA) {
            dma_wait<0>();
        } else {
            unsigned char* to = smem + (st % 2) * kStage + t * 16;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) *reinterpret_cast<u32x4_t*>(to + j * (kThreads * 16)) = held[j];
        }
        __syncthreads();
        if (st + 1 < steps) issue(st + 1);
        compute(st);
    }

    // lane: row li of a block, columns 4 g .. + 3
#pragma unroll
    for (int r = 0; r < kB; ++r)
#pragma unroll
        for (int c = 0; c < kB; ++c) {
            if (!(mask & (1u << (r * kB + c)))) continue;
            const int32_t b = place[(wr * kB + r) * kEdge + wc * kB + c];
            const int32_t row = 16 * (br0 + wr * kB + r) + li, col = 16 * (bc0 + wc * kB + c) + 4 * g;
            Pack<T, 4> o;
#pragma unroll
            for (int q = 0; q < 4; ++q) o.v[q] = (T)(row < a.M && col + q < a.K ? acc[r][c][q] : 0.f);
            *reinterpret_cast<Pack<T, 4>*>(s.dvals + (int64_t)b * 256 + li * 16 + 4 * g) = o;
        }
}

template <typename T>
void launch_sampled_tile(SampledTile<T>& a, bool aligned, hipStream_t s)
{
    a.items = (int64_t)((a.Mb + kEdge - 1) / kEdge) * ((a.Kb + kEdge - 1) / kEdge);
    const int64_t grid = kXcds * xcd_chunk(a.items * a.sides);
    if (grid > 0x7fffffffLL) throw std::invalid_argument("xSpMM: too many blocks for one launch.");
    if (aligned)
        hipLaunchKernelGGL((ff_sampled_tile_kernel<T, true>), dim3((unsigned)grid),
                           dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((ff_sampled_tile_kernel<T, false>), dim3((unsigned)grid),
                           dim3(kThreads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

// Both weights of a gated layer in one launch; false where tiles do not apply.
template <typename T>
bool sampled_tiles(const SampledArgs<T>& f, int weights, hipStream_t s)
{
    if constexpr (is_f32<T>) {
        return false;
    } else {
        const BlockIndex& w = *f.weight[0];
        SampledTile<T> a{};
        a.x = f.x;
        a.M = (int32_t)w.M;
        a.K = (int32_t)w.K;
        a.Mb = (int32_t)w.Mb;
        a.Kb = (int32_t)w.Kb;
        a.N = f.N;
        const int64_t db = narrow_bytes(w.M, f.N, 2), xb = narrow_bytes(w.K, f.N, 2);
        if (db < 0 || xb < 0 || f.N == 0) return false;
        a.dz_bytes = (uint32_t)db;
        a.x_bytes = (uint32_t)xb;
        for (int l = 0; l < weights; ++l) {
            if (!f.dvals[l]) continue;
            if (!f.weight[l]->map) return false;
            a.side[a.sides++] = {f.weight[l]->map, f.dz[l], f.dvals[l]};
        }
        if (a.sides == 0) return true;
        launch_sampled_tile<T>(a, f.N % 8 == 0, s);
        return true;
    }
}

}  // namespace ff

template <typename T>
void sampled_product(const SampledArgs<T>& f, int weights, hipStream_t s)
{
    if (ff::sampled_tiles<T>(f, weights, s)) return;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& w = *f.weight[l];
        if (!f.dvals[l] || w.nnzb == 0) continue;
        if (w.nnzb < 4096 && f.N >= 512)
            hipLaunchKernelGGL((ff::ff_sampled_kernel<T, 4>), dim3((unsigned)w.nnzb), dim3(256), 0, s, w.row, w.col,
                               f.dz[l], f.x, f.dvals[l], w.nnzb, (int32_t)w.M, (int32_t)w.K, f.N);
        else
            hipLaunchKernelGGL((ff::ff_sampled_kernel<T, 1>), dim3((unsigned)((w.nnzb + 3) / 4)), dim3(256), 0, s,
                               w.row, w.col, f.dz[l], f.x, f.dvals[l], w.nnzb, (int32_t)w.M, (int32_t)w.K, f.N);
        XSPMM_LAUNCH_CHECK();
    }
}

template void sampled_product<float>(const SampledArgs<float>&, int, hipStream_t);
template void sampled_product<_Float16>(const SampledArgs<_Float16>&, int, hipStream_t);
template void sampled_product<__bf16>(const SampledArgs<__bf16>&, int, hipStream_t);

}  // namespace detail
}  // namespace xspmm
