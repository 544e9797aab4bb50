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
// One wave per four consecutive blocks (SPLIT waves share their tokens), operands
// straight from memory: for short rows and operands of any size.  A load of 16 rows'
// 16 bytes costs a lookup per row and lane, 64 of them, which is what bounds it
// (14336 x 4096 fp16, one token, 30 % stored: 25 us; 2047 tokens, 3 %: 366).
// ---------------------------------------------------------------------------

constexpr int kGroup = kGroupBlocks;  // stored blocks of a wave

// A weight's blocks by fours; the two weights of a gated layer are the grid's rows.
template <typename T>
struct SampledFours {
    const int32_t* group;
    const int32_t* ptr;
    const int32_t* row;
    const int32_t* col;
    const T* dz;
    T* dvals;
    int64_t nnzb, groups;
};
template <typename T>
struct SampledArray {
    SampledFours<T> side[2];
    const T* x;
    int32_t M, K;
    int64_t N;
    uint32_t dz_bytes, x_bytes;
};

// One step's operands: V tokens of a row per lane
template <typename T, int ROWS>
struct SampledStep {
    u32x4_t d[ROWS], x[kGroup];
};

template <typename T, int SPLIT>
__global__ __launch_bounds__(256) void ff_sampled_kernel(const SampledArray<T> a)
{
    const SampledFours<T>& s = a.side[blockIdx.y];
    const int32_t* const __restrict__ row = s.row;
    const int32_t* const __restrict__ col = s.col;
    const T* const __restrict__ dz = s.dz;
    const T* const __restrict__ x = a.x;
    T* const __restrict__ dvals = s.dvals;
    const int64_t nnzb = s.nnzb, N = a.N;
    const int32_t M = a.M, K = a.K;
    constexpr int V = 16 / sizeof(T);  // tokens a lane takes per step
    constexpr int kStep = 4 * V;
    constexpr int kPer = 4 / SPLIT;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int64_t b0 = ((int64_t)blockIdx.x * kPer + wave / SPLIT) * kGroup;
    const int part = wave % SPLIT;
    if ((int64_t)blockIdx.x * kPer * kGroup >= nnzb) return;  // the other weight has more
    float4_t acc[kGroup];
    int32_t r0[kGroup], c0[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
        const int64_t b = min(b0 + i, nnzb - 1);  // past the last block: the last one again, not stored
        r0[i] = 16 * row[b];
        c0[i] = 16 * col[b];
    }
    // whole: all lanes' tokens are there, without a condition around the load (one
    // makes the wave wait for it before the next)
    auto tokens = [&](const T* p, int64_t n, auto whole) {
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (decltype(whole)::value || n + V <= N) {
            const auto q = global_load<T, V>(p + n);
            v = u32x4_t{q.d[0], q.d[1], q.d[2], q.d[3]};
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (n + i < N) {
                    const uint32_t q = global_load<T, 1>(p + n + i).d[0];
                    if constexpr (is_f32<T>)
                        v[i] = q;
                    else
                        v[i / 2] |= q << (16 * (i % 2));
                }
        }
        return v;
    };
    // ROWS: 1 where the blocks stand in one block-row, else one operand each
    auto run = [&](auto rows) {
        constexpr int ROWS = decltype(rows)::value;
        // rows past the edge read the last one; their results are not kept
        const T *pd[ROWS], *px[kGroup];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) pd[i] = dz + (int64_t)min(r0[i] + li, M - 1) * N;
#pragma unroll
        for (int i = 0; i < kGroup; ++i) px[i] = x + (int64_t)min(c0[i] + li, K - 1) * N;
        auto load = [&](SampledStep<T, ROWS>& s, int64_t st, auto whole) {
            const int64_t n = st * kStep + V * g;
#pragma unroll
            for (int i = 0; i < ROWS; ++i) s.d[i] = tokens(pd[i], n, whole);
#pragma unroll
            for (int i = 0; i < kGroup; ++i) s.x[i] = tokens(px[i], n, whole);
        };
        auto multiply = [&](const SampledStep<T, ROWS>& s) {
#pragma unroll
            for (int i = 0; i < kGroup; ++i) {
                const u32x4_t d = s.d[ROWS == 1 ? 0 : i];
                if constexpr (is_f32<T>) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i] = mfma32(s.x[i][q], d[q], acc[i]);
                } else {
                    acc[i] = mfma16<T>(s.x[i], d, acc[i]);
                }
            }
        };
        const int64_t steps = (N + kStep - 1) / kStep;
        int64_t st = steps * part / SPLIT;
        const int64_t hi = steps * (part + 1) / SPLIT, full = min(hi, N / kStep);
        const std::true_type yes{};
        // whole steps: the loads of one run ahead of the instructions of the last
        if (st < full) {
            SampledStep<T, ROWS> a, b;
            load(a, st, yes);
            for (;; st += 2) {
                load(b, min(st + 1, full - 1), yes);
                multiply(a);
                if (st + 1 >= full) break;
                load(a, min(st + 2, full - 1), yes);
                multiply(b);
                if (st + 2 >= full) break;
            }
            st = full;
        }
        if (st < hi) {
            SampledStep<T, ROWS> a;
            load(a, st, std::false_type{});
            multiply(a);
        }
    };
    if (b0 < nnzb && N > 0) {
        if (r0[0] == r0[kGroup - 1])
            run(std::integral_constant<int, 1>{});
        else
            run(std::integral_constant<int, kGroup>{});
    }
    if constexpr (SPLIT > 1) {
        __shared__ float4_t red[kPer][SPLIT][kGroup][64];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) red[wave / SPLIT][part][i][lane] = acc[i];
        __syncthreads();
        static_assert(SPLIT == kGroup);  // each wave finishes a block
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
            if (i != part) continue;
            acc[i] = red[wave / SPLIT][0][i][lane];
            for (int p = 1; p < SPLIT; ++p) acc[i] += red[wave / SPLIT][p][i][lane];
        }
    }
    // lane: row li of the block, columns 4 g .. + 3
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        if (b0 + i >= nnzb || (SPLIT > 1 && i != part)) continue;
        Pack<T, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = (T)(r0[i] + li < M && c0[i] + 4 * g + q < K ? acc[i][q] : 0.f);
        *reinterpret_cast<Pack<T, 4>*>(dvals + (b0 + i) * 256 + li * 16 + 4 * g) = o;
    }
}

// V tokens of a row from n on, at offset `off` of its array; whole: the row goes on
// past them.  Where the row ends within them they come one by one: what follows is
// another row's, and a load past the array's end gives whole dwords of zeros.
template <typename T>
__device__ __forceinline__ u32x4_t row_chunk(__amdgpu_buffer_rsrc_t b, uint32_t off, int32_t n, int64_t N, bool whole)
{
    constexpr int V = 16 / sizeof(T);
    if (whole || n + V <= N) {
        const auto v = buffer_load<T, V>(b, off);
        return u32x4_t{v.d[0], v.d[1], v.d[2], v.d[3]};
    }
    u32x4_t o = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (n + i < N && off != kNone) {
            const uint32_t q = buffer_load<T, 1>(b, off + (uint32_t)i * (uint32_t)sizeof(T)).d[0];
            if constexpr (is_f32<T>)
                o[i] = q;
            else
                o[i / 2] |= q << (16 * (i % 2));
        }
    return o;
}

// The same for blocks of one block-row: a wave moves 128 bytes of its rows of dz and
// x at a time into LDS of its own, in whole lines (the operands themselves are 16
// bytes of 16 rows, and memory serves one line at a time), while it multiplies the
// 128 bytes before.  It waits for nothing but its own loads.  DMA: rows on 16-byte
// boundaries go straight into LDS; others pass through registers and touch two lines
// for each.  Bound by the L2: four blocks read five blocks' rows, 14336 x 4096 fp16,
// 10 % stored, 2048 tokens 1.9 GB in 102 us, 18 TB/s, 2047 tokens 196 us (883 operand
// by operand); fp32 4096 x 4096, 10 %, 512 tokens 29.4 us (57 without LDS), 58 TFLOP/s.
template <typename T, int SPLIT, bool DMA>
__global__ __launch_bounds__(256, 2) void ff_sampled_wave_kernel(const SampledArray<T> a)
{
    const SampledFours<T>& s = a.side[blockIdx.y];
    constexpr int V = 16 / sizeof(T), kTokens = 128 / (int)sizeof(T);
    constexpr int kUnits = 1 + kGroup, kStage = kUnits * 16 * 128, kLoads = 2 * kUnits;
    constexpr int kPer = 4 / SPLIT;
    constexpr int kStages = DMA ? 2 : 1;
    __shared__ __align__(16) unsigned char smem[4][kStages][kStage];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g = lane >> 4;
    const int64_t items = (s.groups + kPer - 1) / kPer;
    const int64_t item = xcd_item(blockIdx.x, items);
    if (item < 0 || blockIdx.x / kXcds >= xcd_chunk(items)) return;  // the other weight has more
    const int64_t gi = item * kPer + wave / SPLIT;
    const int part = wave % SPLIT;
    const bool live = gi < s.groups;
    const int32_t b0 = live ? s.group[gi] : 0;
    const int32_t br = live ? s.row[b0] : 0;
    const int count = live ? min(s.ptr[br + 1] - b0, kGroup) : 0;
    int32_t c0[kGroup];
    float4_t acc[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
        c0[i] = 16 * s.col[min(b0 + i, b0 + max(count, 1) - 1)];
    }
    if (live) {
        // load j of a stage: rows 8 (j % 2) .. + 7 of unit j / 2 (dz, then the
        // blocks' rows of x); lane l lands at chunk l % 8 of row l / 8 and brings
        // chunk (l % 8) ^ (l / 8), so that an operand's rows are in different banks
        const uint32_t ld = (uint32_t)a.N * (uint32_t)sizeof(T);
        const int chunk = (lane & 7) ^ (lane >> 3);
        uint32_t off[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int32_t r = (j < 2 ? 16 * br : c0[j / 2 - 1 < 0 ? 0 : j / 2 - 1]) + 8 * (j % 2) + (lane >> 3);
            const bool in = j < 2 ? r < a.M : j / 2 <= count && r < a.K;
            off[j] = in ? (uint32_t)r * ld + (uint32_t)chunk * 16u : kNone;
        }
        const i32x4_t bd = dma_buffer(s.dz, a.dz_bytes), bx = dma_buffer(a.x, a.x_bytes);
        const uint32_t lds0 = lds_address(smem[wave]);
        const int32_t steps = (int32_t)((a.N + kTokens - 1) / kTokens);
        const int32_t lo = steps * part / SPLIT, hi = steps * (part + 1) / SPLIT;
        u32x4_t held[DMA ? 1 : kLoads];
        auto issue = [&](int32_t st) {
            const int32_t n = st * kTokens + V * chunk;
            if constexpr (DMA) {
                const uint32_t to = lds0 + (uint32_t)(st & 1) * kStage;
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    dma_to_lds(to + (uint32_t)j * 1024u, n < a.N ? off[j] + (uint32_t)st * 128u : kNone, j < 2 ? bd : bx);
            } else {
                const auto rd = make_buffer(s.dz, a.dz_bytes), rx = make_buffer(a.x, a.x_bytes);
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    held[j] = row_chunk<T>(j < 2 ? rd : rx, off[j] != kNone ? off[j] + (uint32_t)st * 128u : kNone, n, a.N,
                                           st + 1 < steps);
            }
        };
        if (lo < hi) issue(lo);
        for (int32_t st = lo; st < hi; ++st) {
            if constexpr (DMA) {
                // the last reads of the stage that is loaded next are over
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (st + 1 < hi) {
                    issue(st + 1);
                    dma_wait<kLoads>();
                } else {
                    dma_wait<0>();
                }
            } else {
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    *reinterpret_cast<u32x4_t*>(smem[wave][0] + j * 1024 + lane * 16) = held[j];
                if (st + 1 < hi) issue(st + 1);
            }
            const unsigned char* S = smem[wave][DMA ? st & 1 : 0] + li * 128;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int piece = ((4 * h + g) ^ (li & 7)) * 16;
                const u32x4_t d = *reinterpret_cast<const u32x4_t*>(S + piece);
#pragma unroll
                for (int i = 0; i < kGroup; ++i) {
                    const u32x4_t xo = *reinterpret_cast<const u32x4_t*>(S + (1 + i) * 2048 + piece);
                    if constexpr (is_f32<T>) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[i] = mfma32(xo[q], d[q], acc[i]);
                    } else {
                        acc[i] = mfma16<T>(xo, d, acc[i]);
                    }
                }
            }
        }
    }
    if constexpr (SPLIT > 1) {
        static_assert(SPLIT == kGroup && kGroup * 4 * 64 * 16 <= sizeof(smem));
        float4_t(*red)[kGroup][64] = reinterpret_cast<float4_t(*)[kGroup][64]>(&smem[0][0][0]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kGroup; ++i) red[wave][i][lane] = acc[i];
        __syncthreads();
        // each wave finishes a block
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
            if (i == part) {
                acc[i] = red[0][i][lane];
                for (int p = 1; p < SPLIT; ++p) acc[i] += red[p][i][lane];
            }
    }
    // lane: row li of the block, columns 4 g .. + 3
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
        if (i >= count || (SPLIT > 1 && i != part)) continue;
        Pack<T, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = (T)(16 * br + li < a.M && c0[i] + 4 * g + q < a.K ? acc[i][q] : 0.f);
        *reinterpret_cast<Pack<T, 4>*>(s.dvals + (int64_t)(b0 + i) * 256 + li * 16 + 4 * g) = o;
    }
}

template <typename T>
void sampled_fours(const SampledArgs<T>& f, int weights, hipStream_t s)
{
    const BlockIndex& w = *f.weight[0];
    const int64_t db = narrow_bytes(w.M, f.N, sizeof(T)), xb = narrow_bytes(w.K, f.N, sizeof(T));
    SampledArray<T> a{};
    a.x = f.x;
    a.M = (int32_t)w.M;
    a.K = (int32_t)w.K;
    a.N = f.N;
    a.dz_bytes = (uint32_t)db;
    a.x_bytes = (uint32_t)xb;
    unsigned sides = 0;
    int64_t groups = 0, fours = 0, most_groups = 0, most_fours = 0;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *f.weight[l];
        if (!f.dvals[l] || wl.nnzb == 0) continue;
        a.side[sides++] = {wl.group, wl.ptr, wl.row, wl.col, f.dz[l], f.dvals[l], wl.nnzb, wl.groups};
        const int64_t n = (wl.nnzb + kGroup - 1) / kGroup;
        groups += wl.groups;
        fours += n;
        most_groups = wl.groups > most_groups ? wl.groups : most_groups;
        most_fours = n > most_fours ? n : most_fours;
    }
    if (sides == 0) return;
    auto go = [&](auto kernel, int64_t grid) {
        hipLaunchKernelGGL(kernel, launch_grid(grid, 256, sides), dim3(256), 0, s, a);
        XSPMM_LAUNCH_CHECK();
    };
    // rows of at least a line, through LDS (off 16 bytes, 14336 x 4096 fp16, 30 %
    // stored: 75 tokens 56 us and 86 operand by operand, 37 tokens 49 and 46)
    const bool aligned = f.N * sizeof(T) % 16 == 0;
    if (db >= 0 && xb >= 0 && f.N != 0 && (aligned || f.N * sizeof(T) >= 128)) {
        const bool split = groups < 2048 && f.N * sizeof(T) >= 1024;
        const int64_t grid = kXcds * xcd_chunk(split ? most_groups : (most_groups + 3) / 4);
        if (aligned)
            split ? go(ff_sampled_wave_kernel<T, 4, true>, grid) : go(ff_sampled_wave_kernel<T, 1, true>, grid);
        else
            split ? go(ff_sampled_wave_kernel<T, 4, false>, grid) : go(ff_sampled_wave_kernel<T, 1, false>, grid);
    } else if (fours < 2048 && f.N >= 256) {
        go(ff_sampled_kernel<T, 4>, most_fours);
    } else {
        go(ff_sampled_kernel<T, 1>, (most_fours + 3) / 4);
    }
}

// ---------------------------------------------------------------------------
// Tiles: a workgroup takes 128 rows of dz and 128 rows of x, 128 bytes of each at
// a time through LDS, and multiplies where the tile holds a block.  Each of eight
// waves owns 2 x 4 of its positions, with an accumulator for each; two workgroups
// share a CU.  (With four waves of 4 x 4, which read a third less from LDS but are
// two a SIMD, 14336 x 4096 fp16 of 2048 tokens took 222 us at 25 % stored and 270 at
// 100 %; so it is 174 and 245, 980 TFLOP/s.  The loads alone, 3.8 GB at 24 TB/s from
// L2, take 157.)
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

constexpr int kWR = 4, kWC = 2;           // a grid of waves,
constexpr int kBR = 2, kBC = 4;           // the positions of each
constexpr int kEdge = kWR * kBR;          // blocks along either edge of a tile
constexpr int kSide = 16 * kEdge;         // its rows of dz, and of x
constexpr int kThreads = 64 * kWR * kWC;
constexpr int kLine = 128;                // bytes of a row per step, a line of memory
constexpr int kPieces = kLine / 16;
constexpr int kStage = 2 * kSide * kLine;
constexpr int kLoads = 2 * kSide * kPieces / kThreads;  // chunks a thread moves per step
constexpr int kBand = 8;
static_assert(kWR * kBR == kWC * kBC && kEdge * kEdge <= kThreads && kBR * kBC <= 32);

template <typename T, bool DMA>
__global__ __launch_bounds__(kThreads, kThreads / 128) void ff_sampled_tile_kernel(const SampledTile<T> a)
{
    constexpr int V = 16 / sizeof(T);                // tokens of a chunk
    constexpr int kTokens = kLine / (int)sizeof(T);  // of a step
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
    uint32_t mask;  // bit r kBC + c: this wave's block (r, c) is stored
    {
        const int r = lane / kBC, c = lane % kBC;
        const bool there = lane < kBR * kBC && place[(wr * kBR + r) * kEdge + wc * kBC + c] >= 0;
        mask = (uint32_t)__ballot(there);
    }
    if (!__syncthreads_or(mask != 0)) return;

    // Thread t moves, for each j, what lies at chunk t % 8 of tile row
    // t / 8 + j kThreads / 8 (rows of dz, then of x): chunk (t % 8) ^ (row % 8) of
    // the row's piece, so that the rows that an operand read touches lie in
    // different banks.
    auto swizzle = [](int row) { return row % 8; };
    uint32_t base[kLoads];
    constexpr uint32_t kSize = sizeof(T);
    const uint32_t ld = (uint32_t)a.N * kSize;
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
        const int32_t n = st * kTokens + V * chunk;
        if constexpr (DMA) {
            const uint32_t to = lds0 + (uint32_t)(st % 2) * kStage + (uint32_t)wave * 1024u;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const uint32_t off = n < a.N && base[j] != kNone ? base[j] + (uint32_t)n * kSize : kNone;
                dma_to_lds(to + (uint32_t)j * (kThreads * 16u), off, j < kSide * kPieces / kThreads ? dma_dz : dma_x);
            }
        } else {
            const auto bd = make_buffer(s.dz, a.dz_bytes), bx = make_buffer(a.x, a.x_bytes);
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
                held[j] = row_chunk<T>(j < kSide * kPieces / kThreads ? bd : bx,
                                       base[j] != kNone ? base[j] + (uint32_t)n * kSize : kNone, n, a.N, st + 1 < steps);
        }
    };

    float4_t acc[kBR][kBC];
#pragma unroll
    for (int r = 0; r < kBR; ++r)
#pragma unroll
        for (int c = 0; c < kBC; ++c) acc[r][c] = float4_t{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int32_t st) {
#pragma unroll
        for (int h = 0; h < kPieces / 4; ++h) {
            const unsigned char* S =
                smem + (st % 2) * kStage + li * kLine + (((4 * h + g) ^ swizzle(li)) * 16);
            u32x4_t xo[kBC];
#pragma unroll
            for (int c = 0; c < kBC; ++c)
                xo[c] = *reinterpret_cast<const u32x4_t*>(S + (kSide + 16 * (wc * kBC + c)) * kLine);
#pragma unroll
            for (int r = 0; r < kBR; ++r) {
                if (!((mask >> (r * kBC)) & ((1u << kBC) - 1u))) continue;
                const u32x4_t d = *reinterpret_cast<const u32x4_t*>(S + 16 * (wr * kBR + r) * kLine);
#pragma unroll
                for (int c = 0; c < kBC; ++c)
                    if (mask & (1u << (r * kBC + c))) {
                        if constexpr (is_f32<T>) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) acc[r][c] = mfma32(xo[c][q], d[q], acc[r][c]);
                        } else {
                            acc[r][c] = mfma16<T>(xo[c], d, acc[r][c]);
                        }
                    }
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
    for (int r = 0; r < kBR; ++r)
#pragma unroll
        for (int c = 0; c < kBC; ++c) {
            if (!(mask & (1u << (r * kBC + c)))) continue;
            const int32_t b = place[(wr * kBR + r) * kEdge + wc * kBC + c];
            const int32_t row = 16 * (br0 + wr * kBR + r) + li, col = 16 * (bc0 + wc * kBC + c) + 4 * g;
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
    const dim3 grid = launch_grid(kXcds * xcd_chunk(a.items * a.sides), kThreads);
    if (aligned)
        hipLaunchKernelGGL((ff_sampled_tile_kernel<T, true>), grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((ff_sampled_tile_kernel<T, false>), grid, dim3(kThreads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

// Both weights of a gated layer in one launch; false where tiles do not apply.
template <typename T>
bool sampled_tiles(const SampledArgs<T>& f, int weights, hipStream_t s)
{
    const BlockIndex& w = *f.weight[0];
    SampledTile<T> a{};
    a.x = f.x;
    a.M = (int32_t)w.M;
    a.K = (int32_t)w.K;
    a.Mb = (int32_t)w.Mb;
    a.Kb = (int32_t)w.Kb;
    a.N = f.N;
    const int64_t db = narrow_bytes(w.M, f.N, sizeof(T)), xb = narrow_bytes(w.K, f.N, sizeof(T));
    if (db < 0 || xb < 0 || f.N == 0) return false;
    a.dz_bytes = (uint32_t)db;
    a.x_bytes = (uint32_t)xb;
    int64_t blocks = 0;
    for (int l = 0; l < weights; ++l) {
        if (!f.dvals[l]) continue;
        if (!f.weight[l]->map) return false;
        blocks += f.weight[l]->nnzb;
        a.side[a.sides++] = {f.weight[l]->map, f.dz[l], f.dvals[l]};
    }
    if (a.sides == 0) return true;
    if (blocks == 0) return false;
    // The share of stored blocks from which a tile's rows are cheaper than the rows
    // of each four blocks.  On 16 bytes (14336 x 4096 fp16, us by tiles and by fours:
    // 2048 tokens, 15 % stored 169 and 148, 20 % 173 and 194; 256 tokens, 10 % 36 and
    // 15, 30 % 41 and 39; 4096 x 4096 fp32, 512 tokens: 45 % 95 and 86, 60 % 113 and
    // 108, 80 % 128 and 139) and off (fp16, 2047 tokens, 15 % 360 and 289, 20 % 354 and
    // 386; 301, 10 % 86 and 41, 30 % 88 and 102; 37, operand by operand, 30 % 48 and
    // 46; 1, 30 % 39 and 25, 100 % 45 and 69; fp32, 511 tokens, 30 % 84 and 76, 45 % 100
    // and 115; 1, 100 % 25 and 21).
    // Tiles take rounds of two workgroups a CU, and a round of one a CU seven tenths
    // of that; blocks by fours fill the chip sooner (1024 x 1024, 2048 tokens, all
    // stored: fp16 25 us by tiles and 19, fp32 143 and 48).
    const bool aligned = f.N * sizeof(T) % 16 == 0;
    double share;
    if (aligned)
        share = is_f32<T> ? 0.62 : f.N < 512 ? 0.27 : 0.18;
    else if constexpr (is_f32<T>)
        share = f.N < 32 ? 2.0 : 0.4;
    else
        share = f.N < 28 ? 0.45 : f.N < 64 ? 0.35 : 0.2;
    const int64_t tiles = (int64_t)((a.Mb + kEdge - 1) / kEdge) * ((a.Kb + kEdge - 1) / kEdge) * a.sides;
    const int64_t rest = tiles % 512;
    const double rounds = (double)(tiles / 512) + (rest == 0 ? 0.0 : rest <= 256 ? 0.7 : 1.0);
    const double fill = (double)tiles / (512.0 * rounds);
    if ((double)blocks * fill < share * (double)(a.sides * w.Mb * w.Kb)) return false;
    launch_sampled_tile<T>(a, aligned, s);
    return true;
}

}  // namespace ff

template <typename T>
void sampled_product(const SampledArgs<T>& f, int weights, hipStream_t s)
{
    if (!ff::sampled_tiles<T>(f, weights, s)) ff::sampled_fours<T>(f, weights, s);
}

template void sampled_product<float>(const SampledArgs<float>&, int, hipStream_t);
template void sampled_product<_Float16>(const SampledArgs<_Float16>&, int, hipStream_t);
template void sampled_product<__bf16>(const SampledArgs<__bf16>&, int, hipStream_t);

}  // namespace detail
}  // namespace xspmm
