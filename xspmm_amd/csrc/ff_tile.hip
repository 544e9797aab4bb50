// ff_tile.hip -- the products of ff_product.hip for 16-bit values where blocks
// are not rare: a workgroup takes eight block-rows and 128 tokens, 64 rows of x
// at a time.
//
//   forward      eight block-rows of A, or (gated) four of the gate's and the same
//                four of the up projection's
//   transposed   eight block-columns of A; the sum runs over the block-rows of one
//                weight and then of the other
//
// Per step, 64 rows of x (16 KB) and the stored blocks among the 8 x 4 that meet
// them (512 bytes each; absent ones are neither read nor multiplied) go straight
// from memory into LDS, two stages in turn.  A wave owns four block-rows x 64
// tokens and takes the block-columns in pairs.  A lane's operands of a pair are
// four values of the one block and four of the other, so that two stored blocks
// make one v_mfma_f32_16x16x32 and a single one, with the same registers, one
// v_mfma_f32_16x16x16: nothing of x meets a block that is not there.  Rows of x
// are read from memory once for eight block-rows, where the kernel that walks
// single block-rows reads them for every block.  Two workgroups share a CU, so that one
// multiplies while the other waits for its loads.
#include "feed_forward_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

typedef __attribute__((address_space(3))) short4_t lds_short4_t;

template <typename T>
struct TileSide {
    const int32_t* map;
    const T* vals;
    const T* x;
    const T* bias;
    T* keep;
    uint32_t vals_bytes;
};

template <typename T>
struct TileArgs {
    TileSide<T> side[2];
    const T* residual;
    T* y;
    int32_t sides;
    int32_t rows;                   // of the result
    int32_t block_rows, in_blocks;  // of the result, of x
    int32_t map_ld;                 // block-columns of A
    int32_t in_rows;                // of x
    int64_t N;
    uint32_t x_bytes;
    int act;
};

constexpr int kSlots = 8;          // block-rows of a workgroup, half of them a wave's
constexpr int WS = kSlots / 2, WC = 2;
constexpr int kWide = 64 * WC;     // its tokens, 64 of them a wave's
constexpr int kTileThreads = 128 * WC;
constexpr int kDeep = 4;           // blocks of a slot per step
constexpr int kPairs = kDeep / 2;
constexpr int kXRow = 2 * kWide;
constexpr int kABytes = kSlots * kDeep * 512;
constexpr int kTileStage = kABytes + 16 * kDeep * kXRow;
constexpr int kWindow = 256;       // block-columns whose positions are in LDS at a time
constexpr int kPlaceRow = kWindow + kDeep;
constexpr int kTileBand = 8;
constexpr int kOutRow = kWide + 4;  // floats of a row on its way out
constexpr int kTileLds = 2 * kTileStage + kSlots * kPlaceRow * 4;
// two workgroups share a CU; the sums leave through the same LDS
static_assert(kTileLds <= 80 * 1024 && 16 * kSlots * kOutRow * 4 <= kTileLds && kWindow % kDeep == 0);

// Chunk c (16 bytes) of row e of the x stage lies at chunk c ^ x_swizzle(e): the
// rows that one transposed read touches are in different banks.
__device__ __forceinline__ int x_swizzle(int e) { return 2 * (e & 7); }
// Half h (16 bytes) of row r of a block lies at half h ^ a_swizzle(r).
__device__ __forceinline__ int a_swizzle(int r) { return (r >> 3) & 1; }

// Four rows of 16 values (8 bytes of a row per lane): lane l of 16 gets column
// l's four values.
__device__ __forceinline__ u32x2_t read_transposed(const unsigned char* p)
{
    return __builtin_bit_cast(u32x2_t,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)const_cast<unsigned char*>(p)));
}

template <typename T, bool TR, bool GATED, bool DMA>
__global__ __launch_bounds__(kTileThreads, 2) void ff_tile_kernel(const TileArgs<T> a)
{
    constexpr int kOutRows = GATED ? kSlots / 2 : kSlots;  // block-rows of the result
    __shared__ __align__(16) unsigned char smem[kTileLds];
    // byte offsets of the blocks, or kNone
    uint32_t(*const place)[kPlaceRow] = reinterpret_cast<uint32_t(*)[kPlaceRow]>(smem + 2 * kTileStage);
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wr = wave / WC, wc = wave % WC;
    const int li = lane & 15, g = lane >> 4;

    // bands of kTileBand row groups, token tile by token tile
    int32_t br0;
    int64_t first;
    {
        const int64_t tiles = (a.N + kWide - 1) / kWide, groups = (a.block_rows + kOutRows - 1) / kOutRows;
        const int64_t item = xcd_item(blockIdx.x, groups * tiles);
        if (item < 0) return;
        const int64_t band = item / (kTileBand * tiles) * kTileBand;
        const int64_t h = min((int64_t)kTileBand, groups - band), in = item - band * tiles;
        br0 = (int32_t)(band + in % h) * kOutRows;
        first = in / h * kWide;
    }
    // without DMA the last tile moves back into the matrix (and stores its own tokens only)
    const int64_t n0 = !DMA && first + kWide > a.N ? a.N - kWide : first;

    // slot s: block-row br0 + slot_row(s) of side slot_side(s); a wave owns slots
    // WS wr .. + WS - 1, of a gated product half of them of either side
    auto slot_row = [](int s) { return GATED ? s / WS * (WS / 2) + s % (WS / 2) : s; };
    auto slot_side = [](int s) { return GATED ? s / (WS / 2) % 2 : 0; };

    const uint32_t lds0 = lds_address(smem);
    const uint32_t ld = (uint32_t)a.N * 2u;
    constexpr int kAPer = kSlots / (2 * WC);                  // a wave's loads of A per step
    constexpr int kXPer = kDeep;                       // and of x

    // Wave w moves the blocks of kAPer slots from kAPer w on and kRowsPer rows of x
    // from kRowsPer w on, a KB per load.  This lane's bytes: of a block (16 at p = lane % 32), and of x from
    // the first step on; rows past the last are past the end of x.
    const int p = lane & 31;
    const uint32_t a_lane = (uint32_t)((p >> 1) * 32 + (((p & 1) ^ a_swizzle(p >> 1)) * 16));
    constexpr int kRowsPer = 16 * kDeep / (2 * WC);
    uint32_t x_lane[kXPer];
#pragma unroll
    for (int u = 0; u < kXPer; ++u) {
        const int e = kRowsPer * wave + kRowsPer / kXPer * u + lane / (8 * WC);
        const int64_t n = n0 + 8 * (lane % (8 * WC) ^ x_swizzle(e));
        x_lane[u] = n < a.N ? (uint32_t)e * ld + (uint32_t)n * 2u : kNone;
    }
    const uint32_t* const dma_place = &place[kAPer * wave][lane >> 5];
    const uint32_t* const own_place = &place[WS * wr + lane / kDeep % WS][lane % kDeep];

    // Operands: row 4 g + li / 4 of a block (or of x), 8-byte piece li % 4; of A
    // itself row li, values 4 g .. + 3.
    const int r4 = 4 * g + (li >> 2), piece = (li & 3) >> 1;
    uint32_t x_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        x_at[j] = (uint32_t)(kABytes + r4 * kXRow + 8 * (li & 1) + (((2 * (4 * wc + j) + piece) ^ x_swizzle(r4)) * 16));
    const uint32_t a_at = (uint32_t)(WS * wr * kDeep * 512 + (TR ? r4 * 32 + ((piece ^ a_swizzle(r4)) * 16) + 8 * (li & 1)
                                                                : li * 32 + (((g >> 1) ^ a_swizzle(li)) * 16) + 8 * (g & 1)));

    float4_t acc[WS][4];
#pragma unroll
    for (int s = 0; s < WS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[s][j] = float4_t{0.f, 0.f, 0.f, 0.f};

    // The operands of a pair of block-columns.  Those of A^T are read with those of
    // x, of blocks that are not there too (what lies in their places is not used);
    // those of A, whose reads have bank conflicts, at a block's own instructions.
    struct Operands {
        u32x2_t x[kDeep][4], a[kDeep][TR ? WS : 1];
    };
    auto a_operand = [&](const unsigned char* S, int s, int d) {
        const unsigned char* q = S + a_at + (s * kDeep + d) * 512;
        if constexpr (TR)
            return read_transposed(q);
        else
            return *reinterpret_cast<const u32x2_t*>(q);
    };
    auto read = [&](Operands& o, const unsigned char* S, int d) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o.x[d][j] = read_transposed(S + x_at[j] + 16 * d * kXRow);
        if constexpr (TR)
#pragma unroll
            for (int s = 0; s < WS; ++s) o.a[d][s] = a_operand(S, s, d);
    };
    // Blocks d and d + 1 of every slot; stored: bit kDeep s + d, block d of this
    // wave's slot s.  Three conditions of their own, not alternatives: an accumulator
    // with more than one way to its new value is copied on all of them.
    auto multiply = [&](const Operands& o, const unsigned char* S, uint32_t stored, int d) {
        uint32_t pairs = stored & (stored >> 1), firsts = stored & ~(stored >> 1), seconds = ~stored & (stored >> 1);
        asm volatile("" : "+s"(pairs), "+s"(firsts), "+s"(seconds));
        auto operand = [&](int s, int e) { return TR ? o.a[e][TR ? s : 0] : a_operand(S, s, e); };
#pragma unroll
        for (int s = 0; s < WS; ++s) {
            const uint32_t bit = 1u << (kDeep * s + d);
            if (pairs & bit) {
                const u32x2_t p = operand(s, d), q = operand(s, d + 1);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[s][j] = mfma16<T>(u32x4_t{p.x, p.y, q.x, q.y},
                                          u32x4_t{o.x[d][j].x, o.x[d][j].y, o.x[d + 1][j].x, o.x[d + 1][j].y},
                                          acc[s][j]);
            }
            if (firsts & bit) {
                const u32x2_t p = operand(s, d);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[s][j] = mfma16_half<T>(p, o.x[d][j], acc[s][j]);
            }
            if (seconds & bit) {
                const u32x2_t q = operand(s, d + 1);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[s][j] = mfma16_half<T>(q, o.x[d + 1][j], acc[s][j]);
            }
        }
    };

    // Windows of the sum, with the positions of their blocks in LDS.
    for (int which = 0; which < (TR ? a.sides : 1); ++which) {
        const i32x4_t vals0 = dma_buffer(a.side[which].vals, a.side[which].vals_bytes);
        const i32x4_t vals1 = GATED ? dma_buffer(a.side[1].vals, a.side[1].vals_bytes) : vals0;
        const i32x4_t xb = dma_buffer(a.side[which].x, a.x_bytes);
        const auto xr = make_buffer(a.side[which].x, a.x_bytes);
        for (int32_t c0 = 0; c0 < a.in_blocks; c0 += kWindow) {
            __syncthreads();  // the last window's positions and stages have been read
            for (int e = t; e < kSlots * kWindow; e += kTileThreads) {
                // consecutive threads take consecutive entries of the map
                const int s = TR ? e % kSlots : e / kWindow, d = TR ? e / kSlots : e % kWindow;
                const int32_t r = br0 + slot_row(s), c = c0 + d;
                const bool in = r < a.block_rows && c < a.in_blocks;
                const int32_t* map = a.side[GATED ? slot_side(s) : which].map;
                const int32_t b = !in ? -1 : TR ? map[(int64_t)c * a.map_ld + r] : map[(int64_t)r * a.map_ld + c];
                place[s][d] = b < 0 ? kNone : (uint32_t)b * 512u;
            }
            __syncthreads();
            const int32_t steps = min(kWindow, a.in_blocks - c0 + kDeep - 1) / kDeep;
            uint32_t x_off[kXPer];
#pragma unroll
            for (int u = 0; u < kXPer; ++u) x_off[u] = x_lane[u] + (uint32_t)c0 * 16u * ld;
            u32x4_t held[DMA ? 1 : kXPer];
            // what the next step to load needs of the positions, read ahead of it
            uint32_t next_own, next_dma[kAPer * kPairs];
            auto look = [&](int32_t st) {
                next_own = own_place[st * kDeep];
#pragma unroll
                for (int u = 0; u < kAPer * kPairs; ++u)
                    next_dma[u] = dma_place[u / kPairs * (kPlaceRow) + st * kDeep + 2 * (u % kPairs)];
            };
            // the loads of step st; what is stored of this wave's own slots in it
            auto issue = [&](int32_t st) -> uint32_t {
                const uint32_t to = lds0 + (uint32_t)(st & 1) * kTileStage;
                const uint32_t f = (uint32_t)__builtin_amdgcn_readfirstlane(
                    (int)__ballot(lane < kDeep * WS && next_own != kNone));
#pragma unroll
                for (int u = 0; u < kAPer * kPairs; ++u) {
                    const int s = u / kPairs, h = u % kPairs;
                    dma_to_lds(to + (uint32_t)((kAPer * wave + s) * kDeep + 2 * h) * 512u, next_dma[u] + a_lane,
                               GATED && slot_side(kAPer * wave + s) ? vals1 : vals0);
                }
#pragma unroll
                for (int u = 0; u < kXPer; ++u) {
                    if constexpr (DMA) {
                        dma_to_lds(to + kABytes + (uint32_t)(kRowsPer * wave + kRowsPer / kXPer * u) * kXRow, x_off[u],
                                   xb);
                    } else {
                        const auto v = buffer_load<T, 8>(xr, x_off[u]);
                        held[u] = u32x4_t{v.d[0], v.d[1], v.d[2], v.d[3]};
                    }
                    x_off[u] += 16u * kDeep * ld;
                }
                look(st + 1 < steps ? st + 1 : steps - 1);
                return f;
            };
            // until the loads of step st are in LDS, of every wave, and what was read
            // from the other stage in registers
            auto landed = [&](int32_t st) {
                if constexpr (!DMA)
#pragma unroll
                    for (int u = 0; u < kXPer; ++u)
                        *reinterpret_cast<u32x4_t*>(smem + (st & 1) * kTileStage + kABytes +
                                                    (kRowsPer * wave + kRowsPer / kXPer * u) * kXRow + lane * 16) = held[u];
                dma_wait<0>();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __syncthreads();
            };
            look(0);
            uint32_t coming = issue(0);
            if constexpr (TR) {
                // a step is multiplied from registers while the next one's operands are
                // read and the loads of the one after that are under way
                uint32_t stored = coming;
                Operands even, odd;
                landed(0);
                coming = 1 < steps ? issue(1) : 0u;
#pragma unroll
                for (int d = 0; d < kDeep; ++d) read(even, smem, d);
                auto round = [&](int32_t st, const Operands& now, Operands& then) {
                    const uint32_t mine = stored;
                    if (st + 1 < steps) {
                        stored = coming;
                        landed(st + 1);
                        coming = st + 2 < steps ? issue(st + 2) : 0u;
#pragma unroll
                        for (int d = 0; d < kDeep; ++d) read(then, smem + ((st + 1) & 1) * kTileStage, d);
                    }
#pragma unroll
                    for (int d = 0; d < kDeep; d += 2) multiply(now, smem, mine, d);
                };
                for (int32_t st = 0; st < steps; st += 2) {
                    round(st, even, odd);
                    if (st + 1 < steps) round(st + 1, odd, even);
                }
            } else {
                for (int32_t st = 0; st < steps; ++st) {
                    const uint32_t stored = coming;
                    landed(st);
                    if (st + 1 < steps) coming = issue(st + 1);
                    const unsigned char* S = smem + (st & 1) * kTileStage;
                    Operands o;
#pragma unroll
                    for (int d = 0; d < kDeep; d += 2) {
                        read(o, S, d);
                        read(o, S, d + 1);
                        multiply(o, S, stored, d);
                    }
                }
            }
        }
    }

    // The sums leave through LDS, so that the rest is done on eight tokens of a row
    // per thread.
    float* O = reinterpret_cast<float*>(smem);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < WS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                O[(16 * (WS * wr + s) + 4 * g + q) * kOutRow + 64 * wc + 16 * j + li] = acc[s][j][q];
    __syncthreads();
    {
        constexpr int kOut = 16 * kOutRows;
#pragma unroll 1
        for (int v = 0; v < kOut * (kWide / 8) / kTileThreads; ++v) {
            const int at = v * kTileThreads + t, r = at / (kWide / 8), c = at % (kWide / 8) * 8;
            // the block-row's slot, of a gated product the gate's, with the up
            // projection's WS / 2 slots on
            const int from = GATED ? 16 * (r / (8 * WS) * WS) + r % (8 * WS) : r;
            const int64_t row = 16 * (int64_t)br0 + r, n = n0 + c;
            if (row >= a.rows || n + 8 <= first || n >= a.N) continue;
            const bool whole = n >= first && n + 8 <= a.N;
            float z[2][8];
#pragma unroll
            for (int l = 0; l < (GATED ? 2 : 1); ++l) {
                const float4_t lo = *reinterpret_cast<const float4_t*>(O + (from + 8 * WS * l) * kOutRow + c);
                const float4_t hi = *reinterpret_cast<const float4_t*>(O + (from + 8 * WS * l) * kOutRow + c + 4);
                const float bias = !TR && a.side[l].bias ? (float)a.side[l].bias[row] : 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    z[l][q] = lo[q] + bias;
                    z[l][4 + q] = hi[q] + bias;
                }
            }
            auto store = [&](T* o, const float(&w)[8]) {
                if (whole) {
                    Pack<T, 8> k;
#pragma unroll
                    for (int q = 0; q < 8; ++q) k.v[q] = (T)w[q];
                    *reinterpret_cast<Pack<T, 8>*>(o + row * a.N + n) = k;
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (n + q >= first && n + q < a.N) o[row * a.N + n + q] = (T)w[q];
                }
            };
            if constexpr (!TR) {
#pragma unroll
                for (int l = 0; l < (GATED ? 2 : 1); ++l)
                    if (a.side[l].keep) store(a.side[l].keep, z[l]);
                with_act(a.act, [&](auto act) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) z[0][q] = act_value<decltype(act)::value>(z[0][q]);
                });
                if constexpr (GATED)
#pragma unroll
                    for (int q = 0; q < 8; ++q) z[0][q] *= z[1][q];
                if (a.residual) {
                    if (whole) {
                        const Pack<T, 8> k = *reinterpret_cast<const Pack<T, 8>*>(a.residual + row * a.N + n);
#pragma unroll
                        for (int q = 0; q < 8; ++q) z[0][q] += (float)k.v[q];
                    } else {
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            if (n + q >= first && n + q < a.N) z[0][q] += (float)a.residual[row * a.N + n + q];
                    }
                }
            }
            store(a.y, z[0]);
        }
    }
}

template <typename T, bool TR, bool GATED>
void launch_tile(const TileArgs<T>& a, hipStream_t s)
{
    constexpr int rows = GATED ? kSlots / 2 : kSlots;
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + kWide - 1) / kWide);
    const int64_t grid = kXcds * xcd_chunk(items);
    if (grid > 0x7fffffffLL) throw std::invalid_argument("xSpMM: too many tokens for one launch.");
    if (a.N % 8 == 0)
        hipLaunchKernelGGL((ff_tile_kernel<T, TR, GATED, true>), dim3((unsigned)grid), dim3(kTileThreads), 0, s, a);
    else
        hipLaunchKernelGGL((ff_tile_kernel<T, TR, GATED, false>), dim3((unsigned)grid), dim3(kTileThreads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

// Whether the share of stored blocks is one at which tiles are faster than walking
// the block-rows one by one (14336 x 4096 fp16, 2048 tokens, us by tiles and by
// rows: y 25 % 220 and 212, 50 % 257 and 365, all 310 and 640; two weights 25 %
// 416 and 391, 50 % 486 and 717; dx 25 % 192 and 188, 50 % 218 and 353, all 244 and
// 670), of a token tile that may be filled in part, and whether they are enough
// for the chip (a workgroup walks its whole sum).
bool tiles_pay(int64_t blocks, int64_t grid_blocks, int64_t N, int64_t row_groups)
{
    const int64_t tiles = (N + kWide - 1) / kWide;
    if (row_groups * tiles < 256) return false;
    return (double)blocks * (double)N >= 0.28 * (double)grid_blocks * (double)(tiles * kWide);
}

}  // namespace ff

template <typename T>
bool feed_forward_tiles(const ForwardArgs<T>& f, int weights, hipStream_t s)
{
    const BlockIndex& w = *f.weight[0];
    ff::TileArgs<T> a{};
    int64_t blocks = 0;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *f.weight[l];
        const int64_t vb = narrow_bytes(wl.nnzb, 256, 2);
        if (!wl.map || vb < 0) return false;
        a.side[l] = {wl.map, f.vals[l], f.x, f.bias[l], f.keep[l], (uint32_t)vb};
        blocks += wl.nnzb;
    }
    const int64_t xb = narrow_bytes(w.K, f.N, 2);
    if (xb < 0 || (f.N % 8 != 0 && f.N < ff::kWide) ||
        !ff::tiles_pay(blocks, weights * w.Mb * w.Kb, f.N, w.Mb * weights / ff::kSlots))
        return false;
    a.residual = f.residual;
    a.y = f.y;
    a.sides = weights;
    a.rows = (int32_t)w.M;
    a.block_rows = (int32_t)w.Mb;
    a.in_blocks = (int32_t)w.Kb;
    a.map_ld = (int32_t)w.Kb;
    a.in_rows = (int32_t)w.K;
    a.N = f.N;
    a.x_bytes = (uint32_t)xb;
    a.act = f.act;
    if (weights == 2)
        ff::launch_tile<T, false, true>(a, s);
    else
        ff::launch_tile<T, false, false>(a, s);
    return true;
}

template <typename T>
bool transposed_tiles(const TransposedArgs<T>& f, int weights, hipStream_t s)
{
    const BlockIndex& w = *f.weight[0];
    ff::TileArgs<T> a{};
    int64_t blocks = 0;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *f.weight[l];
        const int64_t vb = narrow_bytes(wl.nnzb, 256, 2);
        if (!wl.map || vb < 0) return false;
        a.side[l] = {wl.map, f.vals[l], f.dz[l], nullptr, nullptr, (uint32_t)vb};
        blocks += wl.nnzb;
    }
    const int64_t xb = narrow_bytes(w.M, f.N, 2);
    if (xb < 0 || (f.N % 8 != 0 && f.N < ff::kWide) ||
        !ff::tiles_pay(blocks, weights * w.Mb * w.Kb, f.N, w.Kb / ff::kSlots))
        return false;
    a.y = f.dx;
    a.sides = weights;
    a.rows = (int32_t)w.K;
    a.block_rows = (int32_t)w.Kb;
    a.in_blocks = (int32_t)w.Mb;
    a.map_ld = (int32_t)w.Kb;
    a.in_rows = (int32_t)w.M;
    a.N = f.N;
    a.x_bytes = (uint32_t)xb;
    ff::launch_tile<T, true, false>(a, s);
    return true;
}

#define XSPMM_FF_TILE(T)                                                        \
    template bool feed_forward_tiles<T>(const ForwardArgs<T>&, int, hipStream_t); \
    template bool transposed_tiles<T>(const TransposedArgs<T>&, int, hipStream_t);
XSPMM_FF_TILE(_Float16)
XSPMM_FF_TILE(__bf16)
#undef XSPMM_FF_TILE

}  // namespace detail
}  // namespace xspmm
