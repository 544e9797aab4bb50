// ff_tile.hip -- the products of ff_product.hip for 16-bit values where blocks
// are not rare: a workgroup takes sixteen (or eight) block-rows and 128 tokens, 32
// (or 64) rows of x at a time.
//
//   forward      block-rows of A, or (gated) half of them the gate's and the others
//                the same ones of the up projection's
//   transposed   block-columns of A; the sum runs over the block-rows of one
//                weight and then of the other
//
// Per step, the rows of x (8 or 16 KB) and the stored blocks that meet them (512
// bytes each; absent ones are neither read nor multiplied) go straight from memory
// into LDS, two stages in turn.  Of eight waves each owns four (two) block-rows x 64
// tokens and takes the block-columns in pairs.  A lane's operands of a pair are
// four values of the one block and four of the other, so that two stored blocks
// make one v_mfma_f32_16x16x32 and a single one, with the same registers, one
// v_mfma_f32_16x16x16: nothing of x meets a block that is not there.  Rows of x
// are read from memory once for all the block-rows, where the kernel that walks
// single block-rows reads them for every block.
//
// What bounds it, at 14336 x 4096 and 2048 tokens: the bare steps, with the reads of x
// from LDS and the barriers but neither loads nor matrix instructions, take 73 us (62
// of them the reads, 128 bytes a clock and CU), the loads with them 129, the
// instructions (50 us of the matrix units' time at 25 % stored, 110 at 100 %) 140,
// all 160.  Hence two workgroups of eight waves on a CU, four waves a SIMD, that take
// turns (25 % stored: 175 us; with four waves of four block-rows x 64 tokens each
// 218), and sixteen block-rows where there are enough of them, so that a row of x is
// read from LDS for four block-rows and not for two (158 us).  Measured: y 155 to 165
// us at 25 % stored and 240 to 254 at 100 % (960 TFLOP/s), both of a gated product's
// 283 to 300 and 461 to 482 (1010), dx, by eight, 154 to 162 and 253 to 269.  silu and
// the gelus add 10 to 14, after a workgroup's last step; bias and relu nothing.
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

constexpr int kWide = 128;     // tokens of a workgroup
constexpr int WC = 2, TT = 4;  // waves along them, a wave's tiles of 16
constexpr int kTileWaves = 8;
constexpr int kTileThreads = 64 * kTileWaves;
constexpr int kXRow = 2 * kWide;
constexpr int kWindow = 256;  // block-columns whose positions are in LDS at a time
constexpr int kTileBand = 8;
constexpr int kOutRow = kWide + 4;  // floats of a row on its way out

template <int SLOTS>
struct TileShape {
    static constexpr int kSlots = SLOTS;                       // block-rows
    static constexpr int WS = kSlots / (kTileWaves / WC);      // a wave's
    static constexpr int kDeep = 32 / kSlots;                  // blocks of a slot per step
    static constexpr int kPairs = kDeep / 2;
    static constexpr int kABytes = kSlots * kDeep * 512;
    static constexpr int kStage = kABytes + 16 * kDeep * kXRow;
    static constexpr int kPlaceRow = kWindow + kDeep;
    static constexpr int kPasses = kSlots / 8;                 // of the sums through the same LDS
    static constexpr int kUsed = 2 * kStage + kSlots * kPlaceRow * 4, kOut = 16 * 8 * kOutRow * 4;
    static constexpr int kLds = kUsed > kOut ? kUsed : kOut;
    // two workgroups share a CU
    static_assert(kLds <= 80 * 1024 && kWindow % kDeep == 0);
};

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

template <typename T, int SLOTS, bool TR, bool GATED, bool DMA>
__global__ __launch_bounds__(kTileThreads, 4) void ff_tile_kernel(const TileArgs<T> a)
{
    using Shape = TileShape<SLOTS>;
    constexpr int kSlots = Shape::kSlots, WS = Shape::WS, kDeep = Shape::kDeep, kPairs = Shape::kPairs, kABytes = Shape::kABytes;
    constexpr int kTileStage = Shape::kStage, kPlaceRow = Shape::kPlaceRow, kPasses = Shape::kPasses;
    constexpr int kOutRows = GATED ? kSlots / 2 : kSlots;  // block-rows of the result
    __shared__ __align__(16) unsigned char smem[Shape::kLds];
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
    constexpr int kAPer = kSlots / kTileWaves;                      // slots whose blocks a wave loads
    constexpr int kXPer = 16 * kDeep * kXRow / 1024 / kTileWaves;  // and its loads of x

    // Wave w moves the blocks of kAPer slots from kAPer w on and kRowsPer rows of x
    // from kRowsPer w on, a KB per load.  This lane's bytes: of a block (16 at p =
    // lane % 32), and of x from the first step on; rows past the last are past the
    // end of x.
    const int p = lane & 31;
    const uint32_t a_lane = (uint32_t)((p >> 1) * 32 + (((p & 1) ^ a_swizzle(p >> 1)) * 16));
    constexpr int kRowsPer = 16 * kDeep / kTileWaves;
    uint32_t x_lane[kXPer];
#pragma unroll
    for (int u = 0; u < kXPer; ++u) {
        const int e = kRowsPer * wave + kRowsPer / kXPer * u + lane / (kWide / 8);
        const int64_t n = n0 + 8 * (lane % (kWide / 8) ^ x_swizzle(e));
        x_lane[u] = n < a.N ? (uint32_t)e * ld + (uint32_t)n * 2u : kNone;
    }
    const uint32_t* const dma_place = &place[kAPer * wave][lane >> 5];
    const uint32_t* const own_place = &place[WS * wr + lane / kDeep % WS][lane % kDeep];

    // Operands: row 4 g + li / 4 of a block (or of x), 8-byte piece li % 4; of A
    // itself row li, values 4 g .. + 3.
    const int r4 = 4 * g + (li >> 2), piece = (li & 3) >> 1;
    uint32_t x_at[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j)
        x_at[j] = (uint32_t)(kABytes + r4 * kXRow + 8 * (li & 1) + (((2 * (TT * wc + j) + piece) ^ x_swizzle(r4)) * 16));
    const uint32_t a_at = (uint32_t)(WS * wr * kDeep * 512 + (TR ? r4 * 32 + ((piece ^ a_swizzle(r4)) * 16) + 8 * (li & 1)
                                                                : li * 32 + (((g >> 1) ^ a_swizzle(li)) * 16) + 8 * (g & 1)));

    float4_t acc[WS][TT];
#pragma unroll
    for (int s = 0; s < WS; ++s)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[s][j] = float4_t{0.f, 0.f, 0.f, 0.f};

    auto a_operand = [&](const unsigned char* S, int s, int d) {
        const unsigned char* q = S + a_at + (s * kDeep + d) * 512;
        if constexpr (TR)
            return read_transposed(q);
        else
            return *reinterpret_cast<const u32x2_t*>(q);
    };
    // Blocks d and d + 1 of every slot; stored: bit kDeep s + d, block d of this
    // wave's slot s.  Three conditions of their own, not alternatives: an accumulator
    // with more than one way to its new value is copied on all of them.
    auto multiply = [&](const unsigned char* S, uint32_t stored, int d) {
        u32x2_t x[2][TT];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < TT; ++j) x[e][j] = read_transposed(S + x_at[j] + 16 * (d + e) * kXRow);
        // ahead of the waves that are still on their way from the barrier: the matrix
        // units are not to wait for these (5 % of the time)
        __builtin_amdgcn_s_setprio(1);
        uint32_t pairs = stored & (stored >> 1), firsts = stored & ~(stored >> 1), seconds = ~stored & (stored >> 1);
        asm volatile("" : "+s"(pairs), "+s"(firsts), "+s"(seconds));
#pragma unroll
        for (int s = 0; s < WS; ++s) {
            const uint32_t bit = 1u << (kDeep * s + d);
            if (pairs & bit) {
                const u32x2_t p = a_operand(S, s, d), q = a_operand(S, s, d + 1);
#pragma unroll
                for (int j = 0; j < TT; ++j)
                    acc[s][j] = mfma16<T>(u32x4_t{p.x, p.y, q.x, q.y},
                                          u32x4_t{x[0][j].x, x[0][j].y, x[1][j].x, x[1][j].y}, acc[s][j]);
            }
            if (firsts & bit) {
                const u32x2_t p = a_operand(S, s, d);
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[s][j] = mfma16_half<T>(p, x[0][j], acc[s][j]);
            }
            if (seconds & bit) {
                const u32x2_t q = a_operand(S, s, d + 1);
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[s][j] = mfma16_half<T>(q, x[1][j], acc[s][j]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
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
                    if (__ballot(next_dma[u] != kNone))
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
            for (int32_t st = 0; st < steps; ++st) {
                const uint32_t stored = coming;
                landed(st);
                if (st + 1 < steps) coming = issue(st + 1);
#pragma unroll
                for (int d = 0; d < kDeep; d += 2) multiply(smem + (st & 1) * kTileStage, stored, d);
            }
        }
    }

    // The sums leave through LDS, eight block-rows of a product at a time, so that the
    // rest is done on eight tokens of a row per thread.
    float* O = reinterpret_cast<float*>(smem);
    constexpr int kPassWaves = kTileWaves / WC / kPasses;  // rows of waves of a pass
#pragma unroll 1
    for (int pass = 0; pass < kPasses; ++pass) {
        __syncthreads();
        if (wr / kPassWaves == pass)
#pragma unroll
            for (int s = 0; s < WS; ++s)
#pragma unroll
                for (int j = 0; j < TT; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        O[(16 * (WS * (wr % kPassWaves) + s) + 4 * g + q) * kOutRow + 16 * (TT * wc + j) + li] =
                            acc[s][j][q];
        __syncthreads();
        constexpr int kOut = 16 * kOutRows / kPasses;
        static_assert(kOut * (kWide / 8) % kTileThreads == 0);
#pragma unroll 1
        for (int v = 0; v < kOut * (kWide / 8) / kTileThreads; ++v) {
            const int at = v * kTileThreads + t, r = at / (kWide / 8), c = at % (kWide / 8) * 8;
            // the block-row's slot, of a gated product the gate's, with the up
            // projection's WS / 2 slots on
            const int from = GATED ? 16 * (r / (8 * WS) * WS) + r % (8 * WS) : r;
            const int64_t row = 16 * (int64_t)br0 + kOut * pass + r, n = n0 + c;
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

template <typename T, int SLOTS, bool TR, bool GATED>
void launch_shape(const TileArgs<T>& a, hipStream_t s)
{
    constexpr int rows = GATED ? SLOTS / 2 : SLOTS;
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + kWide - 1) / kWide);
    const dim3 grid = launch_grid(kXcds * xcd_chunk(items), kTileThreads);
    if (a.N % 8 == 0)
        hipLaunchKernelGGL((ff_tile_kernel<T, SLOTS, TR, GATED, true>), grid, dim3(kTileThreads), 0, s, a);
    else
        hipLaunchKernelGGL((ff_tile_kernel<T, SLOTS, TR, GATED, false>), grid, dim3(kTileThreads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

// Block-rows of a workgroup; 0 where walking the block-rows one by one is faster.
//
// The time of tiles goes by the rounds of two workgroups a CU, a last one of one a
// CU taking four fifths as long; that of the walk by what is stored.  Sixteen
// block-rows where there is more than one such workgroup a CU (16-bit, 4096 x 4096
// gated, 25 % stored, us by sixteen and by eight: 2048 tokens 87 and 103, 1024 tokens,
// one workgroup a CU, 75 and 55).  The shares from which tiles of a full round pay are
// from 18 % and 25 % stored, us by tiles and by rows: by sixteen, 14336 x 4096, 2048
// tokens, 148 and 164, 157 and 211, by eight, 4096 x 14336, 154 and 137, 160 and 185;
// all stored 256 and 650, 266 and 655.
double rounds(int64_t workgroups)
{
    const int64_t whole = workgroups / 512, rest = workgroups % 512;
    return (double)whole + (rest == 0 ? 0.0 : rest <= 256 ? 0.8 : 1.0);
}
int tile_slots(int64_t blocks, int64_t grid_blocks, int64_t N, int64_t slots)
{
    const int64_t tiles = (N + kWide - 1) / kWide;
    const int shape = (slots + 15) / 16 * tiles > 256 ? 16 : 8;
    const int64_t n = (slots + shape - 1) / shape * tiles;
    const double filled = (double)blocks * (double)N / ((double)grid_blocks * (double)(tiles * kWide));
    return filled * (double)n >= (shape == 16 ? 0.155 : 0.2) * 512.0 * rounds(n) ? shape : 0;
}

template <typename T, bool TR, bool GATED>
void launch_tile(const TileArgs<T>& a, int slots, hipStream_t s)
{
    if (slots == 16)
        launch_shape<T, 16, TR, GATED>(a, s);
    else
        launch_shape<T, 8, TR, GATED>(a, s);
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
    const int slots = ff::tile_slots(blocks, weights * w.Mb * w.Kb, f.N, w.Mb * weights);
    if (xb < 0 || (f.N % 8 != 0 && f.N < ff::kWide) || slots == 0) return false;
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
        ff::launch_tile<T, false, true>(a, slots, s);
    else
        ff::launch_tile<T, false, false>(a, slots, s);
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
    const int slots = ff::tile_slots(blocks, weights * w.Mb * w.Kb, f.N, w.Kb);
    if (xb < 0 || (f.N % 8 != 0 && f.N < ff::kWide) || slots == 0) return false;
    a.y = f.dx;
    a.sides = weights;
    a.rows = (int32_t)w.K;
    a.block_rows = (int32_t)w.Kb;
    a.in_blocks = (int32_t)w.Mb;
    a.map_ld = (int32_t)w.Kb;
    a.in_rows = (int32_t)w.M;
    a.N = f.N;
    a.x_bytes = (uint32_t)xb;
    ff::launch_tile<T, true, false>(a, slots, s);
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
