// ff_int8_tile.hip -- the products of ff_int8_product.hip where most blocks are stored and
// tokens many: a workgroup of four waves takes 16 block-rows (gated: eight of the gate's
// and the same ones of the up projection's) and 128 tokens, two workgroups a CU.
//
// The tokens' features go straight from memory into LDS, a window of 16 block-columns
// at a time, two in turn.  A wave owns four block-rows and walks the window by four
// block-columns: a row's four blocks (absent ones are zeros and not read) make one
// v_mfma_i32_16x16x64_i8 with each of the eight tiles of 16 tokens, if any of them is
// stored.  A value of x is read from LDS once for four block-rows; a block is read
// from memory by the one wave that needs it, three steps ahead, its position two windows.
//
// 14336 x 4096, all stored, 2048 tokens, fp16, bias and gelu: 140 to 170 us by the clock that
// power leaves, 144 to 150 in the mean, 1.6 to 1.7 Pop/s.  The matrix units are busy for 57 us of that at 2
// GHz; a step's loads, 24 KB a workgroup through the 64 bytes a clock of a CU's L1, take
// three quarters of the matrix instructions' time beside them, and the gelus and the results
// 25 us, of which the other workgroup hides a part (one workgroup of eight waves: 142 where
// four took 140, with gate and up and 25 % stored 204 and 187).
#include "int8_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

constexpr int kI8Wide = kInt8TileTokens;   // of a workgroup
constexpr int kI8Waves = 4, kI8Threads = 64 * kI8Waves;
constexpr int kI8Rows = 4;                 // a wave's block-rows, of both weights
constexpr int kI8Slots = kI8Rows * kI8Waves;
static_assert(kI8Slots == kInt8TileRows);
constexpr int kI8Tiles = kI8Wide / 16;
constexpr int kI8Window = 16;              // block-columns
constexpr int kI8Stage = kI8Window * kI8Wide * 16;
constexpr int kI8OutRow = kI8Wide + 4;     // floats of a row on its way out
constexpr int kI8Out = 2 * 16 * kI8OutRow * 4;  // a wave's bytes on their way out
constexpr int kI8Used = 2 * kI8Stage + 3 * kI8Slots * kI8Window * 4;
constexpr int kI8Lds = kI8Used > kI8Waves * kI8Out ? kI8Used : kI8Waves * kI8Out;
constexpr int kI8Band = 8;

template <typename T, bool GATED>
__global__ __launch_bounds__(kI8Threads, 2) void ff_int8_tile_kernel(const Int8Product<T> a)
{
    constexpr int kOutRows = GATED ? kI8Slots / 2 : kI8Slots;  // block-rows of the result
    __shared__ __align__(16) unsigned char smem[kI8Lds];
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);

    int32_t br0, n0;
    {
        // bands of kI8Band row groups, token tile by token tile
        const uint32_t tiles = (uint32_t)((a.N + kI8Wide - 1) / kI8Wide);
        const uint32_t groups = (uint32_t)(a.block_rows + kOutRows - 1) / kOutRows;
        const uint32_t item = xcd_item32(blockIdx.x, groups * tiles);
        if (item == ~0u) return;
        const uint32_t band = item / (kI8Band * tiles) * kI8Band;
        const uint32_t h = min((uint32_t)kI8Band, groups - band), in = item - band * tiles;
        // (uniform, which the compiler does not see behind the divisions)
        br0 = __builtin_amdgcn_readfirstlane((int32_t)(band + in % h) * kOutRows);
        n0 = __builtin_amdgcn_readfirstlane((int32_t)(in / h) * kI8Wide);
    }
    // slot s of a wave: block-row slot_row(s) of weight slot_side(s)
    auto slot_row = [&](int s) { return br0 + (GATED ? wave * (kI8Rows / 2) + s % (kI8Rows / 2) : wave * kI8Rows + s); };
    auto slot_side = [](int s) { return GATED ? s / (kI8Rows / 2) : 0; };

    // A wave's loads of a window: kI8Window / kI8Waves block-columns, a KB (64 tokens) each.
    constexpr int kPer = kI8Stage / 1024 / kI8Waves;
    const uint32_t lds0 = lds_address(smem);
    const uint32_t column_bytes = (uint32_t)a.N * 16u;
    auto issue = [&](int32_t c0, int stage, int u) {
        const i32x4_t xb = dma_buffer(a.x + ((int64_t)c0 * a.N + n0) * 16, 0x7fffffffu);
        const int at = wave * kPer + u, c = at / 2, n = at % 2 * 64 + lane;
        const bool in = c0 + c < a.in_blocks && n0 + n < a.N;
        dma_to_lds(lds0 + (uint32_t)(stage * kI8Stage + at * 1024),
                   in ? (uint32_t)c * column_bytes + (uint32_t)n * 16u : kNone, xb);
    };
    // Positions: three windows in turn, as byte offsets of blocks, or kNone.
    uint32_t(*const place)[kI8Slots][kI8Window] = reinterpret_cast<uint32_t(*)[kI8Slots][kI8Window]>(smem + 2 * kI8Stage);
    constexpr int kLooks = kI8Slots * kI8Window / kI8Threads;
    auto look = [&](int32_t c0, int32_t (&p)[kLooks]) {
#pragma unroll
        for (int u = 0; u < kLooks; ++u) {
            const int e = u * kI8Threads + t, s = e / kI8Window, c = c0 + e % kI8Window;
            const int32_t r = br0 + (GATED ? s / kI8Rows * (kI8Rows / 2) + s % (kI8Rows / 2) : s);
            const int32_t* map = a.side[GATED ? s / (kI8Rows / 2) % 2 : 0].map;
            p[u] = r < a.block_rows && c < a.in_blocks ? map[(int64_t)r * a.in_blocks + c] : -1;
        }
    };
    auto note = [&](int w, const int32_t (&p)[kLooks]) {
#pragma unroll
        for (int u = 0; u < kLooks; ++u) {
            const int e = u * kI8Threads + t;
            place[w][e / kI8Window][e % kI8Window] = p[u] < 0 ? kNone : (uint32_t)p[u] * 256u;
        }
    };

    int4_t acc[kI8Rows][kI8Tiles];
#pragma unroll
    for (int s = 0; s < kI8Rows; ++s)
#pragma unroll
        for (int j = 0; j < kI8Tiles; ++j) acc[s][j] = int4_t{0, 0, 0, 0};

    const auto v0 = make_buffer(a.side[0].vals, a.vals_bytes[0]);
    const auto v1 = GATED ? make_buffer(a.side[1].vals, a.vals_bytes[1]) : v0;
    // the wave's blocks of four block-columns, and which rows have any
    auto fetch = [&](const uint32_t* at, u32x4_t (&w)[kI8Rows]) -> uint32_t {
        uint32_t any = 0;
#pragma unroll
        for (int s = 0; s < kI8Rows; ++s) {
            const uint32_t p = at[s * kI8Window + g];
            const auto v = buffer_load<float, 4>(slot_side(s) ? v1 : v0, p + (uint32_t)li * 16u);
            w[s] = u32x4_t{v.d[0], v.d[1], v.d[2], v.d[3]};
            if (__ballot(p != kNone)) any |= 1u << s;
        }
        return any;
    };
    // Half a step's operands of x: four tiles of 16 tokens.
    auto read = [&](const unsigned char* S, int half, u32x4_t (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = *reinterpret_cast<const u32x4_t*>(S + (half / 2 * 4 + g) * (kI8Wide * 16) + (16 * (half % 2 * 4 + j) + li) * 16);
    };
    auto multiply = [&](const u32x4_t (&x)[4], const u32x4_t (&w)[kI8Rows], uint32_t any, int h) {
#pragma unroll
        for (int s = 0; s < kI8Rows; ++s)
            if (any & (1u << s))
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[s][h + j] = mfma8(w[s], x[j], acc[s][h + j]);
    };

    // Window by window, four block-columns at a time; blocks are fetched three such steps
    // ahead, so that whole windows are walked (past the last block-column is nothing).
    constexpr int kQuads = kI8Window / 4, kAhead = 3, kRing = kAhead + 1;
    // the next window's x in its first steps: kAhead steps' blocks are fetched after it
    constexpr int kMoves = kQuads - kAhead + 1;
    static_assert(kPer % kMoves == 0);
    const int32_t windows = (a.in_blocks + kI8Window - 1) / kI8Window;
    u32x4_t w[kRing][kI8Rows];
    uint32_t any[kRing];
    int32_t seen[kLooks];
    {
        int32_t second[kLooks];
        look(0, seen);
        look(kI8Window, second);
#pragma unroll
        for (int u = 0; u < kPer; ++u) issue(0, 0, u);
        note(0, seen);
        note(1, second);
        __syncthreads();
    }
    // the rows of `place` that are this wave's
    auto mine = [&](int ring, int quad) { return &place[ring][wave * kI8Rows][4 * quad]; };
#pragma unroll
    for (int q = 0; q < kAhead; ++q) any[q] = fetch(mine(0, q), w[q]);
    int ring = 0;  // of the present window
    for (int32_t i = 0; i < windows; ++i) {
        const int next = ring == 2 ? 0 : ring + 1;
        // the loads of x were under way before the blocks of the last kAhead steps
        dma_wait<kAhead * kI8Rows>();
        __syncthreads();
        const unsigned char* S = smem + (i & 1) * kI8Stage;
        u32x4_t x[2][4];
        read(S, 0, x[0]);
        look((i + 2) * kI8Window, seen);
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            if (q < kMoves && i + 1 < windows)
#pragma unroll
                for (int u = 0; u < kPer / kMoves; ++u)
                    issue((i + 1) * kI8Window, (i + 1) & 1, kPer / kMoves * q + u);
            any[(q + kAhead) % kRing] =
                fetch(q + kAhead < kQuads ? mine(ring, q + kAhead) : mine(next, q + kAhead - kQuads), w[(q + kAhead) % kRing]);
            read(S, 2 * q + 1, x[1]);
            multiply(x[0], w[q % kRing], any[q % kRing], 0);
            if (q + 1 < kQuads) read(S, 2 * q + 2, x[0]);
            multiply(x[1], w[q % kRing], any[q % kRing], 4);
        }
        note(next == 2 ? 0 : next + 1, seen);
        ring = next;
    }

    // The sums leave through LDS, a block-row at a time, so that the rest is done on
    // eight tokens of a row per thread.  What the rest needs is in registers by then: the
    // scales of a lane's tokens, and of a wave's rows one row (16 s + r) per lane.
    constexpr int kSides = GATED ? 2 : 1, kResults = kI8Rows / kSides;
    float xs[8], rs[kSides], bias[kSides];
#pragma unroll
    for (int q = 0; q < 8; ++q) xs[q] = a.x_scale[min((int64_t)n0 + 8 * li + q, a.N - 1)];
    {
        const int64_t row = min(16 * (int64_t)slot_row(lane / 16 % kResults) + li, (int64_t)a.rows - 1);
#pragma unroll
        for (int l = 0; l < kSides; ++l) {
            rs[l] = a.side[l].scale[row];
            bias[l] = a.side[l].bias ? (float)static_cast<const T*>(a.side[l].bias)[row] : 0.f;
        }
    }
    __syncthreads();
    float* O = reinterpret_cast<float*>(smem + wave * kI8Out);
#pragma unroll
    for (int s = 0; s < kResults; ++s) {
#pragma unroll
        for (int l = 0; l < kSides; ++l)
#pragma unroll
            for (int j = 0; j < kI8Tiles; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    O[(l * 16 + 4 * g + q) * kI8OutRow + 16 * j + li] = (float)acc[l * kResults + s][j][q];
        __builtin_amdgcn_wave_barrier();
        int8_rows<T, kSides, kI8Wide>(a, O, 16 * (int64_t)slot_row(s), n0, xs, rs, bias, 16 * s);
        __builtin_amdgcn_wave_barrier();
    }
}

}  // namespace ff

template <typename T>
void int8_tiles(const ff::Int8Product<T>& a, int weights, hipStream_t s)
{
    const int rows = ff::kI8Slots / weights;
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + ff::kI8Wide - 1) / ff::kI8Wide);
    const dim3 grid = launch_grid(ff::kXcds * ff::xcd_chunk(items), ff::kI8Threads);
    if (weights == 2)
        hipLaunchKernelGGL((ff::ff_int8_tile_kernel<T, true>), grid, dim3(ff::kI8Threads), 0, s, a);
    else
        hipLaunchKernelGGL((ff::ff_int8_tile_kernel<T, false>), grid, dim3(ff::kI8Threads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

#define XSPMM_INT8_TILE(T) template void int8_tiles<T>(const ff::Int8Product<T>&, int, hipStream_t);
XSPMM_INT8_TILE(float)
XSPMM_INT8_TILE(_Float16)
XSPMM_INT8_TILE(__bf16)
#undef XSPMM_INT8_TILE

}  // namespace detail
}  // namespace xspmm
