// ff_int8_list.hip -- the products of ff_int8_product.hip for many tokens where most
// blocks are absent: as in ff_int8_tile.hip x goes through LDS by windows, but a wave
// walks what is stored of a block-row in a window, four blocks at a time wherever their
// columns are, so that all that is loaded and multiplied is stored.
//
// A workgroup of eight waves takes 32 block-rows (gated: 16 of either weight) and 64
// tokens; a window is 32 block-columns (32 KB of x), two in turn, two workgroups a CU.
// A wave lists its four block-rows' blocks a window ahead: a lane looks at two entries of
// the weight's map, and the lists are what is stored, pushed together.  Of every row the
// first 4 Q blocks are fetched, two rows ahead, and multiplied without a question (zeros
// where there are fewer); more than that is rare and fetched when it is met.
//
// What bounds it is latency, of a window's x, lists and first blocks one after the other
// (at 5 % stored a window takes 2 us, its instructions a quarter of that): waves of eight
// block-rows with twice the registers, two a SIMD, take 163 us for gate and up of 14336 x
// 4096, 2048 tokens, 25 % stored, bf16, where waves of four, four a SIMD, took 147; those
// take 126 to 135 now, with two fours fetched ahead in place of three.  One product 75 (by
// tiles 100, by the walk 126), 10 % stored 58 (83, 69).
#include "int8_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

constexpr int kListWide = kInt8ListTokens;  // of a workgroup
constexpr int kListTiles = kListWide / 16;
constexpr int kListWaves = 8, kListThreads = 64 * kListWaves;
constexpr int kListRows = 4;     // a wave's block-rows, of both weights
constexpr int kListSlots = kListRows * kListWaves;
static_assert(kListSlots == kInt8ListRows);
constexpr int kListWindow = kInt8ListColumns;
constexpr int kListStage = kListWindow * kListWide * 16;
constexpr int kListAhead = 2;    // rows whose blocks are on their way
constexpr int kListLanes = 64 / kListRows, kListColumns = kListWindow / kListLanes;  // of a row's list
constexpr int kListOut = 2 * 16 * (kListWide + 4) * 4;  // a wave's bytes on their way out
constexpr int kListLds = 2 * kListStage + 2 * kListSlots * kListWindow * 4;
constexpr int kListBand = 8;
static_assert(kListLds <= 80 * 1024 && kListWaves * kListOut <= kListLds);

template <typename T, bool GATED, int Q>
__global__ __launch_bounds__(kListThreads, 4) void ff_int8_list_kernel(const Int8Product<T> a)
{
    constexpr int kSides = GATED ? 2 : 1, kResults = kListRows / kSides;
    constexpr int kOutRows = kListSlots / kSides;  // block-rows of the result
    __shared__ __align__(16) unsigned char smem[kListLds];
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);

    int32_t br0, n0;
    {
        // bands of kListBand row groups, token tile by token tile
        const uint32_t tiles = (uint32_t)((a.N + kListWide - 1) / kListWide);
        const uint32_t groups = (uint32_t)(a.block_rows + kOutRows - 1) / kOutRows;
        const uint32_t item = xcd_item32(blockIdx.x, groups * tiles);
        if (item == ~0u) return;
        const uint32_t band = item / (kListBand * tiles) * kListBand;
        const uint32_t h = min((uint32_t)kListBand, groups - band), in = item - band * tiles;
        br0 = __builtin_amdgcn_readfirstlane((int32_t)(band + in % h) * kOutRows);
        n0 = __builtin_amdgcn_readfirstlane((int32_t)(in / h) * kListWide);
    }
    auto slot_row = [&](int s) { return br0 + wave * kResults + s % kResults; };

    // a wave's loads of a window: a block-column's 64 tokens each
    constexpr int kPer = kListWindow / kListWaves;
    const uint32_t lds0 = lds_address(smem);
    const uint32_t column_bytes = (uint32_t)a.N * 16u;
    auto issue = [&](int32_t c0, int stage) {
        const i32x4_t xb = dma_buffer(a.x + ((int64_t)c0 * a.N + n0) * 16, 0x7fffffffu);
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int c = wave * kPer + u;
            const bool in = c0 + c < a.in_blocks && n0 + lane < a.N;
            dma_to_lds(lds0 + (uint32_t)(stage * kListStage + c * 1024),
                       in ? (uint32_t)c * column_bytes + (uint32_t)lane * 16u : kNone, xb);
        }
    };

    // Lists of this wave's rows, two windows in turn: 256 times a block's position plus its
    // column in the window, or kNone.
    uint32_t* const lists = reinterpret_cast<uint32_t*>(smem + 2 * kListStage) + wave * (2 * kListRows * kListWindow);
    const int mine = lane / kListLanes, at_c = lane % kListLanes * kListColumns;  // what this lane looks at
    const int32_t my_row = br0 + wave * kResults + mine % kResults;
    const int32_t* const my_map =
        a.side[mine / kResults].map + (int64_t)(my_row < a.block_rows ? my_row : 0) * a.in_blocks;
    auto look = [&](int32_t c0, int32_t (&p)[kListColumns]) {
#pragma unroll
        for (int j = 0; j < kListColumns; ++j) {
            const int32_t c = c0 + at_c + j;
            p[j] = my_row < a.block_rows && c < a.in_blocks ? my_map[c] : -1;
        }
    };
    // fours: of every row how many fours of blocks it has, 4 bits each
    auto list = [&](uint32_t* to, const int32_t (&p)[kListColumns]) -> uint32_t {
        constexpr int kEach = kListRows * kListWindow / 64;
        lanes_in_order();
#pragma unroll
        for (int j = 0; j < kEach; ++j) to[kEach * lane + j] = kNone;
        lanes_in_order();
        constexpr uint32_t kRow = (uint32_t)((1ull << kListLanes) - 1);
        int at = mine * kListWindow;
        uint64_t there[kListColumns];
#pragma unroll
        for (int j = 0; j < kListColumns; ++j) {
            there[j] = __ballot(p[j] >= 0);
            const uint32_t row = (uint32_t)(there[j] >> (kListLanes * mine)) & kRow;
            if (p[j] >= 0)
                to[at + __popc(row & ((1u << (lane % kListLanes)) - 1u))] = (uint32_t)p[j] * 256u + (uint32_t)(at_c + j);
            at += __popc(row);
        }
        lanes_in_order();
        uint32_t fours = 0;
#pragma unroll
        for (int s = 0; s < kListRows; ++s) {
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < kListColumns; ++j) n += (uint32_t)__popc((uint32_t)(there[j] >> (kListLanes * s)) & kRow);
            fours |= (n + 3) / 4 << (4 * s);
        }
        return (uint32_t)__builtin_amdgcn_readfirstlane((int)fours);
    };

    const auto v0 = make_buffer(a.side[0].vals, a.vals_bytes[0]);
    const auto v1 = GATED ? make_buffer(a.side[1].vals, a.vals_bytes[1]) : v0;
    auto entry = [&](const uint32_t* from, int s, int k) { return from[s * kListWindow + 4 * k + g]; };
    auto fetch = [&](int s, uint32_t e) {
        const auto v = buffer_load<float, 4>(s / kResults ? v1 : v0, (e & ~255u) + (uint32_t)li * 16u);
        return u32x4_t{v.d[0], v.d[1], v.d[2], v.d[3]};
    };

    int4_t acc[kListRows][kListTiles];
#pragma unroll
    for (int s = 0; s < kListRows; ++s)
#pragma unroll
        for (int j = 0; j < kListTiles; ++j) acc[s][j] = int4_t{0, 0, 0, 0};
    auto multiply = [&](const unsigned char* S, int4_t (&to)[kListTiles], u32x4_t w, uint32_t e) {
        const unsigned char* x = S + (e & 255u) * 1024u + li * 16;
#pragma unroll
        for (int j = 0; j < kListTiles; ++j) to[j] = mfma8(w, *reinterpret_cast<const u32x4_t*>(x + 256 * j), to[j]);
    };

    const int32_t windows = (a.in_blocks + kListWindow - 1) / kListWindow;
    constexpr int kList = kListRows * kListWindow;
    u32x4_t w[kListAhead][Q];
    uint32_t e[kListAhead][Q], following[Q];
    int32_t seen[kListColumns];
    look(0, seen);
    issue(0, 0);
    uint32_t fours = list(lists, seen);
    look(kListWindow, seen);
#pragma unroll
    for (int s = 0; s < kListAhead; ++s)
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            e[s][k] = entry(lists, s, k);
            w[s][k] = fetch(s, e[s][k]);
        }
#pragma unroll
    for (int k = 0; k < Q; ++k) following[k] = entry(lists, kListAhead, k);

    for (int32_t i = 0; i < windows; ++i) {
        // the loads of x were under way before the blocks of the last kListAhead rows
        dma_wait<kListAhead * Q>();
        __syncthreads();
        const unsigned char* S = smem + (i & 1) * kListStage;
        uint32_t *now = lists + (i & 1) * kList, *next = lists + ((i + 1) & 1) * kList;
        const uint32_t coming = list(next, seen);
        look((i + 2) * kListWindow, seen);
        if (i + 1 < windows) issue((i + 1) * kListWindow, (i + 1) & 1);
#pragma unroll
        for (int s = 0; s < kListRows; ++s) {
            constexpr int kRing = kListAhead;
#pragma unroll
            for (int k = 0; k < Q; ++k) multiply(S, acc[s], w[s % kRing][k], e[s % kRing][k]);
            const uint32_t n = fours >> (4 * s) & 15u;
            for (uint32_t k = Q; k < n; ++k) {
                const uint32_t more = entry(now, s, (int)k);
                multiply(S, acc[s], fetch(s, more), more);
            }
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                e[s % kRing][k] = following[k];
                w[s % kRing][k] = fetch((s + kRing) % kListRows, following[k]);
                following[k] = s + kRing + 1 < kListRows ? entry(now, s + kRing + 1, k)
                                                         : entry(next, s + kRing + 1 - kListRows, k);
            }
        }
        fours = coming;
    }

    // the sums leave through LDS, as in the tiles
    constexpr int kFour = (kResults + 3) / 4;
    float xs[8], rs[kFour][kSides], bias[kFour][kSides];
#pragma unroll
    for (int q = 0; q < 8; ++q) xs[q] = a.x_scale[min((int64_t)n0 + 8 * (lane & 7) + q, a.N - 1)];
#pragma unroll
    for (int h = 0; h < kFour; ++h) {
        const int64_t row = min(16 * (int64_t)slot_row(4 * h + lane / 16) + li, (int64_t)a.rows - 1);
#pragma unroll
        for (int l = 0; l < kSides; ++l) {
            rs[h][l] = a.side[l].scale[row];
            bias[h][l] = a.side[l].bias ? (float)static_cast<const T*>(a.side[l].bias)[row] : 0.f;
        }
    }
    __syncthreads();
    float* O = reinterpret_cast<float*>(smem + wave * kListOut);
#pragma unroll
    for (int s = 0; s < kResults; ++s) {
#pragma unroll
        for (int l = 0; l < kSides; ++l)
#pragma unroll
            for (int j = 0; j < kListTiles; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    O[(l * 16 + 4 * g + q) * (kListWide + 4) + 16 * j + li] = (float)acc[l * kResults + s][j][q];
        __builtin_amdgcn_wave_barrier();
        int8_rows<T, kSides, kListWide>(a, O, 16 * (int64_t)slot_row(s), n0, xs, rs[s / 4], bias[s / 4], 16 * (s % 4));
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, int Q>
void launch_list(const Int8Product<T>& a, int weights, int64_t items, hipStream_t s)
{
    const dim3 grid = launch_grid(kXcds * xcd_chunk(items), kListThreads);
    if (weights == 2)
        hipLaunchKernelGGL((ff_int8_list_kernel<T, true, Q>), grid, dim3(kListThreads), 0, s, a);
    else
        hipLaunchKernelGGL((ff_int8_list_kernel<T, false, Q>), grid, dim3(kListThreads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

}  // namespace ff

template <typename T>
void int8_lists(const ff::Int8Product<T>& a, int weights, int fours, hipStream_t s)
{
    const int rows = ff::kListSlots / weights;
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + ff::kListWide - 1) / ff::kListWide);
    if (fours == 1)
        ff::launch_list<T, 1>(a, weights, items, s);
    else if (fours == 2)
        ff::launch_list<T, 2>(a, weights, items, s);
    else
        ff::launch_list<T, 3>(a, weights, items, s);
}

#define XSPMM_INT8_LIST(T) template void int8_lists<T>(const ff::Int8Product<T>&, int, int, hipStream_t);
XSPMM_INT8_LIST(float)
XSPMM_INT8_LIST(_Float16)
XSPMM_INT8_LIST(__bf16)
#undef XSPMM_INT8_LIST

}  // namespace detail
}  // namespace xspmm
