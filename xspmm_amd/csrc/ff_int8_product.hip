// ff_int8_product.hip -- products of block-sparse weights with tokens, both in
// 8-bit integers:
//
//   y = act(A0 x + b0) [* (A1 x + b1)] [+ residual]
//
// A lane's operand of v_mfma_i32_16x16x64_i8 is 16 bytes: one row of a block, or 16
// features of a token.  Lanes 16 g .. + 15 hold block g of four, wherever their
// columns are: four stored blocks of a block-row make one instruction, and absent
// ones of the last four are zeros in A.  Sums are whole numbers and exact in any
// order; a result is float(sum) * row's scale * token's scale, then as in fp32.
//
// Few tokens are bound by latency and the weight's bytes: one token of fp16 4096 x 14336,
// 25 % stored, 6.9 us for 15 MB; gate and up of bf16 14336 x 4096 10.0 us for 29 MB
// (3.1 and 6.0 at the rate of a copy), rounding the token ahead of the blocks.  The walk is
// bound by x, of which L1 brings every stored block its tokens: 45 us at 4 % stored, 14336
// x 4096 and 2048 tokens; 4.4 us at fp32 5003 x 4999, 10 %, 31 tokens.
#include "int8_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

// A wave's share of a block-row times VT tiles of 16 tokens.  Tokens past the last
// read the last one's features, and so do absent blocks (of zeros) the first's.
template <int VT>
struct Int8Step {
    u32x4_t a;
    u32x4_t x[VT];
};

template <typename T, int VT, int NACC, int SPLIT>
__global__ __launch_bounds__(64 * (SPLIT > 4 ? SPLIT : 4)) void ff_int8_walk_kernel(const Int8Product<T> a)
{
    constexpr int kRowsPerGroup = SPLIT > 4 ? 1 : 4 / SPLIT;
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t groups = (uint32_t)(a.block_rows + kRowsPerGroup - 1) / kRowsPerGroup;
    const uint32_t tiles = (uint32_t)((a.N + 16 * VT - 1) / (16 * VT));
    const uint32_t item = xcd_item32(blockIdx.x, groups * tiles);
    if (item == ~0u) return;
    const uint32_t tile = item / groups;
    const int32_t br = (int32_t)(item - tile * groups) * kRowsPerGroup + wave / SPLIT;
    const int part = wave % SPLIT;
    const int64_t n0 = (int64_t)tile * (16 * VT);
    int64_t at[VT];  // this lane's bytes of x at block-column 0
#pragma unroll
    for (int j = 0; j < VT; ++j) at[j] = 16 * min(n0 + 16 * j + li, a.N - 1);
    int4_t acc[NACC][VT];
#pragma unroll
    for (int l = 0; l < NACC; ++l)
#pragma unroll
        for (int j = 0; j < VT; ++j) acc[l][j] = int4_t{0, 0, 0, 0};
    if (br < a.block_rows) {
#pragma unroll
        for (int l = 0; l < NACC; ++l) {
            const Int8Side& s = a.side[l];
            const int32_t b = s.ptr[br], e = s.ptr[br + 1], steps = (e - b + 3) / 4;
            const int32_t lo = b + 4 * (steps * part / SPLIT), hi = min(b + 4 * (steps * (part + 1) / SPLIT), e);
            auto load = [&](Int8Step<VT>& st, int32_t q) {
                const int32_t mine = q + g < hi ? q + g : lo;
                st.a = *reinterpret_cast<const u32x4_t*>(s.vals + (int64_t)mine * 256 + li * 16);
                if (q + g >= hi) st.a = u32x4_t{0u, 0u, 0u, 0u};
                const int8_t* xs = a.x + (int64_t)s.col[mine] * a.N * 16;
#pragma unroll
                for (int j = 0; j < VT; ++j) st.x[j] = *reinterpret_cast<const u32x4_t*>(xs + at[j]);
            };
            for (int32_t q = lo; q < hi; q += 4) {
                Int8Step<VT> st;
                load(st, q);
#pragma unroll
                for (int j = 0; j < VT; ++j)
                    acc[l][j] = mfma8(st.a, st.x[j], acc[l][j]);
            }
        }
    }
    const int64_t row0 = 16 * (int64_t)br + 4 * g;
    if constexpr (SPLIT > 1) {
        __shared__ int red[kRowsPerGroup][SPLIT][NACC][VT][4][64];
#pragma unroll
        for (int l = 0; l < NACC; ++l)
#pragma unroll
            for (int j = 0; j < VT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) red[wave / SPLIT][part][l][j][q][lane] = acc[l][j][q];
        __syncthreads();
        if (part >= 4 || row0 + part >= a.rows) return;
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            const int64_t n = n0 + 16 * j + li;
            if (n >= a.N) break;
            int sum[NACC];
#pragma unroll
            for (int l = 0; l < NACC; ++l) {
                sum[l] = 0;
#pragma unroll
                for (int p = 0; p < SPLIT; ++p) sum[l] += red[wave / SPLIT][p][l][j][part][lane];
            }
            a.y[(row0 + part) * a.N + n] = (T)int8_finish<T, NACC>(a, sum, row0 + part, n, a.x_scale[n]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            const int64_t n = n0 + 16 * j + li;
            if (n >= a.N) break;
            const float xs = a.x_scale[n];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (row0 + q >= a.rows) break;
                int sum[NACC];
#pragma unroll
                for (int l = 0; l < NACC; ++l) sum[l] = acc[l][j][q];
                a.y[(row0 + q) * a.N + n] = (T)int8_finish<T, NACC>(a, sum, row0 + q, n, xs);
            }
        }
    }
}

// Few tokens and few features: a workgroup rounds its (up to 16) tokens itself, into LDS,
// with its first blocks on their way meanwhile, and then walks ROWS block-rows, 16 /
// ROWS waves to each.
constexpr int kFewTokens = kInt8FewTokens, kFewThreads = 1024;
static_assert(kInt8FewPieces == kFewThreads);

// KEPT: such blocks of a thread
template <typename T, int NACC, int ROWS, int KEPT, bool ONE>
__global__ __launch_bounds__(kFewThreads, KEPT == 1 ? 8 : 4) void ff_int8_few_kernel(const Int8Product<T> a)
{
    constexpr int SPLIT = 16 / ROWS, kAhead = KEPT == 1 && NACC == 2 ? 2 : 4;
    __shared__ __align__(16) u32x4_t xs[KEPT * kFewThreads];
    __shared__ int red[ROWS][SPLIT][NACC][4][64];
    __shared__ uint32_t most[16];
    __shared__ float scales[kFewTokens];
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t tiles = (uint32_t)((a.N + kFewTokens - 1) / kFewTokens), group = blockIdx.x / tiles;
    const int32_t br = (int32_t)group * ROWS + wave / SPLIT;
    const int part = wave % SPLIT;
    const int64_t n0 = (int64_t)(blockIdx.x - group * tiles) * kFewTokens;
    const int nt = ONE ? 1 : (int)min((int64_t)kFewTokens, a.N - n0);
    const int blocks = a.in_blocks * nt;

    float v[KEPT][16];
#pragma unroll
    for (int u = 0; u < KEPT; ++u) {
        const int e = t + kFewThreads * u;
        if (e < blocks) {
            if constexpr (ONE) {
                const int32_t k = 16 * e;
                if (k + 16 <= a.in_rows) {
                    const Pack<T, 16> p = *reinterpret_cast<const Pack<T, 16>*>(a.raw + k);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[u][i] = (float)p.v[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[u][i] = k + i < a.in_rows ? (float)a.raw[k + i] : 0.f;
                }
            } else {
                load_features<T>(a.raw, a.in_rows, a.N, e / nt, n0 + e % nt, v[u]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[u][i] = 0.f;
        }
    }

    // this wave's share of its block-row, of either weight
    int32_t lo[NACC], hi[NACC];
    u32x4_t first[NACC][kAhead];
    int32_t column[NACC][kAhead];
    auto load = [&](int l, int32_t q, u32x4_t& w, int32_t& c) {
        const int32_t mine = q + g < hi[l] ? q + g : lo[l];
        w = *reinterpret_cast<const u32x4_t*>(a.side[l].vals + (int64_t)mine * 256 + li * 16);
        if (q + g >= hi[l]) w = u32x4_t{0u, 0u, 0u, 0u};
        c = a.side[l].col[mine];
    };
#pragma unroll
    for (int l = 0; l < NACC; ++l) {
        lo[l] = hi[l] = 0;
        if (br < a.block_rows) {
            const int32_t b = a.side[l].ptr[br], e = a.side[l].ptr[br + 1], steps = (e - b + 3) / 4;
            lo[l] = b + 4 * (steps * part / SPLIT);
            hi[l] = min(b + 4 * (steps * (part + 1) / SPLIT), e);
        }
#pragma unroll
        for (int p = 0; p < kAhead; ++p)
            if (lo[l] + 4 * p < hi[l]) load(l, lo[l] + 4 * p, first[l][p], column[l][p]);
    }

    // the tokens' scales
    if constexpr (ONE) {
        uint32_t m = 0u;
#pragma unroll
        for (int u = 0; u < KEPT; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, magnitude(v[u][i]));
        join<kFewThreads, 1>(m, most);
        const Rounding round(m);
        if (t == 0) scales[0] = round.scale;
#pragma unroll
        for (int u = 0; u < KEPT; ++u)
            if (t + kFewThreads * u < blocks) xs[t + kFewThreads * u] = round_features(v[u], round);
    } else {
        if (t < kFewTokens) most[t] = 0u;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < KEPT; ++u)
            if (t + kFewThreads * u < blocks) {
                uint32_t m = 0u;
#pragma unroll
                for (int i = 0; i < 16; ++i) m = max(m, magnitude(v[u][i]));
                atomicMax(&most[(t + kFewThreads * u) % nt], m);
            }
        __syncthreads();
        if (t < nt) scales[t] = Rounding(most[t]).scale;
#pragma unroll
        for (int u = 0; u < KEPT; ++u)
            if (t + kFewThreads * u < blocks)
                xs[t + kFewThreads * u] = round_features(v[u], Rounding(most[(t + kFewThreads * u) % nt]));
    }
    __syncthreads();

    int4_t acc[NACC];
    const int n = min(li, nt - 1);
#pragma unroll
    for (int l = 0; l < NACC; ++l) {
        acc[l] = int4_t{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < kAhead; ++p)
            if (lo[l] + 4 * p < hi[l]) acc[l] = mfma8(first[l][p], xs[column[l][p] * nt + n], acc[l]);
        for (int32_t q = lo[l] + 4 * kAhead; q < hi[l]; q += 4) {
            u32x4_t w;
            int32_t c;
            load(l, q, w, c);
            acc[l] = mfma8(w, xs[c * nt + n], acc[l]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) red[wave / SPLIT][part][l][q][lane] = acc[l][q];
    }
    __syncthreads();
    const int64_t row = 16 * (int64_t)br + 4 * g + part;
    if (part >= 4 || row >= a.rows || li >= nt) return;
    int sum[NACC];
#pragma unroll
    for (int l = 0; l < NACC; ++l) {
        sum[l] = 0;
#pragma unroll
        for (int p = 0; p < SPLIT; ++p) sum[l] += red[wave / SPLIT][p][l][part][lane];
    }
    a.y[row * a.N + n0 + li] = (T)int8_finish<T, NACC>(a, sum, row, n0 + li, scales[li]);
}

template <typename T, int NACC, int ROWS, int KEPT, bool ONE>
void launch_few(const Int8Product<T>& a, hipStream_t s)
{
    const int64_t items = (int64_t)((a.block_rows + ROWS - 1) / ROWS) * ((a.N + kFewTokens - 1) / kFewTokens);
    hipLaunchKernelGGL((ff_int8_few_kernel<T, NACC, ROWS, KEPT, ONE>), launch_grid(items, kFewThreads), dim3(kFewThreads), 0, s,
                       a);
    XSPMM_LAUNCH_CHECK();
}

template <typename T, int VT, int NACC, int SPLIT>
void launch_walk(const Int8Product<T>& a, hipStream_t s)
{
    constexpr int rows = SPLIT > 4 ? 1 : 4 / SPLIT, threads = 64 * (SPLIT > 4 ? SPLIT : 4);
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + 16 * VT - 1) / (16 * VT));
    hipLaunchKernelGGL((ff_int8_walk_kernel<T, VT, NACC, SPLIT>), launch_grid(kXcds * xcd_chunk(items), threads),
                       dim3(threads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

// What int8_choice has chosen: no other kernels are built.
template <typename T, int NACC>
void launch_few(const Int8Product<T>& a, const Int8Choice& c, hipStream_t s)
{
    auto with = [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        if (a.N > 1)
            launch_few<T, NACC, R, 1, false>(a, s);
        else if (c.b == 1)
            launch_few<T, NACC, R, 1, true>(a, s);
        else
            launch_few<T, NACC, R, 2, true>(a, s);
    };
    if (c.a == 1)
        with(std::integral_constant<int, 1>{});
    else if (c.a == 2)
        with(std::integral_constant<int, 2>{});
    else
        with(std::integral_constant<int, 4>{});
}

template <typename T, int NACC>
void launch_walk(const Int8Product<T>& a, const Int8Choice& c, hipStream_t s)
{
    if (c.a == 4) {
        if (c.b == 4)
            launch_walk<T, 4, NACC, 4>(a, s);
        else
            launch_walk<T, 4, NACC, 1>(a, s);
    } else if (c.b == 16) {
        launch_walk<T, 1, NACC, 16>(a, s);
    } else {
        launch_walk<T, 1, NACC, 4>(a, s);
    }
}

}  // namespace ff

template <typename T>
void int8_product(const Int8Args<T>& f, int weights, hipStream_t s)
{
    const BlockIndex& w = *f.weight[0];
    if (w.Mb == 0 || f.N == 0) return;
    ff::Int8Product<T> a{};
    int64_t blocks[2] = {};
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *f.weight[l];
        a.side[l] = {wl.ptr, wl.col, wl.map, f.vals[l], f.scale[l], f.bias[l]};
        const int64_t vb = narrow_bytes(wl.nnzb, 256, 1);
        a.vals_bytes[l] = vb < 0 ? 0u : (uint32_t)vb;
        blocks[l] = wl.nnzb;
    }
    a.raw = f.raw;
    a.x = f.x;
    a.in_rows = (int32_t)w.K;
    a.in_blocks = (int32_t)w.Kb;
    a.x_scale = f.x_scale;
    a.residual = f.residual;
    a.y = f.y;
    a.rows = (int32_t)w.M;
    a.block_rows = (int32_t)w.Mb;
    a.N = f.N;
    a.act = f.act;
    const Int8Choice c = int8_choice(weights, w.M, w.K, blocks, f.N, (int)sizeof(T), a.raw != nullptr);
    switch (c.kernel) {
    case Int8Kernel::kLists:
        int8_lists<T>(a, weights, c.a, s);
        break;
    case Int8Kernel::kTiles:
        int8_tiles<T>(a, weights, s);
        break;
    case Int8Kernel::kFew:
        weights == 2 ? ff::launch_few<T, 2>(a, c, s) : ff::launch_few<T, 1>(a, c, s);
        break;
    case Int8Kernel::kWalk:
        weights == 2 ? ff::launch_walk<T, 2>(a, c, s) : ff::launch_walk<T, 1>(a, c, s);
        break;
    }
}

#define XSPMM_INT8_PRODUCT(T) template void int8_product<T>(const Int8Args<T>&, int, hipStream_t);
XSPMM_INT8_PRODUCT(float)
XSPMM_INT8_PRODUCT(_Float16)
XSPMM_INT8_PRODUCT(__bf16)
#undef XSPMM_INT8_PRODUCT

}  // namespace detail
}  // namespace xspmm
