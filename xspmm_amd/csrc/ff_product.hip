// ff_product.hip -- products of block-sparse weights with activations:
//
//   forward      y = act(A0 x + b0) [* (A1 x + b1)] [+ residual]
//   transposed   dx = A0^T dz0 [+ A1^T dz1]
//
// Blocks are 16 x 16, x is features x tokens.  A wave owns one block-row of
// the result (block-column of A for the transposed product) and 16 * VEC
// tokens; lane l owns tokens VEC * (l % 16) .. + VEC - 1 of them, so that its
// loads of x, and its stores of y, are VEC consecutive elements.
//
//   16 bits: two blocks of the row make one v_mfma_f32_16x16x32: lanes 0..31
//     hold the first, lanes 32..63 the second, wherever their columns are.  A
//     lane loads its 8 rows of x (VEC tokens each) and v_perm gathers, token
//     by token, the 8 values that the instruction wants in one lane.
//   32 bits: four v_mfma_f32_16x16x4 per block; step s takes row 4 (l / 16) + s,
//     so a lane's four values of A are one load and no value of x moves.
//
// A^T: the same walk over the blocks of a block-column, whose values are
// loaded down the columns of the block.
//
// One token is bound by the weight's bytes: 4096 x 14336 fp16, 25 % stored, 29 MB in
// 6.3 us, 4.7 TB/s; bf16 gate and up of 14336 x 4096 59 MB in 12.1, 4.9 TB/s.  More
// tokens are bound by the rows of x that every block reads anew, through the 64
// bytes a clock of a CU's L1: 14336 x 4096, 10 % stored, 2048 tokens 107 us, 14 TB/s,
// 25 % 210 us, 18 TB/s (there the tiles of ff_tile.hip take over).  With few blocks a
// wave the chain of loads (row pointer, block-column, x) shows: 8192 x 8192, 5 %,
// 256 tokens 13.0 us, of which 4.8 are launch, pointers, the sums of four waves and
// the results.  fp32, 4096 x 4096, 512 tokens, dx: 10 % stored 26 us, 66 TFLOP/s, all
// 165 us, 104.
#include "feed_forward_device.hpp"

namespace xspmm {
namespace detail {
namespace ff {

constexpr int kWaves = 4;
template <typename T>
struct Side {
    const int32_t* ptr;
    const int32_t* other;  // block-columns (transposed: block-rows)
    const int32_t* blk;    // transposed: positions of the blocks
    const T* vals;
    const T* x;
    const T* bias;
    T* keep;
};

template <typename T>
struct ProductArgs {
    Side<T> side[2];
    const T* residual;
    T* y;
    int32_t sides;
    int32_t rows;        // of the result
    int32_t block_rows;
    int32_t in_rows;     // of x
    int64_t N;
    uint32_t x_bytes, vals_bytes[2];
    int act;
};

// What one step multiplies: two blocks of 16-bit values, one of 32-bit values.
template <typename T, int VEC>
struct Step {
    static constexpr int kRows = is_f32<T> ? 4 : 8;
    uint32_t a[4];
    Dwords<kDwords<T, VEC>> b[kRows];
};

// ONE: a single token, whose rows of x are consecutive: one load has them all, and
// the 16 columns of the instruction compute the same.
template <typename T, int VEC, bool TR, bool WIDE, bool ONE>
struct Walk {
    static constexpr int kRows = Step<T, VEC>::kRows;
    static constexpr int kPer = is_f32<T> ? 1 : 2;  // blocks per step

    const Side<T>& s;
    const int64_t N;
    const int64_t n;       // this lane's first token
    const int32_t in_rows;
    const int32_t edge;    // the block-row of x that ends early, or -1
    const int li, g;
    __amdgpu_buffer_rsrc_t xr, vr;

    __device__ __forceinline__ Walk(const ProductArgs<T>& a, int l, int64_t n_, int lane)
        : s(a.side[l]), N(a.N), n(n_), in_rows(a.in_rows), edge(a.in_rows % 16 ? a.in_rows / 16 : -1),
          li(lane & 15), g(lane >> 4)
    {
        if constexpr (!WIDE) {
            xr = make_buffer(s.x, a.x_bytes);
            vr = make_buffer(s.vals, a.vals_bytes[l]);
        }
    }

    // the step at blocks b and b + 1 (the latter absent at `end`)
    __device__ __forceinline__ void load(Step<T, VEC>& st, int32_t b, int32_t end) const
    {
        const bool two = kPer == 1 || b + 1 < end;
        const int32_t c0 = s.other[b], c1 = s.other[two ? b + kPer - 1 : b];
        const bool second = kPer == 2 && g >= 2;
        const int32_t c = second ? c1 : c0;
        const bool absent = second && !two;
        int32_t at;
        if constexpr (TR) {
            const int32_t i0 = s.blk[b], i1 = s.blk[two ? b + kPer - 1 : b];
            at = second ? i1 : i0;
        } else {
            at = second && two ? b + 1 : b;
        }
        // row and column of this lane's values within the block
        const int sub = is_f32<T> ? 4 * g : 8 * (g & 1);
        const int32_t row = 16 * c + sub;
        const bool cut = c0 == edge || c1 == edge;  // rows past the last contribute nothing
        if constexpr (!WIDE) {
            const uint32_t a0 = absent ? kNone : (uint32_t)at * (256u * sizeof(T));
            if constexpr (!TR) {
                const auto v = buffer_load<float, 4>(vr, a0 + (uint32_t)(li * 16 + sub) * (uint32_t)sizeof(T));
#pragma unroll
                for (int i = 0; i < 4; ++i) st.a[i] = v.d[i];
            } else {
#pragma unroll
                for (int i = 0; i < kRows; ++i) put(st, i, buffer_load<T, 1>(vr, a0 + (uint32_t)((sub + i) * 16 + li) * (uint32_t)sizeof(T)).d[0]);
            }
            if constexpr (ONE) {
                load_one(st, row, absent);
                return;
            }
            const uint32_t ld = (uint32_t)N * (uint32_t)sizeof(T);
            const uint32_t x0 = absent ? kNone : (uint32_t)row * ld + (uint32_t)n * (uint32_t)sizeof(T);
            if (!cut) {
#pragma unroll
                for (int i = 0; i < kRows; ++i) st.b[i] = buffer_load<T, VEC>(xr, x0 + (uint32_t)i * ld);
            } else {
#pragma unroll
                for (int i = 0; i < kRows; ++i)
                    st.b[i] = buffer_load<T, VEC>(xr, row + i < in_rows ? x0 + (uint32_t)i * ld : kNone);
            }
        } else {
            const T* v = s.vals + (int64_t)at * 256;
            if constexpr (!TR) {
                const auto q = global_load<float, 4>(reinterpret_cast<const float*>(v + li * 16 + sub));
#pragma unroll
                for (int i = 0; i < 4; ++i) st.a[i] = absent ? 0u : q.d[i];
            } else {
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const uint32_t q = global_load<T, 1>(v + (sub + i) * 16 + li).d[0];
                    put(st, i, absent ? 0u : q);
                }
            }
            // tokens past the last (lanes of a narrow result) read its value
            const int64_t col = n < N - VEC ? n : N - VEC;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const bool there = row + i < in_rows;
                st.b[i] = global_load<T, VEC>(s.x + (int64_t)(there ? row + i : in_rows - 1) * N + col);
                if (absent || !there)
#pragma unroll
                    for (int d = 0; d < kDwords<T, VEC>; ++d) st.b[i].d[d] = 0u;
            }
        }
    }

    // x has one column: the lane's rows in one load (in parts at the edge, as a
    // load past the end gives whole dwords of zeros)
    __device__ __forceinline__ void load_one(Step<T, VEC>& st, int32_t row, bool absent) const
    {
        uint32_t d[4] = {0u, 0u, 0u, 0u};
        if (row + kRows <= in_rows || absent) {
            const auto v = buffer_load<float, 4>(xr, absent ? kNone : (uint32_t)row * (uint32_t)sizeof(T));
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = v.d[i];
        } else {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const uint32_t v =
                    buffer_load<T, 1>(xr, row + i < in_rows ? (uint32_t)(row + i) * (uint32_t)sizeof(T) : kNone).d[0];
                if constexpr (is_f32<T>)
                    d[i] = v;
                else
                    d[i / 2] |= v << (16 * (i % 2));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) st.b[i].d[0] = d[i];
    }

    // element i of a lane's values of A
    static __device__ __forceinline__ void put(Step<T, VEC>& st, int i, uint32_t v)
    {
        if constexpr (is_f32<T>)
            st.a[i] = v;
        else
            st.a[i / 2] = i % 2 ? st.a[i / 2] | (v << 16) : v;
    }

    static __device__ __forceinline__ void multiply(float4_t (&acc)[VEC], const Step<T, VEC>& st)
    {
        if constexpr (is_f32<T>) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VEC; ++c) acc[c] = mfma32(st.a[i], st.b[i].d[c], acc[c]);
        } else {
            const u32x4_t a = {st.a[0], st.a[1], st.a[2], st.a[3]};
            if constexpr (ONE) {
                acc[0] = mfma16<T>(a, u32x4_t{st.b[0].d[0], st.b[1].d[0], st.b[2].d[0], st.b[3].d[0]}, acc[0]);
                return;
            }
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                u32x4_t v;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    v[r] = __builtin_amdgcn_perm(st.b[2 * r + 1].d[c / 2], st.b[2 * r].d[c / 2],
                                                 c % 2 ? 0x07060302u : 0x05040100u);
                acc[c] = mfma16<T>(a, v, acc[c]);
            }
        }
    }

    // acc += blocks [b, end) times x: the loads of kAhead steps run ahead of the
    // instructions of the step before
    static constexpr int kAhead = ONE ? 4 : VEC <= 2 ? 3 : 2;
    __device__ __forceinline__ void run(float4_t (&acc)[VEC], int32_t b, int32_t end) const
    {
        if (b >= end) return;
        const int32_t last = end - 1 - (kPer == 2 ? (end - 1 - b) % 2 : 0);
        Step<T, VEC> s[kAhead];
#pragma unroll
        for (int p = 0; p + 1 < kAhead; ++p) load(s[p], b + p * kPer < last ? b + p * kPer : last, end);
        for (; b < end; b += kAhead * kPer) {
#pragma unroll
            for (int p = 0; p < kAhead; ++p) {
                const int32_t next = b + (p + kAhead - 1) * kPer;
                load(s[(p + kAhead - 1) % kAhead], next < last ? next : last, end);
                // 32-bit products are bound by the matrix units as much as by loads, and
                // a wave with its operands goes first (4096 x 4096 fp32 gated, 30 %
                // stored, 512 tokens 124 -> 109 us; in 16 bits dx loses a tenth)
                if constexpr (is_f32<T>) __builtin_amdgcn_s_setprio(1);
                multiply(acc, s[p]);
                if constexpr (is_f32<T>) __builtin_amdgcn_s_setprio(0);
                if (b + (p + 1) * kPer >= end) return;
            }
        }
    }
};

// The result's rows 4 (l / 16) + q of a wave's block-row and the lane's VEC tokens
template <typename T, int VEC, int NACC, bool TR>
__device__ __forceinline__ void finish(const ProductArgs<T>& a, float (&z)[NACC][VEC], int64_t row, int64_t n,
                                       int64_t first, int64_t end)
{
    const bool whole = n >= first && n + VEC <= end;
    auto store = [&](T* p, const float(&v)[VEC]) {
        if (whole) {
            Pack<T, VEC> o;
#pragma unroll
            for (int c = 0; c < VEC; ++c) o.v[c] = (T)v[c];
            *reinterpret_cast<Pack<T, VEC>*>(p + row * a.N + n) = o;
        } else {
#pragma unroll
            for (int c = 0; c < VEC; ++c)
                if (n + c >= first && n + c < end) p[row * a.N + n + c] = (T)v[c];
        }
    };
    if constexpr (!TR) {
        float r[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) r[c] = 0.f;
        if (a.residual) {
            if (whole) {
                const Pack<T, VEC> k = *reinterpret_cast<const Pack<T, VEC>*>(a.residual + row * a.N + n);
#pragma unroll
                for (int c = 0; c < VEC; ++c) r[c] = (float)k.v[c];
            } else {
#pragma unroll
                for (int c = 0; c < VEC; ++c)
                    if (n + c >= first && n + c < end) r[c] = (float)a.residual[row * a.N + n + c];
            }
        }
#pragma unroll
        for (int l = 0; l < NACC; ++l) {
            const float bias = a.side[l].bias ? (float)a.side[l].bias[row] : 0.f;
#pragma unroll
            for (int c = 0; c < VEC; ++c) z[l][c] += bias;
            if (a.side[l].keep) store(a.side[l].keep, z[l]);
        }
        with_act(a.act, [&](auto act) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) z[0][c] = act_value<decltype(act)::value>(z[0][c]);
        });
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
            if constexpr (NACC == 2) z[0][c] *= z[1][c];
            z[0][c] += r[c];
        }
    }
    store(a.y, z[0]);
}

// NACC accumulators: 2 for the gated forward product.  SPLIT waves share a
// block-row's blocks and add up in LDS, in their order; four of them then finish
// a quarter of its rows each.
template <typename T, int VEC, int NACC, bool TR, int SPLIT, bool WIDE, bool ONE>
__global__ __launch_bounds__(64 * (SPLIT > kWaves ? SPLIT : kWaves)) void ff_product_kernel(const ProductArgs<T> a)
{
    constexpr int kRowsPerGroup = SPLIT > kWaves ? 1 : kWaves / SPLIT;
    constexpr int kTile = ONE ? 1 : 16 * VEC;
    using W = Walk<T, VEC, TR, WIDE, ONE>;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t groups = (a.block_rows + kRowsPerGroup - 1) / kRowsPerGroup;
    const int64_t tiles = (a.N + kTile - 1) / kTile;
    const int64_t item = xcd_item(blockIdx.x, groups * tiles);
    if (item < 0) return;
    const int32_t br = (int32_t)(item % groups) * kRowsPerGroup + wave / SPLIT;
    const int part = wave % SPLIT;
    const int64_t first = item / groups * kTile;  // the tile's first token
    // the last tile moves back into the matrix (and stores its own tokens only)
    const int64_t n0 = first + kTile > a.N && a.N >= kTile ? a.N - kTile : first;
    const int64_t n = ONE ? lane & 15 : n0 + VEC * (lane & 15);

    float4_t acc[NACC][VEC];
#pragma unroll
    for (int l = 0; l < NACC; ++l)
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[l][c] = float4_t{0.f, 0.f, 0.f, 0.f};
    if (br < a.block_rows) {
        auto side = [&](int l, float4_t(&to)[VEC]) {
            const W w(a, l, n, lane);
            const int32_t b = a.side[l].ptr[br], e = a.side[l].ptr[br + 1];
            constexpr int per = W::kPer;
            const int32_t steps = (e - b + per - 1) / per;
            const int32_t lo = b + per * (int32_t)((int64_t)steps * part / SPLIT);
            const int32_t hi = b + per * (int32_t)((int64_t)steps * (part + 1) / SPLIT);
            w.run(to, lo, hi < e ? hi : e);
        };
        side(0, acc[0]);
        if constexpr (NACC == 2)
            side(1, acc[1]);
        else if (a.sides == 2)
            side(1, acc[0]);
    }
    const int64_t row0 = 16 * (int64_t)br + 4 * (lane >> 4);
    float z[NACC][VEC];
    if constexpr (SPLIT > 1) {
        __shared__ float red[kRowsPerGroup][SPLIT][NACC][VEC][4][64];
#pragma unroll
        for (int l = 0; l < NACC; ++l)
#pragma unroll
            for (int c = 0; c < VEC; ++c)
#pragma unroll
                for (int q = 0; q < 4; ++q) red[wave / SPLIT][part][l][c][q][lane] = acc[l][c][q];
        __syncthreads();
        if (part >= 4) return;
#pragma unroll
        for (int l = 0; l < NACC; ++l)
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                z[l][c] = 0.f;
#pragma unroll
                for (int p = 0; p < SPLIT; ++p) z[l][c] += red[wave / SPLIT][p][l][c][part][lane];
            }
        if (row0 + part < a.rows && n + VEC > first && n < a.N)
            finish<T, VEC, NACC, TR>(a, z, row0 + part, n, first, a.N);
    } else {
        if (n + VEC <= first || n >= a.N) return;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (row0 + q >= a.rows) break;
#pragma unroll
            for (int l = 0; l < NACC; ++l)
#pragma unroll
                for (int c = 0; c < VEC; ++c) z[l][c] = acc[l][c][q];
            finish<T, VEC, NACC, TR>(a, z, row0 + q, n, first, a.N);
        }
    }
}

template <typename T, int VEC, int NACC, bool TR, int SPLIT, bool WIDE, bool ONE = false>
void launch(const ProductArgs<T>& a, hipStream_t s)
{
    constexpr int rows = SPLIT > kWaves ? 1 : kWaves / SPLIT, threads = 64 * (SPLIT > kWaves ? SPLIT : kWaves);
    constexpr int tile = ONE ? 1 : 16 * VEC;
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + tile - 1) / tile);
    hipLaunchKernelGGL((ff_product_kernel<T, VEC, NACC, TR, SPLIT, WIDE, ONE>),
                       launch_grid(kXcds * xcd_chunk(items), threads), dim3(threads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

template <typename T, int VEC, int NACC, bool TR>
void launch_split(const ProductArgs<T>& a, int split, hipStream_t s)
{
    if (split == 1)
        launch<T, VEC, NACC, TR, 1, false>(a, s);
    else if (split == 4 || VEC > 2)
        launch<T, VEC, NACC, TR, 4, false>(a, s);
    else if constexpr (VEC <= 2)
        launch<T, VEC, NACC, TR, 16, false>(a, s);
}

template <typename T, int NACC, bool TR>
void launch_product(const ProductArgs<T>& a, int64_t blocks, bool wide, hipStream_t s)
{
    if (a.block_rows == 0 || a.N == 0) return;
    constexpr int most = is_f32<T> ? 4 : 8;
    int vec = most;
    while (vec > 1 && 16 * vec > a.N) vec /= 2;
    if (wide) {
        if (vec == 1)
            launch<T, 1, NACC, TR, 4, true>(a, s);
        else if (a.N >= 64)
            launch<T, 4, NACC, TR, 1, true>(a, s);
        else
            launch<T, 2, NACC, TR, 4, true>(a, s);
        return;
    }
    // Wide tiles while they leave enough waves for the chip, with four waves to a
    // block-row if need be (8192 x 8192, 5 % of the blocks, 256 tokens: 14.1 us with
    // 8 x 16 tokens a wave, 16.8 with 4 x 16); narrow ones where even those are few
    // (1024 x 1024, 20 %, 64 tokens: 5.6 us with 16 tokens a wave, 6.5 with 64).
    auto waves = [&](int v) { return (int64_t)a.block_rows * ((a.N + 16 * v - 1) / (16 * v)); };
    while (vec > 4 && waves(vec) < 1024) vec /= 2;
    while (vec > 1 && waves(vec) < 256) vec /= 2;
    const int64_t each = blocks / a.block_rows;  // blocks of a wave without a split
    const int split = waves(vec) <= 512 && each >= 64 ? 16 : waves(vec) < 4096 && each >= 8 ? 4 : 1;
    if (a.N == 1) {
        if (split == 16)
            launch<T, 1, NACC, TR, 16, false, true>(a, s);
        else
            launch<T, 1, NACC, TR, 4, false, true>(a, s);
        return;
    }
    switch (vec) {
    case 8:
        if constexpr (!is_f32<T>) launch_split<T, 8, NACC, TR>(a, split, s);
        break;
    case 4: launch_split<T, 4, NACC, TR>(a, split, s); break;
    case 2: launch_split<T, 2, NACC, TR>(a, split, s); break;
    default: launch_split<T, 1, NACC, TR>(a, split, s); break;
    }
}

}  // namespace ff

template <typename T>
void feed_forward(const ForwardArgs<T>& f, int weights, hipStream_t s)
{
    if constexpr (!ff::is_f32<T>)
        if (feed_forward_tiles<T>(f, weights, s)) return;
    const BlockIndex& w = *f.weight[0];
    ff::ProductArgs<T> a{};
    int64_t blocks = 0;
    bool wide = false;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *f.weight[l];
        a.side[l] = {wl.ptr, wl.col, nullptr, f.vals[l], f.x, f.bias[l], f.keep[l]};
        const int64_t vb = narrow_bytes(wl.nnzb, 256, sizeof(T));
        wide |= vb < 0;
        a.vals_bytes[l] = (uint32_t)vb;
        blocks += wl.nnzb;
    }
    const int64_t xb = narrow_bytes(w.K, f.N, sizeof(T));
    wide |= xb < 0;
    a.x_bytes = (uint32_t)xb;
    a.residual = f.residual;
    a.y = f.y;
    a.sides = weights;
    a.rows = (int32_t)w.M;
    a.block_rows = (int32_t)w.Mb;
    a.in_rows = (int32_t)w.K;
    a.N = f.N;
    a.act = f.act;
    if (weights == 2)
        ff::launch_product<T, 2, false>(a, blocks, wide, s);
    else
        ff::launch_product<T, 1, false>(a, blocks, wide, s);
}

template <typename T>
void transposed_product(const TransposedArgs<T>& t, int weights, hipStream_t s)
{
    if constexpr (!ff::is_f32<T>)
        if (transposed_tiles<T>(t, weights, s)) return;
    const BlockIndex& w = *t.weight[0];
    ff::ProductArgs<T> a{};
    int64_t blocks = 0;
    bool wide = false;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *t.weight[l];
        a.side[l] = {wl.tptr, wl.trow, wl.tblk, t.vals[l], t.dz[l], nullptr, nullptr};
        const int64_t vb = narrow_bytes(wl.nnzb, 256, sizeof(T));
        wide |= vb < 0;
        a.vals_bytes[l] = (uint32_t)vb;
        blocks += wl.nnzb;
    }
    const int64_t xb = narrow_bytes(w.M, t.N, sizeof(T));
    wide |= xb < 0;
    a.x_bytes = (uint32_t)xb;
    a.y = t.dx;
    a.sides = weights;
    a.rows = (int32_t)w.K;
    a.block_rows = (int32_t)w.Kb;
    a.in_rows = (int32_t)w.M;
    a.N = t.N;
    ff::launch_product<T, 1, true>(a, blocks, wide, s);
}

#define XSPMM_FF_PRODUCT(T)                                               \
    template void feed_forward<T>(const ForwardArgs<T>&, int, hipStream_t); \
    template void transposed_product<T>(const TransposedArgs<T>&, int, hipStream_t);
XSPMM_FF_PRODUCT(float)
XSPMM_FF_PRODUCT(_Float16)
XSPMM_FF_PRODUCT(__bf16)
#undef XSPMM_FF_PRODUCT

}  // namespace detail
}  // namespace xspmm
