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

template <typename T, int VEC, bool TR, bool WIDE>
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
            for (int c = 0; c < VEC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[c] = mfma32(st.a[i], st.b[i].d[c], acc[c]);
        } else {
            const u32x4_t a = {st.a[0], st.a[1], st.a[2], st.a[3]};
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

    // acc += blocks [b, end) times x: the loads of a step run ahead of the
    // instructions of the step before
    __device__ __forceinline__ void run(float4_t (&acc)[VEC], int32_t b, int32_t end) const
    {
        if (b >= end) return;
        const int32_t last = end - 1 - (kPer == 2 ? (end - 1 - b) % 2 : 0);
        Step<T, VEC> s0, s1;
        load(s0, b, end);
        for (; b < end; b += 2 * kPer) {
            load(s1, b + kPer < last ? b + kPer : last, end);
            multiply(acc, s0);
            if (b + kPer >= end) break;
            load(s0, b + 2 * kPer < last ? b + 2 * kPer : last, end);
            multiply(acc, s1);
        }
    }
};

// NACC accumulators: 2 for the gated forward product.  SPLIT waves share a
// block-row's blocks and add up in LDS, in their order.
template <typename T, int VEC, int NACC, bool TR, int SPLIT, bool WIDE>
__global__ __launch_bounds__(64 * kWaves) void ff_product_kernel(const ProductArgs<T> a)
{
    constexpr int kRowsPerGroup = kWaves / SPLIT;
    constexpr int kTile = 16 * VEC;
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
    const int64_t n = n0 + VEC * (lane & 15);

    float4_t acc[NACC][VEC];
#pragma unroll
    for (int l = 0; l < NACC; ++l)
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[l][c] = float4_t{0.f, 0.f, 0.f, 0.f};
    if (br < a.block_rows) {
        auto side = [&](int l, float4_t(&to)[VEC]) {
            const Walk<T, VEC, TR, WIDE> w(a, l, n, lane);
            const int32_t b = a.side[l].ptr[br], e = a.side[l].ptr[br + 1];
            constexpr int per = Walk<T, VEC, TR, WIDE>::kPer;
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
    if constexpr (SPLIT > 1) {
        __shared__ float4_t red[kRowsPerGroup][SPLIT - 1][NACC][VEC][64];
        if (part > 0) {
#pragma unroll
            for (int l = 0; l < NACC; ++l)
#pragma unroll
                for (int c = 0; c < VEC; ++c) red[wave / SPLIT][part - 1][l][c][lane] = acc[l][c];
        }
        __syncthreads();
        if (part > 0) return;
        for (int p = 0; p < SPLIT - 1; ++p)
#pragma unroll
            for (int l = 0; l < NACC; ++l)
#pragma unroll
                for (int c = 0; c < VEC; ++c) acc[l][c] += red[wave / SPLIT][p][l][c][lane];
    }
    if (br >= a.block_rows) return;

    // lane l: rows 4 (l / 16) + q of the block-row, its VEC tokens
    const bool whole = n >= first && n + VEC <= a.N;
    const bool any = n + VEC > first && n < a.N;
    if (!any) return;
    auto store = [&](T* p, const float(&v)[VEC], int64_t row) {
        if (whole) {
            Pack<T, VEC> o;
#pragma unroll
            for (int c = 0; c < VEC; ++c) o.v[c] = (T)v[c];
            *reinterpret_cast<Pack<T, VEC>*>(p + row * a.N + n) = o;
        } else {
#pragma unroll
            for (int c = 0; c < VEC; ++c)
                if (n + c >= first && n + c < a.N) p[row * a.N + n + c] = (T)v[c];
        }
    };
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t row = 16 * (int64_t)br + 4 * (lane >> 4) + q;
        if (row >= a.rows) continue;
        float z[NACC][VEC];
#pragma unroll
        for (int l = 0; l < NACC; ++l) {
            const float bias = !TR && a.side[l].bias ? (float)a.side[l].bias[row] : 0.f;
#pragma unroll
            for (int c = 0; c < VEC; ++c) z[l][c] = TR ? acc[l][c][q] : acc[l][c][q] + bias;
            if (!TR && a.side[l].keep) store(a.side[l].keep, z[l], row);
        }
        if constexpr (!TR) {
            with_act(a.act, [&](auto act) {
#pragma unroll
                for (int c = 0; c < VEC; ++c) z[0][c] = act_value<decltype(act)::value>(z[0][c]);
            });
            if constexpr (NACC == 2)
#pragma unroll
                for (int c = 0; c < VEC; ++c) z[0][c] *= z[1][c];
            if (a.residual) {
                if (whole) {
                    const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(a.residual + row * a.N + n);
#pragma unroll
                    for (int c = 0; c < VEC; ++c) z[0][c] += (float)r.v[c];
                } else {
#pragma unroll
                    for (int c = 0; c < VEC; ++c)
                        if (n + c >= first && n + c < a.N) z[0][c] += (float)a.residual[row * a.N + n + c];
                }
            }
        }
        store(a.y, z[0], row);
    }
}

template <typename T, int VEC, int NACC, bool TR, int SPLIT, bool WIDE>
void launch(const ProductArgs<T>& a, hipStream_t s)
{
    constexpr int rows = kWaves / SPLIT;
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + 16 * VEC - 1) / (16 * VEC));
    const int64_t grid = kXcds * xcd_chunk(items);
    if (grid > 0x7fffffffLL) throw std::invalid_argument("xSpMM: too many tokens for one launch.");
    hipLaunchKernelGGL((ff_product_kernel<T, VEC, NACC, TR, SPLIT, WIDE>), dim3((unsigned)grid), dim3(64 * kWaves), 0,
                       s, a);
    XSPMM_LAUNCH_CHECK();
}

template <typename T, int VEC, int NACC, bool TR, bool WIDE>
void launch_split(const ProductArgs<T>& a, int split, hipStream_t s)
{
    if (split == 4)
        launch<T, VEC, NACC, TR, 4, WIDE>(a, s);
    else
        launch<T, VEC, NACC, TR, 1, WIDE>(a, s);
}

template <typename T, int NACC, bool TR>
void launch_product(const ProductArgs<T>& a, int64_t blocks, bool wide, hipStream_t s)
{
    if (a.block_rows == 0 || a.N == 0) return;
    constexpr int most = is_f32<T> ? 4 : 8;
    int vec = most;
    while (vec > 1 && 16 * vec > a.N) vec /= 2;
    auto waves = [&](int v) { return (int64_t)a.block_rows * ((a.N + 16 * v - 1) / (16 * v)); };
    while (vec > 4 && waves(vec) < 2048) vec /= 2;
    const int split = waves(vec) < 2048 && blocks >= 8 * a.block_rows ? 4 : 1;
    if (wide) {
        if (vec == 1)
            launch_split<T, 1, NACC, TR, true>(a, split, s);
        else if (a.N >= 64)
            launch_split<T, 4, NACC, TR, true>(a, split, s);
        else
            launch_split<T, 2, NACC, TR, true>(a, split, s);
        return;
    }
    switch (vec) {
    case 8:
        if constexpr (!is_f32<T>) launch_split<T, 8, NACC, TR, false>(a, split, s);
        break;
    case 4: launch_split<T, 4, NACC, TR, false>(a, split, s); break;
    case 2: launch_split<T, 2, NACC, TR, false>(a, split, s); break;
    default: launch_split<T, 1, NACC, TR, false>(a, split, s); break;
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
