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
#include "feed_forward_device.hpp"
#include "int8.hpp"

namespace xspmm {
namespace detail {
namespace ff {

typedef int int4_t __attribute__((ext_vector_type(4)));

struct Int8Side {
    const int32_t* ptr;
    const int32_t* col;
    const int8_t* vals;
    const float* scale;
    const void* bias;
};

template <typename T>
struct Int8Product {
    Int8Side side[2];
    const int8_t* x;
    const float* x_scale;
    const T* residual;
    T* y;
    int32_t rows, block_rows;
    int64_t N;
    int act;
};

template <typename T, int NACC>
__device__ __forceinline__ float int8_finish(const Int8Product<T>& a, const int (&sum)[NACC], int64_t row, int64_t n,
                                             float x_scale)
{
    float z[NACC];
#pragma unroll
    for (int l = 0; l < NACC; ++l) {
        z[l] = (float)sum[l] * a.side[l].scale[row] * x_scale;
        if (a.side[l].bias) z[l] += (float)static_cast<const T*>(a.side[l].bias)[row];
    }
    with_act(a.act, [&](auto act) { z[0] = act_value<decltype(act)::value>(z[0]); });
    if constexpr (NACC == 2) z[0] *= z[1];
    if (a.residual) z[0] += (float)a.residual[row * a.N + n];
    return z[0];
}

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
    const int64_t groups = (a.block_rows + kRowsPerGroup - 1) / kRowsPerGroup;
    const int64_t tiles = (a.N + 16 * VT - 1) / (16 * VT);
    const int64_t item = xcd_item(blockIdx.x, groups * tiles);
    if (item < 0) return;
    const int32_t br = (int32_t)(item % groups) * kRowsPerGroup + wave / SPLIT;
    const int part = wave % SPLIT;
    const int64_t n0 = item / groups * (16 * VT);
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
            const int32_t lo = b + 4 * (int32_t)((int64_t)steps * part / SPLIT);
            const int32_t hi = min(b + 4 * (int32_t)((int64_t)steps * (part + 1) / SPLIT), e);
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
                    acc[l][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4_t, st.a),
                                                                      __builtin_bit_cast(int4_t, st.x[j]), acc[l][j],
                                                                      0, 0, 0);
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

template <typename T, int VT, int NACC, int SPLIT>
void launch_walk(const Int8Product<T>& a, hipStream_t s)
{
    constexpr int rows = SPLIT > 4 ? 1 : 4 / SPLIT, threads = 64 * (SPLIT > 4 ? SPLIT : 4);
    const int64_t items = (int64_t)((a.block_rows + rows - 1) / rows) * ((a.N + 16 * VT - 1) / (16 * VT));
    hipLaunchKernelGGL((ff_int8_walk_kernel<T, VT, NACC, SPLIT>), launch_grid(kXcds * xcd_chunk(items), threads),
                       dim3(threads), 0, s, a);
    XSPMM_LAUNCH_CHECK();
}

template <typename T, int NACC>
void launch_int8(const Int8Product<T>& a, int64_t blocks, hipStream_t s)
{
    auto waves = [&](int v) { return (int64_t)a.block_rows * ((a.N + 16 * v - 1) / (16 * v)); };
    int vt = 4;
    while (vt > 1 && (16 * vt >= 2 * a.N || waves(vt) < 256)) vt /= 2;
    const int64_t each = blocks / a.block_rows;
    if (vt == 4) {
        if (waves(4) < 4096 && each >= 16)
            launch_walk<T, 4, NACC, 4>(a, s);
        else
            launch_walk<T, 4, NACC, 1>(a, s);
    } else if (waves(1) <= 512 && each >= 64) {
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
    int64_t blocks = 0;
    for (int l = 0; l < weights; ++l) {
        const BlockIndex& wl = *f.weight[l];
        a.side[l] = {wl.ptr, wl.col, f.vals[l], f.scale[l], f.bias[l]};
        blocks += wl.nnzb;
    }
    a.x = f.x;
    a.x_scale = f.x_scale;
    a.residual = f.residual;
    a.y = f.y;
    a.rows = (int32_t)w.M;
    a.block_rows = (int32_t)w.Mb;
    a.N = f.N;
    a.act = f.act;
    if (weights == 2)
        ff::launch_int8<T, 2>(a, blocks, s);
    else
        ff::launch_int8<T, 1>(a, blocks, s);
}

#define XSPMM_INT8_PRODUCT(T) template void int8_product<T>(const Int8Args<T>&, int, hipStream_t);
XSPMM_INT8_PRODUCT(float)
XSPMM_INT8_PRODUCT(_Float16)
XSPMM_INT8_PRODUCT(__bf16)
#undef XSPMM_INT8_PRODUCT

}  // namespace detail
}  // namespace xspmm
