// feed_forward.hpp -- the feed-forward layer on block-sparse weights: what the
// C entry points and the kernels share (not installed).
//
// Activations are features x tokens, row-major, as the B and C of the SpMM.
// Weights are BCSR matrices of 16x16 blocks.
#pragma once

#include <cstdint>

#include "internal.hpp"

namespace xspmm {
namespace detail {

// Where the blocks of a weight stand, laid out once per weight: by block-row
// (as in the BCSR matrix) and by block-column, for the products with A^T.
// Indices are 32-bit: nnzb < 2^31 is checked when it is made.
struct BlockIndex {
    int64_t M = 0, K = 0, Mb = 0, Kb = 0, nnzb = 0;
    // device
    int32_t* ptr = nullptr;   // [Mb + 1]
    int32_t* col = nullptr;   // [nnzb]
    int32_t* row = nullptr;   // [nnzb] block-row of each block
    int64_t groups = 0;
    int32_t* group = nullptr; // [groups] first blocks of runs of up to 4 within a block-row
    int32_t* tptr = nullptr;  // [Kb + 1]
    int32_t* trow = nullptr;  // [nnzb] block-rows by block-column, ascending
    int32_t* tblk = nullptr;  // [nnzb] and their positions in the BCSR order
    int32_t* map = nullptr;   // [Mb * Kb] position of each block, or -1; null on large grids of few blocks
    void* memory = nullptr;   // the one allocation behind them

    BlockIndex() = default;
    BlockIndex(const BlockIndex&) = delete;
    BlockIndex& operator=(const BlockIndex&) = delete;
    ~BlockIndex() {
        if (memory) (void)hipFree(memory);
    }
};

constexpr int kGroupBlocks = 4;

// Fills `out` from BCSR arrays on the device; synchronizes `s`.  Throws
// std::invalid_argument where they are no BCSR matrix with strictly ascending
// columns.
template <typename I>
void build_block_index(BlockIndex& out, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnzb, const I* brp,
                       const I* bci, hipStream_t s);

enum Activation { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

// y = act(A0 x + bias0) [* (A1 x + bias1)] [+ residual], keep_i = A_i x + bias_i
template <typename T>
struct ForwardArgs {
    const BlockIndex* weight[2];
    const T* vals[2];
    const T* bias[2];
    const T* x;
    const T* residual;
    T* y;
    T* keep[2];
    int64_t N;
    int act;
};
template <typename T>
void feed_forward(const ForwardArgs<T>& a, int weights, hipStream_t s);

// dx = sum_i A_i^T dz_i
template <typename T>
struct TransposedArgs {
    const BlockIndex* weight[2];
    const T* vals[2];
    const T* dz[2];
    T* dx;
    int64_t N;
};
template <typename T>
void transposed_product(const TransposedArgs<T>& a, int weights, hipStream_t s);

// The same by tiles, for 16-bit values: false where that does not apply or pay.
template <typename T>
bool feed_forward_tiles(const ForwardArgs<T>& a, int weights, hipStream_t s);
template <typename T>
bool transposed_tiles(const TransposedArgs<T>& a, int weights, hipStream_t s);

// dvals_i = (dz_i x^T) at the stored blocks, zero past the edges of A_i; a null
// dvals is not wanted
template <typename T>
struct SampledArgs {
    const BlockIndex* weight[2];
    const T* dz[2];
    const T* x;
    T* dvals[2];
    int64_t N;
};
template <typename T>
void sampled_product(const SampledArgs<T>& a, int weights, hipStream_t s);

// A launch holds less than 2^32 threads along its first dimension.
inline dim3 launch_grid(int64_t groups, int threads, unsigned sides = 1)
{
    if (groups > 0xffffffffLL / threads)
        throw std::invalid_argument("xSpMM: too many tokens or blocks for one launch.");
    return dim3((unsigned)groups, sides);
}

// Whether a weight has a map of its grid of blocks.
bool has_block_map(int64_t Mb, int64_t Kb, int64_t nnzb);

// Bytes of `rows` rows of N elements where those of whole blocks of rows stay
// below 2^31, else -1.
inline int64_t narrow_bytes(int64_t rows, int64_t N, int64_t size)
{
    const __int128 b = (__int128)((rows + 15) / 16 * 16) * N * size;
    return b < ((int64_t)1 << 31) ? rows * N * size : -1;
}

// linear (up null): dz = dy act'(z);  gated: dz = dy up act'(z), dup = dy act(z).
// dz / dup may be null (sums only).  bias sums over the tokens where not null.
template <typename T>
void activation_backward(const T* z, const T* up, const T* dy, T* dz, T* dup, T* dbias, T* dbias_up, int act,
                         int64_t M, int64_t N, hipStream_t s);

// size: bytes of a value
int64_t layer_norm_scratch(int64_t K, int64_t N, int64_t size, int backward);
template <typename T>
void layer_norm(const T* x, const T* weight, const T* bias, float eps, T* y, float* mean, float* rstd, int64_t K,
                int64_t N, void* scratch, hipStream_t s);
template <typename T>
void layer_norm_backward(const T* dy, const T* x, const T* weight, const float* mean, const float* rstd, T* dx,
                         T* dweight, T* dbias, int64_t K, int64_t N, void* scratch, hipStream_t s);

}  // namespace detail
}  // namespace xspmm
