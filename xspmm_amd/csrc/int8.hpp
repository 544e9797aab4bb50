// int8.hpp -- the feed-forward layer's products in 8-bit integers: what the C
// entry points and the kernels share (not installed).
//
// A weight's whole numbers stand at its blocks as its values do (256 of a block,
// row by row), tokens' as features by sixteen: ceil(K / 16) x N x 16, so that 16
// consecutive bytes are what a block multiplies of one token.
#pragma once

#include "feed_forward.hpp"

namespace xspmm {
namespace detail {

// The sums of a row are 32-bit integers: 127 * 127 * K stays below 2^31.
constexpr int64_t kInt8MostFeatures = 133136;

// q = round(127 v / most) of every row's values (half to even), scale = most / 127
template <typename T>
void int8_weight(const BlockIndex& w, const T* vals, int8_t* q, float* scale, hipStream_t s);

// The same of every token's.  scratch: largest magnitudes of slices of the features.
int64_t quantize_tokens_scratch(int64_t K, int64_t N);
template <typename T>
void quantize_tokens(const T* x, int8_t* q, float* scale, int64_t K, int64_t N, void* scratch, hipStream_t s);

// y = act(A0 x + bias0) [* (A1 x + bias1)] [+ residual]
template <typename T>
struct Int8Args {
    const BlockIndex* weight[2];
    const int8_t* vals[2];
    const float* scale[2];  // of the rows
    const T* bias[2];
    const T* raw;  // activations that the product rounds itself, or null
    const int8_t* x;
    const float* x_scale;
    const T* residual;
    T* y;
    int64_t N;
    int act;
};
// Whether a product of N tokens rounds them itself, without memory for the result.
bool int8_rounds_itself(int64_t M, int64_t K, int64_t N);

// What the kernels take at a time: few tokens' workgroups 16 tokens and 1024 pieces of 16
// features; lists and tiles some block-rows (of both weights), tokens and block-columns.
constexpr int kInt8FewTokens = 16, kInt8FewPieces = 1024;
constexpr int kInt8ListRows = 32, kInt8ListTokens = 64, kInt8ListColumns = 32;
constexpr int kInt8TileRows = 16, kInt8TileTokens = 128, kInt8TileColumns = 4;

// Which kernel a product takes, by its sizes alone.
enum class Int8Kernel {
    kFew,    // tokens rounded within: `a` block-rows a workgroup, `b` pieces of a token a thread
    kWalk,   // `a` tiles of 16 tokens a wave, `b` waves to a block-row
    kLists,  // the first `a` fours of blocks of a row are fetched ahead
    kTiles
};
struct Int8Choice {
    Int8Kernel kernel;
    int a, b;
};
// M x K, blocks of each weight, N tokens, bytes of a result; whether the product rounds them
Int8Choice int8_choice(int weights, int64_t M, int64_t K, const int64_t* blocks, int64_t N, int size, bool rounds);
template <typename T>
void int8_product(const Int8Args<T>& a, int weights, hipStream_t s);

}  // namespace detail
}  // namespace xspmm
