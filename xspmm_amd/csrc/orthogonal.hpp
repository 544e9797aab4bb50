// orthogonal.hpp -- orthogonalised updates of a block-sparse weight: what the C
// entry point and the kernels share (not installed).
#pragma once

#include "feed_forward.hpp"

namespace xspmm {
namespace detail {

struct OrthogonalArgs {
    float a, b, c;  // of X <- a X + (b S + c S S) X
    float eps;
    int steps;
};

// Sides of a weight whose update may be orthogonalised.
constexpr int64_t kOrthogonalMostSide = int64_t(1) << 20;

template <typename T>
int64_t orthogonal_scratch(const BlockIndex& w);
template <typename T>
void orthogonalize(const BlockIndex& w, const T* update, T* out, const OrthogonalArgs& o, void* scratch, hipStream_t s);

}  // namespace detail
}  // namespace xspmm
