// ff_weight.hip -- the block index of a weight: the BCSR arrays in 32 bits, the
// block-row of every block, and the blocks in block-column order.
//
// Once per weight, so built for determinism rather than speed: the columns of a
// block-row ascend, so whether block-row i holds block-column j is one binary
// search.  One wave per block-column asks all block-rows, 64 at a time, first
// to count and, after a scan of the counts, to list them in ascending order.
#include "feed_forward.hpp"
#include "scan.hpp"

namespace xspmm {
namespace detail {

namespace {

// bit 0: the pointers are not those of nnzb blocks; bit 1: a column is outside
// the matrix or not above its left neighbour
constexpr int kBadPtr = 1, kBadCol = 2;

template <typename I>
__global__ __launch_bounds__(256) void ff_check_ptr_kernel(const I* __restrict__ brp, int64_t Mb, int64_t nnzb,
                                                           int32_t* __restrict__ ptr, int* bad)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i > Mb) return;
    const int64_t p = (int64_t)brp[i];
    bool ok = p >= 0 && p <= nnzb;
    if (i == 0) ok &= p == 0;
    if (i == Mb) ok &= p == nnzb;
    if (i < Mb) ok &= (int64_t)brp[i + 1] >= p;
    if (!ok) atomicOr(bad, kBadPtr);
    ptr[i] = ok ? (int32_t)p : 0;
}

// one wave per block-row
template <typename I>
__global__ __launch_bounds__(256) void ff_check_col_kernel(const int32_t* __restrict__ ptr, const I* __restrict__ bci,
                                                           int64_t Mb, int64_t Kb, const int* bad_in,
                                                           int32_t* __restrict__ col, int32_t* __restrict__ row,
                                                           int32_t* __restrict__ map, int* bad)
{
    if (*bad_in & kBadPtr) return;
    const int64_t br = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (br >= Mb) return;
    const int32_t b0 = ptr[br], b1 = ptr[br + 1];
    for (int32_t b = b0 + (int32_t)(threadIdx.x & 63); b < b1; b += 64) {
        const int64_t c = (int64_t)bci[b];
        const bool ok = c >= 0 && c < Kb && (b == b0 || (int64_t)bci[b - 1] < c);
        if (!ok) atomicOr(bad, kBadCol);
        col[b] = ok ? (int32_t)c : 0;
        row[b] = (int32_t)br;
        if (map && ok) map[br * Kb + c] = b;
    }
}

// position of column j in block-row i, or -1
__device__ __forceinline__ int32_t find(const int32_t* ptr, const int32_t* col, int64_t i, int32_t j)
{
    int32_t lo = ptr[i], hi = ptr[i + 1];
    const int32_t end = hi;
    while (lo < hi) {
        const int32_t mid = lo + (hi - lo) / 2;
        if (col[mid] < j)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo < end && col[lo] == j ? lo : -1;
}

// one wave per block-column
template <bool FILL>
__global__ __launch_bounds__(256) void ff_transpose_kernel(const int32_t* __restrict__ ptr,
                                                           const int32_t* __restrict__ col, int64_t Mb, int64_t Kb,
                                                           const int* __restrict__ bad, int32_t* __restrict__ counts,
                                                           const int32_t* __restrict__ tptr,
                                                           int32_t* __restrict__ trow, int32_t* __restrict__ tblk)
{
    const int lane = threadIdx.x & 63;
    const int64_t j = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (j >= Kb) return;
    if (*bad) {  // nothing to list: the host reports it
        if (!FILL && lane == 0) counts[j] = 0;
        return;
    }
    int32_t at = FILL ? tptr[j] : 0;
    for (int64_t i0 = 0; i0 < Mb; i0 += 64) {
        const int64_t i = i0 + lane;
        const int32_t b = i < Mb ? find(ptr, col, i, (int32_t)j) : -1;
        const uint64_t there = __ballot(b >= 0);
        if (FILL && b >= 0) {
            const int32_t o = at + __popcll(there & ((1ull << lane) - 1));
            trow[o] = (int32_t)i;
            tblk[o] = b;
        }
        at += __popcll(there);
    }
    if (!FILL && lane == 0) counts[j] = at;
}

__global__ __launch_bounds__(256) void ff_group_count_kernel(const int32_t* __restrict__ ptr, int64_t Mb,
                                                             int32_t* __restrict__ counts)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    // pointers that do not ascend count for nothing: the host reports them
    if (i < Mb) counts[i] = max(ptr[i + 1] - ptr[i] + kGroupBlocks - 1, 0) / kGroupBlocks;
}

__global__ __launch_bounds__(256) void ff_group_kernel(const int32_t* __restrict__ ptr, const int32_t* __restrict__ gptr,
                                                       const int* __restrict__ bad, int64_t Mb,
                                                       int32_t* __restrict__ group)
{
    const int64_t br = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (*bad || br >= Mb) return;
    const int32_t g0 = gptr[br], g1 = gptr[br + 1], b0 = ptr[br];
    for (int32_t g = g0 + (int32_t)(threadIdx.x & 63); g < g1; g += 64) group[g] = b0 + (g - g0) * kGroupBlocks;
}

// exclusive prefix sum of n counts in place, n + 1 results; one workgroup
__global__ __launch_bounds__(kScanThreads) void ff_scan_kernel(int32_t* __restrict__ v, int64_t n)
{
    __shared__ int64_t red[kScanThreads / 64];
    int64_t carry = 0;
    for (int64_t i0 = 0; i0 <= n; i0 += kScanThreads) {
        const int64_t i = i0 + threadIdx.x;
        const int64_t x = i < n ? v[i] : 0;
        int64_t total;
        const int64_t before = block_exclusive_scan(x, &total, red);
        if (i <= n) v[i] = (int32_t)(carry + before);
        carry += total;
    }
}

__global__ __launch_bounds__(256) void ff_fill_kernel(int32_t* __restrict__ p, int64_t n, int32_t v)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = v;
}

}  // namespace

// The tile kernels' map costs 4 bytes for every block of the grid, stored or
// not: worth it up to 64 MB where at least one block in 64 is stored.
bool has_block_map(int64_t Mb, int64_t Kb, int64_t nnzb)
{
    return Mb * Kb <= (1 << 24) && nnzb * 64 >= Mb * Kb && nnzb > 0;
}

template <typename I>
void build_block_index(BlockIndex& out, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnzb, const I* brp,
                       const I* bci, hipStream_t s)
{
    auto require = [](bool ok, const char* what) {
        if (!ok) throw std::invalid_argument(what);
    };
    require(M >= 0 && K >= 0 && nnzb >= 0, "xSpMM: weight dimensions must be non-negative.");
    // a wave per block-row, and per block-column, of one launch
    require(M <= (1LL << 30) - 64 && K <= (1LL << 30) - 64, "xSpMM: a weight has at most 2^30 - 64 rows and columns.");
    require(Mb == (M + 15) / 16 && Kb == (K + 15) / 16, "xSpMM: a weight's block grid must cover it with 16x16 blocks.");
    require(nnzb < 0x7fffffffLL, "xSpMM: a weight has at most 2^31 - 2 blocks.");
    require(brp != nullptr && (nnzb == 0 || bci != nullptr), "xSpMM: null weight array.");
    out.M = M;
    out.K = K;
    out.Mb = Mb;
    out.Kb = Kb;
    out.nnzb = nnzb;
    Carve c;
    const size_t o_ptr = c.take((size_t)(Mb + 1) * 4), o_tptr = c.take((size_t)(Kb + 1) * 4);
    const size_t o_col = c.take((size_t)nnzb * 4), o_row = c.take((size_t)nnzb * 4);
    const size_t o_trow = c.take((size_t)nnzb * 4), o_tblk = c.take((size_t)nnzb * 4);
    const size_t o_bad = c.take(4);
    const size_t o_gptr = c.take((size_t)(Mb + 1) * 4);
    const size_t o_group = c.take((size_t)(nnzb / kGroupBlocks + (Mb < nnzb ? Mb : nnzb)) * 4);
    const bool map = has_block_map(Mb, Kb, nnzb);
    const size_t o_map = c.take(map ? (size_t)(Mb * Kb) * 4 : 0);
    XSPMM_HIP_CHECK(hipMalloc(&out.memory, c.end));
    char* p = static_cast<char*>(out.memory);
    out.ptr = reinterpret_cast<int32_t*>(p + o_ptr);
    out.tptr = reinterpret_cast<int32_t*>(p + o_tptr);
    out.col = reinterpret_cast<int32_t*>(p + o_col);
    out.row = reinterpret_cast<int32_t*>(p + o_row);
    out.trow = reinterpret_cast<int32_t*>(p + o_trow);
    out.tblk = reinterpret_cast<int32_t*>(p + o_tblk);
    if (map) out.map = reinterpret_cast<int32_t*>(p + o_map);
    out.group = reinterpret_cast<int32_t*>(p + o_group);
    int32_t* gptr = reinterpret_cast<int32_t*>(p + o_gptr);
    int* bad = reinterpret_cast<int*>(p + o_bad);

    auto groups = [](int64_t n, int64_t per) { return dim3((unsigned)((n + per - 1) / per)); };
    hipLaunchKernelGGL(ff_fill_kernel, dim3(1), dim3(256), 0, s, bad, (int64_t)1, 0);
    if (map)
        hipLaunchKernelGGL(ff_fill_kernel, dim3(1024), dim3(256), 0, s, out.map, Mb * Kb, -1);
    hipLaunchKernelGGL((ff_check_ptr_kernel<I>), groups(Mb + 1, 256), dim3(256), 0, s, brp, Mb, nnzb, out.ptr, bad);
    if (Mb > 0)
        hipLaunchKernelGGL((ff_check_col_kernel<I>), groups(Mb, 4), dim3(256), 0, s, out.ptr, bci, Mb, Kb, bad,
                           out.col, out.row, out.map, bad);
    if (Kb > 0)
        hipLaunchKernelGGL((ff_transpose_kernel<false>), groups(Kb, 4), dim3(256), 0, s, out.ptr, out.col, Mb, Kb,
                           bad, out.tptr, nullptr, nullptr, nullptr);
    hipLaunchKernelGGL(ff_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, out.tptr, Kb);
    if (Kb > 0 && nnzb > 0)
        hipLaunchKernelGGL((ff_transpose_kernel<true>), groups(Kb, 4), dim3(256), 0, s, out.ptr, out.col, Mb, Kb, bad,
                           nullptr, out.tptr, out.trow, out.tblk);
    if (Mb > 0)
        hipLaunchKernelGGL(ff_group_count_kernel, groups(Mb, 256), dim3(256), 0, s, out.ptr, Mb, gptr);
    hipLaunchKernelGGL(ff_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, gptr, Mb);
    if (Mb > 0 && nnzb > 0)
        hipLaunchKernelGGL(ff_group_kernel, groups(Mb, 4), dim3(256), 0, s, out.ptr, gptr, bad, Mb, out.group);
    XSPMM_LAUNCH_CHECK();
    int found = 0;
    int32_t made = 0;
    XSPMM_HIP_CHECK(hipMemcpyAsync(&found, bad, 4, hipMemcpyDeviceToHost, s));
    XSPMM_HIP_CHECK(hipMemcpyAsync(&made, gptr + Mb, 4, hipMemcpyDeviceToHost, s));
    XSPMM_HIP_CHECK(hipStreamSynchronize(s));
    out.groups = made;
    require(!(found & kBadPtr), "xSpMM: a weight's row pointers must ascend from 0 to the number of blocks.");
    require(!(found & kBadCol), "xSpMM: a weight's block columns must lie in the grid and ascend within a row.");
}

template void build_block_index<int32_t>(BlockIndex&, int64_t, int64_t, int64_t, int64_t, int64_t, const int32_t*,
                                         const int32_t*, hipStream_t);
template void build_block_index<int64_t>(BlockIndex&, int64_t, int64_t, int64_t, int64_t, int64_t, const int64_t*,
                                         const int64_t*, hipStream_t);

}  // namespace detail
}  // namespace xspmm
