// capi.cpp -- extern "C" entry points declared in include/xspmm_capi.h.
// Each maps type codes onto the internal launchers and turns exceptions into
// error codes (std::invalid_argument -> XSPMM_ERR_INVALID, "HIP Error" ->
// XSPMM_ERR_HIP, any other failure -> XSPMM_ERR_UNSUPPORTED).
#include <hip/hip_fp16.h>

#include <cstring>
#include <memory>
#include <string>
#include <utility>

#include "feed_forward.hpp"
#include "internal.hpp"
#include "xspmm_capi.h"

using namespace xspmm::detail;

// The opaque handles of the C ABI.
struct xspmm_plan_s {
    PlanBase* impl;
};
struct xspmm_mtx_s {
    MtxData data;
};
struct xspmm_weight_s {
    BlockIndex index;
};

namespace {

thread_local std::string g_last_error;

template <typename F>
int guarded(F&& f)
{
    try {
        f();
        g_last_error.clear();
        return XSPMM_OK;
    } catch (const std::invalid_argument& e) {
        g_last_error = e.what();
        return XSPMM_ERR_INVALID;
    } catch (const MtxError& e) {
        g_last_error = e.what();
        return XSPMM_ERR_IO;
    } catch (const std::exception& e) {
        g_last_error = e.what();
        return std::strncmp(e.what(), "HIP Error", 9) == 0 ? XSPMM_ERR_HIP : XSPMM_ERR_UNSUPPORTED;
    } catch (...) {
        g_last_error = "unknown error";
        return XSPMM_ERR_UNSUPPORTED;
    }
}

template <typename T>
struct Tag { using type = T; };

// Calls f(Tag<value>, Tag<index>) for the requested type codes.
template <typename F>
void with_types(int vtype, int itype, F&& f)
{
    if (itype != XSPMM_I32 && itype != XSPMM_I64) throw std::invalid_argument("unknown index type code");
    if (vtype != XSPMM_F32 && vtype != XSPMM_F16) throw std::invalid_argument("unknown value type code");
    if (vtype == XSPMM_F16) {
        if (itype == XSPMM_I32) f(Tag<uint16_t>{}, Tag<int32_t>{});
        else f(Tag<uint16_t>{}, Tag<int64_t>{});
    } else {
        if (itype == XSPMM_I32) f(Tag<float>{}, Tag<int32_t>{});
        else f(Tag<float>{}, Tag<int64_t>{});
    }
}

template <typename F>
void with_index(int itype, F&& f)
{
    if (itype == XSPMM_I32) f(Tag<int32_t>{});
    else if (itype == XSPMM_I64) f(Tag<int64_t>{});
    else throw std::invalid_argument("unknown index type code");
}

// Calls f(Tag<value>) for the value types of the feed-forward layer.
template <typename F>
void with_layer_type(int vtype, F&& f)
{
    if (vtype == XSPMM_F32) f(Tag<float>{});
    else if (vtype == XSPMM_F16) f(Tag<_Float16>{});
    else if (vtype == XSPMM_BF16) f(Tag<__bf16>{});
    else throw std::invalid_argument("unknown value type code");
}

hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

void require(bool ok, const char* what)
{
    if (!ok) throw std::invalid_argument(what);
}

// A dense operand of the feed-forward layer: there unless it is empty, and on
// a 16-byte boundary.
template <typename T>
const T* operand(const void* p, bool needed, const char* what)
{
    if (p == nullptr && needed) throw std::invalid_argument(std::string("xSpMM: ") + what + " is null.");
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
        throw std::invalid_argument(std::string("xSpMM: ") + what + " must start on a 16-byte boundary.");
    return static_cast<const T*>(p);
}

template <typename T>
T* result(void* p, bool needed, const char* what)
{
    return const_cast<T*>(operand<T>(p, needed, what));
}

void require_layer(int act, int64_t N)
{
    require(act >= XSPMM_ACT_NONE && act <= XSPMM_ACT_GELU_TANH, "unknown activation code");
    require(N >= 0, "xSpMM: negative N.");
    // a weight has less than 2^30 rows: two fp32 arrays of a pass stay below 2^63 bytes
    require(N <= (int64_t(1) << 30), "xSpMM: at most 2^30 tokens.");
}

// 256-byte aligned bytes of one M x N array of a backward pass
int64_t layer_array(int vtype, int64_t M, int64_t N)
{
    const int64_t size = vtype == XSPMM_F32 ? 4 : 2;
    return (M * N * size + 255) / 256 * 256;
}

void require_scratch(const void* p, int64_t have, int64_t need)
{
    require(have >= need && (need == 0 || p != nullptr), "xSpMM: the scratch is smaller than its query says.");
    require(reinterpret_cast<uintptr_t>(p) % 256 == 0 || need == 0, "xSpMM: scratch must start on a 256-byte boundary.");
}

}  // namespace

extern "C" {

const char* xspmm_last_error(void) { return g_last_error.c_str(); }

int xspmm_abi_version(void) { return 4; }

int xspmm_bcsr_spmm(int vtype, int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb,
                    int64_t nnzb, const void* brp, const void* bci, const void* bvals,
                    const void* B, float* C, int64_t N, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            bcsr_spmm<T, I>(M, K, Mb, Kb, nnzb, static_cast<const I*>(brp), static_cast<const I*>(bci),
                            static_cast<const T*>(bvals), static_cast<const T*>(B), C, N,
                            as_stream(stream), kNoAllocScratchBytes);
        });
    });
}

int xspmm_bcsr_spmm_noalloc(int vtype, int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb,
                            int64_t nnzb, const void* brp, const void* bci, const void* bvals,
                            const void* B, float* C, int64_t N, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            bcsr_spmm_noalloc<T, I>(M, K, Mb, Kb, nnzb, static_cast<const I*>(brp),
                                    static_cast<const I*>(bci), static_cast<const T*>(bvals),
                                    static_cast<const T*>(B), C, N, as_stream(stream));
        });
    });
}

int64_t xspmm_noalloc_scratch_bytes(void) { return (int64_t)kNoAllocScratchBytes; }

int xspmm_bcsr_dispatch_order(int itype, int64_t Mb, const void* brp, int32_t* order,
                              int* written, void* stream)
{
    return guarded([&] {
        if (Mb < 0) throw std::invalid_argument("xSpMM: negative number of block-rows.");
        if (!written) throw std::invalid_argument("xSpMM: written must not be NULL.");
        *written = 0;
        if (!spmm_order_wanted(Mb)) return;
        if (!brp || !order) throw std::invalid_argument("xSpMM: brp and order must not be NULL.");
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            spmm_dispatch_order<I>(static_cast<const I*>(brp), Mb, order, as_stream(stream));
        });
        *written = 1;
    });
}

int xspmm_bcsr_dispatch_order_cols(int itype, int64_t Mb, const void* brp, const void* bci,
                                   int32_t* order, int* written, void* stream)
{
    return guarded([&] {
        if (Mb < 0) throw std::invalid_argument("xSpMM: negative number of block-rows.");
        if (!written) throw std::invalid_argument("xSpMM: written must not be NULL.");
        *written = 0;
        if (!spmm_order_cols_wanted(Mb)) return;
        if (!brp || !bci || !order)
            throw std::invalid_argument("xSpMM: brp, bci and order must not be NULL.");
        bool used = false;
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            used = spmm_dispatch_order_cols<I>(static_cast<const I*>(brp), static_cast<const I*>(bci), Mb,
                                               order, as_stream(stream));
        });
        *written = used ? 1 : 0;
    });
}

int xspmm_bcsr_spmm_ordered(int vtype, int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb,
                            int64_t nnzb, const void* brp, const void* bci, const void* bvals,
                            const void* B, float* C, int64_t N, const int32_t* order, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            (void)bcsr_spmm_ex<T, I>(M, K, Mb, Kb, nnzb, static_cast<const I*>(brp),
                                     static_cast<const I*>(bci), static_cast<const T*>(bvals),
                                     static_cast<const T*>(B), C, N, order, nullptr,
                                     as_stream(stream), kNoAllocScratchBytes);
        });
    });
}

int xspmm_bcsr_band_rows(int vtype, int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnz,
                         int64_t nnzb, const void* brp, const void* bci, int* band, void* stream)
{
    return guarded([&] {
        if (!band) throw std::invalid_argument("xSpMM: band must not be NULL.");
        *band = 0;
        if (vtype != XSPMM_F16 && vtype != XSPMM_F32) throw std::invalid_argument("xSpMM: unknown value type.");
        if (M < 0 || K < 0 || Mb < 0 || Kb < 0 || nnzb < 0)
            throw std::invalid_argument("xSpMM: negative size passed to BCSR SpMM.");
        if (Mb == 0 || nnzb == 0) return;
        if (!brp || !bci) throw std::invalid_argument("xSpMM: brp and bci must not be NULL.");
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            *band = spmm_band_wanted<I>(static_cast<const I*>(brp), static_cast<const I*>(bci), M, K, Mb, Kb,
                                        nnz, nnzb, 0, vtype == XSPMM_F16 ? 2 : 4, as_stream(stream))
                        ? 1
                        : 0;
        });
    });
}

int xspmm_bcsr_spmm_band(int vtype, int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnzb,
                         const void* brp, const void* bci, const void* bvals, const void* B, float* C,
                         int64_t N, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            bcsr_spmm_band<T, I>(M, K, Mb, Kb, nnzb, static_cast<const I*>(brp), static_cast<const I*>(bci),
                                 static_cast<const T*>(bvals), static_cast<const T*>(B), C, N, as_stream(stream));
        });
    });
}

int xspmm_bcsr_spmm_auto(int vtype, int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnzb,
                         const void* brp, const void* bci, const void* bvals, const void* B, float* C, int64_t N,
                         const int32_t* order, int band, void* scratch, int64_t scratch_bytes, void* stream)
{
    return guarded([&] {
        if (scratch_bytes < 0 || (reinterpret_cast<uintptr_t>(scratch) & 255) != 0)
            throw std::invalid_argument("xSpMM: scratch must be 256-byte aligned, its size not negative.");
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            bcsr_spmm_auto<T, I>(M, K, Mb, Kb, nnzb, static_cast<const I*>(brp), static_cast<const I*>(bci),
                                 static_cast<const T*>(bvals), static_cast<const T*>(B), C, N, order, band != 0,
                                 scratch, (size_t)scratch_bytes, as_stream(stream));
        });
    });
}

int xspmm_bcsr_spmm_scratch(int vtype, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnzb, const void* B,
                            const float* C, int64_t N, int ordered, int band, int64_t* bytes)
{
    return guarded([&] {
        require(bytes != nullptr, "bytes is null");
        if (vtype != XSPMM_F16 && vtype != XSPMM_F32) throw std::invalid_argument("xSpMM: unknown value type.");
        *bytes = (int64_t)bcsr_spmm_scratch(vtype == XSPMM_F16 ? 2 : 4, M, K, Mb, Kb, nnzb, B, C, N, ordered != 0,
                                            band != 0);
    });
}

int xspmm_csr_to_bcsr_count(int itype, int64_t M, int64_t K, int64_t nnz, const void* rp,
                            const void* ci, int64_t r_block, int64_t c_block,
                            void* bcsr_row_ptr, int64_t* nnzb_out, void* stream)
{
    return guarded([&] {
        require(nnzb_out != nullptr, "nnzb_out is null");
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            *nnzb_out = csr_to_bcsr_count<I>(M, K, nnz, static_cast<const I*>(rp),
                                             static_cast<const I*>(ci), r_block, c_block,
                                             static_cast<I*>(bcsr_row_ptr), as_stream(stream));
        });
    });
}

int xspmm_csr_to_bcsr_fill(int vtype, int itype, int64_t M, int64_t K, int64_t nnz,
                           const void* rp, const void* ci, const void* vals,
                           int64_t r_block, int64_t c_block, const void* bcsr_row_ptr,
                           void* bcsr_col_ind, void* bcsr_vals, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            csr_to_bcsr_fill<T, I>(M, K, nnz, static_cast<const I*>(rp), static_cast<const I*>(ci),
                                   static_cast<const T*>(vals), r_block, c_block,
                                   static_cast<const I*>(bcsr_row_ptr), static_cast<I*>(bcsr_col_ind),
                                   static_cast<T*>(bcsr_vals), as_stream(stream));
        });
    });
}

int xspmm_apply_permutation(int vtype, int itype, int64_t M, int64_t nnz, const void* rp,
                            const void* ci, const void* vals, const void* perm,
                            void* new_rp, void* new_ci, void* new_vals, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            apply_permutation<T, I>(M, nnz, static_cast<const I*>(rp), static_cast<const I*>(ci),
                                    static_cast<const T*>(vals), static_cast<const I*>(perm),
                                    static_cast<I*>(new_rp), static_cast<I*>(new_ci),
                                    static_cast<T*>(new_vals), as_stream(stream));
        });
    });
}

int xspmm_unpermute_dense(int itype, const float* in, float* out, const void* perm, int64_t M,
                          int64_t N, void* stream)
{
    return guarded([&] {
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            unpermute_dense<I>(in, out, static_cast<const I*>(perm), M, N, as_stream(stream));
        });
    });
}

int xspmm_jaccard_clustering_host(int itype, int64_t M, int64_t K, const void* rp,
                                  const void* ci, float dist_thresh, int64_t block_width,
                                  void* perm_out, int nthreads)
{
    return guarded([&] {
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            jaccard_clustering_host<I>(M, K, static_cast<const I*>(rp), static_cast<const I*>(ci),
                                       dist_thresh, block_width, static_cast<I*>(perm_out), nthreads);
        });
    });
}

int xspmm_jaccard_clustering(int itype, int64_t M, int64_t K, int64_t nnz, const void* rp,
                             const void* ci, float dist_thresh, int64_t block_width,
                             void* perm_out, int* engine_used, void* stream)
{
    return guarded([&] {
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            jaccard_clustering_device<I>(M, K, nnz, static_cast<const I*>(rp),
                                         static_cast<const I*>(ci), dist_thresh, block_width,
                                         static_cast<I*>(perm_out), as_stream(stream), engine_used);
        });
    });
}

int xspmm_spmm_pipeline(int vtype, int itype, int64_t M, int64_t K, int64_t nnz,
                        const void* rp, const void* ci, const void* vals, const void* B,
                        float* C, int64_t N, int64_t hw_block_size, int optimize_pattern,
                        double* timings, void* stream)
{
    return guarded([&] {
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            require(M >= 0 && K >= 0 && nnz >= 0 && N >= 0, "CSR dimensions must be non-negative.");
            require(hw_block_size == 16,
                    "xSpMM: the MFMA tile kernel requires hw_block_size == 16.");
            spmm_pipeline<T, I>(M, K, nnz, static_cast<const I*>(rp), static_cast<const I*>(ci),
                                static_cast<const T*>(vals), static_cast<const T*>(B), C, N,
                                hw_block_size, optimize_pattern != 0, timings, as_stream(stream));
        });
    });
}

int xspmm_pipeline_temp_bytes(int64_t* bytes_out)
{
    return guarded([&] {
        require(bytes_out != nullptr, "xspmm_pipeline_temp_bytes: bytes_out is null.");
        *bytes_out = (int64_t)last_pipeline_temp_bytes();
    });
}

int xspmm_pipeline_last_form(int* packed_out)
{
    return guarded([&] {
        require(packed_out != nullptr, "xspmm_pipeline_last_form: packed_out is null.");
        *packed_out = last_pipeline_packed() ? 1 : 0;
    });
}

int xspmm_plan_create(int vtype, int itype, int64_t M, int64_t K, int64_t nnz, const void* rp,
                      const void* ci, const void* vals, int64_t hw_block_size,
                      int optimize_pattern, double* timings, void* stream, xspmm_plan_t* plan_out)
{
    return guarded([&] {
        require(plan_out != nullptr, "xspmm_plan_create: plan_out is null.");
        *plan_out = nullptr;
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            require(M >= 0 && K >= 0 && nnz >= 0, "CSR dimensions must be non-negative.");
            require(hw_block_size == 16,
                    "xSpMM: the MFMA tile kernel requires hw_block_size == 16.");
            PlanBase* impl = make_plan<T, I>(M, K, nnz, static_cast<const I*>(rp),
                                             static_cast<const I*>(ci), static_cast<const T*>(vals),
                                             hw_block_size, optimize_pattern != 0, timings,
                                             as_stream(stream));
            *plan_out = new xspmm_plan_s{impl};
        });
    });
}

int xspmm_plan_execute(xspmm_plan_t plan, const void* B, float* C, int64_t N, void* stream)
{
    return guarded([&] {
        require(plan != nullptr, "xspmm_plan_execute: null plan.");
        require(N >= 0, "xSpMM: negative N.");
        plan->impl->execute(B, C, N, as_stream(stream));
    });
}

int xspmm_plan_info(xspmm_plan_t plan, int64_t* num_blocks, int64_t* num_block_rows,
                    int* clustered, const void** perm)
{
    return guarded([&] {
        require(plan != nullptr, "xspmm_plan_info: null plan.");
        if (num_blocks) *num_blocks = plan->impl->num_blocks();
        if (num_block_rows) *num_block_rows = plan->impl->num_block_rows();
        if (clustered) *clustered = plan->impl->clustered() ? 1 : 0;
        if (perm) *perm = plan->impl->permutation();
    });
}

int xspmm_plan_packed_batches(xspmm_plan_t plan, int64_t* batches)
{
    return guarded([&] {
        require(plan != nullptr && batches != nullptr, "xspmm_plan_packed_batches: null argument.");
        *batches = plan->impl->num_packed_batches();
    });
}

int xspmm_plan_destroy(xspmm_plan_t plan)
{
    return guarded([&] {
        if (!plan) return;
        delete plan->impl;
        delete plan;
    });
}

int xspmm_mtx_read(const char* path, xspmm_mtx_t* out)
{
    return guarded([&] {
        require(out != nullptr && path != nullptr, "xspmm_mtx_read: null argument.");
        *out = nullptr;
        auto* m = new xspmm_mtx_s{read_matrix_market(path)};
        *out = m;
    });
}

int xspmm_mtx_info(xspmm_mtx_t m, int64_t* rows, int64_t* cols, int64_t* nnz)
{
    return guarded([&] {
        require(m != nullptr, "xspmm_mtx_info: null handle.");
        if (rows) *rows = m->data.rows;
        if (cols) *cols = m->data.cols;
        if (nnz) *nnz = (int64_t)m->data.values.size();
    });
}

int xspmm_mtx_export(xspmm_mtx_t m, int itype, int vtype, void* row_ptr, void* col_ind,
                     void* values)
{
    return guarded([&] {
        require(m != nullptr, "xspmm_mtx_export: null handle.");
        const MtxData& d = m->data;
        const size_t nnz = d.values.size();
        require(row_ptr != nullptr && (nnz == 0 || (col_ind != nullptr && values != nullptr)),
                "xspmm_mtx_export: null output array.");
        with_types(vtype, itype, [&](auto tv, auto ti) {
            using T = typename decltype(tv)::type;
            using I = typename decltype(ti)::type;
            I* rp = static_cast<I*>(row_ptr);
            I* ci = static_cast<I*>(col_ind);
            for (size_t i = 0; i < d.row_ptr.size(); ++i) rp[i] = (I)d.row_ptr[i];
            for (size_t k = 0; k < nnz; ++k) ci[k] = (I)d.col_ind[k];
            T* v = static_cast<T*>(values);
            for (size_t k = 0; k < nnz; ++k) {
                if constexpr (sizeof(T) == 2) {
                    const __half h = __float2half(d.values[k]);  // round to nearest even
                    std::memcpy(&v[k], &h, 2);
                } else {
                    v[k] = d.values[k];
                }
            }
        });
    });
}

int xspmm_mtx_free(xspmm_mtx_t m)
{
    return guarded([&] { delete m; });
}

int xspmm_weight_create(int itype, int64_t M, int64_t K, int64_t Mb, int64_t Kb, int64_t nnzb, const void* brp,
                        const void* bci, void* stream, xspmm_weight_t* weight_out)
{
    return guarded([&] {
        require(weight_out != nullptr, "xspmm_weight_create: weight_out is null.");
        *weight_out = nullptr;
        with_index(itype, [&](auto ti) {
            using I = typename decltype(ti)::type;
            auto w = std::make_unique<xspmm_weight_s>();
            build_block_index<I>(w->index, M, K, Mb, Kb, nnzb, static_cast<const I*>(brp),
                                 static_cast<const I*>(bci), as_stream(stream));
            *weight_out = w.release();
        });
    });
}

int xspmm_weight_destroy(xspmm_weight_t weight)
{
    return guarded([&] { delete weight; });
}

int xspmm_linear(xspmm_weight_t weight, int vtype, int act, const void* vals, const void* x, const void* bias,
                 const void* residual, void* y, void* keep, int64_t N, void* stream)
{
    return guarded([&] {
        require(weight != nullptr, "xspmm_linear: null weight.");
        const BlockIndex& w = weight->index;
        require_layer(act, N);
        with_layer_type(vtype, [&](auto tv) {
            using T = typename decltype(tv)::type;
            const bool any = w.M > 0 && N > 0;
            ForwardArgs<T> a{};
            a.weight[0] = &w;
            a.vals[0] = operand<T>(vals, any && w.nnzb > 0, "vals");
            a.x = operand<T>(x, any && w.nnzb > 0, "x");
            a.bias[0] = static_cast<const T*>(bias);
            a.residual = operand<T>(residual, false, "residual");
            a.y = result<T>(y, any, "y");
            a.keep[0] = result<T>(keep, false, "keep");
            a.N = N;
            a.act = act;
            if (any) feed_forward<T>(a, 1, as_stream(stream));
        });
    });
}

int xspmm_gated(xspmm_weight_t gate, xspmm_weight_t up, int vtype, int act, const void* gate_vals,
                const void* up_vals, const void* x, const void* gate_bias, const void* up_bias, void* h,
                void* keep_gate, void* keep_up, int64_t N, void* stream)
{
    return guarded([&] {
        require(gate != nullptr && up != nullptr, "xspmm_gated: null weight.");
        const BlockIndex &g = gate->index, &u = up->index;
        require(g.M == u.M && g.K == u.K, "xspmm_gated: gate and up differ in shape.");
        require_layer(act, N);
        with_layer_type(vtype, [&](auto tv) {
            using T = typename decltype(tv)::type;
            const bool any = g.M > 0 && N > 0;
            ForwardArgs<T> a{};
            a.weight[0] = &g;
            a.weight[1] = &u;
            a.vals[0] = operand<T>(gate_vals, any && g.nnzb > 0, "gate_vals");
            a.vals[1] = operand<T>(up_vals, any && u.nnzb > 0, "up_vals");
            a.x = operand<T>(x, any && g.nnzb + u.nnzb > 0, "x");
            a.bias[0] = static_cast<const T*>(gate_bias);
            a.bias[1] = static_cast<const T*>(up_bias);
            a.y = result<T>(h, any, "h");
            a.keep[0] = result<T>(keep_gate, false, "keep_gate");
            a.keep[1] = result<T>(keep_up, false, "keep_up");
            a.N = N;
            a.act = act;
            if (any) feed_forward<T>(a, 2, as_stream(stream));
        });
    });
}

int xspmm_linear_backward_scratch(xspmm_weight_t weight, int vtype, int act, int64_t N, int64_t* bytes)
{
    return guarded([&] {
        require(weight != nullptr && bytes != nullptr, "xspmm_linear_backward_scratch: null argument.");
        require_layer(act, N);
        with_layer_type(vtype, [](auto) {});
        *bytes = act == XSPMM_ACT_NONE ? 0 : layer_array(vtype, weight->index.M, N);
    });
}

int xspmm_linear_backward(xspmm_weight_t weight, int vtype, int act, const void* vals, const void* x,
                          const void* keep, const void* dy, void* dx, void* dvals, void* dbias, int64_t N,
                          void* scratch, int64_t scratch_bytes, void* stream)
{
    return guarded([&] {
        require(weight != nullptr, "xspmm_linear_backward: null weight.");
        const BlockIndex& w = weight->index;
        require_layer(act, N);
        with_layer_type(vtype, [&](auto tv) {
            using T = typename decltype(tv)::type;
            const bool any = w.M > 0 && N > 0, act_too = act != XSPMM_ACT_NONE;
            require_scratch(scratch, scratch_bytes, any && act_too ? layer_array(vtype, w.M, N) : 0);
            const T* z = operand<T>(keep, any && act_too, "keep");
            const T* g = operand<T>(dy, any, "dy");
            const T* v = operand<T>(vals, any && dx != nullptr && w.nnzb > 0, "vals");
            const T* xs = operand<T>(x, any && dvals != nullptr && w.nnzb > 0, "x");
            T* out_x = result<T>(dx, false, "dx");
            T* out_v = result<T>(dvals, false, "dvals");
            T* out_b = static_cast<T*>(dbias);
            const hipStream_t s = as_stream(stream);
            T* dz = act_too ? static_cast<T*>(scratch) : nullptr;
            if (act_too || out_b) activation_backward<T>(z, nullptr, g, dz, nullptr, out_b, nullptr, act, w.M, N, s);
            const T* d = act_too ? dz : g;
            if (out_x && w.K > 0 && N > 0) {
                TransposedArgs<T> t{};
                t.weight[0] = &w;
                t.vals[0] = v;
                t.dz[0] = d;
                t.dx = out_x;
                t.N = N;
                transposed_product<T>(t, 1, s);
            }
            if (out_v) {
                SampledArgs<T> t{};
                t.weight[0] = &w;
                t.dz[0] = d;
                t.x = xs;
                t.dvals[0] = out_v;
                t.N = N;
                sampled_product<T>(t, 1, s);
            }
        });
    });
}

int xspmm_gated_backward_scratch(xspmm_weight_t gate, int vtype, int64_t N, int64_t* bytes)
{
    return guarded([&] {
        require(gate != nullptr && bytes != nullptr, "xspmm_gated_backward_scratch: null argument.");
        require_layer(XSPMM_ACT_NONE, N);
        with_layer_type(vtype, [](auto) {});
        *bytes = 2 * layer_array(vtype, gate->index.M, N);
    });
}

int xspmm_gated_backward(xspmm_weight_t gate, xspmm_weight_t up, int vtype, int act, const void* gate_vals,
                         const void* up_vals, const void* x, const void* keep_gate, const void* keep_up,
                         const void* dh, void* dx, void* dgate_vals, void* dup_vals, void* dgate_bias, void* dup_bias,
                         int64_t N, void* scratch, int64_t scratch_bytes, void* stream)
{
    return guarded([&] {
        require(gate != nullptr && up != nullptr, "xspmm_gated_backward: null weight.");
        const BlockIndex &wg = gate->index, &wu = up->index;
        require(wg.M == wu.M && wg.K == wu.K, "xspmm_gated_backward: gate and up differ in shape.");
        require_layer(act, N);
        with_layer_type(vtype, [&](auto tv) {
            using T = typename decltype(tv)::type;
            const bool any = wg.M > 0 && N > 0;
            const int64_t each = layer_array(vtype, wg.M, N);
            require_scratch(scratch, scratch_bytes, any ? 2 * each : 0);
            const T* zg = operand<T>(keep_gate, any, "keep_gate");
            const T* zu = operand<T>(keep_up, any, "keep_up");
            const T* g = operand<T>(dh, any, "dh");
            const T* vg = operand<T>(gate_vals, any && dx != nullptr && wg.nnzb > 0, "gate_vals");
            const T* vu = operand<T>(up_vals, any && dx != nullptr && wu.nnzb > 0, "up_vals");
            const T* xs = operand<T>(x, any && ((dgate_vals && wg.nnzb > 0) || (dup_vals && wu.nnzb > 0)), "x");
            T* out_x = result<T>(dx, false, "dx");
            T* out_g = result<T>(dgate_vals, false, "dgate_vals");
            T* out_u = result<T>(dup_vals, false, "dup_vals");
            const hipStream_t s = as_stream(stream);
            T* dg = static_cast<T*>(scratch);
            T* du = any ? reinterpret_cast<T*>(static_cast<char*>(scratch) + each) : nullptr;
            if (any)
                activation_backward<T>(zg, zu, g, dg, du, static_cast<T*>(dgate_bias), static_cast<T*>(dup_bias), act,
                                       wg.M, N, s);
            else  // sums over no tokens
                for (void* b : {dgate_bias, dup_bias})
                    if (b)
                        activation_backward<T>(nullptr, nullptr, nullptr, nullptr, nullptr, static_cast<T*>(b),
                                               nullptr, XSPMM_ACT_NONE, wg.M, N, s);
            if (out_x && wg.K > 0 && N > 0) {
                TransposedArgs<T> t{};
                t.weight[0] = &wg;
                t.weight[1] = &wu;
                t.vals[0] = vg;
                t.vals[1] = vu;
                t.dz[0] = dg;
                t.dz[1] = du;
                t.dx = out_x;
                t.N = N;
                transposed_product<T>(t, 2, s);
            }
            if (out_g || out_u) {
                SampledArgs<T> t{};
                t.weight[0] = &wg;
                t.weight[1] = &wu;
                t.dz[0] = dg;
                t.dz[1] = du;
                t.x = xs;
                t.dvals[0] = out_g;
                t.dvals[1] = out_u;
                t.N = N;
                sampled_product<T>(t, 2, s);
            }
        });
    });
}

int xspmm_layer_norm_scratch(int vtype, int64_t K, int64_t N, int backward, int64_t* bytes)
{
    return guarded([&] {
        require(bytes != nullptr, "xspmm_layer_norm_scratch: bytes is null.");
        require(K >= 0 && N >= 0 && K <= 0x7fffffffLL && N <= (int64_t(1) << 30), "xSpMM: bad size of a norm.");
        with_layer_type(vtype, [&](auto tv) {
            *bytes = layer_norm_scratch(K, N, sizeof(typename decltype(tv)::type), backward);
        });
    });
}

int xspmm_layer_norm(int vtype, int64_t K, int64_t N, const void* x, const void* weight, const void* bias, float eps,
                     void* y, float* mean, float* rstd, void* scratch, int64_t scratch_bytes, void* stream)
{
    return guarded([&] {
        require(K >= 0 && N >= 0 && K <= 0x7fffffffLL && N <= (int64_t(1) << 30), "xSpMM: bad size of a norm.");
        require(eps >= 0.f, "xSpMM: a norm's eps is not negative.");
        require((mean == nullptr) == (rstd == nullptr), "xSpMM: a norm keeps both statistics or none.");
        with_layer_type(vtype, [&](auto tv) {
            using T = typename decltype(tv)::type;
            const bool any = K > 0 && N > 0;
            require_scratch(scratch, scratch_bytes, layer_norm_scratch(K, N, sizeof(T), 0));
            layer_norm<T>(operand<T>(x, any, "x"), static_cast<const T*>(weight), static_cast<const T*>(bias), eps,
                          result<T>(y, any, "y"), mean, rstd, K, N, scratch, as_stream(stream));
        });
    });
}

int xspmm_layer_norm_backward(int vtype, int64_t K, int64_t N, const void* dy, const void* x, const void* weight,
                              const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                              void* scratch, int64_t scratch_bytes, void* stream)
{
    return guarded([&] {
        require(K >= 0 && N >= 0 && K <= 0x7fffffffLL && N <= (int64_t(1) << 30), "xSpMM: bad size of a norm.");
        with_layer_type(vtype, [&](auto tv) {
            using T = typename decltype(tv)::type;
            const bool any = K > 0 && N > 0;
            require(!any || (mean != nullptr && rstd != nullptr), "xSpMM: a norm's gradient needs its statistics.");
            require_scratch(scratch, scratch_bytes, layer_norm_scratch(K, N, sizeof(T), 1));
            layer_norm_backward<T>(operand<T>(dy, any, "dy"), operand<T>(x, any, "x"), static_cast<const T*>(weight),
                                   mean, rstd, result<T>(dx, false, "dx"), static_cast<T*>(dweight),
                                   static_cast<T*>(dbias), K, N, scratch, as_stream(stream));
        });
    });
}

}  // extern "C"
