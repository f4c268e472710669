// The residual norm: a branch added to the residual stream, through dropout and
// scaled, and the sum normed for the next branch, in one pass.
//
//   forward   s = x + scale drop(branch), y = (s - mean) rstd w + b
//   backward  ds as the layer norm's dx (dres: the gradient of s past the norm),
//             dx = ds, dbranch = scale drop(ds), dw, db
//
// The kernels are the layer norm's (layer_norm.cuh) with the branch: 4 tensors
// forward (x, branch, s, y) and 5 backward (dy, s, dres, dx, dbranch), or 1 + 1/32
// bytes per element for s as a checkpoint.  s is normed and checkpointed before its
// rounding: y is that of the sum in fp32.
#include "layer_norm.cuh"

namespace rwkv {
namespace {

template <typename T, bool CK>
int launch_rn_fwd(const LnFwdArgs& a, cudaStream_t st) {
    // threads, vectors per thread and rows as in the layer norm
    constexpr int R = CK ? 1 : 2;
    const int nvec = a.D / Vec16<T>::N;
    if (nvec <= 64) launch_ln_fwd_t<T, 64, 1, 2, CK, true>(a, st);
    else if (nvec <= 64 * 2) launch_ln_fwd_t<T, 64, 2, 2, CK, true>(a, st);
    else if (nvec <= 64 * 3) launch_ln_fwd_t<T, 64, 3, 2, CK, true>(a, st);
    else if (nvec <= 128 * 2) launch_ln_fwd_t<T, 128, 2, 2, CK, true>(a, st);
    else if (nvec <= 64 * 5) launch_ln_fwd_t<T, 64, 5, R, CK, true>(a, st);
    else if (nvec <= 256 * 2) launch_ln_fwd_t<T, 256, 2, R, CK, true>(a, st);
    else if (nvec <= 256 * 5) launch_ln_fwd_t<T, 256, 5, R, CK, true>(a, st);
    else launch_ln_fwd_t<T, 512, 3, 1, CK, true>(a, st);
    return check_launch("ln_fwd_kernel (residual)");
}

template <typename T, bool CK>
int launch_rn_bwd(const LnBwdArgs& a, void* dw, void* db, cudaStream_t st) {
    constexpr int R = CK ? 1 : 2;
    const int nvec = a.D / Vec16<T>::N;
    int blocks;
    cudaError_t e = nvec > 1024  ? launch_ln_bwd_t<T, CK, 3, 1, 512, 1, false, true>(a, &blocks, st)
                    : nvec > 512 ? launch_ln_bwd_t<T, CK, 2, 1, 512, 1, false, true>(a, &blocks, st)
                    : nvec > 320 ? launch_ln_bwd_t<T, CK, 1, R, 512, 1, false, true>(a, &blocks, st)
                                 : launch_ln_bwd_t<T, CK, 1, R, 320, 2, false, true>(a, &blocks, st);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "ln_bwd_kernel (residual): %s", cudaGetErrorString(e));
    if (int rc = check_launch("ln_bwd_kernel (residual)")) return rc;
    if (!a.part) return ok();
    e = launch_pdl(ln_bwd_params_kernel, dim3(ceil_div(2 * (int64_t)a.D, 32)), dim3(1024), 0, st, (const float*)a.part,
                   blocks, a.D, dw, db, a.wdtype);
    if (e != cudaSuccess) return fail(RWKV_E_CUDA, "ln_bwd_params_kernel: %s", cudaGetErrorString(e));
    return ok();
}

int check_sizes(int dtype, int wdtype, int rows, int D, double p, double scale, const char* fn) {
    RWKV_REQUIRE(valid_dtype(dtype) && valid_dtype(wdtype), RWKV_E_DTYPE, "%s: dtypes x=%d w=%d", fn, dtype, wdtype);
    const int most = dtype == RWKV_F32 ? LN_BWD_VECTORS * 4 : LN_BWD_VECTORS * 8;
    RWKV_REQUIRE(rows >= 1 && D >= 1, RWKV_E_SHAPE, "%s: rows=%d D=%d", fn, rows, D);
    RWKV_REQUIRE(D % 8 == 0 && D <= most, RWKV_E_UNSUPPORTED, "%s: D=%d must be a multiple of 8, at most %d", fn, D, most);
    RWKV_REQUIRE(p >= 0.0 && p <= 1.0, RWKV_E_SHAPE, "%s: p=%g must be in 0..1", fn, p);
    RWKV_REQUIRE(std::isfinite(make_dropout(p, scale, 0, 0, nullptr).scale), RWKV_E_SHAPE,
                 "%s: scale=%g over 1 - p must be finite in fp32", fn, scale);
    return RWKV_OK;
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_residual_norm_forward(int dtype, const void* x, const void* branch, double scale, double p,
                                          uint64_t seed, uint64_t offset, const int64_t* state, int wdtype,
                                          const void* weight, const void* bias, float eps, void* sum, void* y,
                                          float* mean, float* rstd, int8_t* codes, uint8_t* exps, int rows, int D,
                                          rwkv_stream_t stream) {
    const char* fn = "rwkv_residual_norm_forward";
    if (int rc = check_sizes(dtype, wdtype, rows, D, p, scale, fn)) return rc;
    RWKV_REQUIRE(x && branch && weight && bias && sum && y, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(!mean == !rstd, RWKV_E_NULL, "%s: give both mean and rstd or neither", fn);
    RWKV_REQUIRE(!codes == !exps, RWKV_E_NULL, "%s: give both codes and exps or neither", fn);
    RWKV_REQUIRE(eps >= 0.f, RWKV_E_SHAPE, "%s: eps=%g must be >= 0", fn, eps);
    RWKV_REQUIRE(al(x, 16) && al(branch, 16) && al(weight, 16) && al(bias, 16) && al(sum, 16) && al(y, 16) &&
                     al(codes, 8) && al(state, 8) && al(mean, 4) && al(rstd, 4),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned (codes, state: 8; mean, rstd: 4)", fn);
    const LnFwdArgs a{x,  weight, bias, y, mean, rstd, codes, exps, wdtype, rows, D, ceil_div(D, CK_GROUP),
                      eps, branch, sum, make_dropout(p, scale, seed, offset, state)};
    return dispatch_dtype(dtype, [&]<typename T>() {
        return codes ? launch_rn_fwd<T, true>(a, (cudaStream_t)stream) : launch_rn_fwd<T, false>(a, (cudaStream_t)stream);
    });
}

extern "C" int64_t rwkv_residual_norm_backward_workspace_size(int rows, int D) {
    return D <= LN_BWD_VECTORS * 8 ? rwkv_layer_norm_backward_workspace_size(rows, D) : 0;
}

extern "C" int rwkv_residual_norm_backward(int dtype, const void* dy, const void* sum, const int8_t* codes,
                                           const uint8_t* exps, int wdtype, const void* weight, const float* mean,
                                           const float* rstd, const void* dres, double scale, double p, uint64_t seed,
                                           uint64_t offset, const int64_t* state, void* dx, void* dbranch,
                                           void* dweight, void* dbias, int rows, int D, void* workspace,
                                           int64_t workspace_bytes, rwkv_stream_t stream) {
    const char* fn = "rwkv_residual_norm_backward";
    if (int rc = check_sizes(dtype, wdtype, rows, D, p, scale, fn)) return rc;
    RWKV_REQUIRE(dy && weight && mean && rstd && dx && dbranch, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(sum ? !codes && !exps : codes && exps, RWKV_E_NULL, "%s: give either sum or codes and exps", fn);
    RWKV_REQUIRE(!dweight == !dbias, RWKV_E_NULL, "%s: give both dweight and dbias or neither", fn);
    RWKV_REQUIRE(al(dy, 16) && al(sum, 16) && al(codes, 8) && al(dres, 16) && al(dx, 16) && al(dbranch, 16) &&
                     al(weight, 16) && al(dweight, elem(wdtype)) && al(dbias, elem(wdtype)) && al(state, 8) &&
                     al(mean, 4) && al(rstd, 4),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned (codes, state: 8; others: their element)", fn);
    if (dweight) {
        const int64_t need = rwkv_residual_norm_backward_workspace_size(rows, D);
        RWKV_REQUIRE(workspace && workspace_bytes >= need, RWKV_E_WORKSPACE, "%s: workspace of %lld bytes, need %lld",
                     fn, (long long)workspace_bytes, (long long)need);
        RWKV_REQUIRE(al(workspace, 16), RWKV_E_UNSUPPORTED, "%s: workspace not 16-byte aligned", fn);
    }
    const LnBwdArgs a{dy,   sum,  codes, exps, weight, mean, rstd, dres, dx, dweight ? static_cast<float*>(workspace) : nullptr,
                      wdtype, rows, D, ceil_div(D, CK_GROUP), dbranch, make_dropout(p, scale, seed, offset, state)};
    return dispatch_dtype(dtype, [&]<typename T>() {
        return codes ? launch_rn_bwd<T, true>(a, dweight, dbias, (cudaStream_t)stream)
                     : launch_rn_bwd<T, false>(a, dweight, dbias, (cudaStream_t)stream);
    });
}
