// Trainable projections: y = act(x W^T + bias) + residual, dX and dW, over the
// tcgen05 kernel of gemm_proj.cuh, and the weight-streaming kernel of
// gemv_proj.cuh for a forward of a few rows.
#include "gemv_proj.cuh"

namespace rwkv {

// qaffine.cu
int gemm_wait_record(cudaStream_t st, const char* fn, int** err, int** err_host, int* sm_count);

namespace {

// What dW needs before its product, in one launch: blocks below `first` sum slices of
// dY's columns (few and long, so they start first), the others write act(X) in the
// operands' type (from the dense pre-activation or its checkpoint).
//
// Restoring the operand in a pass of its own reads and writes it once (8192 x 8192: 50
// us, of 232 with the product for 2048 outputs); decoding inside the product would
// repeat the work for every 256 outputs of dW, 8 times here (not measured).
struct DwPrep {
    const void* x;         // dense, or
    const int8_t* codes;   // its checkpoint
    const uint8_t* exps;
    void* operand;         // [rows, IN] or NULL
    int act, IN;
    int64_t units;         // of 8 channels
    const void* dy;        // [rows, OUT]
    float* part;           // [slices][OUT] or NULL
    int rows, OUT, slices, bf16;
    int first;
};
constexpr int PREP_T = 256, PREP_U = 4, CS_COLS = 256;
constexpr int CS_DIRECT = 128;  // rows of dY summed without slices: 32 per warp, one launch less

// FLAT: whole groups per row (IN % 32 == 0, or a dense x), nothing is divided.
template <bool CK, bool FLAT>
__device__ __forceinline__ void restore_operand(const DwPrep& a) {
    const int64_t i0 = ((int)blockIdx.x - a.first) * (int64_t)(PREP_T * PREP_U) + threadIdx.x;
    const int G = (a.IN + CK_GROUP - 1) / CK_GROUP, per = a.IN / 8;
    uint4 raw[PREP_U];
    uint32_t e[PREP_U];
#pragma unroll
    for (int j = 0; j < PREP_U; j++) {
        const int64_t i = min(i0 + j * PREP_T, a.units - 1);
        if constexpr (CK) {
            const uint2 w = __ldcs(reinterpret_cast<const uint2*>(a.codes + 8 * i));
            raw[j] = make_uint4(w.x, w.y, 0, 0);
            int64_t group = i >> 2;
            if constexpr (!FLAT) {
                const int64_t row = a.units < (1ll << 32) ? (uint32_t)i / (uint32_t)per : i / per;
                group = row * G + ((int)(i - row * per) >> 2);
            }
            e[j] = a.exps[group];
        } else {
            raw[j] = __ldcs(static_cast<const uint4*>(a.x) + i);
        }
    }
    with_act(a.act, [&]<int ACT>() {
#pragma unroll
        for (int j = 0; j < PREP_U; j++) {
            float v[8];
            if constexpr (CK) {
                const float s = ck_scale(e[j]);
                ck_unpack4(raw[j].x, s, v);
                ck_unpack4(raw[j].y, s, v + 4);
            } else {
                floats8_16(raw[j], a.bf16, v);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = act_t<ACT, true>(v[k]);
            if (i0 + j * PREP_T < a.units) static_cast<uint4*>(a.operand)[i0 + j * PREP_T] = pack8_16(v, a.bf16);
        }
    });
}

// A block sums 256 columns of every (8 slices)th group of 8 rows: a thread takes 8
// columns of one row of each group, the 8 row lanes meet in shared memory.
__device__ __forceinline__ void sum_columns(const DwPrep& a, int block) {
    __shared__ float red[8][CS_COLS];
    const int cv = threadIdx.x & 31, rl = threadIdx.x >> 5, cblocks = (a.OUT + CS_COLS - 1) / CS_COLS;
    const int slice = block / cblocks, c0 = (block - slice * cblocks) * CS_COLS, col = c0 + cv * 8;
    float s[8] = {};
    if (col < a.OUT)
#pragma unroll 4
        for (int64_t r = (int64_t)slice * 8 + rl; r < a.rows; r += 8 * (int64_t)a.slices) {
            float v[8];
            load8_16(a.dy, r * a.OUT + col, a.bf16, v);
#pragma unroll
            for (int k = 0; k < 8; k++) s[k] += v[k];
        }
#pragma unroll
    for (int k = 0; k < 8; k++) red[rl][cv * 8 + k] = s[k];
    __syncthreads();
    const int c = c0 + threadIdx.x;
    if (c < a.OUT) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) t += red[k][threadIdx.x];
        a.part[(int64_t)slice * a.OUT + c] = t;
    }
}
__global__ void __launch_bounds__(PREP_T, 1) dw_prep_kernel(const DwPrep a) {
    if ((int)blockIdx.x < a.first) sum_columns(a, (int)blockIdx.x);
    else if (!a.codes) restore_operand<false, true>(a);
    else if (a.IN % CK_GROUP == 0) restore_operand<true, true>(a);
    else restore_operand<true, false>(a);
}
int col_slices(int rows, int OUT) {
    return std::max(1, std::min(ceil_div(rows, 64), 148 * 4 / ceil_div(OUT, CS_COLS)));
}

template <typename F>
cudaError_t by_kind(const ProjEpi& e, F&& f) {
    const bool fast = e.fast();
    switch (e.kind()) {
        case PJ_GRAD: return fast ? f.template operator()<PJ_GRAD, true>() : f.template operator()<PJ_GRAD, false>();
        case PJ_FWD_CK: return fast ? f.template operator()<PJ_FWD_CK, true>() : f.template operator()<PJ_FWD_CK, false>();
        case PJ_FWD: return fast ? f.template operator()<PJ_FWD, true>() : f.template operator()<PJ_FWD, false>();
        default: return f.template operator()<PJ_PLAIN, true>();
    }
}

int64_t al256(int64_t n) { return (n + 255) / 256 * 256; }
bool al(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_common(int dtype, int rows, int OUT, int IN, const char* fn) {
    RWKV_REQUIRE(dtype == RWKV_BF16 || dtype == RWKV_F16, RWKV_E_DTYPE, "%s: dtype %d (bf16 or fp16)", fn, dtype);
    RWKV_REQUIRE(rows >= 1 && OUT >= 1 && IN >= 1, RWKV_E_SHAPE, "%s: rows=%d OUT=%d IN=%d must be >= 1", fn, rows, OUT,
                 IN);
    RWKV_REQUIRE(IN % 8 == 0 && OUT % 8 == 0, RWKV_E_UNSUPPORTED, "%s: IN=%d and OUT=%d must be multiples of 8", fn,
                 IN, OUT);
    RWKV_REQUIRE(rows <= 1 << 24 && OUT <= 1 << 20 && IN <= 1 << 20 &&
                     (int64_t)ceil_div(rows, 128) * ceil_div(std::max(OUT, IN), 64) < 1 << 30,
                 RWKV_E_SHAPE, "%s: rows=%d OUT=%d IN=%d too large", fn, rows, OUT, IN);
    return RWKV_OK;
}
int check_ws(const void* ws, int64_t bytes, int64_t need, const char* fn) {
    RWKV_REQUIRE(need == 0 || (ws && bytes >= need), RWKV_E_WORKSPACE, "%s: workspace of %lld bytes, need %lld", fn,
                 (long long)bytes, (long long)need);
    RWKV_REQUIRE(need == 0 || al(ws, 16), RWKV_E_UNSUPPORTED, "%s: workspace not 16-byte aligned", fn);
    return RWKV_OK;
}
// stream the weights (gemv_proj.cuh)
bool few_rows(int rows, int IN) { return rows <= GP_ROWS && IN <= GP_IN; }
bool out_ok(int out, int dtype) { return out == dtype || out == RWKV_F32; }

bool sizes_ok(int rows, int OUT, int IN) {
    return check_common(RWKV_BF16, rows, OUT, IN, "workspace_size") == RWKV_OK;
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int64_t rwkv_projection_forward_workspace_size(int rows, int OUT, int IN) {
    return sizes_ok(rows, OUT, IN) && !few_rows(rows, IN) ? proj_plan(rows, OUT, IN).ws_bytes : 0;
}

extern "C" int rwkv_projection_forward(int dtype, const void* x, const void* w, int bdtype, const void* bias, int act,
                                       int ydtype, const void* residual, void* y, void* z, int8_t* codes,
                                       uint8_t* exps, int rows, int OUT, int IN, void* workspace,
                                       int64_t workspace_bytes, rwkv_stream_t stream) {
    const char* fn = "rwkv_projection_forward";
    if (int rc = check_common(dtype, rows, OUT, IN, fn)) return rc;
    RWKV_REQUIRE(x && w && y, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(!codes == !exps, RWKV_E_NULL, "%s: give both codes and exps or neither", fn);
    RWKV_REQUIRE(out_ok(ydtype, dtype) && (!bias || valid_dtype(bdtype)), RWKV_E_DTYPE, "%s: dtypes y=%d bias=%d", fn,
                 ydtype, bdtype);
    RWKV_REQUIRE(valid_act(act), RWKV_E_UNSUPPORTED, "%s: activation %d", fn, act);
    RWKV_REQUIRE(al(x, 16) && al(w, 16) && al(y, 16) && al(residual, 16) && al(z, 16) && al(codes, 16) &&
                     al(bias, 16),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned", fn);
    const bool few = few_rows(rows, IN);
    if (!few)
        if (int rc = check_ws(workspace, workspace_bytes, proj_plan(rows, OUT, IN).ws_bytes, fn)) return rc;
    int *err, *err_host, sms;
    if (int rc = gemm_wait_record((cudaStream_t)stream, fn, &err, &err_host, &sms)) return rc;
    ProjEpi e{};
    e.bf16 = dtype == RWKV_BF16;
    e.out_f32 = ydtype == RWKV_F32;
    e.act = act;
    e.bias = bias;
    e.bias_dtype = bdtype;
    e.add = residual;
    e.codes = codes;
    e.exps = exps;
    e.z = z;
    const cudaError_t rc =
        few ? launch_gemv_proj(GemvProjArgs{x, w, y, e, rows, OUT, IN}, sms, (cudaStream_t)stream)
            : by_kind(e, [&]<int KIND, bool FAST>() {
                  return proj_gemm<false, false, KIND == PJ_GRAD ? PJ_PLAIN : KIND, KIND == PJ_GRAD || FAST>(  // no gradient
                      x, w, y, rows, OUT, IN, e, static_cast<float*>(workspace), err, err_host, sms, (cudaStream_t)stream);
              });
    if (rc != cudaSuccess) return fail(RWKV_E_CUDA, "%s: %s", fn, cudaGetErrorString(rc));
    return ok();
}

extern "C" int64_t rwkv_projection_dx_workspace_size(int rows, int OUT, int IN) {
    return sizes_ok(rows, OUT, IN) ? proj_plan(rows, IN, OUT).ws_bytes : 0;
}

extern "C" int rwkv_projection_dx(int dtype, const void* dy, const void* w, int act, const void* z,
                                  const int8_t* codes, const uint8_t* exps, int dxdtype, const void* addend, void* dx,
                                  int rows, int OUT, int IN, void* workspace, int64_t workspace_bytes,
                                  rwkv_stream_t stream) {
    const char* fn = "rwkv_projection_dx";
    if (int rc = check_common(dtype, rows, OUT, IN, fn)) return rc;
    RWKV_REQUIRE(dy && w && dx, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(valid_act(act), RWKV_E_UNSUPPORTED, "%s: activation %d", fn, act);
    RWKV_REQUIRE(!codes == !exps && !(z && codes), RWKV_E_NULL, "%s: z, or codes and exps, or neither", fn);
    RWKV_REQUIRE(z || codes || act == RWKV_ACT_NONE, RWKV_E_NULL, "%s: the activation needs its pre-activation", fn);
    RWKV_REQUIRE(out_ok(dxdtype, dtype), RWKV_E_DTYPE, "%s: dX dtype %d", fn, dxdtype);
    RWKV_REQUIRE(al(dy, 16) && al(w, 16) && al(z, 16) && al(codes, 16) && al(addend, 16) && al(dx, 16),
                 RWKV_E_UNSUPPORTED, "%s: a tensor is not 16-byte aligned", fn);
    if (int rc = check_ws(workspace, workspace_bytes, proj_plan(rows, IN, OUT).ws_bytes, fn)) return rc;
    int *err, *err_host, sms;
    if (int rc = gemm_wait_record((cudaStream_t)stream, fn, &err, &err_host, &sms)) return rc;
    ProjEpi e{};
    e.bf16 = dtype == RWKV_BF16;
    e.out_f32 = dxdtype == RWKV_F32;
    e.act = act;
    e.grad = act != RWKV_ACT_NONE;
    e.pre = z;
    e.pre_codes = codes;
    e.pre_exps = exps;
    e.add = addend;
    const cudaError_t rc = by_kind(e, [&]<int KIND, bool FAST>() {
        // (never keeps a checkpoint; an activation only as its gradient)
        return proj_gemm<false, true, KIND == PJ_FWD_CK ? PJ_FWD : KIND, KIND != PJ_GRAD || FAST>(
            dy, w, dx, rows, IN, OUT, e, static_cast<float*>(workspace), err, err_host, sms, (cudaStream_t)stream);
    });
    if (rc != cudaSuccess) return fail(RWKV_E_CUDA, "%s: %s", fn, cudaGetErrorString(rc));
    return ok();
}

namespace {
// dW's workspace: the restored operand, the split-K partials, the partial column sums
struct DwPlan {
    int64_t operand, parts, total;
    int slices;
};
DwPlan dw_plan(int rows, int OUT, int IN, bool restore) {
    DwPlan p{};
    p.operand = restore ? al256((int64_t)rows * IN * 2) : 0;
    p.parts = al256(proj_plan(OUT, IN, rows).ws_bytes);
    p.slices = col_slices(rows, OUT);
    p.total = p.operand + p.parts + al256((int64_t)p.slices * OUT * 4);
    return p;
}
}  // namespace

extern "C" int64_t rwkv_projection_dw_workspace_size(int rows, int OUT, int IN, int restore) {
    return sizes_ok(rows, OUT, IN) ? dw_plan(rows, OUT, IN, restore != 0).total : 0;
}

extern "C" int rwkv_projection_dw(int dtype, const void* dy, int act, const void* x, const int8_t* codes,
                                  const uint8_t* exps, int dwdtype, void* dw, float* db, int rows, int OUT, int IN,
                                  void* workspace, int64_t workspace_bytes, rwkv_stream_t stream) {
    const char* fn = "rwkv_projection_dw";
    if (int rc = check_common(dtype, rows, OUT, IN, fn)) return rc;
    RWKV_REQUIRE(dy && (dw || db), RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(!dw || (x ? !codes && !exps : codes && exps), RWKV_E_NULL, "%s: give either x or codes and exps", fn);
    RWKV_REQUIRE(valid_act(act), RWKV_E_UNSUPPORTED, "%s: activation %d", fn, act);
    RWKV_REQUIRE(out_ok(dwdtype, dtype), RWKV_E_DTYPE, "%s: dW dtype %d", fn, dwdtype);
    RWKV_REQUIRE(al(dy, 16) && al(x, 16) && al(codes, 16) && al(dw, 16) && al(db, 4), RWKV_E_UNSUPPORTED,
                 "%s: a tensor is not 16-byte aligned", fn);
    const bool restore = dw && (codes || act != RWKV_ACT_NONE);
    const DwPlan p = dw_plan(rows, OUT, IN, restore);
    if (int rc = check_ws(workspace, workspace_bytes, p.total, fn)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    int *err, *err_host, sms;
    if (int rc = gemm_wait_record(st, fn, &err, &err_host, &sms)) return rc;
    char* ws = static_cast<char*>(workspace);
    DwPrep q{};
    q.x = x;
    q.codes = codes;
    q.exps = exps;
    q.operand = ws;
    q.act = act;
    q.IN = IN;
    q.units = (int64_t)rows * IN / 8;
    q.dy = dy;
    q.part = reinterpret_cast<float*>(ws + p.operand + p.parts);
    q.rows = rows;
    q.OUT = OUT;
    q.slices = p.slices;
    q.bf16 = dtype == RWKV_BF16;
    const bool direct = rows <= CS_DIRECT;  // summed beside the join, from dY itself
    q.first = db && !direct ? ceil_div(OUT, CS_COLS) * p.slices : 0;
    const int grid = q.first + (restore ? ceil_div(q.units, PREP_T * PREP_U) : 0);
    if (grid) {
        dw_prep_kernel<<<grid, PREP_T, 0, st>>>(q);
        if (int rc = check_launch("dw_prep_kernel")) return rc;
    }
    const ColJoin cols{direct ? nullptr : q.part, dy, db, OUT, direct ? rows : p.slices, q.bf16};
    cudaError_t rc;
    if (dw) {
        ProjEpi e{};
        e.bf16 = q.bf16;
        e.out_f32 = dwdtype == RWKV_F32;
        rc = proj_gemm<true, true, PJ_PLAIN, true>(dy, restore ? ws : x, dw, OUT, IN, rows, e, reinterpret_cast<float*>(ws + p.operand),
                                   err, err_host, sms, st, grid != 0, db ? &cols : nullptr);
    } else {
        rc = launch_pdl(proj_join_kernel<PJ_PLAIN, true>, dim3(ceil_div(OUT, 32)), dim3(PJ_JOIN_T), 0, st, ProjJoin{}, cols, 0);
    }
    if (rc != cudaSuccess) return fail(RWKV_E_CUDA, "%s: %s", fn, cudaGetErrorString(rc));
    return ok();
}
