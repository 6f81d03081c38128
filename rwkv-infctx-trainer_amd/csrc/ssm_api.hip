// C ABI of the state space operators and of sampling: argument checks and dispatch (a translation unit of its own).
#include "../../include/rwkv_wkv_hip.h"
#include "common.h"
#include "ssm_conv.hip"
#include "ssm_norm.hip"
#include "ssm_scan.hip"
#include "sampling.hip"

using namespace wkv;

namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t element(int dtype) { return dtype == WKV_F32 ? 4 : 2; }
bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int finished(hipError_t e) { return e == hipSuccess ? WKV_OK : WKV_ERR_LAUNCH; }
int dtype_ok(int dtype) { return dtype < WKV_F32 || dtype > WKV_F16 ? WKV_ERR_DTYPE : WKV_OK; }

#define BY_DTYPE(dtype, CALL) ((dtype) == WKV_BF16 ? CALL(bf16) : (dtype) == WKV_F16 ? CALL(f16) : CALL(float))

bool overlaps(const void *a, const void *b, size_t bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + bytes && y < x + bytes;
}

int check_streams(int B, int T, int D, int dtype) {
    if (B <= 0 || T <= 0 || D <= 0 || B > 65535) return WKV_ERR_DIMS;
    if ((long long)B * T * D >= (1ll << 40) || (long long)T * D >= (1ll << 40) || T > (1 << 24) || (long long)B * D >= (1ll << 28)) return WKV_ERR_DIMS;
    return dtype_ok(dtype);
}

// ---- convolution
int check_conv(int B, int T, int D, int W, int dtype, int param_dtype) {
    if (W < conv::MIN_TAPS || W > conv::MAX_TAPS || T > 65535 * conv::RUNS * 8) return WKV_ERR_DIMS;
    if (int st = check_streams(B, T, D, dtype)) return st;
    return param_dtype == WKV_F32 || param_dtype == dtype ? WKV_OK : WKV_ERR_DTYPE;
}
conv::Call conv_call(int B, int T, int D, int param_dtype, int silu, const wkv_rows *x, const void *weight, const void *bias, const void *state_in,
                     const int *lengths) {
    conv::Call k = {};
    k.B = B; k.T = T; k.D = D;
    k.silu = silu; k.w32 = param_dtype == WKV_F32;
    k.x = x->p; k.batch = x->batch; k.token = x->token;
    k.weight = weight; k.bias = bias; k.state_in = state_in; k.lengths = lengths;
    return k;
}
// how many channels a lane may take at once
int conv_piece(const wkv_rows *x, int D, int dtype) {
    for (int v : {4, 2})
        if (D % v == 0 && aligned_to(x->p, v * element(dtype)) && x->batch % v == 0 && x->token % v == 0) return v;
    return 1;
}

// ---- scan
int check_scan(int B, int T, int D, int N, int G, int dtype) {
    if (N <= 0 || N > scan::MAX_STATES || G <= 0 || D % G != 0 || D >= scan::MAX_TOKEN_STRIDE || (long long)D * N >= (1ll << 30)) return WKV_ERR_DIMS;
    if (int st = check_streams(B, T, D, dtype)) return st;
    // (grids: at most 64 segments of workgroups of 16 channels)
    return (long long)B * G * ((D / G + 15) / 16) * 64 >= (1ll << 31) || (long long)B * T * G * N >= (1ll << 31) ? WKV_ERR_DIMS : WKV_OK;
}
scan::Rows rows_of(const wkv_rows *r) { return r ? scan::Rows{r->p, r->batch, r->token, r->group} : scan::Rows{}; }
int check_scan_operands(int dtype, const wkv_rows *x, const wkv_rows *dt, const wkv_rows *z, const wkv_rows *b, const wkv_rows *c, const float *A) {
    if (!x || !dt || !b || !c || !A) return WKV_ERR_NULL;
    for (const wkv_rows *r : {x, dt, z, b, c}) {
        if (r && !r->p) return WKV_ERR_NULL;
        if (r && !aligned_to(r->p, element(dtype))) return WKV_ERR_ALIGN;
        if (r && (r->token < 0 || r->token >= scan::MAX_TOKEN_STRIDE)) return WKV_ERR_DIMS;
    }
    return WKV_OK;
}
scan::Call scan_call(int B, int T, int D, int N, int G, const wkv_rows *x, const wkv_rows *dt, const wkv_rows *z, const wkv_rows *b, const wkv_rows *c,
                     const float *A, const float *skip, const float *bias, const float *state_in, const int *lengths, float *checkpoints) {
    scan::Call k = {};
    k.B = B; k.T = T; k.D = D; k.N = N; k.G = G; k.Dg = D / G;
    k.x = rows_of(x); k.dt = rows_of(dt); k.z = rows_of(z); k.b = rows_of(b); k.c = rows_of(c);
    k.A = A; k.skip = skip; k.bias = bias; k.state_in = state_in; k.lengths = lengths;
    k.checkpoints = checkpoints;
    return k;
}

// ---- norm
int check_norm(int rows, int C, int dtype, int residual_dtype, int weight_dtype) {
    if (rows <= 0 || C <= 0 || C > (1 << 24)) return WKV_ERR_DIMS;
    if (int st = dtype_ok(dtype)) return st;
    if (residual_dtype != WKV_F32 && residual_dtype != dtype) return WKV_ERR_DTYPE;
    return weight_dtype == WKV_F32 || weight_dtype == dtype ? WKV_OK : WKV_ERR_DTYPE;
}
// elements per piece of a row, as its width, its strides and the addresses allow
int norm_piece(int C, long long xs, long long rs, const void *x, const void *residual, int dtype, int residual_dtype) {
    if (C % 8 == 0 && xs % 8 == 0 && rs % 8 == 0 && aligned16(x) && aligned16(residual)) return 8;
    return C % 2 == 0 && xs % 2 == 0 && rs % 2 == 0 && aligned_to(x, 2 * element(dtype)) && aligned_to(residual, 2 * element(residual_dtype)) ? 2 : 1;
}

}  // namespace

extern "C" {

int wkv_causal_conv_forward(void *stream, int B, int T, int D, int W, int dtype, int param_dtype, int silu, const wkv_rows *x, const void *weight,
                            const void *bias, const void *state_in, const int *lengths, void *y, void *state_out) {
    if (int st = check_conv(B, T, D, W, dtype, param_dtype)) return st;
    if (!x || !x->p || !weight || !y || !state_out) return WKV_ERR_NULL;
    for (const void *p : {weight, bias, state_in, (const void *)y, (const void *)state_out})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (!aligned_to(x->p, element(dtype))) return WKV_ERR_ALIGN;
    if (overlaps(state_in, state_out, (size_t)B * (W - 1) * D * element(dtype)) && !(T == 1 && state_in == state_out)) return WKV_ERR_ALIAS;
    conv::Call k = conv_call(B, T, D, param_dtype, silu, x, weight, bias, state_in, lengths);
    k.y = y; k.state_out = state_out;
    const int piece = conv_piece(x, D, dtype);
#define CALL(TY) conv::forward_t<TY>((hipStream_t)stream, W, k, piece)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_causal_conv_backward_workspace(int B, int T, int D, int W, int dtype) {
    return check_conv(B, T, D, W, dtype, WKV_F32) ? 0 : conv::backward_scratch(B, T, D, W);
}

int wkv_causal_conv_backward(void *stream, int B, int T, int D, int W, int dtype, int param_dtype, int silu, const wkv_rows *x, const void *weight,
                             const void *bias, const void *state_in, const int *lengths, const void *gy, const void *gstate_out, void *gx,
                             void *gweight, void *gbias, void *gstate_in, void *workspace, size_t workspace_bytes) {
    if (int st = check_conv(B, T, D, W, dtype, param_dtype)) return st;
    if (!x || !x->p || !weight || !gy || !gx || !gweight || !workspace) return WKV_ERR_NULL;
    for (const void *p : {weight, bias, state_in, gy, gstate_out, (const void *)gx, (const void *)gweight, (const void *)gbias, (const void *)gstate_in,
                          (const void *)workspace})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (!aligned_to(x->p, element(dtype))) return WKV_ERR_ALIGN;
    if (workspace_bytes < conv::backward_scratch(B, T, D, W)) return WKV_ERR_WORKSPACE;
    if (overlaps(gstate_out, gstate_in, (size_t)B * (W - 1) * D * element(dtype))) return WKV_ERR_ALIAS;
    conv::Call k = conv_call(B, T, D, param_dtype, silu, x, weight, bias, state_in, lengths);
    k.gy = gy; k.gstate_out = gstate_out; k.gx = gx; k.gstate_in = gstate_in;
    k.part = static_cast<float *>(workspace);
    const int piece = conv_piece(x, D, dtype);
#define CALL(TY) conv::backward_t<TY>((hipStream_t)stream, W, k, piece, gweight, gbias)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_selective_scan_checkpoint_bytes(int B, int T, int D, int N, int G, int dtype) {
    return check_scan(B, T, D, N, G, dtype) ? 0 : scan::checkpoint_bytes(B, T, D, N);
}
size_t wkv_selective_scan_forward_workspace(int B, int T, int D, int N, int G, int dtype) {
    return check_scan(B, T, D, N, G, dtype) ? 0 : scan::forward_scratch(B, T, D, N, G);
}

int wkv_selective_scan_forward(void *stream, int B, int T, int D, int N, int G, int dtype, const wkv_rows *x, const wkv_rows *dt, const float *A,
                               const wkv_rows *b, const wkv_rows *c, const float *skip, const wkv_rows *z, const float *dt_bias, const float *state_in,
                               const int *lengths, void *y, float *state_out, float *checkpoints, void *workspace, size_t workspace_bytes) {
    if (int st = check_scan(B, T, D, N, G, dtype)) return st;
    if (int st = check_scan_operands(dtype, x, dt, z, b, c, A)) return st;
    if (!y || !state_out) return WKV_ERR_NULL;
    for (const void *p : {(const void *)A, (const void *)skip, (const void *)dt_bias, (const void *)state_in, (const void *)y, (const void *)state_out,
                          (const void *)checkpoints, (const void *)workspace})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (overlaps(state_in, state_out, (size_t)B * D * N * 4) && !(T == 1 && !checkpoints && state_in == state_out)) return WKV_ERR_ALIAS;
    const size_t need = T == 1 && !checkpoints ? 0 : scan::forward_scratch(B, T, D, N, G);
    if (need && !workspace) return WKV_ERR_NULL;
    if (workspace_bytes < need) return WKV_ERR_WORKSPACE;
    scan::Call k = scan_call(B, T, D, N, G, x, dt, z, b, c, A, skip, dt_bias, state_in, lengths, checkpoints);
    k.y = y; k.state_out = state_out;
#define CALL(TY) scan::forward_t<TY>((hipStream_t)stream, k, workspace)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_selective_scan_backward_workspace(int B, int T, int D, int N, int G, int dtype) {
    return check_scan(B, T, D, N, G, dtype) ? 0 : scan::backward_scratch(B, T, D, N, G);
}

int wkv_selective_scan_backward(void *stream, int B, int T, int D, int N, int G, int dtype, const wkv_rows *x, const wkv_rows *dt, const float *A,
                                const wkv_rows *b, const wkv_rows *c, const float *skip, const wkv_rows *z, const float *dt_bias, const int *lengths,
                                const float *checkpoints, const void *gy, const float *gstate_out, void *gx, void *gdt, float *gA, void *gb, void *gc,
                                float *gskip, void *gz, float *gdt_bias, float *gstate_in, void *workspace, size_t workspace_bytes) {
    if (int st = check_scan(B, T, D, N, G, dtype)) return st;
    if (int st = check_scan_operands(dtype, x, dt, z, b, c, A)) return st;
    if (!checkpoints || !gy || !gx || !gdt || !gA || !gb || !gc || (z && !gz) || !workspace) return WKV_ERR_NULL;
    for (const void *p : {(const void *)A, (const void *)skip, (const void *)dt_bias, (const void *)checkpoints, gy, (const void *)gstate_out,
                          (const void *)gx, (const void *)gdt, (const void *)gA, (const void *)gb, (const void *)gc, (const void *)gskip,
                          (const void *)gz, (const void *)gdt_bias, (const void *)gstate_in, (const void *)workspace})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (workspace_bytes < scan::backward_scratch(B, T, D, N, G)) return WKV_ERR_WORKSPACE;
    if (overlaps(gstate_out, gstate_in, (size_t)B * D * N * 4)) return WKV_ERR_ALIAS;
    scan::Call k = scan_call(B, T, D, N, G, x, dt, z, b, c, A, skip, dt_bias, nullptr, lengths, const_cast<float *>(checkpoints));
    k.gy = gy; k.gstate_out = gstate_out;
    k.gx = gx; k.gdt = gdt; k.gz = gz; k.gstate_in = gstate_in;
    const scan::Gradients to = {gb, gc, gA, gskip, gdt_bias};
#define CALL(TY) scan::backward_t<TY>((hipStream_t)stream, k, to, workspace)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

int wkv_rms_norm_forward(void *stream, int rows, int C, int dtype, int residual_dtype, int weight_dtype, float eps, const void *x, long long x_stride,
                         const void *residual, long long residual_stride, const void *weight, void *y, void *q, float *scale, void *residual_out,
                         float *rstd) {
    if (int st = check_norm(rows, C, dtype, residual_dtype, weight_dtype)) return st;
    if (!x || !weight || (!y && !q) || (q && !scale)) return WKV_ERR_NULL;
    for (const void *p : {weight, (const void *)y, (const void *)q, (const void *)scale, (const void *)residual_out, (const void *)rstd})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (!aligned_to(x, element(dtype)) || !aligned_to(residual, element(residual_dtype))) return WKV_ERR_ALIGN;
    norm::Call k = {};
    k.rows = rows; k.C = C; k.w32 = weight_dtype == WKV_F32;
    k.xs = x_stride; k.rs = residual_stride; k.eps = eps;
    k.x = x; k.residual = residual; k.weight = weight;
    k.y = q ? nullptr : y; k.q = q; k.scale = scale; k.out = residual_out; k.rstd = rstd;
    const int piece = norm_piece(C, x_stride, residual ? residual_stride : 0, x, residual, dtype, residual_dtype);
#define CALL(TY) (residual_dtype == WKV_F32 ? norm::forward_t<TY, float>((hipStream_t)stream, k, piece) : norm::forward_t<TY, TY>((hipStream_t)stream, k, piece))
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_rms_norm_backward_workspace(int rows, int C) {
    return check_norm(rows, C, WKV_F32, WKV_F32, WKV_F32) ? 0 : (size_t)norm::backward_groups(rows, C) * C * 4;
}

int wkv_rms_norm_backward(void *stream, int rows, int C, int dtype, int residual_dtype, int weight_dtype, const void *x, long long x_stride,
                          const void *residual, long long residual_stride, const void *weight, const float *rstd, const void *gy,
                          const void *gresidual_out, void *gx, void *gresidual, void *gweight, void *workspace, size_t workspace_bytes) {
    if (int st = check_norm(rows, C, dtype, residual_dtype, weight_dtype)) return st;
    if ((!x && !residual) || !weight || !rstd || !gy || !gx || !gweight || !workspace) return WKV_ERR_NULL;
    for (const void *p : {weight, (const void *)rstd, gy, gresidual_out, (const void *)gx, (const void *)gresidual, (const void *)gweight, (const void *)workspace})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (!aligned_to(x, element(dtype)) || !aligned_to(residual, element(residual_dtype))) return WKV_ERR_ALIGN;
    if (workspace_bytes < wkv_rms_norm_backward_workspace(rows, C)) return WKV_ERR_WORKSPACE;
    norm::Call k = {};
    k.rows = rows; k.C = C; k.w32 = weight_dtype == WKV_F32;
    k.xs = x_stride; k.rs = residual_stride;
    k.x = x; k.residual = residual; k.weight = weight; k.rstd = const_cast<float *>(rstd);
    k.gy = gy; k.gout = gresidual_out; k.gx = gx; k.gres = gresidual;
    k.part = static_cast<float *>(workspace);
    const int piece = norm_piece(C, x ? x_stride : 0, residual ? residual_stride : 0, x, residual, dtype, residual_dtype);
#define CALL(TY) (residual_dtype == WKV_F32 ? norm::backward_t<TY, float>((hipStream_t)stream, k, piece, gweight) : norm::backward_t<TY, TY>((hipStream_t)stream, k, piece, gweight))
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

int wkv_sample(void *stream, int rows, int V, int dtype, const void *logits, long long stride, const float *u, const float *temperature,
               float temperature_value, const int *top_k, int top_k_value, const float *top_p, float top_p_value, const float *min_p, float min_p_value,
               long long *token, float *logprob) {
    if (rows <= 0 || V <= 0 || V > sampling::MAX_VOCABULARY) return WKV_ERR_DIMS;
    if (int st = dtype_ok(dtype)) return st;
    if (!logits || !u || !token || !logprob) return WKV_ERR_NULL;
    if (!aligned_to(logits, element(dtype))) return WKV_ERR_ALIGN;
    for (const void *p : {(const void *)u, (const void *)temperature, (const void *)top_k, (const void *)top_p, (const void *)min_p, (const void *)logprob})
        if (!aligned_to(p, 4)) return WKV_ERR_ALIGN;
    if (!aligned_to(token, 8)) return WKV_ERR_ALIGN;
    const sampling::Call k = {rows, V, stride, logits, u, temperature, top_p, min_p, top_k, temperature_value, top_p_value, min_p_value, top_k_value, token, logprob};
#define CALL(TY) sampling::launch<TY>((hipStream_t)stream, k)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

}  // extern "C"
