// C ABI of the operators of a gated recurrence model: argument checks and dispatch (a translation unit of its own).
#include "../../include/rwkv_wkv_hip.h"
#include "common.h"
#include "gated_scan.hip"
#include "gated_product.hip"
#include "embedding.hip"

using namespace wkv;

namespace {

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t element(int dtype) { return dtype == WKV_F32 ? 4 : 2; }
int finished(hipError_t e) { return e == hipSuccess ? WKV_OK : WKV_ERR_LAUNCH; }
int dtype_ok(int dtype) { return dtype < WKV_F32 || dtype > WKV_F16 ? WKV_ERR_DTYPE : WKV_OK; }

#define BY_DTYPE(dtype, CALL) ((dtype) == WKV_BF16 ? CALL(bf16) : (dtype) == WKV_F16 ? CALL(f16) : CALL(float))

bool aligned16(const void *p) { return aligned_to(p, 16); }
bool overlaps(const void *a, const void *b, size_t bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + bytes && y < x + bytes;
}

// ---- gated recurrence
int check_recurrence(int B, int T, int D, int dtype) {
    if (B <= 0 || T <= 0 || D <= 0 || B > 65535 || T > (1 << 24) || D >= gated::MAX_TOKEN_STRIDE) return WKV_ERR_DIMS;
    if ((long long)B * T * D >= (1ll << 40) || (long long)B * D >= (1ll << 30)) return WKV_ERR_DIMS;
    return dtype_ok(dtype);
}
int check_operands(int T, int D, int dtype, const wkv_rows *x, const wkv_rows *r, const wkv_rows *i, const wkv_rows *z, const float *decay) {
    if (!x || !r || !i || !decay) return WKV_ERR_NULL;
    for (const wkv_rows *o : {x, r, i, z}) {
        if (o && !o->p) return WKV_ERR_NULL;
        if (o && !aligned_to(o->p, element(dtype))) return WKV_ERR_ALIGN;
        if (o && T > 1 && (o->token < D || o->token >= gated::MAX_TOKEN_STRIDE)) return WKV_ERR_DIMS;
    }
    return aligned16(decay) ? WKV_OK : WKV_ERR_ALIGN;
}
// (of a single token the stride means nothing: that of rows side by side, so that what lies behind it is out of its range)
gated::Rows rows_of(const wkv_rows *o, int T, int D) { return o ? gated::Rows{o->p, o->batch, T > 1 ? o->token : D} : gated::Rows{}; }
gated::Call recurrence_call(int B, int T, int D, float scale, const wkv_rows *x, const wkv_rows *r, const wkv_rows *i, const wkv_rows *z, const float *decay,
                            const int *lengths, const float *checkpoints, void *workspace) {
    gated::Call k = {};
    k.B = B; k.T = T; k.D = D; k.scale = scale;
    k.x = rows_of(x, T, D); k.r = rows_of(r, T, D); k.i = rows_of(i, T, D); k.z = rows_of(z, T, D);
    k.decay = decay; k.lengths = lengths;
    k.checkpoints = const_cast<float *>(checkpoints);
    k.pairs = static_cast<float *>(workspace);
    return k;
}
// whether a lane may take two channels at once
bool recurrence_pairs(int D, int dtype, const wkv_rows *x, const wkv_rows *r, const wkv_rows *i, const wkv_rows *z) {
    for (const wkv_rows *o : {x, r, i, z})
        if (o && (D % 2 || !aligned_to(o->p, 2 * element(dtype)) || o->batch % 2 || o->token % 2)) return false;
    return true;
}

// ---- embedding
int check_embedding(long long count, int V, int C, int dtype, int index_bytes) {
    if (count <= 0 || V <= 0 || C <= 0 || count > (1 << 28) || V > (1 << 24) || C > (1 << 23)) return WKV_ERR_DIMS;
    // (a grid has fewer than 2^32 threads)
    if (count * C >= (1ll << 33) || (long long)V * C >= (1ll << 36)) return WKV_ERR_DIMS;
    if (index_bytes != 4 && index_bytes != 8) return WKV_ERR_DTYPE;
    return dtype_ok(dtype);
}

// ---- gated feed-forward.  256 rows of an operand lie within the 2^31 bytes of a buffer's range.
constexpr int MAX_WIDTH = 1 << 20, MAX_ROWS = 1 << 21;
int check_product(int rows, int C, int F, int dtype, int activation) {
    if (int st = dtype_ok(dtype)) return st;
    if (rows <= 0 || C <= 0 || F <= 0 || rows > MAX_ROWS || C > MAX_WIDTH || F > MAX_WIDTH - ffn::ROUND) return WKV_ERR_DIMS;
    // (a grid of the smallest tiles has fewer than 2^32 threads, as has the one that lays rows out in whole pieces)
    if (C % (16 / (int)element(dtype)) && (rows + 2ll * F) * ffn::rounded(C) >= (1ll << 34)) return WKV_ERR_DIMS;
    if ((long long)rows * F >= (1ll << 35) || (long long)rows * C >= (1ll << 35) || (long long)F * C >= (1ll << 34)) return WKV_ERR_DIMS;
    return activation < 0 || activation >= ffn::ACTIVATIONS ? WKV_ERR_ALGO : WKV_OK;
}
// what is read in whole pieces is aligned to them
int check_pieces(const void *p, long long stride, int C, int dtype) {
    if (!p) return WKV_ERR_NULL;
    if (stride < C || stride > MAX_ROWS) return WKV_ERR_DIMS;          // (256 rows of a tile within 2^31 bytes)
    const bool whole = C % (16 / (int)element(dtype)) == 0;
    return aligned_to(p, whole ? 16 : element(dtype)) && (!whole || stride * element(dtype) % 16 == 0) ? WKV_OK : WKV_ERR_ALIGN;
}

}  // namespace

extern "C" {

size_t wkv_gated_recurrence_checkpoint_bytes(int B, int T, int D, int dtype) {
    return check_recurrence(B, T, D, dtype) ? 0 : gated::checkpoint_bytes(B, T, D);
}
size_t wkv_gated_recurrence_forward_workspace(int B, int T, int D, int dtype) {
    return check_recurrence(B, T, D, dtype) ? 0 : gated::forward_scratch(B, T, D);
}

int wkv_gated_recurrence_forward(void *stream, int B, int T, int D, int dtype, float scale, const wkv_rows *x, const wkv_rows *r, const wkv_rows *i,
                                 const float *decay, const wkv_rows *z, const float *state_in, const int *lengths, void *y, float *state_out,
                                 float *checkpoints, void *workspace, size_t workspace_bytes) {
    if (int st = check_recurrence(B, T, D, dtype)) return st;
    if (int st = check_operands(T, D, dtype, x, r, i, z, decay)) return st;
    if (!y || !state_out) return WKV_ERR_NULL;
    for (const void *p : {(const void *)state_in, (const void *)y, (const void *)state_out, (const void *)checkpoints, (const void *)workspace})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (overlaps(state_in, state_out, (size_t)B * D * 4) && !(T == 1 && !checkpoints && state_in == state_out)) return WKV_ERR_ALIAS;
    const size_t need = gated::forward_scratch(B, T, D);
    if (need && !workspace) return WKV_ERR_NULL;
    if (workspace_bytes < need) return WKV_ERR_WORKSPACE;
    gated::Call k = recurrence_call(B, T, D, scale, x, r, i, z, decay, lengths, checkpoints, workspace);
    k.state_in = state_in; k.y = y; k.state_out = state_out;
    const bool two = recurrence_pairs(D, dtype, x, r, i, z);
#define CALL(TY) gated::forward_t<TY>((hipStream_t)stream, k, two)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_gated_recurrence_backward_workspace(int B, int T, int D, int dtype) {
    return check_recurrence(B, T, D, dtype) ? 0 : gated::backward_scratch(B, T, D);
}

int wkv_gated_recurrence_backward(void *stream, int B, int T, int D, int dtype, float scale, const wkv_rows *x, const wkv_rows *r, const wkv_rows *i,
                                  const float *decay, const wkv_rows *z, const int *lengths, const float *checkpoints, const void *gy, const float *gstate_out,
                                  void *gx, void *gr, void *gi, float *gdecay, void *gz, float *gstate_in, void *workspace, size_t workspace_bytes) {
    if (int st = check_recurrence(B, T, D, dtype)) return st;
    if (int st = check_operands(T, D, dtype, x, r, i, z, decay)) return st;
    if (!checkpoints || !gy || !gx || !gr || !gi || !gdecay || (z && !gz) || !workspace) return WKV_ERR_NULL;
    for (const void *p : {(const void *)checkpoints, gy, (const void *)gstate_out, (const void *)gx, (const void *)gr, (const void *)gi, (const void *)gdecay,
                          (const void *)gz, (const void *)gstate_in, (const void *)workspace})
        if (!aligned16(p)) return WKV_ERR_ALIGN;
    if (overlaps(gstate_out, gstate_in, (size_t)B * D * 4)) return WKV_ERR_ALIAS;
    if (workspace_bytes < gated::backward_scratch(B, T, D)) return WKV_ERR_WORKSPACE;
    gated::Call k = recurrence_call(B, T, D, scale, x, r, i, z, decay, lengths, checkpoints, workspace);
    k.gy = gy; k.gstate_out = gstate_out;
    k.gx = gx; k.gr = gr; k.gi = gi; k.gz = gz; k.gstate_in = gstate_in;
    const bool two = recurrence_pairs(D, dtype, x, r, i, z);
#define CALL(TY) gated::backward_t<TY>((hipStream_t)stream, k, two, gdecay)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

int wkv_embedding_forward(void *stream, long long count, int V, int C, int dtype, int index_bytes, float scale, const void *tokens, const void *table,
                          void *out) {
    if (int st = check_embedding(count, V, C, dtype, index_bytes)) return st;
    if (!tokens || !table || !out) return WKV_ERR_NULL;
    if (!aligned_to(tokens, index_bytes) || !aligned16(table) || !aligned16(out)) return WKV_ERR_ALIGN;
    const embedding::Lookup k = {(size_t)count, V, C, C, scale, tokens, table, out};
    const bool whole = C % (16 / (int)element(dtype)) == 0;
#define CALL(TY) (index_bytes == 8 ? embedding::forward_t<TY, long long>((hipStream_t)stream, k, whole) : embedding::forward_t<TY, int>((hipStream_t)stream, k, whole))
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_embedding_backward_workspace(long long count, int V, int C) {
    return check_embedding(count, V, C, WKV_F32, 4) ? 0 : embedding::regions((int)count, V, C).all;
}

int wkv_embedding_backward(void *stream, long long count, int V, int C, int dtype, int index_bytes, float scale, const void *tokens, const void *gout,
                           long long gout_stride, void *gtable, void *workspace, size_t workspace_bytes) {
    if (int st = check_embedding(count, V, C, dtype, index_bytes)) return st;
    if (!tokens || !gout || !gtable || !workspace) return WKV_ERR_NULL;
    if (!aligned_to(tokens, index_bytes) || !aligned_to(gout, element(dtype)) || !aligned16(gtable) || !aligned16(workspace)) return WKV_ERR_ALIGN;
    if (workspace_bytes < wkv_embedding_backward_workspace(count, V, C)) return WKV_ERR_WORKSPACE;
    embedding::Gradient k = {};
    k.count = (int)count; k.V = V; k.C = C; k.gs = gout_stride; k.scale = scale;
    k.gout = gout; k.out = gtable;
    const bool whole = C % (16 / (int)element(dtype)) == 0 && aligned16(gout) && gout_stride * element(dtype) % 16 == 0;
#define CALL(TY) embedding::backward_t<TY>((hipStream_t)stream, k, tokens, index_bytes == 8, whole, workspace)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_gated_product_kept_bytes(int rows, int C, int F, int dtype) {
    return check_product(rows, C, F, dtype, 0) ? 0 : (size_t)rows * 2 * ffn::rounded(F) * 4;
}
size_t wkv_gated_product_forward_workspace(int rows, int C, int F, int dtype) {
    if (check_product(rows, C, F, dtype, 0)) return 0;
#define CALL(TY) ffn::forward_scratch<TY>(rows, C, F)
    return BY_DTYPE(dtype, CALL);
#undef CALL
}

int wkv_gated_product_forward(void *stream, int rows, int C, int F, int dtype, int activation, const void *x, long long x_stride, const void *w_gate,
                              const void *w_up, void *h, float *kept, void *workspace, size_t workspace_bytes) {
    if (int st = check_product(rows, C, F, dtype, activation)) return st;
    if (!h) return WKV_ERR_NULL;
    if (int st = check_pieces(x, x_stride, C, dtype)) return st;
    for (const void *w : {w_gate, w_up})
        if (int st = check_pieces(w, C, C, dtype)) return st;
    if (!aligned_to(h, 16) || !aligned_to(kept, 16) || !aligned_to(workspace, 16)) return WKV_ERR_ALIGN;
    const size_t need = wkv_gated_product_forward_workspace(rows, C, F, dtype);
    if (need && !workspace) return WKV_ERR_NULL;
    if (workspace_bytes < need) return WKV_ERR_WORKSPACE;
    const ffn::Forward k = {rows, C, F, activation, x, w_gate, w_up, x_stride, C, h, kept, F, ffn::rounded(F)};
#define CALL(TY) ffn::forward_t<TY>((hipStream_t)stream, k, workspace)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

size_t wkv_gated_product_backward_workspace(int rows, int C, int F, int dtype, int want_x, int want_w) {
    if (check_product(rows, C, F, dtype, 0)) return 0;
#define CALL(TY) ffn::regions<TY>(rows, C, F, want_x, want_w).all
    return BY_DTYPE(dtype, CALL);
#undef CALL
}

int wkv_gated_product_backward(void *stream, int rows, int C, int F, int dtype, int activation, const void *x, long long x_stride, const void *w_gate,
                               const void *w_up, const float *kept, const void *gh, void *gx, void *gw_gate, void *gw_up, void *workspace,
                               size_t workspace_bytes) {
    if (int st = check_product(rows, C, F, dtype, activation)) return st;
    if (!kept || !gh || (!gx && !gw_gate) || !gw_gate != !gw_up || !workspace) return WKV_ERR_NULL;
    if (int st = check_pieces(x, x_stride, C, dtype)) return st;
    for (const void *w : {w_gate, w_up})
        if (int st = check_pieces(w, C, C, dtype)) return st;
    for (const void *p : {(const void *)kept, gh, (const void *)gx, (const void *)gw_gate, (const void *)gw_up, (const void *)workspace})
        if (!aligned_to(p, 16)) return WKV_ERR_ALIGN;
    if (workspace_bytes < wkv_gated_product_backward_workspace(rows, C, F, dtype, gx != nullptr, gw_gate != nullptr)) return WKV_ERR_WORKSPACE;
    const ffn::Backward k = {rows, C, F, activation, x, w_gate, w_up, gh, kept, x_stride, C, gx, gw_gate, gw_up};
#define CALL(TY) ffn::backward_t<TY>((hipStream_t)stream, k, workspace)
    return finished(BY_DTYPE(dtype, CALL));
#undef CALL
}

}  // extern "C"
