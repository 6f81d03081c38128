// The state space operators and sampling: checks, allocation and autograd nodes over the entry points of csrc/ssm_api.hip.
// (Part of host.cpp.)

// A new tensor on the current device, straight from its caching allocator: through the dispatcher it takes half as long again, and
// a single token's call makes two or three of them.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
    static c10::Allocator *const allocator = at::cuda::getCUDADeviceAllocator();
    return at::detail::empty_generic(sizes, allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}
Tensor fresh_bytes(size_t n) { return fresh({(int64_t)std::max<size_t>(n, 16)}, at::kByte); }

// ---- operands
void same_device(const Tensor &x, std::initializer_list<const Tensor *> others) {
    on_gpu(x);
    for (const Tensor *t : others) {
        on_gpu(*t);
        REQUIRE(!t->defined() || t->device() == x.device());
    }
}
// what the kernels read in whole pieces
Tensor plain(const Tensor &t) {
    if (!t.defined()) return t;
    const Tensor c = t.contiguous();
    return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}
Tensor plain_float(const Tensor &t) { return t.defined() ? plain(as_float(t)) : t; }
// a parameter: read in fp32 or in the streams' type, whichever it has
Tensor plain_parameter(const Tensor &t, at::ScalarType streams) {
    return !t.defined() || t.scalar_type() == streams ? plain(t) : plain_float(t);
}
// a stream or vector operand: any strides over a contiguous last dimension (a tile's tokens have to lie within 32-bit offsets)
Tensor strided(const Tensor &t) {
    if (!t.defined() || ((t.stride(-1) == 1 || t.size(-1) == 1) && (t.size(1) == 1 || t.stride(1) < (1 << 24)))) return t;
    return t.contiguous();
}
wkv_rows rows_of(const Tensor &t) {
    if (!t.defined()) return wkv_rows{};
    auto step = [&](int64_t d) { return t.size(d) > 1 ? (long long)t.stride(d) : 0; };          // (that of a single element means nothing)
    return wkv_rows{t.data_ptr(), step(0), step(1), t.dim() == 4 ? step(2) : 0};
}
Tensor lengths_of(const Tensor &t, int64_t B) {
    if (!t.defined()) return t;
    REQUIRE(t.dim() == 1 && t.size(0) == B && !t.is_floating_point());
    return as_type(t, at::kInt).contiguous();
}
const int *iptr(const Tensor &t) { return static_cast<const int *>(ptr(t)); }
bool has_shape(const Tensor &t, std::initializer_list<int64_t> shape) { return t.sizes().equals(at::IntArrayRef(shape.begin(), shape.size())); }
// the caller's buffer for a new state: written as it is, so exactly what the kernel writes
void check_out_state(const Tensor &out, std::initializer_list<int64_t> shape, at::ScalarType type, bool recorded) {
    if (!out.defined()) return;
    REQUIRE(!recorded);          // (a backward would need the state it replaces)
    REQUIRE(has_shape(out, shape) && out.scalar_type() == type && out.is_contiguous() && (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15) == 0);
}
// a kernel has written the caller's buffer: whoever saved it for a backward is to notice (inference tensors have no version)
void written(const Tensor &out) {
    if (out.defined() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}
int fits_int(int64_t n) {
    if (n > INT_MAX) raise(PyExc_ValueError, "size out of range");
    return (int)n;
}

// an autograd node's input that may be left out
typedef std::optional<Tensor> Maybe;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor given(const Maybe &t) { return t ? *t : Tensor(); }

// ---- the short causal convolution
class CausalConv : public torch::autograd::Function<CausalConv> {
public:
    // ctx NULL: no gradient is recorded
    static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &weight, const Maybe &bias_, const Maybe &state_, const Maybe &lengths_,
                                 bool silu, const Maybe &out_state_) {
        const Tensor bias = given(bias_), state = given(state_), lengths = given(lengths_), out_state = given(out_state_);
        const Tensor x = strided(x_), s = plain(state);
        // (the kernels take both parameters in one type: fp32 unless both have the streams')
        const bool narrow = weight.scalar_type() == x.scalar_type() && (!bias.defined() || bias.scalar_type() == x.scalar_type());
        const Tensor w = narrow ? plain(weight) : plain_float(weight), b = narrow ? plain(bias) : plain_float(bias);
        const int B = fits_int(x.size(0)), T = fits_int(x.size(1)), D = fits_int(x.size(2)), W = fits_int(w.size(1)), dt = dtype_code(x);
        OnDevice dev(x);
        const Tensor y = fresh({B, T, D}, x.scalar_type()), out = out_state.defined() ? out_state : fresh({B, W - 1, D}, x.scalar_type());
        const wkv_rows rows = rows_of(x);
        check(abi.wkv_causal_conv_forward(dev.stream(), B, T, D, W, dt, dtype_code(w), silu, &rows, ptr(w), ptr(b), ptr(s), iptr(lengths), ptr(y), ptr(out)),
              "wkv_causal_conv_forward");
        if (ctx) {
            ctx->set_materialize_grads(false);
            ctx->saved_data["call"] = std::vector<int64_t>{silu, (int64_t)weight.scalar_type(), bias.defined() ? (int64_t)bias.scalar_type() : 0};
            ctx->save_for_backward({x, w, b, s, lengths});
        }
        return {y, out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const std::vector<int64_t> c = ctx->saved_data["call"].toIntVector();
        const variable_list v = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &x = v[0], &w = v[1], &b = v[2], &s = v[3];
        const int B = x.size(0), T = x.size(1), D = x.size(2), W = w.size(1), dt = dtype_code(x);
        OnDevice dev(x);
        const Tensor gy = grads[0].defined() ? plain(grads[0]) : at::zeros({B, T, D}, x.options()), gout = plain(grads[1]);
        const Tensor gx = fresh({B, T, D}, x.scalar_type()), gw = fresh(w.sizes(), w.scalar_type()), gb = b.defined() ? fresh(b.sizes(), b.scalar_type()) : Tensor();
        const Tensor gs = s.defined() ? fresh(s.sizes(), s.scalar_type()) : Tensor(), ws = fresh_bytes(abi.wkv_causal_conv_backward_workspace(B, T, D, W, dt));
        const wkv_rows rows = rows_of(x);
        check(abi.wkv_causal_conv_backward(dev.stream(), B, T, D, W, dt, dtype_code(w), c[0], &rows, ptr(w), ptr(b), ptr(s), iptr(v[4]), ptr(gy), ptr(gout),
                                           ptr(gx), ptr(gw), ptr(gb), ptr(gs), ptr(ws), ws.numel()), "wkv_causal_conv_backward");
        return {gx, as_type(gw, (at::ScalarType)c[1]), b.defined() ? as_type(gb, (at::ScalarType)c[2]) : Tensor(), gs, Tensor(), Tensor(), Tensor()};
    }
};

// causal_conv(x, weight, bias or None, state or None, lengths or None, silu, out_state or None) -> (y, new_state); None: traced
PyObject *py_causal_conv(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 7);
    if (traced()) Py_RETURN_NONE;
    const Tensor x = tensor(a[0]), w = tensor(a[1]), b = maybe_tensor(a[2]), s = maybe_tensor(a[3]), l = maybe_tensor(a[4]), out = maybe_tensor(a[6]);
    const bool silu = a[5] == Py_True;
    variable_list o;
    {
        NoLock no_lock;
        same_device(x, {&w, &b, &s, &l, &out});
        dtype_code(x);
        REQUIRE(x.dim() == 3 && w.dim() == 2 && w.size(0) == x.size(2));
        REQUIRE(!b.defined() || has_shape(b, {x.size(2)}));
        REQUIRE(!s.defined() || (has_shape(s, {x.size(0), w.size(1) - 1, x.size(2)}) && s.scalar_type() == x.scalar_type()));
        const bool recorded = seen_by_autograd({&x, &w, &b, &s});
        check_out_state(out, {x.size(0), w.size(1) - 1, x.size(2)}, x.scalar_type(), recorded);
        const Tensor lengths = lengths_of(l, x.size(0));
        if (recorded) {
            o = CausalConv::apply(x, w, maybe(b), maybe(s), maybe(lengths), silu, Maybe());
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            o = CausalConv::forward(nullptr, x, w, maybe(b), maybe(s), maybe(lengths), silu, maybe(out));
            written(out);
        }
    }
    return tuple(o[0], o[1]);
    END_HANDLE_TH_ERRORS
}

// ---- the selective scan
enum { SX, SDT, SA, SB, SC, SD, SZ, SBIAS, SSTATE, SCAN_INPUTS };
class SelectiveScan : public torch::autograd::Function<SelectiveScan> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &dt_, const Tensor &A_, const Tensor &B_, const Tensor &C_,
                                 const Maybe &D__, const Maybe &z__, const Maybe &bias__, const Maybe &state__, const Maybe &lengths_, const Maybe &out_state_) {
        const Tensor D_ = given(D__), z_ = given(z__), bias_ = given(bias__), state_ = given(state__), lengths = given(lengths_), out_state = given(out_state_);
        const Tensor x = strided(x_), dt = strided(dt_), z = strided(z_), A = plain_float(A_), skip = plain_float(D_), bias = plain_float(bias_);
        const Tensor b = strided(B_.dim() == 3 ? B_.unsqueeze(2) : B_), c = strided(C_.dim() == 3 ? C_.unsqueeze(2) : C_), s = plain_float(state_);
        const int B = fits_int(x.size(0)), T = fits_int(x.size(1)), D = fits_int(x.size(2)), N = fits_int(A.size(1)), G = fits_int(b.size(2)), t = dtype_code(x);
        OnDevice dev(x);
        const Tensor y = fresh({B, T, D}, x.scalar_type()), out = out_state.defined() ? out_state : fresh({B, D, N}, at::kFloat);
        const Tensor kept = ctx ? fresh_bytes(abi.wkv_selective_scan_checkpoint_bytes(B, T, D, N, G, t)) : Tensor();
        const size_t need = abi.wkv_selective_scan_forward_workspace(B, T, D, N, G, t);
        const Tensor ws = need ? fresh_bytes(need) : Tensor();
        const wkv_rows rx = rows_of(x), rdt = rows_of(dt), rz = rows_of(z), rb = rows_of(b), rc = rows_of(c);
        check(abi.wkv_selective_scan_forward(dev.stream(), B, T, D, N, G, t, &rx, &rdt, fptr(A), &rb, &rc, fptr(skip), z.defined() ? &rz : nullptr, fptr(bias),
                                             fptr(s), iptr(lengths), ptr(y), fptr(out), fptr(kept), ptr(ws), need), "wkv_selective_scan_forward");
        if (ctx) {
            ctx->set_materialize_grads(false);
            auto type = [](const Tensor &v) { return v.defined() ? (int64_t)v.scalar_type() : 0; };
            ctx->saved_data["call"] = std::vector<int64_t>{type(A_), type(D_), type(bias_), type(state_), B_.dim(), state_.defined() && state_.requires_grad()};
            ctx->save_for_backward({x, dt, A, b, c, skip, z, bias, lengths, kept});
        }
        return {y, out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const std::vector<int64_t> k = ctx->saved_data["call"].toIntVector();
        const variable_list v = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &x = v[0], &dt = v[1], &A = v[2], &b = v[3], &c = v[4], &skip = v[5], &z = v[6], &bias = v[7], &lengths = v[8], &kept = v[9];
        const int B = x.size(0), T = x.size(1), D = x.size(2), N = A.size(1), G = b.size(2), t = dtype_code(x);
        OnDevice dev(x);
        auto like_x = [&] { return fresh({B, T, D}, x.scalar_type()); };
        const Tensor gy = grads[0].defined() ? plain(grads[0]) : at::zeros({B, T, D}, x.options()), gout = plain_float(grads[1]);
        const Tensor gx = like_x(), gdt = like_x(), gz = z.defined() ? like_x() : Tensor(), gA = fresh(A.sizes(), at::kFloat);
        const Tensor gb = fresh({B, T, G, N}, x.scalar_type()), gc = fresh({B, T, G, N}, x.scalar_type());
        const Tensor gskip = skip.defined() ? fresh(skip.sizes(), at::kFloat) : Tensor(), gbias = bias.defined() ? fresh(bias.sizes(), at::kFloat) : Tensor();
        const Tensor gs = k[5] ? fresh({B, D, N}, at::kFloat) : Tensor();
        const Tensor ws = fresh_bytes(abi.wkv_selective_scan_backward_workspace(B, T, D, N, G, t));
        const wkv_rows rx = rows_of(x), rdt = rows_of(dt), rz = rows_of(z), rb = rows_of(b), rc = rows_of(c);
        check(abi.wkv_selective_scan_backward(dev.stream(), B, T, D, N, G, t, &rx, &rdt, fptr(A), &rb, &rc, fptr(skip), z.defined() ? &rz : nullptr, fptr(bias),
                                              iptr(lengths), fptr(kept), ptr(gy), fptr(gout), ptr(gx), ptr(gdt), fptr(gA), ptr(gb), ptr(gc), fptr(gskip),
                                              ptr(gz), fptr(gbias), fptr(gs), ptr(ws), ws.numel()), "wkv_selective_scan_backward");
        auto back = [&](const Tensor &g, int i) { return g.defined() ? as_type(g, (at::ScalarType)k[i]) : g; };
        const bool three = k[4] == 3;
        return {gx, gdt, back(gA, 0), three ? gb.squeeze(2) : gb, three ? gc.squeeze(2) : gc, back(gskip, 1), gz, back(gbias, 2), back(gs, 3), Tensor(), Tensor()};
    }
};

// selective_scan(x, dt, A, B, C, D or None, z or None, dt_bias or None, state or None, lengths or None, out_state or None) -> (y, new_state); None: traced
PyObject *py_selective_scan(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 11);
    if (traced()) Py_RETURN_NONE;
    Tensor v[SCAN_INPUTS];
    for (int i = 0; i < SCAN_INPUTS; i++) v[i] = i <= SC ? tensor(a[i]) : maybe_tensor(a[i]);
    const Tensor l = maybe_tensor(a[9]), out = maybe_tensor(a[10]);
    variable_list o;
    {
        NoLock no_lock;
        const Tensor &x = v[SX];
        same_device(x, {&v[SDT], &v[SA], &v[SB], &v[SC], &v[SD], &v[SZ], &v[SBIAS], &v[SSTATE], &l, &out});
        dtype_code(x);
        REQUIRE(x.dim() == 3 && v[SA].dim() == 2 && v[SA].size(0) == x.size(2));
        const int64_t B = x.size(0), T = x.size(1), D = x.size(2), N = v[SA].size(1);
        for (int i : {SDT, SZ}) REQUIRE(!v[i].defined() || (v[i].sizes().equals(x.sizes()) && v[i].scalar_type() == x.scalar_type()));
        for (int i : {SB, SC})
            REQUIRE((v[i].dim() == 3 || v[i].dim() == 4) && v[i].size(0) == B && v[i].size(1) == T && v[i].size(-1) == N && v[i].scalar_type() == x.scalar_type());
        REQUIRE(v[SB].sizes().equals(v[SC].sizes()));
        for (int i : {SD, SBIAS}) REQUIRE(!v[i].defined() || has_shape(v[i], {D}));
        REQUIRE(!v[SSTATE].defined() || has_shape(v[SSTATE], {B, D, N}));
        const bool recorded = seen_by_autograd({&v[0], &v[1], &v[2], &v[3], &v[4], &v[5], &v[6], &v[7], &v[8]});
        check_out_state(out, {B, D, N}, at::kFloat, recorded);
        const Tensor lengths = lengths_of(l, B);
        if (recorded) {
            o = SelectiveScan::apply(v[0], v[1], v[2], v[3], v[4], maybe(v[5]), maybe(v[6]), maybe(v[7]), maybe(v[8]), maybe(lengths), Maybe());
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            o = SelectiveScan::forward(nullptr, v[0], v[1], v[2], v[3], v[4], maybe(v[5]), maybe(v[6]), maybe(v[7]), maybe(v[8]), maybe(lengths), maybe(out));
            written(out);
        }
    }
    return tuple(o[0], o[1]);
    END_HANDLE_TH_ERRORS
}

// ---- the residual's addition and the norm
// rows of C elements at one distance, or a copy that has them
Tensor as_rows(const Tensor &t) {
    if (!t.defined()) return t;
    const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
int64_t row_stride(const Tensor &t) { return t.defined() ? t.stride(0) : 0; }
struct NormOperands {
    Tensor x, residual, weight;
    int rows, C, dt, rt, wt;
    NormOperands(const Tensor &x_, const Tensor &weight_, const Tensor &residual_)
        : x(as_rows(x_)), residual(as_rows(residual_)), weight(plain_parameter(weight_, x_.scalar_type())) {
        rows = fits_int(x.size(0)); C = fits_int(x.size(1));
        dt = dtype_code(x); wt = dtype_code(weight);
        rt = residual.defined() ? dtype_code(residual) : dt;
    }
};
class RmsNorm : public torch::autograd::Function<RmsNorm> {
public:
    // (y), or (y, sum) where there is a residual
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Maybe &residual_, double eps) {
        const Tensor residual = given(residual_);
        const NormOperands v(x, weight, residual);
        OnDevice dev(v.x);
        const Tensor y = fresh(x.sizes(), x.scalar_type()), sum = residual.defined() ? fresh(residual.sizes(), residual.scalar_type()) : Tensor();
        const Tensor rstd = ctx ? fresh({v.rows}, at::kFloat) : Tensor();
        check(abi.wkv_rms_norm_forward(dev.stream(), v.rows, v.C, v.dt, v.rt, v.wt, (float)eps, ptr(v.x), row_stride(v.x), ptr(v.residual),
                                       row_stride(v.residual), ptr(v.weight), ptr(y), nullptr, nullptr, ptr(sum), fptr(rstd)), "wkv_rms_norm_forward");
        if (ctx) {
            // an fp32 sum is what was normalised; a rounded one is not, and is added up again
            const bool whole = residual.defined() && residual.scalar_type() == at::kFloat;
            ctx->set_materialize_grads(false);
            ctx->saved_data["call"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)weight.scalar_type(), residual.defined()};
            ctx->save_for_backward({whole ? Tensor() : x, whole ? sum : residual, v.weight, rstd});
        }
        if (residual.defined()) return {y, sum};
        return {y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const std::vector<int64_t> k = ctx->saved_data["call"].toIntVector();
        const variable_list saved = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const at::ScalarType type = (at::ScalarType)k[0];
        const bool has_residual = k[2];
        const Tensor &weight = saved[2], &rstd = saved[3], &some = saved[0].defined() ? saved[0] : saved[1];
        const Tensor x = as_rows(saved[0]), residual = as_rows(saved[1]);
        OnDevice dev(some);
        const auto options = some.options().dtype(type);
        const Tensor gy = grads[0].defined() ? plain(grads[0]) : at::zeros(some.sizes(), options), gsum = has_residual ? plain(grads[1]) : Tensor();
        const Tensor gx = fresh(some.sizes(), type), gw = fresh(weight.sizes(), weight.scalar_type());
        const bool two = has_residual && saved[1].scalar_type() != type;
        const Tensor gres = two ? fresh(some.sizes(), saved[1].scalar_type()) : has_residual ? gx : Tensor();
        const int C = weight.size(0), R = rstd.size(0);
        const Tensor ws = fresh_bytes(abi.wkv_rms_norm_backward_workspace(R, C));
        check(abi.wkv_rms_norm_backward(dev.stream(), R, C, dtype_code(gx), has_residual ? dtype_code(saved[1]) : dtype_code(gx), dtype_code(weight), ptr(x),
                                        row_stride(x), ptr(residual), row_stride(residual), ptr(weight), fptr(rstd), ptr(gy), ptr(gsum), ptr(gx),
                                        two ? ptr(gres) : nullptr, ptr(gw), ptr(ws), ws.numel()), "wkv_rms_norm_backward");
        return {gx, as_type(gw, (at::ScalarType)k[1]), gres, Tensor()};
    }
};
void check_norm(const Tensor &x, const Tensor &weight, const Tensor &residual) {
    same_device(x, {&weight, &residual});
    dtype_code(x);
    REQUIRE(x.dim() >= 1 && x.numel() > 0 && has_shape(weight, {x.size(-1)}));
    REQUIRE(!residual.defined() || (residual.sizes().equals(x.sizes()) &&
                                    (residual.scalar_type() == x.scalar_type() || residual.scalar_type() == at::kFloat)));
}
double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

// rms_norm(x, weight, eps, residual or None) -> (y, the sum, or x itself); None: traced
PyObject *py_rms_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 4);
    if (traced()) Py_RETURN_NONE;
    const Tensor x = tensor(a[0]), w = tensor(a[1]), r = maybe_tensor(a[3]);
    const double eps = number(a[2]);
    variable_list o;
    {
        NoLock no_lock;
        check_norm(x, w, r);
        if (seen_by_autograd({&x, &w, &r})) {
            o = RmsNorm::apply(x, w, maybe(r), eps);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            o = RmsNorm::forward(nullptr, x, w, maybe(r), eps);
        }
    }
    return tuple(o[0], o.size() > 1 ? o[1] : x);
    END_HANDLE_TH_ERRORS
}

// rms_norm_fp8(x, weight, eps, residual or None) -> (q, scale, the sum, or x itself); None: traced
PyObject *py_rms_norm_fp8(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 4);
    if (traced()) Py_RETURN_NONE;
    const Tensor x = tensor(a[0]), w = tensor(a[1]), r = maybe_tensor(a[3]);
    const double eps = number(a[2]);
    Tensor q, scale, sum;
    {
        NoLock no_lock;
        check_norm(x, w, r);
        if (seen_by_autograd({&x, &w, &r})) raise(wkv_error, "rms_norm_fp8 has no gradient: call it under torch.no_grad()");
        at::AutoDispatchBelowADInplaceOrView below;
        const NormOperands v(x, w, r);
        OnDevice dev(v.x);
        std::vector<int64_t> one = x.sizes().vec();
        one.back() = 1;
        q = fresh(x.sizes(), at::kFloat8_e4m3fn);
        scale = fresh(one, at::kFloat);
        sum = r.defined() ? fresh(r.sizes(), r.scalar_type()) : Tensor();
        check(abi.wkv_rms_norm_forward(dev.stream(), v.rows, v.C, v.dt, v.rt, v.wt, (float)eps, ptr(v.x), row_stride(v.x), ptr(v.residual),
                                       row_stride(v.residual), ptr(v.weight), nullptr, ptr(q), fptr(scale), ptr(sum), nullptr), "wkv_rms_norm_forward");
    }
    return tuple(q, scale, r.defined() ? sum : x);
    END_HANDLE_TH_ERRORS
}

// ---- sampling
// a setting: one number for all rows or a tensor with one per row
struct Setting {
    Tensor rows;
    double value = 0.0;
    Setting(PyObject *o) {
        if (THPVariable_Check(o)) rows = THPVariable_Unpack(o);
        else value = number(o);
    }
    void settle(const Tensor &logits, at::ScalarType type) {
        if (!rows.defined()) return;
        REQUIRE(rows.is_cuda() && rows.device() == logits.device() && has_shape(rows, {logits.size(0)}));
        rows = as_type(rows.detach(), type).contiguous();
    }
};

// sample(logits, u, temperature, top_k, top_p, min_p) -> (tokens, logprobs); None: traced
PyObject *py_sample(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 6);
    if (traced()) Py_RETURN_NONE;
    Tensor l = tensor(a[0]), u = tensor(a[1]);
    Setting temperature(a[2]), top_k(a[3]), top_p(a[4]), min_p(a[5]);
    Tensor token, logprob;
    {
        NoLock no_lock;
        same_device(l, {&u});
        if (seen_by_autograd({&l})) raise(wkv_error, "sample has no gradient: call it under torch.no_grad() or with logits.detach()");
        at::AutoDispatchBelowADInplaceOrView below;
        const int dt = dtype_code(l);
        REQUIRE(l.dim() == 2 && has_shape(u, {l.size(0)}));
        OnDevice dev(l);
        l = l.stride(1) == 1 || l.size(1) == 1 ? l : l.contiguous();
        u = as_float(u).contiguous();
        for (Setting *s : {&temperature, &top_p, &min_p}) s->settle(l, at::kFloat);
        top_k.settle(l, at::kInt);
        const int rows = fits_int(l.size(0));
        token = fresh({rows}, at::kLong);
        logprob = fresh({rows}, at::kFloat);
        check(abi.wkv_sample(dev.stream(), rows, fits_int(l.size(1)), dt, ptr(l), l.stride(0), fptr(u), fptr(temperature.rows), (float)temperature.value,
                             iptr(top_k.rows), (int)std::max(0.0, std::min(top_k.value, 2147483647.0)), fptr(top_p.rows), (float)top_p.value, fptr(min_p.rows),
                             (float)min_p.value, static_cast<long long *>(ptr(token)), fptr(logprob)), "wkv_sample");
    }
    return tuple(token, logprob);
    END_HANDLE_TH_ERRORS
}
