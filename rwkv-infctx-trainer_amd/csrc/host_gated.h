// The operators of a gated recurrence model: checks, allocation and autograd nodes over the entry points of csrc/gated_api.hip.
// (Part of host.cpp, after host_ssm.h.)

// ---- the gated linear recurrence
// as strided(), and a token's row behind the one before it
Tensor apart(const Tensor &t) {
    const Tensor s = strided(t);
    return s.defined() && s.size(1) > 1 && s.stride(1) < s.size(2) ? s.contiguous() : s;
}
enum { GX, GR, GI, GDECAY, GZ, GSTATE, RECURRENCE_INPUTS };
class GatedRecurrence : public torch::autograd::Function<GatedRecurrence> {
public:
    // ctx NULL: no gradient is recorded
    static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &r_, const Tensor &i_, const Tensor &decay_, const Maybe &z__, const Maybe &state__,
                                 const Maybe &lengths_, double scale, const Maybe &out_state_) {
        const Tensor z_ = given(z__), state_ = given(state__), lengths = given(lengths_), out_state = given(out_state_);
        const Tensor x = apart(x_), r = apart(r_), i = apart(i_), z = apart(z_), decay = plain_float(decay_), s = plain_float(state_);
        const int B = fits_int(x.size(0)), T = fits_int(x.size(1)), D = fits_int(x.size(2)), dt = dtype_code(x);
        OnDevice dev(x);
        const Tensor y = fresh({B, T, D}, x.scalar_type()), out = out_state.defined() ? out_state : fresh({B, D}, at::kFloat);
        const Tensor kept = ctx ? fresh_bytes(abi.wkv_gated_recurrence_checkpoint_bytes(B, T, D, dt)) : Tensor();
        const size_t need = abi.wkv_gated_recurrence_forward_workspace(B, T, D, dt);
        const Tensor ws = need ? fresh_bytes(need) : Tensor();
        const wkv_rows rx = rows_of(x), rr = rows_of(r), ri = rows_of(i), rz = rows_of(z);
        check(abi.wkv_gated_recurrence_forward(dev.stream(), B, T, D, dt, (float)scale, &rx, &rr, &ri, fptr(decay), z.defined() ? &rz : nullptr, fptr(s), iptr(lengths),
                                               ptr(y), fptr(out), fptr(kept), ptr(ws), need), "wkv_gated_recurrence_forward");
        if (ctx) {
            ctx->set_materialize_grads(false);
            ctx->saved_data["call"] = std::vector<int64_t>{(int64_t)decay_.scalar_type(), state_.defined() ? (int64_t)state_.scalar_type() : 0,
                                                           state_.defined() && state_.requires_grad()};
            ctx->saved_data["scale"] = scale;
            ctx->save_for_backward({x, r, i, decay, z, lengths, kept});
        }
        return {y, out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const std::vector<int64_t> c = ctx->saved_data["call"].toIntVector();
        const double scale = ctx->saved_data["scale"].toDouble();
        const variable_list v = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &x = v[0], &r = v[1], &i = v[2], &decay = v[3], &z = v[4], &lengths = v[5], &kept = v[6];
        const int B = x.size(0), T = x.size(1), D = x.size(2), dt = dtype_code(x);
        OnDevice dev(x);
        auto like_x = [&] { return fresh({B, T, D}, x.scalar_type()); };
        const Tensor gy = grads[0].defined() ? plain(grads[0]) : at::zeros({B, T, D}, x.options()), gout = plain_float(grads[1]);
        const Tensor gx = like_x(), gr = like_x(), gi = like_x(), gz = z.defined() ? like_x() : Tensor(), gd = fresh({D}, at::kFloat);
        const Tensor gs = c[2] ? fresh({B, D}, at::kFloat) : Tensor(), ws = fresh_bytes(abi.wkv_gated_recurrence_backward_workspace(B, T, D, dt));
        const wkv_rows rx = rows_of(x), rr = rows_of(r), ri = rows_of(i), rz = rows_of(z);
        check(abi.wkv_gated_recurrence_backward(dev.stream(), B, T, D, dt, (float)scale, &rx, &rr, &ri, fptr(decay), z.defined() ? &rz : nullptr, iptr(lengths),
                                                fptr(kept), ptr(gy), fptr(gout), ptr(gx), ptr(gr), ptr(gi), fptr(gd), ptr(gz), fptr(gs), ptr(ws), ws.numel()),
              "wkv_gated_recurrence_backward");
        return {gx, gr, gi, as_type(gd, (at::ScalarType)c[0]), gz, gs.defined() ? as_type(gs, (at::ScalarType)c[1]) : gs, Tensor(), Tensor(), Tensor()};
    }
};

// gated_recurrence(x, r, i, decay, z or None, state or None, lengths or None, scale, out_state or None) -> (y, new_state); None: traced
PyObject *py_gated_recurrence(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 9);
    if (traced()) Py_RETURN_NONE;
    Tensor v[RECURRENCE_INPUTS];
    for (int j = 0; j < RECURRENCE_INPUTS; j++) v[j] = j <= GDECAY ? tensor(a[j]) : maybe_tensor(a[j]);
    const Tensor l = maybe_tensor(a[6]), out = maybe_tensor(a[8]);
    const double scale = number(a[7]);
    variable_list o;
    {
        NoLock no_lock;
        const Tensor &x = v[GX];
        same_device(x, {&v[GR], &v[GI], &v[GDECAY], &v[GZ], &v[GSTATE], &l, &out});
        dtype_code(x);
        REQUIRE(x.dim() == 3 && has_shape(v[GDECAY], {x.size(2)}));
        for (int j : {GR, GI, GZ}) REQUIRE(!v[j].defined() || (v[j].sizes().equals(x.sizes()) && v[j].scalar_type() == x.scalar_type()));
        REQUIRE(!v[GSTATE].defined() || has_shape(v[GSTATE], {x.size(0), x.size(2)}));
        const bool recorded = seen_by_autograd({&v[0], &v[1], &v[2], &v[3], &v[4], &v[5]});
        check_out_state(out, {x.size(0), x.size(2)}, at::kFloat, recorded);
        const Tensor lengths = lengths_of(l, x.size(0));
        if (recorded) {
            o = GatedRecurrence::apply(x, v[GR], v[GI], v[GDECAY], maybe(v[GZ]), maybe(v[GSTATE]), maybe(lengths), scale, Maybe());
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            o = GatedRecurrence::forward(nullptr, x, v[GR], v[GI], v[GDECAY], maybe(v[GZ]), maybe(v[GSTATE]), maybe(lengths), scale, maybe(out));
            written(out);
        }
    }
    return tuple(o[0], o[1]);
    END_HANDLE_TH_ERRORS
}

// ---- rows of a table by token
class Embedding : public torch::autograd::Function<Embedding> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &tokens_, const Tensor &table_, double scale) {
        const Tensor tokens = tokens_.contiguous(), table = plain(table_);
        const int V = fits_int(table.size(0)), C = fits_int(table.size(1));
        OnDevice dev(table);
        std::vector<int64_t> shape = tokens.sizes().vec();
        shape.push_back(C);
        const Tensor out = fresh(shape, table.scalar_type());
        check(abi.wkv_embedding_forward(dev.stream(), tokens.numel(), V, C, dtype_code(table), (int)tokens.element_size(), (float)scale, ptr(tokens), ptr(table),
                                        ptr(out)), "wkv_embedding_forward");
        if (ctx) {
            ctx->saved_data["call"] = std::vector<int64_t>{V, C, (int64_t)table.scalar_type()};
            ctx->saved_data["scale"] = scale;
            ctx->save_for_backward({tokens});
        }
        return {out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const std::vector<int64_t> c = ctx->saved_data["call"].toIntVector();
        const double scale = ctx->saved_data["scale"].toDouble();
        const Tensor tokens = ctx->get_saved_variables()[0];
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor g = as_rows(grads[0]);
        const int V = (int)c[0], C = (int)c[1];
        OnDevice dev(tokens);
        const Tensor gt = fresh({V, C}, (at::ScalarType)c[2]), ws = fresh_bytes(abi.wkv_embedding_backward_workspace(tokens.numel(), V, C));
        check(abi.wkv_embedding_backward(dev.stream(), tokens.numel(), V, C, dtype_code(gt), (int)tokens.element_size(), (float)scale, ptr(tokens), ptr(g),
                                         row_stride(g), ptr(gt), ptr(ws), ws.numel()), "wkv_embedding_backward");
        return {Tensor(), gt, Tensor()};
    }
};

// embedding(tokens, table, scale) -> rows; None: traced
PyObject *py_embedding(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 3);
    if (traced()) Py_RETURN_NONE;
    const Tensor tokens = tensor(a[0]), table = tensor(a[1]);
    const double scale = number(a[2]);
    variable_list o;
    {
        NoLock no_lock;
        same_device(table, {&tokens});
        dtype_code(table);
        REQUIRE(table.dim() == 2 && tokens.numel() > 0 && (tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt));
        if (seen_by_autograd({&table})) {
            o = Embedding::apply(tokens, table, scale);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            o = Embedding::forward(nullptr, tokens, table, scale);
        }
    }
    return wrapped(o[0]);
    END_HANDLE_TH_ERRORS
}

// ---- the gated feed-forward's first half
// rows of C elements that the kernels may read in whole pieces of 16 bytes where C is made of them
Tensor whole_rows(const Tensor &t) {
    const Tensor r = as_rows(t);
    const int64_t size = r.element_size(), C = r.size(1);
    if (r.size(0) > 1 && (r.stride(0) < C || r.stride(0) > (1 << 21))) return plain(r);          // (rows that share memory, or lie too far apart)
    const bool there = (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) == 0 && (r.size(0) == 1 || r.stride(0) * size % 16 == 0);
    return C * size % 16 != 0 || there ? r : plain(r);
}
// (that of a single row means nothing)
int64_t whole_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
class GatedProduct : public torch::autograd::Function<GatedProduct> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_gate, const Tensor &w_up, int64_t activation) {
        const Tensor x = whole_rows(x_), wg = plain(w_gate), wu = plain(w_up);
        const int R = fits_int(x.size(0)), C = fits_int(x.size(1)), F = fits_int(wg.size(0)), dt = dtype_code(x);
        OnDevice dev(x);
        std::vector<int64_t> shape = x_.sizes().vec();
        shape.back() = F;
        const Tensor h = fresh(shape, x.scalar_type()), kept = ctx ? fresh_bytes(abi.wkv_gated_product_kept_bytes(R, C, F, dt)) : Tensor();
        const size_t need = abi.wkv_gated_product_forward_workspace(R, C, F, dt);
        const Tensor ws = need ? fresh_bytes(need) : Tensor();
        check(abi.wkv_gated_product_forward(dev.stream(), R, C, F, dt, (int)activation, ptr(x), whole_stride(x), ptr(wg), ptr(wu), ptr(h), fptr(kept), ptr(ws), need),
              "wkv_gated_product_forward");
        if (ctx) {
            ctx->saved_data["call"] = std::vector<int64_t>{activation};
            ctx->saved_data["shape"] = x_.sizes().vec();
            ctx->save_for_backward({x, wg, wu, kept});
        }
        return {h};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const int activation = (int)ctx->saved_data["call"].toIntVector()[0];
        const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
        const variable_list v = ctx->get_saved_variables();
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor &x = v[0], &wg = v[1], &wu = v[2], &kept = v[3];
        const int R = x.size(0), C = x.size(1), F = wg.size(0), dt = dtype_code(x);
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
        OnDevice dev(x);
        const Tensor gh = plain(grads[0]);
        const Tensor gx = want_x ? fresh(shape, x.scalar_type()) : Tensor(), gg = want_w ? fresh({F, C}, x.scalar_type()) : Tensor();
        const Tensor gu = want_w ? fresh({F, C}, x.scalar_type()) : Tensor();
        const Tensor ws = fresh_bytes(abi.wkv_gated_product_backward_workspace(R, C, F, dt, want_x, want_w));
        check(abi.wkv_gated_product_backward(dev.stream(), R, C, F, dt, activation, ptr(x), whole_stride(x), ptr(wg), ptr(wu), fptr(kept), ptr(gh), ptr(gx), ptr(gg),
                                             ptr(gu), ptr(ws), ws.numel()), "wkv_gated_product_backward");
        return {gx, gg, gu, Tensor()};
    }
};

// Operands of different types under autocast, as fp32 weights behind a projection's 16-bit output are: in autocast's type, as torch.nn.functional.linear takes them (a weight's
// copy is kept for as long as autocast keeps it, but none made where no gradient is recorded: a recorded call after it would take that copy and lose the gradient).  Operands of
// one type are taken as they come.
void cast_by_autocast(std::initializer_list<Tensor *> operands) {
    if (!at::autocast::is_autocast_enabled(at::kCUDA)) return;
    const at::ScalarType first = (*operands.begin())->scalar_type();
    if (std::all_of(operands.begin(), operands.end(), [&](const Tensor *t) { return t->scalar_type() == first; })) return;
    const at::ScalarType type = at::autocast::get_autocast_dtype(at::kCUDA);
    for (Tensor *t : operands) {
        if (at::GradMode::is_enabled()) *t = at::autocast::cached_cast(type, *t, at::kCUDA);
        else if (t->is_floating_point() && t->scalar_type() != at::kDouble) *t = as_type(*t, type);
    }
}

// gated_product(x, w_gate, w_up, activation) -> h; None: traced
PyObject *py_gated_product(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 4);
    if (traced()) Py_RETURN_NONE;
    Tensor x = tensor(a[0]), wg = tensor(a[1]), wu = tensor(a[2]);
    const int activation = integer(a[3]);
    variable_list o;
    {
        NoLock no_lock;
        same_device(x, {&wg, &wu});
        cast_by_autocast({&x, &wg, &wu});
        dtype_code(x);
        REQUIRE(x.dim() >= 1 && x.numel() > 0 && wg.dim() == 2 && wg.size(1) == x.size(-1) && wu.sizes().equals(wg.sizes()));
        REQUIRE(wg.scalar_type() == x.scalar_type() && wu.scalar_type() == x.scalar_type());
        if (seen_by_autograd({&x, &wg, &wu})) {
            o = GatedProduct::apply(x, wg, wu, activation);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            o = GatedProduct::forward(nullptr, x, wg, wu, activation);
        }
    }
    return wrapped(o[0]);
    END_HANDLE_TH_ERRORS
}
