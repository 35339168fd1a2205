// What stands around the layer in a block - the normalisation with the residual stream, the gated feed-forward block - with and without gradients
// (included by gdn_host.cpp).  Through Python a training step of either took 150 us of host time, whatever the size of the tensors.

// Gradients that a second derivative is asked of raise when it is taken (there are kernels for the first one only).
variable_list differentiable_once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list present;
    for (auto& g : grads)
        if (g.defined()) present.push_back(g.detach().requires_grad_(true));
    if (present.empty()) return grads;
    const auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int)present.size());
    present = (*error)(std::move(present));
    size_t at = 0;
    for (auto& g : grads)
        if (g.defined()) g = present[at++];
    return grads;
}

// A saved tensor as the kernels take it (`saved`), of the type and the number of elements that it had: hooks may have handed back something else.
at::Tensor restored(const at::Tensor& t, at::ScalarType type, c10::Device dev, int64_t elements) {
    TORCH_CHECK_VALUE(!t.defined() || t.numel() == elements, "a saved tensor of ", elements, " elements came back with ", t.numel());
    return saved(t, type, dev);
}

// ---- normalisation ----
struct NormCall {
    int64_t rows, D;
    double eps;
    int w_code;
    bool rms, prenorm, own_stream;     // own_stream: the stream is a tensor of its own, in stream_type
    at::ScalarType stream_type;
};

// y and, where it is a tensor of its own, the stream; mean and rstd where `statistics`
void norm_forward(const NormCall& c, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual, bool statistics,
                  at::Tensor& y, at::Tensor& stream, at::Tensor& mean, at::Tensor& rstd) {
    const c10::Device dev = x.device();
    y = empty_on(dev, x.scalar_type(), x.sizes());
    if (c.own_stream) stream = empty_on(dev, c.stream_type, x.sizes());
    if (statistics) {
        rstd = empty_on(dev, at::kFloat, {c.rows});
        if (!c.rms) mean = empty_on(dev, at::kFloat, {c.rows});
    }
    check_rc(p_layer_norm_fwd(x.data_ptr(), ptr_of(residual), ptr_of(weight), ptr_of(bias), y.data_ptr(), ptr_of(stream), ptr_of<float>(mean), ptr_of<float>(rstd),
                              c.rows, c.D, (float)c.eps, code_of(x.scalar_type()), code_of(c.stream_type), c.w_code, c.rms, stream_of(dev)), "gdn_layer_norm_fwd");
}

struct NormTrain : torch::autograd::Function<NormTrain> {
    typedef std::optional<at::Tensor> Maybe;
    static variable_list forward(AutogradContext* ctx, const Variable& x, const Maybe& weight_, const Maybe& bias_, const Maybe& residual_, const NormCall& c) {
        const at::Tensor weight = weight_.value_or(at::Tensor()), bias = bias_.value_or(at::Tensor()), residual = residual_.value_or(at::Tensor());
        at::Tensor y, stream, mean, rstd;
        norm_forward(c, x, weight, bias, residual, true, y, stream, mean, rstd);
        ctx->save_for_backward({c.own_stream ? stream : x, weight, mean, rstd});
        ctx->saved_data["call"] = std::vector<int64_t>{c.rows, c.D, c.w_code, c.rms, (int64_t)c.stream_type, (int64_t)x.scalar_type(), weight.defined(), bias.defined(),
                                                       residual.defined(), (int64_t)(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : at::kFloat)};
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["device"] = x.device();
        ctx->set_materialize_grads(false);
        if (!c.prenorm) return {y};
        return {y, stream};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const at::Tensor none;
        if (!grads[0].defined() && (grads.size() < 2 || !grads[1].defined())) return {none, none, none, none, none};
        const c10::Device dev = ctx->saved_data["device"].toDevice();
        const c10::DeviceGuard guard(dev);
        const std::vector<int64_t> n = ctx->saved_data["call"].toIntVector(), shape = ctx->saved_data["shape"].toIntVector();
        const int64_t rows = n[0], D = n[1];
        const at::ScalarType stream_type = (at::ScalarType)n[4], type = (at::ScalarType)n[5];
        const at::ScalarType ptype = (at::ScalarType)n[9];            // (weight and bias are of one type)
        auto s = ctx->get_saved_variables();
        s[0] = restored(s[0], stream_type, dev, rows * D);
        s[1] = restored(s[1], ptype, dev, D);
        for (int i = 2; i < 4; ++i) s[i] = restored(s[i], at::kFloat, dev, rows);
        const at::Tensor &r = s[0], &weight = s[1], &mean = s[2], &rstd = s[3];
        // (inputs that were absent have no edge)
        size_t edge = 0;
        const bool need_x = ctx->needs_input_grad(edge++), need_w = n[6] && ctx->needs_input_grad(edge++), need_b = n[7] && ctx->needs_input_grad(edge++),
                   need_res = n[8] && ctx->needs_input_grad(edge++), shared = stream_type == type;
        const at::Tensor dy = grads[0].defined() ? grads[0].to(type).contiguous() : at::zeros(shape, at::TensorOptions().dtype(type).device(dev));
        const at::Tensor dstream = grads.size() > 1 && grads[1].defined() ? grads[1].to(stream_type).contiguous() : none;
        at::Tensor dx, dres, part, dw, db;
        if (need_x || (need_res && shared)) dx = empty_on(dev, type, shape);
        if (need_res && !shared) dres = empty_on(dev, stream_type, shape);
        const int64_t kinds = (int)need_w + (int)need_b, parts = p_layer_norm_bwd_parts(rows, D, code_of(type));
        if (kinds) part = empty_on(dev, at::kFloat, {parts, kinds, D});
        void* stream = stream_of(dev);
        check_rc(p_layer_norm_bwd(dy.data_ptr(), r.data_ptr(), ptr_of(weight), ptr_of<float>(mean), ptr_of<float>(rstd), ptr_of(dstream), ptr_of(dx), ptr_of(dres),
                                  ptr_of<float>(part), rows, D, parts, need_w, need_b, code_of(type), code_of(stream_type), (int)n[2], (int)n[3], stream), "gdn_layer_norm_bwd");
        if (kinds) {
            const at::Tensor sums = sum_rows(part, ptype, {kinds, D}, stream);
            if (need_w) dw = sums.select(0, 0);
            if (need_b) db = sums.select(0, kinds - 1);
        }
        return differentiable_once({need_x ? dx : none, dw, db, need_res ? (shared ? dx : dres) : none, none});
    }
};

// Dual tensors of forward-mode differentiation, with a gradient asked for or not: the Python path refuses them.
bool has_tangent(std::initializer_list<const Arg*> args) {
    for (const Arg* a : args)
        if (*a && (*a)->_fw_grad(0).defined()) return true;
    return false;
}
bool needs_grad(std::initializer_list<const Arg*> args) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Arg* a : args)
        if (*a && (*a)->requires_grad()) return true;
    return false;
}

// (x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm) -> y or (y, stream); None: not a call for the native path
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "gdn_host.layer_norm takes 8 arguments"); return nullptr; }
    const Arg x(a[0]), weight(a[1]), bias(a[2]), residual(a[3]);
    const bool prenorm = truth(a[5]), in_fp32 = truth(a[6]), rms = truth(a[7]);
    if (!x || !x->is_cuda() || x->dim() < 1 || x->numel() == 0 || (!PyFloat_Check(a[4]) && !PyLong_Check(a[4]))) Py_RETURN_NONE;
    const c10::Device dev = x->device();
    const at::ScalarType type = x->scalar_type();
    if (dev.index() != c10::hip::current_device() || !plain(x, dev) || !plain(weight, dev) || !plain(bias, dev) || !plain(residual, dev) || code_of(type) < 0) Py_RETURN_NONE;
    NormCall c{};
    c.D = x->size(-1); c.rows = x->numel() / c.D; c.rms = rms; c.prenorm = prenorm;
    c.eps = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) return nullptr;
    if (c.D * (int64_t)x->element_size() >= GDN_NORM_MAX_ROW_BYTES || c.rows >= (1ll << 31)) Py_RETURN_NONE;
    if (residual && (residual->sizes() != x->sizes() || (residual->scalar_type() != type && residual->scalar_type() != at::kFloat))) Py_RETURN_NONE;
    c.w_code = GDN_DTYPE_F32;
    for (const Arg* p : {&weight, &bias}) {
        if (!*p) continue;
        if ((*p)->dim() != 1 || (*p)->numel() != c.D || ((*p)->scalar_type() != type && (*p)->scalar_type() != at::kFloat)) Py_RETURN_NONE;
        c.w_code = code_of((*p)->scalar_type());
    }
    if (weight && bias && weight->scalar_type() != bias->scalar_type()) Py_RETURN_NONE;
    c.stream_type = residual ? residual->scalar_type() : in_fp32 ? at::kFloat : type;
    c.own_stream = residual || c.stream_type != type;
    if (has_tangent({&x, &weight, &bias, &residual})) Py_RETURN_NONE;
    if (prenorm && !c.own_stream) Py_RETURN_NONE;                  // (the stream is x: the Python path says how it leaves)
    at::Tensor y, stream;
    if (needs_grad({&x, &weight, &bias, &residual})) {
        auto var = [](const Arg& t) { return t ? NormTrain::Maybe(*t.t) : NormTrain::Maybe(); };
        const NoGil free;
        variable_list r = NormTrain::apply(*x.t, var(weight), var(bias), var(residual), c);
        y = r[0];
        if (prenorm) stream = r[1];
    } else {
        at::Tensor mean, rstd;
        auto is = [](const Arg& t) { return t ? *t.t : at::Tensor(); };
        const NoGil free;
        norm_forward(c, *x.t, is(weight), is(bias), is(residual), false, y, stream, mean, rstd);
    }
    return prenorm ? pair(y, stream) : THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// ---- feed-forward block ----
struct MlpDims { int64_t M, D, F; int act, code; };

at::Tensor mlp_workspace(const MlpDims& d, int backward, c10::Device dev) {
    return empty_on(dev, at::kByte, {(int64_t)p_gated_mlp_workspace_bytes(d.M, d.D, d.F, backward)});
}
// The kernels take rows of a multiple of 8 elements: copies with zeros up to there, and cut off again, several matrices in a launch.
int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
struct Resize {
    gdn_pad_segment seg[GDN_PAD_SEGMENTS];
    int n = 0;
    c10::Device dev;
    explicit Resize(c10::Device d) : dev(d) {}
    // t [..][cols] as [rows_to][cols_to]: itself where it is that already
    at::Tensor operator()(const at::Tensor& t, int64_t rows, int64_t cols, int64_t rows_to, int64_t cols_to) {
        if (!t.defined() || (rows == rows_to && cols == cols_to)) return t;
        const at::Tensor out = empty_on(dev, t.scalar_type(), {rows_to, cols_to});
        seg[n++] = {t.data_ptr(), out.data_ptr(), rows, cols, rows_to, cols_to};
        return out;
    }
    void run() {
        if (n) check_rc(p_pad_rows(seg, n, stream_of(dev)), "gdn_pad_rows");
    }
};
// s, a: undefined where no backward follows that needs them; x [M][D]
at::Tensor mlp_forward(const MlpDims& d, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, bool keep, at::Tensor& s, at::Tensor& a, at::Tensor& h) {
    const c10::Device dev = x.device();
    const at::ScalarType type = x.scalar_type();
    const at::Tensor y = empty_on(dev, type, {d.M, d.D}), ws = mlp_workspace(d, 0, dev);
    h = empty_on(dev, type, {d.M, d.F});
    if (keep) { s = empty_on(dev, type, {d.M, d.F}); a = empty_on(dev, type, {d.M, d.F}); }
    check_rc(p_gated_mlp_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), y.data_ptr(), ptr_of(s), ptr_of(a), h.data_ptr(), ws.data_ptr(), (size_t)ws.numel(),
                             d.M, d.D, d.F, d.act, d.code, stream_of(dev)), "gdn_gated_mlp_fwd");
    return y;
}

struct MlpTrain : torch::autograd::Function<MlpTrain> {
    // (x and the weights as they are; d: their sizes as the kernels take them)
    static variable_list forward(AutogradContext* ctx, const Variable& x, const Variable& wg, const Variable& wu, const Variable& wd, const MlpDims& d) {
        const bool need_x = x.requires_grad(), weights = wg.requires_grad() || wu.requires_grad(), inner = need_x || weights;
        const int64_t D = wg.size(1), F = wg.size(0);
        Resize pad(x.device()), cut(x.device());
        const at::Tensor xk = pad(x, d.M, D, d.M, d.D), gk = pad(wg, F, D, d.F, d.D), uk = pad(wu, F, D, d.F, d.D), dk = pad(wd, D, F, d.D, d.F), none;
        pad.run();
        at::Tensor s, a, h;
        const at::Tensor yk = mlp_forward(d, xk, gk, uk, dk, inner, s, a, h), y = cut(yk, d.M, d.D, d.M, D).view(x.sizes());
        cut.run();
        ctx->save_for_backward({weights ? xk : none, need_x ? gk : none, need_x ? uk : none, inner ? dk : none, s, a, wd.requires_grad() ? h : none});
        ctx->saved_data["dims"] = std::vector<int64_t>{d.M, d.D, d.F, d.code, D, F};
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["device"] = x.device();
        ctx->set_materialize_grads(false);
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const at::Tensor none;
        if (!grads[0].defined()) return {none, none, none, none, none};
        const c10::Device dev = ctx->saved_data["device"].toDevice();
        const c10::DeviceGuard guard(dev);
        const std::vector<int64_t> n = ctx->saved_data["dims"].toIntVector(), shape = ctx->saved_data["shape"].toIntVector();
        const MlpDims d{n[0], n[1], n[2], 0, (int)n[3]};
        const at::ScalarType type = d.code == GDN_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
        auto s = ctx->get_saved_variables();
        const int64_t D = n[4], F = n[5], elements[] = {d.M * d.D, d.F * d.D, d.F * d.D, d.D * d.F, d.M * d.F, d.M * d.F, d.M * d.F};
        for (int i = 0; i < 7; ++i) s[i] = restored(s[i], type, dev, elements[i]);
        Resize pad(dev), cut(dev);
        const at::Tensor whole = saved(grads[0], type, dev), dy = pad(whole, d.M, D, d.M, d.D);
        pad.run();
        auto room = [&](bool need, at::IntArrayRef sizes) { return need ? empty_on(dev, type, sizes) : at::Tensor(); };
        const bool need_x = ctx->needs_input_grad(0), need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2), inner = need_x || need_g || need_u;
        const at::Tensor dx = room(need_x, {d.M, d.D}), dwg = room(need_g, {d.F, d.D}), dwu = room(need_u, {d.F, d.D}), dwd = room(ctx->needs_input_grad(3), {d.D, d.F});
        const at::Tensor dg = room(inner, {d.M, d.F}), du = room(inner, {d.M, d.F}), ws = mlp_workspace(d, 1, dev);
        check_rc(p_gated_mlp_bwd(dy.data_ptr(), ptr_of(s[0]), ptr_of(s[1]), ptr_of(s[2]), ptr_of(s[3]), ptr_of(s[4]), ptr_of(s[5]), ptr_of(s[6]), ptr_of(dg), ptr_of(du),
                                 ptr_of(dx), ptr_of(dwg), ptr_of(dwu), ptr_of(dwd), ws.data_ptr(), (size_t)ws.numel(), d.M, d.D, d.F, d.code, stream_of(dev)), "gdn_gated_mlp_bwd");
        const at::Tensor dx1 = cut(dx, d.M, d.D, d.M, D), dwg1 = cut(dwg, d.F, d.D, F, D), dwu1 = cut(dwu, d.F, d.D, F, D), dwd1 = cut(dwd, d.D, d.F, D, F);
        cut.run();
        return differentiable_once({need_x ? dx1.view(shape) : none, dwg1, dwu1, dwd1, none});
    }
};

// (x, gate_weight, up_weight, down_weight, activation code) -> y; None: not a call for the native path
PyObject* gated_mlp(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) { PyErr_SetString(PyExc_TypeError, "gdn_host.gated_mlp takes 5 arguments"); return nullptr; }
    const Arg x(a[0]), wg(a[1]), wu(a[2]), wd(a[3]);
    if (!x || !wg || !wu || !wd || !x->is_cuda() || x->dim() < 1 || x->numel() == 0 || wg->dim() != 2 || wd->dim() != 2) Py_RETURN_NONE;
    const c10::Device dev = x->device();
    const at::ScalarType type = x->scalar_type();
    if (dev.index() != c10::hip::current_device() || (type != at::kBFloat16 && type != at::kHalf)) Py_RETURN_NONE;
    for (const Arg* t : {&x, &wg, &wu, &wd})
        if (!plain(*t, dev) || (*t)->scalar_type() != type) Py_RETURN_NONE;
    const int64_t D = x->size(-1), F = wg->size(0);
    if (wg->size(1) != D || wu->sizes() != wg->sizes() || wd->size(0) != D || wd->size(1) != F || F == 0) Py_RETURN_NONE;
    if (has_tangent({&x, &wg, &wu, &wd})) Py_RETURN_NONE;
    const bool train = needs_grad({&x, &wg, &wu, &wd});
    MlpDims d{};
    d.M = x->numel() / D;
    const bool few = !train && d.M <= GDN_MLP_FEW_ROWS;             // (a step of a few rows: of any width, at any address)
    d.D = few ? D : up8(D); d.F = few ? F : up8(F); d.code = code_of(type);
    d.act = (int)PyLong_AsLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    if (!few)
        for (const Arg* t : {&x, &wg, &wu, &wd})
            if (!aligned16(t->ptr())) Py_RETURN_NONE;
    at::Tensor y;
    if (train) {
        const NoGil free;
        y = MlpTrain::apply(*x.t, *wg.t, *wu.t, *wd.t, d)[0];
    } else {
        at::Tensor s, act, h;
        const NoGil free;
        Resize pad(dev), cut(dev);
        const at::Tensor xk = pad(*x.t, d.M, D, d.M, d.D), gk = pad(*wg.t, F, D, d.F, d.D), uk = pad(*wu.t, F, D, d.F, d.D), dk = pad(*wd.t, D, F, d.D, d.F);
        pad.run();
        const at::Tensor yk = mlp_forward(d, xk, gk, uk, dk, false, s, act, h);
        y = cut(yk, d.M, d.D, d.M, D).view(x->sizes());
        cut.run();
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}
