// A serving step over a paged cache - rotary positions (with gradients), the cache's upkeep, attention, verification of drafts - for the calls that need no conversion
// (included by gdn_host.cpp).  Through Python and ctypes a call took 15 to 25 us of host time, of which the kernels of a step are three to ten.

// Present or absent, on this device; of any strides.
bool placed(const Arg& a, c10::Device dev) { return !a.bad && (!a || a->device() == dev); }
bool in_rows(const at::Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1; }
bool whole_numbers(const Arg& a, at::IntArrayRef shape) {
    return a && a->is_contiguous() && a->sizes() == shape && (a->scalar_type() == at::kInt || a->scalar_type() == at::kLong);
}
bool is_int32(const at::Tensor& t) { return t.defined() && t.scalar_type() == at::kInt; }
at::Tensor tensor_of(const Arg& a) { return a ? *a.t : at::Tensor(); }
// An index out of Python: -1 with no error set is not one for this path.
bool int_of(PyObject* o, int64_t& to) {
    if (!PyLong_CheckExact(o)) return false;
    to = PyLong_AsLongLong(o);
    if (PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}
void changed(const Arg& a) {
    if (!a->is_inference()) a->unsafeGetTensorImpl()->bump_version();
}

// ---- rotary positions ----
gdn_rotary_rows rotary_rows(const at::Tensor& x, const at::Tensor& y) {
    gdn_rotary_rows r = {x.data_ptr(), y.defined() ? y.data_ptr() : nullptr, x.size(2), {}, {}};
    for (int i = 0; i < 3; ++i) { r.x_stride[i] = x.stride(i); r.y_stride[i] = y.defined() ? y.stride(i) : 0; }
    return r;
}
struct RotaryTables { at::Tensor cos, sin, positions, offsets, cu; int64_t offset = 0; bool interleaved = false, back = false; };
gdn_rotary_call rotary_call(const RotaryTables& t, const at::Tensor& x) {
    gdn_rotary_call c = {};
    c.cos = ptr_of(t.cos); c.sin = ptr_of(t.sin); c.positions = ptr_of(t.positions); c.offsets = ptr_of(t.offsets); c.cu_seqlens = ptr_of(t.cu);
    c.offset = t.offset; c.B = x.size(0); c.T = x.size(1); c.D = x.size(3); c.N = t.cu.defined() ? t.cu.numel() - 1 : c.B;
    c.dtype = c.table_dtype = code_of(x.scalar_type());
    if (t.cos.defined()) { c.table_rows = t.cos.size(0); c.table_stride = t.cos.stride(0); c.rotary_dim = 2 * t.cos.size(1); c.table_dtype = code_of(t.cos.scalar_type()); }
    c.flags = (t.interleaved ? GDN_ROTARY_INTERLEAVED : 0) | (t.back ? GDN_ROTARY_BACK : 0) | (is_int32(t.positions) ? GDN_ROTARY_POSITIONS_INT32 : 0) |
              (is_int32(t.offsets) ? GDN_ROTARY_OFFSETS_INT32 : 0) | (is_int32(t.cu) ? GDN_FLAG_CU_INT32 : 0);
    return c;
}
variable_list turn(const RotaryTables& t, const variable_list& xs) {
    gdn_rotary_rows rows[2];
    variable_list ys;
    for (auto& x : xs) {
        ys.push_back(empty_on(x.device(), x.scalar_type(), x.sizes()));
        rows[ys.size() - 1] = rotary_rows(x, ys.back());
    }
    const gdn_rotary_call c = rotary_call(t, xs[0]);
    check_rc(p_rotary(rows, (int)xs.size(), &c, stream_of(xs[0].device())), "gdn_rotary");
    return ys;
}

// The gradient is the turn back: this function again, and so differentiable itself.
struct RotaryTrain : torch::autograd::Function<RotaryTrain> {
    typedef std::optional<at::Tensor> Maybe;
    static variable_list forward(AutogradContext* ctx, const Variable& a, const Maybe& b, const RotaryTables& t) {
        variable_list xs = {a};
        if (b) xs.push_back(*b);
        ctx->save_for_backward({t.cos, t.sin, t.positions, t.offsets, t.cu});
        std::vector<int64_t> call = {t.offset, t.interleaved, t.back, (int64_t)a.scalar_type(), (int64_t)b.has_value(), t.cos.size(1)};
        for (const at::Tensor* s : {&t.cos, &t.sin, &t.positions, &t.offsets, &t.cu}) {
            call.push_back(s->defined() ? (int64_t)s->scalar_type() : 0);
            call.push_back(s->defined() ? s->numel() : 0);
        }
        ctx->saved_data["call"] = std::move(call);
        ctx->saved_data["device"] = a.device();
        ctx->set_materialize_grads(false);
        return turn(t, xs);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const std::vector<int64_t> n = ctx->saved_data["call"].toIntVector();
        const c10::Device dev = ctx->saved_data["device"].toDevice();
        const c10::DeviceGuard guard(dev);
        const bool two = n[4];
        variable_list out(3), dys;
        const auto saved = ctx->get_saved_variables();
        // (in the type and the place that they had: saved-tensor hooks may hand back others)
        auto here = [&](int i) {
            const at::Tensor& x = saved[i];
            if (!x.defined()) return x;
            TORCH_CHECK_VALUE(x.numel() == n[7 + 2 * i], "a saved tensor of ", n[7 + 2 * i], " elements came back with ", x.numel());
            return x.to(dev, (at::ScalarType)n[6 + 2 * i]);
        };
        RotaryTables t{here(0), here(1), here(2), here(3), here(4), n[0], (bool)n[1], !n[2]};
        TORCH_CHECK_VALUE(t.cos.sizes() == t.sin.sizes() && t.cos.dim() == 2 && t.cos.size(1) == n[5], "saved tables of rotary positions came back with other sizes");
        if (!in_rows(t.cos) || !in_rows(t.sin) || t.cos.stride(0) != t.sin.stride(0) || t.cos.stride(0) < t.cos.size(1)) { t.cos = t.cos.contiguous(); t.sin = t.sin.contiguous(); }
        for (at::Tensor* index : {&t.positions, &t.offsets, &t.cu})
            if (index->defined()) *index = index->contiguous();
        for (size_t i = 0; i < (two ? 2u : 1u); ++i)
            if (grads[i].defined()) {
                at::Tensor dy = grads[i].to((at::ScalarType)n[3]);
                dys.push_back(in_rows(dy) ? dy : dy.contiguous());
            }
        if (dys.empty()) return out;
        const variable_list dxs = at::GradMode::is_enabled() ? RotaryTrain::apply(dys[0], dys.size() > 1 ? Maybe(dys[1]) : Maybe(), t) : turn(t, dys);
        for (size_t i = 0, j = 0; i < (two ? 2u : 1u); ++i)
            if (grads[i].defined()) out[i] = dxs[j++];
        return out;
    }
};

// cos, sin as the kernels take them beside rows of `type` and `dim` elements
bool tables(const Arg& cos, const Arg& sin, c10::Device dev, at::ScalarType type, int64_t dim) {
    return cos && sin && placed(cos, dev) && placed(sin, dev) && cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->size(1) > 0 && 2 * cos->size(1) <= dim && cos->size(0) > 0 &&
           cos->scalar_type() == sin->scalar_type() && (cos->scalar_type() == type || cos->scalar_type() == at::kFloat) && in_rows(*cos.t) && in_rows(*sin.t) &&
           cos->stride(0) == sin->stride(0) && cos->stride(0) >= cos->size(1);
}

// (q, k or None, cos, sin, interleaved, seqlen_offsets, cu_seqlens, max_seqlen, positions) -> (q, k) or (q,); None: not a call for the native path
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "gdn_host.rotary takes 9 arguments"); return nullptr; }
    const Arg q(a[0]), k(a[1]), cos(a[2]), sin(a[3]), cu(a[6]), positions(a[8]);
    if (!q || !q->is_cuda() || q->dim() != 4 || q->numel() == 0 || k.bad || (k && (k->dim() != 4 || k->numel() == 0))) Py_RETURN_NONE;
    const c10::Device dev = q->device();
    const at::ScalarType type = q->scalar_type();
    const int64_t B = q->size(0), T = q->size(1), D = q->size(3);
    if (dev.index() != c10::hip::current_device() || code_of(type) < 0 || !in_rows(*q.t) || !tables(cos, sin, dev, type, D) || cu.bad || positions.bad) Py_RETURN_NONE;
    if (k && (!placed(k, dev) || k->scalar_type() != type || k->size(0) != B || k->size(1) != T || k->size(3) != D || !in_rows(*k.t))) Py_RETURN_NONE;
    RotaryTables t{*cos.t, *sin.t};
    t.interleaved = truth(a[4]);
    int64_t longest = T, N = B;
    if (cu) {
        if (B != 1 || cu->dim() != 1 || cu->numel() < 2 || cu->device() != dev || !whole_numbers(cu, cu->sizes()) || !int_of(a[7], longest)) Py_RETURN_NONE;
        N = cu->numel() - 1;
        t.cu = *cu.t;
    }
    if (positions) {
        if (positions->device() != dev || !whole_numbers(positions, {B, T}) || !int_of(a[5], t.offset) || t.offset) Py_RETURN_NONE;
        t.positions = *positions.t;
    } else if (int_of(a[5], t.offset)) {
        if (t.offset < 0 || t.offset + longest > cos->size(0)) Py_RETURN_NONE;
    } else {
        const Arg offsets(a[5]);
        if (!offsets || offsets->device() != dev || !whole_numbers(offsets, {N})) Py_RETURN_NONE;
        t.offsets = *offsets.t;
    }
    if (has_tangent({&q, &k, &cos, &sin}) || needs_grad({&cos, &sin})) Py_RETURN_NONE;
    variable_list ys;
    const bool train = needs_grad({&q, &k});
    {
        const NoGil free;
        if (train) ys = RotaryTrain::apply(*q.t, k ? RotaryTrain::Maybe(*k.t) : RotaryTrain::Maybe(), t);
        else if (k) ys = turn(t, {*q.t, *k.t});
        else ys = turn(t, {*q.t});
    }
    if (k) return pair(ys[0], ys[1]);
    PyObject* y = THPVariable_Wrap(ys[0]);
    PyObject* r = y ? PyTuple_Pack(1, y) : nullptr;
    Py_XDECREF(y);
    return r;
    END_HANDLE_TH_ERRORS
}

// ---- the cache ----
bool paged_cache(const Arg& k, const Arg& v, const Arg& table, const Arg& context, int64_t N, bool writes, gdn_paged_cache& c) {
    const c10::Device dev = k->device();
    if (!v || !table || !context || k->dim() != 4 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() || code_of(k->scalar_type()) < 0 || k->numel() == 0 ||
        !in_rows(*k.t) || !in_rows(*v.t) || v->device() != dev || table->device() != dev || context->device() != dev || has_tangent({&k, &v}) || needs_grad({&k, &v}))
        return false;
    if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) != N || table->size(1) < 1 || !in_rows(*table.t) || (N > 1 && table->stride(0) < table->size(1)) ||
        !whole_numbers(context, {N}))
        return false;
    c = {k->data_ptr(), v->data_ptr(), (const int32_t*)table->data_ptr(), context->data_ptr(), {}, {}, k->size(0), k->size(1), k->size(2), k->size(3), table->size(1),
         N > 1 ? table->stride(0) : table->size(1), code_of(k->scalar_type()), context->scalar_type() == at::kInt};
    for (int i = 0; i < 3; ++i) {
        c.k_stride[i] = k->stride(i); c.v_stride[i] = v->stride(i);
        if (writes && k->size(i) > 1 && (k->stride(i) == 0 || v->stride(i) == 0)) return false;
    }
    return true;
}
// cu_seqlens with max_seqlen (its boundaries are not looked at), or neither
bool sequences(const Arg& x, const Arg& cu, PyObject* longest, int64_t& N, int64_t& rows) {
    N = x->size(0); rows = x->size(1);
    if (cu.bad) return false;
    if (!cu) return true;
    if (N != 1 || cu->dim() != 1 || cu->numel() < 2 || cu->device() != x->device() || !whole_numbers(cu, cu->sizes()) || !int_of(longest, rows)) return false;
    N = cu->numel() - 1;
    rows = std::max<int64_t>(0, std::min(rows, x->size(1)));
    return true;
}
bool on_current_gpu(const Arg& x) { return x && x->is_cuda() && x->dim() == 4 && x->numel() > 0 && x->device().index() == c10::hip::current_device(); }

// (k, v, k_cache, v_cache, page_table, context_lens, cu_seqlens, max_seqlen, q, cos, sin, positions, interleaved) -> (q or None,); None: not a call for the native path
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13) { PyErr_SetString(PyExc_TypeError, "gdn_host.paged_append takes 13 arguments"); return nullptr; }
    const Arg k(a[0]), v(a[1]), kc(a[2]), vc(a[3]), table(a[4]), context(a[5]), cu(a[6]), q(a[8]), cos(a[9]), sin(a[10]), positions(a[11]);
    if (!on_current_gpu(k) || !v || !kc || q.bad || cos.bad || sin.bad || positions.bad) Py_RETURN_NONE;
    const c10::Device dev = k->device();
    const at::ScalarType type = k->scalar_type();
    const int64_t D = k->size(3);
    int64_t N, longest;
    gdn_paged_cache cache;
    if (kc->device() != dev || !sequences(k, cu, a[7], N, longest) || !paged_cache(kc, vc, table, context, N, true, cache)) Py_RETURN_NONE;
    if (kc->scalar_type() != type || v->scalar_type() != type || v->sizes() != k->sizes() || v->device() != dev || k->size(2) != kc->size(2) || D != kc->size(3) || !in_rows(*k.t) || !in_rows(*v.t))
        Py_RETURN_NONE;
    if (q && (q->dim() != 4 || q->numel() == 0 || q->device() != dev || q->scalar_type() != type || q->size(0) != k->size(0) || q->size(1) != k->size(1) || q->size(3) != D || !in_rows(*q.t)))
        Py_RETURN_NONE;
    if ((bool)cos != (bool)sin || (cos && !tables(cos, sin, dev, type, D)) || (positions && (!cos || positions->device() != dev || !whole_numbers(positions, {k->size(0), k->size(1)})))) Py_RETURN_NONE;
    if (has_tangent({&k, &v, &q, &cos, &sin}) || needs_grad({&k, &v, &q, &cos, &sin})) Py_RETURN_NONE;
    RotaryTables t{tensor_of(cos), tensor_of(sin), tensor_of(positions), at::Tensor(), tensor_of(cu)};
    t.interleaved = truth(a[12]);
    at::Tensor out;
    {
        const NoGil free;
        if (q) out = empty_on(dev, type, q->sizes());
        const gdn_rotary_call call = rotary_call(t, *k.t);
        const gdn_rotary_rows kr = rotary_rows(*k.t, at::Tensor()), vr = rotary_rows(*v.t, at::Tensor()), qr = q ? rotary_rows(*q.t, out) : gdn_rotary_rows{};
        check_rc(p_paged_append(&cache, q ? &qr : nullptr, &kr, &vr, &call, stream_of(dev)), "gdn_paged_append");
        changed(kc); changed(vc);
    }
    PyObject* y = q ? THPVariable_Wrap(out) : (Py_INCREF(Py_None), Py_None);
    PyObject* r = y ? PyTuple_Pack(1, y) : nullptr;
    Py_XDECREF(y);
    return r;
    END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, page_table, context_lens, tree_mask, scale, cu_seqlens, max_seqlen) -> o; None: not a call for the native path
PyObject* paged_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "gdn_host.paged_attn takes 9 arguments"); return nullptr; }
    const Arg q(a[0]), kc(a[1]), vc(a[2]), table(a[3]), context(a[4]), mask(a[5]), cu(a[7]);
    if (!on_current_gpu(q) || !kc || mask.bad) Py_RETURN_NONE;
    const c10::Device dev = q->device();
    int64_t N, longest;
    gdn_paged_cache cache;
    if (kc->device() != dev || !sequences(q, cu, a[8], N, longest) || !paged_cache(kc, vc, table, context, N, false, cache)) Py_RETURN_NONE;
    const int64_t B = q->size(0), T = q->size(1), HQ = q->size(2), D = q->size(3);
    if (kc->scalar_type() != q->scalar_type() || kc->size(3) != D || HQ % kc->size(2) || !in_rows(*q.t) || has_tangent({&q}) || needs_grad({&q})) Py_RETURN_NONE;
    gdn_paged_attn_call c = {};
    if (!scale_of(a[6], D, c.scale)) { if (PyErr_Occurred()) return nullptr; Py_RETURN_NONE; }
    if (mask) {
        if (mask->scalar_type() != at::kBool || mask->device() != dev || mask->dim() < 2 || mask->dim() > 3 || (mask->dim() == 3 && (cu || mask->size(0) != B)) ||
            mask->size(-2) != T || mask->size(-1) < 1 || !in_rows(*mask.t))
            Py_RETURN_NONE;
        c.mask = (const uint8_t*)mask->data_ptr();
        c.mask_cols = mask->size(-1); c.mask_row_stride = mask->stride(-2); c.mask_seq_stride = mask->dim() == 3 ? mask->stride(0) : 0;
    }
    at::Tensor o;
    {
        const NoGil free;
        o = empty_on(dev, q->scalar_type(), q->sizes());
        c.q = q->data_ptr(); c.o = o.data_ptr(); c.cu_seqlens = cu.ptr();
        for (int i = 0; i < 3; ++i) c.q_stride[i] = q->stride(i);
        c.B = B; c.T = T; c.N = N; c.HQ = HQ; c.max_rows = longest;
        c.flags = cu && cu->scalar_type() == at::kInt ? GDN_FLAG_CU_INT32 : 0;
        const at::Tensor ws = empty_on(dev, at::kByte, {(int64_t)p_paged_attn_workspace_bytes(&cache, &c)});
        check_rc(p_paged_attn(&cache, &c, ws.data_ptr(), (size_t)ws.numel(), stream_of(dev)), "gdn_paged_attn");
    }
    return THPVariable_Wrap(o);
    END_HANDLE_TH_ERRORS
}

// (k_cache, v_cache, page_table, context_lens, rows, num_kept) -> True; None: not a call for the native path
PyObject* paged_keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) { PyErr_SetString(PyExc_TypeError, "gdn_host.paged_keep takes 6 arguments"); return nullptr; }
    const Arg kc(a[0]), vc(a[1]), table(a[2]), context(a[3]), rows(a[4]), kept(a[5]);
    if (!on_current_gpu(kc) || !rows || !kept || rows->dim() != 2 || rows->numel() == 0) Py_RETURN_NONE;
    const c10::Device dev = kc->device();
    const int64_t N = rows->size(0), R = rows->size(1);
    gdn_paged_cache cache;
    if (!paged_cache(kc, vc, table, context, N, true, cache) || rows->device() != dev || kept->device() != dev || rows->scalar_type() != at::kInt || kept->scalar_type() != at::kInt ||
        !rows->is_contiguous() || !whole_numbers(kept, {N}))
        Py_RETURN_NONE;
    check_rc(p_paged_keep(&cache, (const int32_t*)rows->data_ptr(), R, R, (const int32_t*)kept->data_ptr(), N, stream_of(dev)), "gdn_paged_keep");
    changed(kc); changed(vc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (target_probs, draft_tokens, uniforms, parents, draft_probs, lengths) -> (next_token, num_accepted, rows); None: not a call for the native path
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) { PyErr_SetString(PyExc_TypeError, "gdn_host.verify_drafts takes 6 arguments"); return nullptr; }
    const Arg p(a[0]), tokens(a[1]), u(a[2]), parents(a[3]), q(a[4]), lengths(a[5]);
    if (!p || !p->is_cuda() || p->dim() != 3 || p->numel() == 0 || p->device().index() != c10::hip::current_device()) Py_RETURN_NONE;
    const c10::Device dev = p->device();
    const int64_t N = p->size(0), R = p->size(1), V = p->size(2);
    for (const Arg* t : {&p, &tokens, &u, &parents, &q, &lengths})
        if (!placed(*t, dev)) Py_RETURN_NONE;
    if (code_of(p->scalar_type()) < 0 || !in_rows(*p.t) || (q && (q->sizes() != p->sizes() || q->scalar_type() != p->scalar_type() || !in_rows(*q.t))) || !whole_numbers(tokens, {N, R})) Py_RETURN_NONE;
    if (!u || u->scalar_type() != at::kFloat || !u->is_contiguous() || u->dim() != 2 || u->size(0) != N || u->size(1) != R) Py_RETURN_NONE;
    if (parents && (parents->scalar_type() != at::kInt || !(whole_numbers(parents, {R}) || whole_numbers(parents, {N, R})))) Py_RETURN_NONE;
    if (lengths && (lengths->scalar_type() != at::kInt || !whole_numbers(lengths, {N}))) Py_RETURN_NONE;
    gdn_drafts_call c = {};
    at::Tensor token, accepted, rows;
    {
        const NoGil free;
        token = empty_on(dev, at::kLong, {N});
        accepted = empty_on(dev, at::kInt, {N});
        rows = empty_on(dev, at::kInt, {N, R});
        c.p = p->data_ptr(); c.q = q.ptr(); c.tokens = tokens->data_ptr(); c.uniforms = (const float*)u->data_ptr(); c.parents = (const int32_t*)parents.ptr(); c.lengths = (const int32_t*)lengths.ptr();
        c.next_token = (int64_t*)token.data_ptr(); c.accepted = (int32_t*)accepted.data_ptr(); c.rows = (int32_t*)rows.data_ptr();
        for (int i = 0; i < 2; ++i) { c.p_stride[i] = p->stride(i); c.q_stride[i] = q ? q->stride(i) : 0; }
        c.parents_stride = parents && parents->dim() == 2 ? R : 0;
        c.N = N; c.R = R; c.V = V; c.p_dtype = c.q_dtype = code_of(p->scalar_type());
        c.flags = tokens->scalar_type() == at::kLong ? GDN_DRAFTS_TOKENS_INT64 : 0;
        const int64_t need = (int64_t)p_verify_drafts_workspace_bytes(&c);
        at::Tensor ws;
        if (need) ws = empty_on(dev, at::kByte, {need});
        check_rc(p_verify_drafts(&c, ptr_of(ws), (size_t)need, stream_of(dev)), "gdn_verify_drafts");
    }
    PyObject* out[3] = {THPVariable_Wrap(token), THPVariable_Wrap(accepted), THPVariable_Wrap(rows)};
    PyObject* r = out[0] && out[1] && out[2] ? PyTuple_Pack(3, out[0], out[1], out[2]) : nullptr;
    for (PyObject* o : out) Py_XDECREF(o);
    return r;
    END_HANDLE_TH_ERRORS
}
