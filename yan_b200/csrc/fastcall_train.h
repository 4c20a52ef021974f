// Native front of the training operators; part of fastcall.cpp, behind its helpers.  The same rules: what is not the ordinary case is left
// to the Python path, which raises the error.

struct TrainEntries {
    decltype(&yan_b200_fp8_linear_wgrad_workspace_bytes) wgrad_workspace_bytes;
    decltype(&yan_b200_fp8_linear_wgrad) wgrad;
    decltype(&yan_b200_k_grouped_fp8_linear_wgrad) grouped_wgrad;
    decltype(&yan_b200_adamw_step) adamw;
    decltype(&yan_b200_moe_balance_loss_workspace_bytes) balance_workspace_bytes;
    decltype(&yan_b200_moe_balance_loss) balance;
};
TrainEntries g_train = {};

bool element_type(const at::Tensor& t, int* code) {
    if (t.scalar_type() == at::kFloat) *code = YAN_B200_F32;
    else if (t.scalar_type() == at::kBFloat16) *code = YAN_B200_BF16;
    else return false;
    return true;
}

// [..., rows, cols] with contiguous rows that do not overlap: elements from one row to the next.
bool row_stride(const at::Tensor& t, int64_t* stride) {
    const int64_t rows = t.size(-2), cols = t.size(-1);
    if (cols != 1 && t.stride(-1) != 1) return false;
    *stride = rows > 1 ? t.stride(-2) : std::max(t.stride(-2), cols);
    return *stride >= cols;
}

// `given`, if it is a tensor that will do, or new scratch from torch's allocator.
bool scratch(PyObject* given, size_t need, const at::Tensor& like, at::Tensor* ws) {
    if (given == Py_None) {
        *ws = at::empty({static_cast<int64_t>(need)}, like.options().dtype(at::kByte));
        return true;
    }
    const at::Tensor* t = cuda_tensor(given);
    if (!t || t->scalar_type() != at::kByte || !t->is_contiguous() || static_cast<size_t>(t->numel()) < need || !aligned(t->data_ptr(), 256))
        return false;
    *ws = *t;
    return true;
}

bool on_current_device(const at::Tensor& t) { return t.get_device() == c10::cuda::current_device(); }
bool same_device(const at::Tensor& a, const at::Tensor& b) { return a.get_device() == b.get_device(); }

// wgrad(dy, x, out, accumulate, workspace or None, num_sms, group_starts or None, group_sizes or None)
PyObject* wgrad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        long num_sms;
        if (nargs != 8 || !g_train.wgrad || !as_long(args[5], &num_sms)) return code(kNotTaken);
        const at::Tensor *dy = cuda_tensor(args[0]), *x = cuda_tensor(args[1]), *out = cuda_tensor(args[2]);
        if (!dy || !x || !out || dy->dim() != 2 || x->dim() != 2) return code(kNotTaken);
        if (dy->scalar_type() != at::kBFloat16 || x->scalar_type() != at::kBFloat16) return code(kNotTaken);
        if (!on_current_device(*dy) || !same_device(*dy, *x) || !same_device(*dy, *out)) return code(kNotTaken);
        const bool grouped = args[6] != Py_None;
        const at::Tensor *starts = nullptr, *sizes = nullptr;
        int64_t groups = 0;
        if (grouped) {
            starts = cuda_tensor(args[6]), sizes = cuda_tensor(args[7]);
            if (!starts || !sizes || sizes->dim() != 1 || starts->dim() != 1) return code(kNotTaken);
            groups = sizes->size(0);
            if (groups < 1 || groups > 512 || starts->size(0) != groups) return code(kNotTaken);
            for (const at::Tensor* t : {starts, sizes})
                if (t->scalar_type() != at::kInt || !t->is_contiguous() || !same_device(*dy, *t)) return code(kNotTaken);
        }
        const int64_t m = dy->size(0), n = dy->size(1), k = x->size(1);
        int64_t dy_ld, x_ld, out_ld, out_group = 0;
        int dtype;
        if (m > INT32_MAX || x->size(0) != m || !fits_int(n) || !fits_int(k) || out->dim() != (grouped ? 3 : 2)) return code(kNotTaken);
        if (out->size(-2) != n || out->size(-1) != k || (grouped && out->size(0) != groups) || !element_type(*out, &dtype)) return code(kNotTaken);
        if (!row_stride(*dy, &dy_ld) || !row_stride(*x, &x_ld) || !row_stride(*out, &out_ld)) return code(kNotTaken);
        if (grouped) {
            out_group = groups > 1 ? out->stride(0) : n * out_ld;
            if (out_group < (n - 1) * out_ld + k) return code(kNotTaken);
        }
        const int accumulate = PyObject_IsTrue(args[3]) == 1;
        const size_t need = g_train.wgrad_workspace_bytes(static_cast<int>(m), static_cast<int>(n), static_cast<int>(k),
                                                          static_cast<int>(groups), static_cast<int>(num_sms));
        at::Tensor ws;
        if (!scratch(args[4], need, *dy, &ws)) return code(kNotTaken);
        const void *pdy = dy->data_ptr(), *px = x->data_ptr();
        void *pout = out->data_ptr(), *pws = ws.data_ptr(), *stream = current_stream();
        const int* pstarts = grouped ? starts->data_ptr<int>() : nullptr;
        const int* psizes = grouped ? sizes->data_ptr<int>() : nullptr;
        const size_t ws_bytes = static_cast<size_t>(ws.numel());
        int rc = 0;
        Py_BEGIN_ALLOW_THREADS
        if (grouped)
            g_train.grouped_wgrad(pdy, px, pout, pstarts, psizes, static_cast<int>(groups), static_cast<int>(m), static_cast<int>(n),
                                  static_cast<int>(k), dy_ld, x_ld, out_ld, out_group, dtype, accumulate, pws, ws_bytes, stream,
                                  static_cast<int>(num_sms), &rc);
        else
            g_train.wgrad(pdy, px, pout, static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), dy_ld, x_ld, out_ld, dtype,
                          accumulate, pws, ws_bytes, stream, static_cast<int>(num_sms), &rc);
        Py_END_ALLOW_THREADS
        return code(rc);
    } catch (...) {
        return code(kNotTaken);
    }
}

// A list or tuple as an array of borrowed references; they stay while the interpreter runs nothing else, which is until the last
// tensor has been looked at.
bool items(PyObject* o, PyObject*** array, Py_ssize_t* count) {
    if (PyList_CheckExact(o)) {
        *array = reinterpret_cast<PyListObject*>(o)->ob_item;
        *count = PyList_GET_SIZE(o);
        return true;
    }
    if (PyTuple_CheckExact(o)) {
        *array = reinterpret_cast<PyTupleObject*>(o)->ob_item;
        *count = PyTuple_GET_SIZE(o);
        return true;
    }
    return false;
}

bool number(PyObject* o, double* v) {
    if (PyFloat_CheckExact(o)) {
        *v = PyFloat_AS_DOUBLE(o);
        return true;
    }
    long l;
    if (!as_long(o, &l)) return false;
    *v = static_cast<double>(l);
    return true;
}

// The tensors of a list, of which there may be hundreds: the first is looked at in full, the others have to be of the same kind (dispatch
// keys: device type, layout, subclass; element type, device).  A full look at each took 30 ns, this 8.
class AlikeTensors {
public:
    explicit AlikeTensors(at::ScalarType type, int device) : type_(c10::scalarTypeToTypeMeta(type)), device_(device) {}

    // Address of a contiguous tensor of `elements`; false for anything else.
    bool take(PyObject* o, int64_t elements, void** address) {
        if (!THPVariable_CheckExact(o)) return false;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!known_) {
            const at::Tensor* first = cuda_tensor(o);
            if (!first) return false;
            keys_ = first->key_set();
            known_ = true;
        }
        c10::TensorImpl* impl = t.unsafeGetTensorImpl();
        if (impl->key_set() != keys_ || impl->dtype() != type_ || impl->numel() != elements || !impl->is_contiguous()) return false;
        if (impl->device().index() != device_ || !impl->has_storage()) return false;
        *address = impl->mutable_data();
        return true;
    }

private:
    caffe2::TypeMeta type_;
    int device_;
    bool known_ = false;
    c10::DispatchKeySet keys_;
};

// The values (codes) and scales of a moment.
struct Moments {
    AlikeTensors values, scales;
    bool eight_bit;

    Moments(bool eight_bit, int device)
        : values(eight_bit ? at::kFloat8_e4m3fn : at::kFloat, device), scales(at::kFloat, device), eight_bit(eight_bit) {}
    bool take(PyObject* o, int64_t elements, void** value, float** scale) {
        *scale = nullptr;
        if (!eight_bit) return values.take(o, elements, value);
        void* s;
        if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 2 || !values.take(PyTuple_GET_ITEM(o, 0), elements, value) ||
            !scales.take(PyTuple_GET_ITEM(o, 1), ceil_div(elements, 128), &s))
            return false;
        *scale = static_cast<float*>(s);
        return true;
    }
};

// adamw(params, grads, exp_avgs, exp_avg_sqs, weight_decay (number or list), copies or None, grad_scale or None, lr, beta1, beta2, eps, step)
PyObject* adamw(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        if (nargs != 12 || !g_train.adamw) return code(kNotTaken);
        PyObject **p, **g, **m, **v, **w = nullptr, **c = nullptr;
        Py_ssize_t count, sizes[5];
        if (!items(args[0], &p, &count) || count == 0 || count > INT32_MAX) return code(kNotTaken);
        if (!items(args[1], &g, sizes) || !items(args[2], &m, sizes + 1) || !items(args[3], &v, sizes + 2)) return code(kNotTaken);
        if (sizes[0] != count || sizes[1] != count || sizes[2] != count) return code(kNotTaken);
        double decay = 0.0, lr, beta1, beta2, eps;
        if (!number(args[4], &decay) && (!items(args[4], &w, sizes + 3) || sizes[3] != count)) return code(kNotTaken);
        if (args[5] != Py_None && (!items(args[5], &c, sizes + 4) || sizes[4] != count)) return code(kNotTaken);
        long step;
        if (!number(args[7], &lr) || !number(args[8], &beta1) || !number(args[9], &beta2) || !number(args[10], &eps) || !as_long(args[11], &step))
            return code(kNotTaken);
        if (step < 1 || !(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0)) return code(kNotTaken);
        const at::Tensor *first = cuda_tensor(p[0]), *first_grad = cuda_tensor(g[0]);
        int param_dtype, grad_dtype;
        if (!first || !first_grad || !on_current_device(*first) || !element_type(*first, &param_dtype) || !element_type(*first_grad, &grad_dtype))
            return code(kNotTaken);
        const int device = first->get_device();
        const float* grad_scale = nullptr;
        if (args[6] != Py_None) {
            const at::Tensor* t = cuda_tensor(args[6]);
            if (!t || t->scalar_type() != at::kFloat || t->numel() != 1 || t->get_device() != device) return code(kNotTaken);
            grad_scale = t->data_ptr<float>();
        }
        const bool eight_bit = PyTuple_CheckExact(m[0]);
        AlikeTensors params(first->scalar_type(), device), grads(first_grad->scalar_type(), device), copies(at::kBFloat16, device);
        Moments exp_avgs(eight_bit, device), exp_avg_sqs(eight_bit, device);
        std::vector<yan_b200_adamw_tensor> table(static_cast<size_t>(count));
        for (Py_ssize_t i = 0; i < count; ++i) {
            yan_b200_adamw_tensor& t = table[static_cast<size_t>(i)];
            void* address;
            if (!THPVariable_CheckExact(p[i])) return code(kNotTaken);
            t.numel = THPVariable_Unpack(p[i]).unsafeGetTensorImpl()->numel();
            if (!params.take(p[i], t.numel, &t.param) || !grads.take(g[i], t.numel, &address)) return code(kNotTaken);
            t.grad = address;
            if (!exp_avgs.take(m[i], t.numel, &t.exp_avg, &t.exp_avg_scale) || !exp_avg_sqs.take(v[i], t.numel, &t.exp_avg_sq, &t.exp_avg_sq_scale))
                return code(kNotTaken);
            t.copy = nullptr;
            if (c != nullptr && !copies.take(c[i], t.numel, &t.copy)) return code(kNotTaken);
            t.weight_decay = decay;
            if (w != nullptr && !number(w[i], &t.weight_decay)) return code(kNotTaken);
        }
        for (Py_ssize_t i = 0; i < count; ++i) {  // autograd notices that the parameters changed
            const at::Tensor& t = THPVariable_Unpack(p[i]);
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
        void* stream = current_stream();
        int rc = 0;
        Py_BEGIN_ALLOW_THREADS
        g_train.adamw(table.data(), static_cast<int>(count), param_dtype, grad_dtype, eight_bit ? 8 : 32, lr, beta1, beta2, eps, step, grad_scale,
                      stream, &rc);
        Py_END_ALLOW_THREADS
        return code(rc);
    } catch (...) {
        return code(kNotTaken);
    }
}

// balance(logits, expert_ids, token_mask or None, cu_seqlens or None, coef, score, num_sms): (loss, counts, grad), a return code, or -1
PyObject* balance(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        long score, num_sms;
        double coef;
        if (nargs != 7 || !g_train.balance || !number(args[4], &coef) || !as_long(args[5], &score) || !as_long(args[6], &num_sms))
            return code(kNotTaken);
        const at::Tensor *logits = cuda_tensor(args[0]), *ids = cuda_tensor(args[1]);
        if (!logits || !ids || logits->dim() != 2 || ids->dim() != 2 || !on_current_device(*logits) || !same_device(*logits, *ids))
            return code(kNotTaken);
        const int64_t t = logits->size(0), e = logits->size(1), top = ids->size(1);
        int dtype;
        int64_t ld;
        if (t > INT32_MAX || e < 1 || e > 1024 || ids->size(0) != t || top < 1 || top > 65535 || !element_type(*logits, &dtype) || !row_stride(*logits, &ld))
            return code(kNotTaken);
        const bool wide = ids->scalar_type() == at::kLong;
        if ((!wide && ids->scalar_type() != at::kInt) || !ids->is_contiguous()) return code(kNotTaken);
        const void* mask = nullptr;
        if (args[2] != Py_None) {
            const at::Tensor* k = cuda_tensor(args[2]);
            if (!k || k->scalar_type() != at::kBool || k->dim() != 1 || k->size(0) != t || !k->is_contiguous() || !same_device(*logits, *k))
                return code(kNotTaken);
            mask = k->data_ptr();
        }
        const int* cu = nullptr;
        int64_t sequences = 1;
        if (args[3] != Py_None) {
            const at::Tensor* k = cuda_tensor(args[3]);
            if (!k || k->scalar_type() != at::kInt || k->dim() != 1 || k->size(0) < 2 || k->size(0) > 65536 || !k->is_contiguous() ||
                !same_device(*logits, *k))
                return code(kNotTaken);
            cu = k->data_ptr<int>();
            sequences = k->size(0) - 1;
        }
        const auto options = logits->options().requires_grad(false);
        at::Tensor loss = at::empty({}, options.dtype(at::kFloat)), counts = at::empty({sequences, e}, options.dtype(at::kInt));
        at::Tensor grad = at::empty({t, e}, options);
        const size_t need = g_train.balance_workspace_bytes(static_cast<int>(t), static_cast<int>(e), static_cast<int>(sequences), 1,
                                                            static_cast<int>(num_sms));
        at::Tensor ws;
        if (need != 0) ws = at::empty({static_cast<int64_t>(need)}, options.dtype(at::kByte));
        const void *plogits = logits->data_ptr(), *pids = ids->data_ptr();
        void* stream = current_stream();
        float* ploss = loss.data_ptr<float>();
        int* pcounts = counts.data_ptr<int>();
        void *pgrad = grad.data_ptr(), *pws = need != 0 ? ws.data_ptr() : nullptr;
        int rc = 0;
        Py_BEGIN_ALLOW_THREADS
        g_train.balance(plogits, pids, mask, cu, ploss, pcounts, pgrad, static_cast<int>(t), static_cast<int>(e), static_cast<int>(top),
                        static_cast<int>(sequences), ld, e, dtype, wide, static_cast<int>(score), static_cast<float>(coef), pws, need, stream,
                        static_cast<int>(num_sms), &rc);
        Py_END_ALLOW_THREADS
        if (rc != 0) return code(rc);
        PyObject *a = THPVariable_Wrap(loss), *b = THPVariable_Wrap(counts), *c = THPVariable_Wrap(grad);
        PyObject* result = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
        Py_XDECREF(a);
        Py_XDECREF(b);
        Py_XDECREF(c);
        return result;
    } catch (...) {
        PyErr_Clear();
        return code(kNotTaken);
    }
}

// bind_train(six addresses, in the order of TrainEntries)
PyObject* bind_train(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 6) {
        PyErr_SetString(PyExc_TypeError, "bind_train takes six addresses");
        return nullptr;
    }
    void* p[6];
    for (int i = 0; i < 6; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (p[i] == nullptr) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
            return nullptr;
        }
    }
    g_train.wgrad_workspace_bytes = reinterpret_cast<decltype(g_train.wgrad_workspace_bytes)>(p[0]);
    g_train.wgrad = reinterpret_cast<decltype(g_train.wgrad)>(p[1]);
    g_train.grouped_wgrad = reinterpret_cast<decltype(g_train.grouped_wgrad)>(p[2]);
    g_train.adamw = reinterpret_cast<decltype(g_train.adamw)>(p[3]);
    g_train.balance_workspace_bytes = reinterpret_cast<decltype(g_train.balance_workspace_bytes)>(p[4]);
    g_train.balance = reinterpret_cast<decltype(g_train.balance)>(p[5]);
    Py_RETURN_NONE;
}
