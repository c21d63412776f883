// The native host path of the operators over whole sequences and of clipping: the same contract as native.cc (None whenever the
// call is not the plain case), but rows may be strided, and there is no other path: the Python operators check, convert and call
// again.
#include "native_rows.h"

#include <vector>

namespace {

// ---- state_scan -----------------------------------------------------------------------------------------------------
struct Scan {
    const Tensor *x, *delta, *A, *B, *C, *D, *z, *bias, *indptr, *initial;
    Rows rows;
    bpl_state_scan_descriptor d;
    int64_t sequences;

    // args: x, delta, A, B, C, D, z, delta_bias, softplus
    bool read(PyObject *const *args) {
        return operand(args[0], x) && operand(args[1], delta) && operand(args[2], A) && operand(args[3], B) &&
               operand(args[4], C) && operand(args[5], D, true) && operand(args[6], z, true) && operand(args[7], bias, true) &&
               check(truth(args[8]));
    }
    // tensors that have passed the checks once
    void set(const Tensor &x_, const Tensor &delta_, const Tensor &A_, const Tensor &B_, const Tensor &C_, const Tensor &D_, const Tensor &z_,
             const Tensor &bias_, const Tensor &indptr_, const Tensor &initial_, bool softplus) {
        auto given = [](const Tensor &t) { return t.defined() ? &t : nullptr; };
        x = &x_; delta = &delta_; A = &A_; B = &B_; C = &C_;
        D = given(D_); z = given(z_); bias = given(bias_); indptr = given(indptr_); initial = given(initial_);
        TORCH_CHECK(check(softplus) && check_sequences(), "state_scan: operands changed between the passes");
    }
    bool check(bool softplus) {
        const int dtype = dtype_of(*x);
        Rows r;
        if (dtype < 0 || !rows_of(*x, 1, rows) || A->dim() != 2) return false;
        const int64_t channels = x->size(-1), state = A->size(1);
        std::memset(&d, 0, sizeof(d));
        d.x_stride = rows.stride;
        if (delta->scalar_type() != x->scalar_type() || delta->sizes() != x->sizes() || !rows_of(*delta, 1, r)) return false;
        d.delta_stride = r.stride;
        if (z) {
            if (z->scalar_type() != x->scalar_type() || z->sizes() != x->sizes() || !rows_of(*z, 1, r)) return false;
            d.z_stride = r.stride;
        }
        // B and C: (rows, state) for one group, (rows, groups, state) for several
        const int64_t lead = rows.batched ? 2 : 1;
        const int64_t inner = B->dim() - lead;
        if ((inner != 1 && inner != 2) || B->sizes() != C->sizes() || B->scalar_type() != x->scalar_type() ||
            C->scalar_type() != x->scalar_type() || B->size(-1) != state)
            return false;
        const int64_t groups = inner == 2 ? B->size(lead) : 1;
        if (!rows_of(*B, inner, r) || !same_rows(r, rows)) return false;
        d.B_stride = r.stride;
        d.B_group_stride = inner == 2 ? B->stride(lead) : 0;
        if (!rows_of(*C, inner, r)) return false;
        d.C_stride = r.stride;
        d.C_group_stride = inner == 2 ? C->stride(lead) : 0;
        if (groups < 1 || channels % groups != 0 || state < 1 || state > 128 || channels > 0x7fffffffll ||
            rows.rows >= (1ll << 31) || !dense(A, at::kFloat, {channels, state}, *x))
            return false;
        if ((D && !dense(D, at::kFloat, {channels}, *x)) || (bias && !dense(bias, at::kFloat, {channels}, *x))) return false;
        for (const Tensor *t : {delta, z, B, C})
            if (t && t->device() != x->device()) return false;
        d.tokens = static_cast<uint32_t>(rows.rows);
        d.length = static_cast<uint32_t>(rows.length);
        d.channels = static_cast<uint32_t>(channels);
        d.groups = static_cast<uint32_t>(groups);
        d.state = static_cast<uint32_t>(state);
        d.dtype = static_cast<uint32_t>(dtype);
        d.flags = softplus ? BPL_SCAN_SOFTPLUS : 0;
        return true;
    }
    bool read_sequences(PyObject *p, PyObject *i) {
        return operand(p, indptr, true) && operand(i, initial, true) && check_sequences();
    }
    bool check_sequences() {
        sequences = rows.batch;
        if (indptr) {
            if (rows.batched || indptr->scalar_type() != at::kInt || indptr->dim() != 1 || indptr->size(0) < 1 ||
                indptr->stride(0) != 1 || indptr->device() != x->device())
                return false;
            sequences = indptr->size(0) - 1;
        }
        if (sequences >= (1ll << 31)) return false;
        d.sequences = static_cast<uint32_t>(sequences);
        return !initial || dense(initial, at::kFloat, {sequences, x->size(-1), A->size(1)}, *x);
    }
    bool wants() const {
        for (const Tensor *t : {x, delta, A, B, C, D, z, bias, initial})
            if (t && wants_grad(*t)) return true;
        return false;
    }
};

// ---- short_conv -----------------------------------------------------------------------------------------------------
struct Conv {
    const Tensor *x, *weight, *bias, *indptr, *initial;
    Rows rows;
    bpl_short_conv_descriptor d;
    int64_t sequences, channels, width;

    // args: x, weight, bias, silu
    bool read(PyObject *const *args) {
        return operand(args[0], x) && operand(args[1], weight) && operand(args[2], bias, true) && check(truth(args[3]));
    }
    void set(const Tensor &x_, const Tensor &weight_, const Tensor &bias_, const Tensor &indptr_, const Tensor &initial_, bool silu) {
        auto given = [](const Tensor &t) { return t.defined() ? &t : nullptr; };
        x = &x_; weight = &weight_;
        bias = given(bias_); indptr = given(indptr_); initial = given(initial_);
        TORCH_CHECK(check(silu) && check_sequences(), "short_conv: operands changed between the passes");
    }
    bool check(bool silu) {
        const int dtype = dtype_of(*x), weight_dtype = dtype_of(*weight);
        if (dtype < 0 || !rows_of(*x, 1, rows) || weight->dim() != 2) return false;
        channels = x->size(-1);
        width = weight->size(1);
        if ((weight_dtype != dtype && weight_dtype != BPL_FLOAT) || width < 1 || width > 8 || channels > 0x7fffffffll ||
            rows.rows >= (1ll << 31) || !dense(weight, weight->scalar_type(), {channels, width}, *x) ||
            (bias && !dense(bias, weight->scalar_type(), {channels}, *x)))
            return false;
        std::memset(&d, 0, sizeof(d));
        d.tokens = static_cast<uint32_t>(rows.rows);
        d.length = static_cast<uint32_t>(rows.length);
        d.channels = static_cast<uint32_t>(channels);
        d.width = static_cast<uint32_t>(width);
        d.dtype = static_cast<uint32_t>(dtype);
        d.weight_dtype = static_cast<uint32_t>(weight_dtype);
        d.flags = silu ? BPL_CONV_SILU : 0;
        d.x_stride = rows.stride;
        return true;
    }
    bool read_sequences(PyObject *p, PyObject *i) {
        return operand(p, indptr, true) && operand(i, initial, true) && check_sequences();
    }
    bool check_sequences() {
        sequences = rows.batch;
        if (indptr) {
            if (rows.batched || indptr->scalar_type() != at::kInt || indptr->dim() != 1 || indptr->size(0) < 1 ||
                indptr->stride(0) != 1 || indptr->device() != x->device())
                return false;
            sequences = indptr->size(0) - 1;
        }
        if (sequences >= (1ll << 31)) return false;
        d.sequences = static_cast<uint32_t>(sequences);
        return !initial || dense(initial, x->scalar_type(), {sequences, channels, width - 1}, *x);
    }
    bool wants() const {
        for (const Tensor *t : {x, weight, bias, initial})
            if (t && wants_grad(*t)) return true;
        return false;
    }
};

// ---- both passes ------------------------------------------------------------------------------------------------------
struct ScanResult {
    Tensor y, last, saved;
};
ScanResult scan_forward(const Scan &s, bool want_last, bool save) {
    NoGil no_gil;
    OnDevice on(*s.x);
    const int64_t channels = s.x->size(-1), state = s.A->size(1);
    ScanResult r;
    r.y = new_tensor(s.x->sizes(), s.x->scalar_type(), s.x->device());
    if (want_last) r.last = new_tensor({s.sequences, channels, state}, at::kFloat, s.x->device());
    if (save) r.saved = new_tensor({(s.rows.rows + 15) / 16, channels, state}, at::kFloat, s.x->device());
    const char *opaque = reinterpret_cast<const char *>(&s.d);
    Scratch ws(bpl_workspace_bytes("state_scan", opaque, sizeof(s.d)), on.stream);
    void *buffers[14] = {ptr(*s.x), ptr(*s.delta), ptr(*s.A), ptr(*s.B), ptr(*s.C), ptr_of(s.D), ptr_of(s.z),
                         ptr_of(s.bias), ptr_of(s.indptr), ptr_of(s.initial), ptr(r.y), at_or_null(r.last),
                         at_or_null(r.saved), ws.ptr};
    state_scan(on.stream, buffers, opaque, sizeof(s.d));
    check_status();
    return r;
}

struct ScanFn : public torch::autograd::Function<ScanFn> {
    using Maybe = std::optional<Tensor>;
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &B,
                                 const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &bias, const Maybe &initial,
                                 const Maybe &indptr, bool softplus, bool want_last) {
        const Tensor d = value(D), zz = value(z), b = value(bias), i = value(initial), p = value(indptr);
        Scan s;
        s.set(x, delta, A, B, C, d, zz, b, p, i, softplus);
        ScanResult r = scan_forward(s, want_last, true);
        ctx->save_for_backward({x, delta, A, B, C, d, zz, b, i, p, r.saved});
        ctx->saved_data["s"] = softplus;
        ctx->set_materialize_grads(false);
        return want_last ? variable_list{r.y, r.last} : variable_list{r.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0];
        if (!grads[0].defined() && (grads.size() < 2 || !grads[1].defined())) return variable_list(12);
        Scan s;
        s.set(x, saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], saved[9], saved[8], ctx->saved_data["s"].toBool());
        const Tensor dy = cotangent(grads[0], x);
        const Tensor d_last = grads.size() > 1 && grads[1].defined() ? cotangent(grads[1], grads[1]) : Tensor();
        NoGil no_gil;
        OnDevice on(x);
        const auto type = x.scalar_type();
        const auto device = x.device();
        const Tensor dx = new_tensor(x.sizes(), type, device), d_delta = new_tensor(x.sizes(), type, device),
                     dA = new_tensor(s.A->sizes(), at::kFloat, device), dB = new_tensor(s.B->sizes(), type, device),
                     dC = new_tensor(s.B->sizes(), type, device),
                     dD = s.D ? new_tensor(s.D->sizes(), at::kFloat, device) : Tensor(),
                     dz = s.z ? new_tensor(x.sizes(), type, device) : Tensor(),
                     d_bias = s.bias ? new_tensor(s.bias->sizes(), at::kFloat, device) : Tensor(),
                     d_initial = s.initial ? new_tensor(s.initial->sizes(), at::kFloat, device) : Tensor();
        const char *opaque = reinterpret_cast<const char *>(&s.d);
        Scratch ws(bpl_workspace_bytes("state_scan_backward", opaque, sizeof(s.d)), on.stream);
        void *buffers[23] = {ptr(x), ptr(*s.delta), ptr(*s.A), ptr(*s.B), ptr(*s.C), ptr_of(s.D), ptr_of(s.z),
                             ptr_of(s.bias), ptr_of(s.indptr), ptr_of(s.initial), ptr(saved[10]), ptr(dy), at_or_null(d_last),
                             ptr(dx), ptr(d_delta), ptr(dA), ptr(dB), ptr(dC), at_or_null(dD), at_or_null(dz),
                             at_or_null(d_bias), at_or_null(d_initial), ws.ptr};
        state_scan_backward(on.stream, buffers, opaque, sizeof(s.d));
        check_status();
        return differentiable_once({dx, d_delta, dA, dB, dC, dD, dz, d_bias, d_initial, Tensor(), Tensor(), Tensor()}, "state_scan");
    }
};

struct ConvResult {
    Tensor y, last;
};
ConvResult conv_forward(const Conv &s, bool want_last) {
    NoGil no_gil;
    OnDevice on(*s.x);
    ConvResult r;
    r.y = new_tensor(s.x->sizes(), s.x->scalar_type(), s.x->device());
    if (want_last) r.last = new_tensor({s.sequences, s.channels, s.width - 1}, s.x->scalar_type(), s.x->device());
    void *buffers[7] = {ptr(*s.x), ptr(*s.weight), ptr_of(s.bias), ptr_of(s.indptr), ptr_of(s.initial), ptr(r.y), at_or_null(r.last)};
    short_conv(on.stream, buffers, reinterpret_cast<const char *>(&s.d), sizeof(s.d));
    check_status();
    return r;
}

struct ConvFn : public torch::autograd::Function<ConvFn> {
    using Maybe = std::optional<Tensor>;
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Maybe &bias, const Maybe &initial,
                                 const Maybe &indptr, bool silu, bool want_last) {
        const Tensor b = value(bias), i = value(initial), p = value(indptr);
        Conv s;
        s.set(x, weight, b, p, i, silu);
        ConvResult r = conv_forward(s, want_last);
        ctx->save_for_backward({x, weight, b, i, p});
        ctx->saved_data["s"] = silu;
        ctx->set_materialize_grads(false);
        return want_last ? variable_list{r.y, r.last} : variable_list{r.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0];
        if (!grads[0].defined() && (grads.size() < 2 || !grads[1].defined())) return variable_list(7);
        Conv s;
        s.set(x, saved[1], saved[2], saved[4], saved[3], ctx->saved_data["s"].toBool());
        const Tensor dy = cotangent(grads[0], x);
        const Tensor d_last = grads.size() > 1 && grads[1].defined() ? cotangent(grads[1], grads[1]) : Tensor();
        NoGil no_gil;
        OnDevice on(x);
        const Tensor dx = new_tensor(x.sizes(), x.scalar_type(), x.device()),
                     d_weight = new_tensor(s.weight->sizes(), s.weight->scalar_type(), x.device()),
                     d_bias = s.bias ? new_tensor(s.bias->sizes(), s.weight->scalar_type(), x.device()) : Tensor(),
                     d_initial = s.initial ? new_tensor(s.initial->sizes(), x.scalar_type(), x.device()) : Tensor();
        const char *opaque = reinterpret_cast<const char *>(&s.d);
        Scratch ws(bpl_workspace_bytes("short_conv_backward", opaque, sizeof(s.d)), on.stream);
        // (an initial state of no inputs has no address, and no gradient to write)
        void *buffers[12] = {ptr(x), ptr(*s.weight), ptr_of(s.bias), ptr_of(s.indptr), ptr_of(s.initial), ptr(dy), at_or_null(d_last),
                             ptr(dx), ptr(d_weight), at_or_null(d_bias), at_or_null(d_initial), ws.ptr};
        short_conv_backward(on.stream, buffers, opaque, sizeof(s.d));
        check_status();
        return differentiable_once({dx, d_weight, d_bias, d_initial, Tensor(), Tensor(), Tensor()}, "short_conv");
    }
};

}  // namespace

// state_scan(x, delta, A, B, C, D, z, delta_bias, softplus, indptr, initial_state, return_state) -> y, or (y, last)
PyObject *py_state_scan(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    NONE_UNLESS(nargs == 12 && plain_thread() && is_flag(args[8]) && is_flag(args[11]));
    Scan s;
    NONE_UNLESS(s.read(args) && s.read_sequences(args[9], args[10]));
    const bool want_last = truth(args[11]);
    if (s.wants())
        return one_or_two(ScanFn::apply(*s.x, *s.delta, *s.A, *s.B, *s.C, maybe(s.D), maybe(s.z), maybe(s.bias), maybe(s.initial),
                                        maybe(s.indptr), truth(args[8]), want_last));
    const ScanResult r = scan_forward(s, want_last, false);
    return want_last ? tuple_of({r.y, r.last}) : wrap(r.y);
    END_HANDLE_TH_ERRORS
}

// state_scan_step(x, delta, A, B, C, D, z, delta_bias, softplus, state, slots) -> y
PyObject *py_state_scan_step(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    NONE_UNLESS(nargs == 11 && plain_thread() && is_flag(args[8]));
    Scan s;
    const Tensor *state, *slots;
    NONE_UNLESS(s.read(args) && !s.rows.batched && operand(args[9], state) && operand(args[10], slots, true));
    s.initial = nullptr;
    NONE_UNLESS(!s.wants() && !wants_grad(*state) && state->dim() == 3 && state->size(0) < (1ll << 31) &&
                dense(state, at::kFloat, {state->size(0), s.x->size(1), s.A->size(1)}, *s.x) && s.rows.rows <= 65535);
    if (slots) NONE_UNLESS(dense(slots, at::kInt, {s.rows.rows}, *s.x));
    else NONE_UNLESS(s.rows.rows == state->size(0));
    s.d.sequences = static_cast<uint32_t>(state->size(0));
    Tensor y;
    {
        NoGil no_gil;
        OnDevice on(*s.x);
        y = new_tensor(s.x->sizes(), s.x->scalar_type(), s.x->device());
        void *buffers[11] = {ptr(*s.x), ptr(*s.delta), ptr(*s.A), ptr(*s.B), ptr(*s.C), ptr_of(s.D), ptr_of(s.z),
                             ptr_of(s.bias), ptr_of(slots), ptr(*state), ptr(y)};
        state_scan_step(on.stream, buffers, reinterpret_cast<const char *>(&s.d), sizeof(s.d));
        check_status();
        written(*state);
    }
    return wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// short_conv(x, weight, bias, silu, indptr, initial_state, return_state) -> y, or (y, last)
PyObject *py_short_conv(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    NONE_UNLESS(nargs == 7 && plain_thread() && is_flag(args[3]) && is_flag(args[6]));
    Conv s;
    NONE_UNLESS(s.read(args) && s.read_sequences(args[4], args[5]));
    const bool want_last = truth(args[6]);
    if (s.wants())
        return one_or_two(ConvFn::apply(*s.x, *s.weight, maybe(s.bias), maybe(s.initial), maybe(s.indptr), truth(args[3]), want_last));
    const ConvResult r = conv_forward(s, want_last);
    return want_last ? tuple_of({r.y, r.last}) : wrap(r.y);
    END_HANDLE_TH_ERRORS
}

// short_conv_step(x, weight, bias, silu, state, slots) -> y
PyObject *py_short_conv_step(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    NONE_UNLESS(nargs == 6 && plain_thread() && is_flag(args[3]));
    Conv s;
    const Tensor *state, *slots;
    NONE_UNLESS(s.read(args) && !s.rows.batched && operand(args[4], state) && operand(args[5], slots, true));
    s.initial = nullptr;
    NONE_UNLESS(!s.wants() && !wants_grad(*state) && state->dim() == 3 && state->size(0) < (1ll << 31) &&
                dense(state, s.x->scalar_type(), {state->size(0), s.channels, s.width - 1}, *s.x) && s.rows.rows <= 65535);
    if (slots) NONE_UNLESS(dense(slots, at::kInt, {s.rows.rows}, *s.x));
    else NONE_UNLESS(s.rows.rows == state->size(0));
    s.d.sequences = static_cast<uint32_t>(state->size(0));
    Tensor y;
    {
        NoGil no_gil;
        OnDevice on(*s.x);
        y = new_tensor(s.x->sizes(), s.x->scalar_type(), s.x->device());
        void *buffers[6] = {ptr(*s.x), ptr(*s.weight), ptr_of(s.bias), ptr_of(slots), ptr(*state), ptr(y)};
        short_conv_step(on.stream, buffers, reinterpret_cast<const char *>(&s.d), sizeof(s.d));
        check_status();
        written(*state);
    }
    return wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// references to Python objects, taken and given back with the lock held
struct Held {
    std::vector<PyObject *> objects;
    explicit Held(size_t most) { objects.reserve(most); }
    ~Held() {
        for (PyObject *o : objects) Py_DECREF(o);
    }
    Held(const Held &) = delete;
    Held &operator=(const Held &) = delete;
    void add(PyObject *o) {
        Py_INCREF(o);
        objects.push_back(o);
    }
};

// clip_gradients(grads: list, out: list | None, max_norm, norm_type) -> norm; without `out` only the norm is computed, with the
// same list twice the gradients are overwritten
PyObject *py_clip_gradients(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    double max_norm, norm_type;
    NONE_UNLESS(nargs == 4 && plain_thread() && PyList_CheckExact(args[0]) && (args[1] == Py_None || PyList_CheckExact(args[1])) &&
                number_of(args[2], max_norm) && number_of(args[3], norm_type));
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    const bool write = args[1] != Py_None;
    NONE_UNLESS(n >= 1 && n < (1 << 30) && (!write || PyList_GET_SIZE(args[1]) == n));
    std::vector<void *> buffers(2 * static_cast<size_t>(n) + 2, nullptr);
    std::vector<char> opaque(sizeof(bpl_clip_descriptor) + static_cast<size_t>(n) * sizeof(bpl_clip_tensor), 0);
    auto *d = reinterpret_cast<bpl_clip_descriptor *>(opaque.data());
    auto *tensors = reinterpret_cast<bpl_clip_tensor *>(opaque.data() + sizeof(bpl_clip_descriptor));
    const Tensor *first = nullptr;
    bool any_double = false, in_place = write;
    // (the objects are held by themselves: without the lock another thread may change the lists)
    Held held((write ? 2 : 1) * static_cast<size_t>(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor *g, *o;
        NONE_UNLESS(operand(PyList_GET_ITEM(args[0], i), g) && !wants_grad(*g) && g->is_non_overlapping_and_dense() &&
                    g->layout() == at::kStrided);
        const int dtype = g->scalar_type() == at::kDouble ? BPL_DOUBLE : dtype_of(*g);
        held.add(PyList_GET_ITEM(args[0], i));
        if (first == nullptr) first = g;
        NONE_UNLESS(dtype >= 0 && g->device() == first->device());
        any_double |= dtype == BPL_DOUBLE;
        tensors[i].elements = static_cast<uint64_t>(g->numel());
        tensors[i].dtype = static_cast<uint32_t>(dtype);
        buffers[i] = ptr(*g);
        if (write) {
            NONE_UNLESS(operand(PyList_GET_ITEM(args[1], i), o) && !wants_grad(*o));
            NONE_UNLESS(o->scalar_type() == g->scalar_type() && o->sizes() == g->sizes() && o->strides() == g->strides() &&
                        o->device() == g->device());
            held.add(PyList_GET_ITEM(args[1], i));
            buffers[n + i] = ptr(*o);
            in_place &= ptr(*o) == ptr(*g);
        }
    }
    d->tensors = static_cast<uint32_t>(n);
    d->norm_type = static_cast<uint32_t>(norm_type);
    d->norm_dtype = any_double ? BPL_DOUBLE : BPL_FLOAT;
    d->flags = (write ? BPL_CLIP_WRITE : 0) | (in_place ? BPL_CLIP_IN_PLACE : 0);
    d->max_norm = max_norm;
    Tensor norm;
    {
        NoGil no_gil;
        OnDevice on(*first);
        norm = new_tensor({}, any_double ? at::kDouble : at::kFloat, first->device());
        Scratch ws(bpl_workspace_bytes("clip_gradients", opaque.data(), opaque.size()), on.stream);
        buffers[2 * n] = ptr(norm);
        buffers[2 * n + 1] = ws.ptr;
        clip_gradients(on.stream, buffers.data(), opaque.data(), opaque.size());
        char message[256];
        if (bpl_last_status(message, sizeof(message)) == BPL_ERR_ARGUMENT) {
            bpl_clear_status();
            TORCH_CHECK_VALUE(false, message);
        }
        check_status();
    }
    if (write)
        for (size_t i = 1; i < held.objects.size(); i += 2) written(THPVariable_Unpack(held.objects[i]));
    return wrap(std::move(norm));
    END_HANDLE_TH_ERRORS
}
