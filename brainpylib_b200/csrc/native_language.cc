// The native host path of the layers of language models (embedding, norm_rotate, decay_attention and its single step): the contract of
// native_sequence.cc.
#include "native_rows.h"

#include <cmath>
#include <limits>
#include <vector>

namespace {

// (tokens, heads, size) or (batch, length, heads, size) with neighbouring elements of a head next to one another
bool heads_of(const Tensor &t, Rows &r, int64_t &heads, int64_t &size, int64_t &head_stride) {
    if (t.dim() < 3 || !rows_of(t, 2, r)) return false;
    heads = t.size(-2);
    size = t.size(-1);
    head_stride = heads > 1 ? t.stride(-2) : 0;
    return heads <= 65535 && r.rows < (1ll << 31);
}
bool is_int(const Tensor &t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
// (what is no number the Python operators refuse)
bool as_float(PyObject *o, float &v) {
    double d;
    if (!number_of(o, d) || d != d) return false;
    v = static_cast<float>(d);
    return true;
}

// ---- embedding --------------------------------------------------------------------------------------------------------
struct Lookup {
    const Tensor *ids, *weight;
    bpl_embedding_descriptor d;

    bool check(float scale) {
        const int dtype = dtype_of(*weight);
        if (dtype < 0 || weight->dim() != 2 || !is_int(*ids) || !ids->is_contiguous() || ids->device() != weight->device() ||
            (weight->size(1) > 1 && weight->stride(1) != 1))
            return false;
        if (ids->numel() >= (1ll << 31) || weight->size(0) >= (1ll << 31) || weight->size(1) >= (1ll << 28)) return false;
        std::memset(&d, 0, sizeof(d));
        d.tokens = static_cast<uint32_t>(ids->numel());
        d.vocabulary = static_cast<uint32_t>(weight->size(0));
        d.width = static_cast<uint32_t>(weight->size(1));
        d.dtype = static_cast<uint32_t>(dtype);
        d.wide_ids = ids->scalar_type() == at::kLong;
        d.scale = scale;
        d.weight_stride = weight->numel() ? weight->stride(0) : 0;
        return true;
    }
};

Tensor lookup(const Lookup &s) {
    NoGil no_gil;
    OnDevice on(*s.weight);
    std::vector<int64_t> sizes(s.ids->sizes().begin(), s.ids->sizes().end());
    sizes.push_back(s.weight->size(1));
    const Tensor y = new_tensor(sizes, s.weight->scalar_type(), s.weight->device());
    void *buffers[3] = {ptr(*s.ids), ptr(*s.weight), ptr(y)};
    embedding(on.stream, buffers, reinterpret_cast<const char *>(&s.d), sizeof(s.d));
    check_status();
    return y;
}

struct EmbeddingFn : public torch::autograd::Function<EmbeddingFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &weight, const Tensor &ids, double scale) {
        Lookup s{&ids, &weight, {}};
        TORCH_CHECK(s.check(static_cast<float>(scale)), "embedding: operands changed between the passes");
        ctx->save_for_backward({ids});
        ctx->saved_data["d"] = scale;
        ctx->saved_data["n"] = std::vector<int64_t>{weight.size(0), weight.size(1)};
        return {lookup(s)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        if (!grads[0].defined()) return variable_list(3);
        const auto saved = ctx->get_saved_variables();
        const Tensor &ids = saved[0];
        if (!plain_cotangent_keys(grads[0])) throw std::runtime_error("gradients of embedding are plain CUDA tensors only");
        const Tensor dy = grads[0].contiguous();
        const std::vector<int64_t> sizes = ctx->saved_data["n"].toIntVector();
        NoGil no_gil;
        OnDevice on(ids);
        const Tensor dw = new_tensor(sizes, dy.scalar_type(), ids.device());
        Lookup s{&ids, &dw, {}};
        TORCH_CHECK(s.check(static_cast<float>(ctx->saved_data["d"].toDouble())), "embedding: operands changed between the passes");
        const char *opaque = reinterpret_cast<const char *>(&s.d);
        Scratch ws(bpl_workspace_bytes("embedding_backward", opaque, sizeof(s.d)), on.stream);
        void *buffers[4] = {ptr(ids), ptr(dy), ptr(dw), ws.ptr};
        embedding_backward(on.stream, buffers, opaque, sizeof(s.d));
        check_status();
        return differentiable_once({dw, Tensor(), Tensor()}, "embedding");
    }
};

// ---- norm_rotate ------------------------------------------------------------------------------------------------------
struct Rotate {
    const Tensor *q, *k, *positions, *frequencies, *q_weight, *k_weight;
    bpl_norm_rotate_descriptor d;

    // args: q, k, positions, frequencies, q_weight, k_weight
    bool read(PyObject *const *args, float eps, bool interleaved) {
        return operand(args[0], q) && operand(args[1], k) && operand(args[2], positions) && operand(args[3], frequencies) &&
               operand(args[4], q_weight, true) && operand(args[5], k_weight, true) && check(eps, interleaved);
    }
    void set(const Tensor &q_, const Tensor &k_, const Tensor &positions_, const Tensor &frequencies_, const Tensor &q_weight_,
             const Tensor &k_weight_, float eps, bool interleaved) {
        q = &q_; k = &k_; positions = &positions_; frequencies = &frequencies_;
        q_weight = or_null(q_weight_); k_weight = or_null(k_weight_);
        TORCH_CHECK(check(eps, interleaved), "norm_rotate: operands changed between the passes");
    }
    bool check(float eps, bool interleaved) {
        const int dtype = dtype_of(*q);
        Rows r, rk;
        int64_t heads, k_heads, size, k_size, stride, k_stride;
        if (dtype < 0 || k->scalar_type() != q->scalar_type() || !heads_of(*q, r, heads, size, stride) ||
            !heads_of(*k, rk, k_heads, k_size, k_stride) || !same_rows(r, rk) || size != k_size || size < 2 || size > 256 || size % 2 != 0)
            return false;
        if (!is_int(*positions) || !positions->is_contiguous() || positions->dim() != (r.batched ? 2 : 1) || positions->numel() != r.rows ||
            positions->size(0) != (r.batched ? r.batch : r.rows))
            return false;
        if (frequencies->scalar_type() != at::kFloat || frequencies->dim() != 1 || !frequencies->is_contiguous() ||
            2 * frequencies->numel() > size || wants_grad(*frequencies))
            return false;
        int weight_dtype = dtype;
        for (const Tensor *w : {q_weight, k_weight}) {
            if (w == nullptr) continue;
            weight_dtype = dtype_of(*w);
            if ((weight_dtype != dtype && weight_dtype != BPL_FLOAT) || !dense(w, w->scalar_type(), {size}, *q)) return false;
        }
        if (q_weight && k_weight && q_weight->scalar_type() != k_weight->scalar_type()) return false;
        for (const Tensor *t : {k, positions, frequencies})
            if (t->device() != q->device()) return false;
        std::memset(&d, 0, sizeof(d));
        d.tokens = static_cast<uint32_t>(r.rows);
        d.q_heads = static_cast<uint32_t>(heads);
        d.k_heads = static_cast<uint32_t>(k_heads);
        d.size = static_cast<uint32_t>(size);
        d.rotated = static_cast<uint32_t>(2 * frequencies->numel());
        d.dtype = static_cast<uint32_t>(dtype);
        d.weight_dtype = static_cast<uint32_t>(weight_dtype);
        d.flags = (interleaved ? BPL_ROTATE_INTERLEAVED : 0) | (positions->scalar_type() == at::kLong ? BPL_ROTATE_WIDE_POSITIONS : 0);
        d.eps = eps;
        d.q_stride = r.stride; d.q_head_stride = stride;
        d.k_stride = rk.stride; d.k_head_stride = k_stride;
        return true;
    }
    bool wants() const {
        for (const Tensor *t : {q, k, q_weight, k_weight})
            if (t && wants_grad(*t)) return true;
        return false;
    }
};

variable_list rotate_forward(const Rotate &s) {
    NoGil no_gil;
    OnDevice on(*s.q);
    const Tensor q = new_tensor(s.q->sizes(), s.q->scalar_type(), s.q->device()), k = new_tensor(s.k->sizes(), s.k->scalar_type(), s.k->device());
    void *buffers[8] = {ptr(*s.q), ptr(*s.k), ptr(*s.positions), ptr(*s.frequencies), ptr_of(s.q_weight), ptr_of(s.k_weight), ptr(q), ptr(k)};
    norm_rotate(on.stream, buffers, reinterpret_cast<const char *>(&s.d), sizeof(s.d));
    check_status();
    return {q, k};
}

struct RotateFn : public torch::autograd::Function<RotateFn> {
    using Maybe = std::optional<Tensor>;
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Maybe &q_weight, const Maybe &k_weight,
                                 const Tensor &positions, const Tensor &frequencies, double eps, bool interleaved) {
        const Tensor wq = value(q_weight), wk = value(k_weight);
        Rotate s;
        s.set(q, k, positions, frequencies, wq, wk, static_cast<float>(eps), interleaved);
        ctx->save_for_backward({q, k, positions, frequencies, wq, wk});
        ctx->saved_data["e"] = eps;
        ctx->saved_data["i"] = interleaved;
        ctx->set_materialize_grads(false);
        return rotate_forward(s);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(8);
        Rotate s;
        s.set(saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], static_cast<float>(ctx->saved_data["e"].toDouble()),
              ctx->saved_data["i"].toBool());
        const Tensor gq = cotangent(grads[0], *s.q), gk = cotangent(grads[1], *s.k);
        NoGil no_gil;
        OnDevice on(*s.q);
        const auto type = s.q->scalar_type();
        const auto device = s.q->device();
        const Tensor dq = new_tensor(s.q->sizes(), type, device), dk = new_tensor(s.k->sizes(), type, device),
                     dwq = s.q_weight ? new_tensor(s.q_weight->sizes(), s.q_weight->scalar_type(), device) : Tensor(),
                     dwk = s.k_weight ? new_tensor(s.k_weight->sizes(), s.k_weight->scalar_type(), device) : Tensor();
        const char *opaque = reinterpret_cast<const char *>(&s.d);
        Scratch ws(bpl_workspace_bytes("norm_rotate_backward", opaque, sizeof(s.d)), on.stream);
        void *buffers[13] = {ptr(*s.q), ptr(*s.k), ptr(*s.positions), ptr(*s.frequencies), ptr_of(s.q_weight), ptr_of(s.k_weight), ptr(gq), ptr(gk),
                             ptr(dq), ptr(dk), at_or_null(dwq), at_or_null(dwk), ws.ptr};
        norm_rotate_backward(on.stream, buffers, opaque, sizeof(s.d));
        check_status();
        return differentiable_once({dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor()}, "norm_rotate");
    }
};

// ---- decay_attention ----------------------------------------------------------------------------------------------------
struct Attend {
    const Tensor *q, *k, *v, *log_decay, *indptr, *initial;
    Rows rows;
    bpl_decay_attention_descriptor d;
    int64_t sequences;

    // args: q, k, v, log_decay
    bool read(PyObject *const *args, double scale) {
        return operand(args[0], q) && operand(args[1], k) && operand(args[2], v) && operand(args[3], log_decay) && check(scale);
    }
    void set(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &log_decay_, const Tensor &indptr_, const Tensor &initial_,
             double scale) {
        q = &q_; k = &k_; v = &v_; log_decay = &log_decay_;
        indptr = or_null(indptr_); initial = or_null(initial_);
        TORCH_CHECK(check(scale) && check_sequences(), "decay_attention: operands changed between the passes");
    }
    // (NaN stands for the default scale, which a given one cannot be)
    bool check(double scale) {
        const int dtype = dtype_of(*q);
        Rows rk, rv;
        int64_t heads, k_heads, v_heads, key, k_size, value;
        std::memset(&d, 0, sizeof(d));
        if (dtype < 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
            !heads_of(*q, rows, heads, key, d.q_head_stride) || !heads_of(*k, rk, k_heads, k_size, d.k_head_stride) ||
            !heads_of(*v, rv, v_heads, value, d.v_head_stride) || !same_rows(rows, rk) || !same_rows(rows, rv) || k_size != key ||
            v_heads != k_heads || k_heads < 1 || heads < 1 || heads % k_heads != 0 || key < 1 || key > 256 || value < 1 || value > 256)
            return false;
        for (const Tensor *t : {k, v})
            if (t->device() != q->device()) return false;
        if (!dense(log_decay, at::kFloat, {heads}, *q) || wants_grad(*log_decay)) return false;
        d.tokens = static_cast<uint32_t>(rows.rows);
        d.length = static_cast<uint32_t>(rows.length);
        d.heads = static_cast<uint32_t>(heads);
        d.kv_heads = static_cast<uint32_t>(k_heads);
        d.key = static_cast<uint32_t>(key);
        d.value = static_cast<uint32_t>(value);
        d.dtype = static_cast<uint32_t>(dtype);
        d.scale = static_cast<float>(scale != scale ? 1.0 / std::sqrt(static_cast<double>(key)) : scale);
        d.q_stride = rows.stride; d.k_stride = rk.stride; d.v_stride = rv.stride;
        return true;
    }
    bool read_sequences(PyObject *p, PyObject *i) {
        return operand(p, indptr, true) && operand(i, initial, true) && check_sequences();
    }
    bool check_sequences() {
        sequences = rows.batch;
        if (indptr) {
            if (rows.batched || indptr->scalar_type() != at::kInt || indptr->dim() != 1 || indptr->size(0) < 1 ||
                (indptr->size(0) > 1 && indptr->stride(0) != 1) || indptr->device() != q->device())
                return false;
            sequences = indptr->size(0) - 1;
        }
        if (sequences >= (1ll << 31)) return false;
        d.sequences = static_cast<uint32_t>(sequences);
        return !initial || dense(initial, at::kFloat, state_sizes(), *q);
    }
    std::vector<int64_t> state_sizes() const { return {sequences, q->size(-2), q->size(-1), v->size(-1)}; }
    std::vector<int64_t> out_sizes() const {
        std::vector<int64_t> s(q->sizes().begin(), q->sizes().end());
        s.back() = v->size(-1);
        return s;
    }
    bool wants() const {
        for (const Tensor *t : {q, k, v, initial})
            if (t && wants_grad(*t)) return true;
        return false;
    }
};
bool scale_of(PyObject *o, double &v) {
    if (o == Py_None) {
        v = std::numeric_limits<double>::quiet_NaN();
        return true;
    }
    return number_of(o, v) && v == v;
}

struct AttendResult {
    Tensor y, last;
};
AttendResult attend_forward(const Attend &s, bool want_last) {
    NoGil no_gil;
    OnDevice on(*s.q);
    AttendResult r;
    r.y = new_tensor(s.out_sizes(), s.q->scalar_type(), s.q->device());
    if (want_last) r.last = new_tensor(s.state_sizes(), at::kFloat, s.q->device());
    const char *opaque = reinterpret_cast<const char *>(&s.d);
    Scratch ws(bpl_workspace_bytes("decay_attention", opaque, sizeof(s.d)), on.stream);
    void *buffers[9] = {ptr(*s.q), ptr(*s.k), ptr(*s.v), ptr(*s.log_decay), ptr_of(s.indptr), ptr_of(s.initial), ptr(r.y), at_or_null(r.last), ws.ptr};
    decay_attention(on.stream, buffers, opaque, sizeof(s.d));
    check_status();
    return r;
}

struct AttendFn : public torch::autograd::Function<AttendFn> {
    using Maybe = std::optional<Tensor>;
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Maybe &initial,
                                 const Tensor &log_decay, const Maybe &indptr, double scale, bool want_last) {
        const Tensor i = value(initial), p = value(indptr);
        Attend s;
        s.set(q, k, v, log_decay, p, i, scale);
        AttendResult r = attend_forward(s, want_last);
        ctx->save_for_backward({q, k, v, log_decay, i, p});
        ctx->saved_data["s"] = scale;
        ctx->set_materialize_grads(false);
        return want_last ? variable_list{r.y, r.last} : variable_list{r.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        if (!grads[0].defined() && (grads.size() < 2 || !grads[1].defined())) return variable_list(8);
        Attend s;
        s.set(saved[0], saved[1], saved[2], saved[3], saved[5], saved[4], ctx->saved_data["s"].toDouble());
        const Tensor dy = grads[0].defined() ? cotangent(grads[0], grads[0]) : at::zeros(s.out_sizes(), s.q->options());
        const Tensor d_last = grads.size() > 1 && grads[1].defined() ? cotangent(grads[1], grads[1]) : Tensor();
        NoGil no_gil;
        OnDevice on(*s.q);
        const auto type = s.q->scalar_type();
        const auto device = s.q->device();
        const Tensor dq = new_tensor(s.q->sizes(), type, device), dk = new_tensor(s.k->sizes(), type, device),
                     dv = new_tensor(s.v->sizes(), type, device),
                     d_initial = s.initial ? new_tensor(s.initial->sizes(), at::kFloat, device) : Tensor();
        const char *opaque = reinterpret_cast<const char *>(&s.d);
        Scratch ws(bpl_workspace_bytes("decay_attention_backward", opaque, sizeof(s.d)), on.stream);
        void *buffers[13] = {ptr(*s.q), ptr(*s.k), ptr(*s.v), ptr(*s.log_decay), ptr_of(s.indptr), ptr_of(s.initial), ptr(dy), at_or_null(d_last),
                             ptr(dq), ptr(dk), ptr(dv), at_or_null(d_initial), ws.ptr};
        decay_attention_backward(on.stream, buffers, opaque, sizeof(s.d));
        check_status();
        return differentiable_once({dq, dk, dv, d_initial, Tensor(), Tensor(), Tensor(), Tensor()}, "decay_attention");
    }
};

}  // namespace

// embedding(ids, weight, scale) -> y
PyObject *py_embedding(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Lookup s;
    float scale;
    NONE_UNLESS(nargs == 3 && plain_thread() && operand(args[0], s.ids) && operand(args[1], s.weight) && as_float(args[2], scale) && s.check(scale));
    if (wants_grad(*s.weight)) return wrap(EmbeddingFn::apply(*s.weight, *s.ids, static_cast<double>(scale))[0]);
    return wrap(lookup(s));
    END_HANDLE_TH_ERRORS
}

// norm_rotate(q, k, positions, frequencies, q_weight, k_weight, eps, interleaved) -> (q, k)
PyObject *py_norm_rotate(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Rotate s;
    float eps;
    NONE_UNLESS(nargs == 8 && plain_thread() && as_float(args[6], eps) && is_flag(args[7]) && s.read(args, eps, truth(args[7])));
    const variable_list r = s.wants() ? RotateFn::apply(*s.q, *s.k, maybe(s.q_weight), maybe(s.k_weight), *s.positions, *s.frequencies,
                                                        static_cast<double>(eps), truth(args[7]))
                                      : rotate_forward(s);
    return tuple_of({r[0], r[1]});
    END_HANDLE_TH_ERRORS
}

// decay_attention(q, k, v, log_decay, scale, indptr, initial_state, return_state) -> y, or (y, last)
PyObject *py_decay_attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Attend s;
    double scale;
    NONE_UNLESS(nargs == 8 && plain_thread() && scale_of(args[4], scale) && is_flag(args[7]) && s.read(args, scale) &&
                s.read_sequences(args[5], args[6]));
    const bool want_last = truth(args[7]);
    if (s.wants())
        return one_or_two(AttendFn::apply(*s.q, *s.k, *s.v, maybe(s.initial), *s.log_decay, maybe(s.indptr), scale, want_last));
    const AttendResult r = attend_forward(s, want_last);
    return want_last ? tuple_of({r.y, r.last}) : wrap(r.y);
    END_HANDLE_TH_ERRORS
}

// decay_attention_step(q, k, v, log_decay, state, scale, slots) -> y
PyObject *py_decay_attention_step(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Attend s;
    double scale;
    const Tensor *state, *slots;
    NONE_UNLESS(nargs == 7 && plain_thread() && scale_of(args[5], scale) && s.read(args, scale) && !s.rows.batched && operand(args[4], state) &&
                operand(args[6], slots, true));
    s.initial = nullptr;
    NONE_UNLESS(!s.wants() && !wants_grad(*state) && state->dim() == 4 && state->size(0) < (1ll << 31) && s.rows.rows <= 65535 &&
                dense(state, at::kFloat, {state->size(0), s.q->size(1), s.q->size(2), s.v->size(2)}, *s.q));
    if (slots) NONE_UNLESS(dense(slots, at::kInt, {s.rows.rows}, *s.q));
    else NONE_UNLESS(s.rows.rows == state->size(0));
    s.d.sequences = static_cast<uint32_t>(state->size(0));
    Tensor y;
    {
        NoGil no_gil;
        OnDevice on(*s.q);
        y = new_tensor(s.out_sizes(), s.q->scalar_type(), s.q->device());
        void *buffers[7] = {ptr(*s.q), ptr(*s.k), ptr(*s.v), ptr(*s.log_decay), ptr_of(slots), ptr(*state), ptr(y)};
        decay_attention_step(on.stream, buffers, reinterpret_cast<const char *>(&s.d), sizeof(s.d));
        check_status();
        written(*state);
    }
    return wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}
