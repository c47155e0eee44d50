// torch-library shim of the operators of a mixer with heads and of a model's answer: rotary positions, linear attention,
// sampling from logits.  Checks, allocation and autograd; the kernels are behind the C ABI of libbutterfly_hip.so.  Device tensors
// only: the Python functions of the same names compose them from tensor operations for host tensors.

#include "shim.hpp"

namespace {

// ---- rotary positions -----------------------------------------------------------------------------------

Tensor rotary_op(const Tensor &x, const Tensor &positions, const Tensor &frequencies, bool interleaved, double magnitude, bool back);

Tensor rotary_run(const Tensor &input, const Tensor &positions, const Tensor &frequencies, bool interleaved, double magnitude, bool back)
{
    const char *who = "rotary";
    const Guard guard(input.device());
    const Tensor where = plain(positions), f = dense(frequencies);
    Tensor x = plain(input);
    bf_rotary d = {};
    d.dtype = dtype_code(x, false, who);
    d.interleaved = interleaved;
    d.heads = x.size(-2);
    d.features = x.size(-1);
    d.rotated = 2 * f.size(0);
    d.magnitude = magnitude;
    // (batch, steps) from whatever leads
    const int64_t lead = x.dim() - 2;
    Tensor at = where;
    if (lead != 2) {
        const int64_t last = lead > 0 ? x.size(lead - 1) : 1, rest = lead > 0 ? row_count(where) : 1;
        x = x.reshape({rest, last, d.heads, d.features});
        at = where.reshape({rest, last});
    }
    if (d.features > 1 && x.stride(3) != 1) x = x.contiguous();
    d.batch = x.size(0);
    d.steps = x.size(1);
    for (int i = 0; i < 3; ++i) d.x_stride[i] = x.size(i) > 1 ? x.stride(i) : 0;
    for (int i = 0; i < 2; ++i) d.position_stride[i] = at.size(i) > 1 ? at.stride(i) : 0;
    Tensor y = at::empty(input.sizes(), input.options());
    check_rc(bf_rotary_apply(&d, x.data_ptr(), static_cast<const int64_t *>(at.data_ptr()), static_cast<const double *>(f.data_ptr()),
                             y.data_ptr(), back, current_stream()),
             who);
    return y;
}

struct RotaryNode : public torch::autograd::Node {
    SavedSlot positions, frequencies;
    bool interleaved = false, back = false;
    double magnitude = 1.0;

    // edge: x.  The gradient is the operator itself, turned the other way, with derivatives of its own.
    variable_list apply(variable_list &&grads) override
    {
        variable_list out(num_outputs());
        if (!grads[0].defined()) return out;
        std::lock_guard<std::mutex> lock(mutex_);
        const auto self = getptr();
        out[0] = rotary_op(grads[0], positions.get(self), frequencies.get(self), interleaved, magnitude, !back);
        return out;
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedSlot *s : {&positions, &frequencies}) s->drop();
    }

    std::string name() const override { return "RotaryBackward"; }
};

Tensor rotary_op(const Tensor &x, const Tensor &positions, const Tensor &frequencies, bool interleaved, double magnitude, bool back)
{
    refuse_tangents({x}, "rotary");
    if (!any_wants_grad({x})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return rotary_run(x, positions, frequencies, interleaved, magnitude, back);
    }
    std::shared_ptr<RotaryNode> node(new RotaryNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = rotary_run(x, positions, frequencies, interleaved, magnitude, back);
    }
    node->positions.set(positions);
    node->frequencies.set(frequencies);
    node->interleaved = interleaved;
    node->magnitude = magnitude;
    node->back = back;
    torch::autograd::set_history(y, node);
    return y;
}

Tensor rotary(Tensor x, Tensor positions, Tensor frequencies, bool interleaved, double magnitude)
{
    const char *who = "rotary";
    require_device(x, who);
    require_beside(positions, x, "positions", who);
    require_beside(frequencies, x, "frequencies", who);
    TORCH_CHECK(x.dim() >= 2, who, ": x must have shape (*, heads, features)");
    dtype_code(x, false, who);
    TORCH_CHECK(positions.scalar_type() == at::kLong, who, ": positions must be int64");
    TORCH_CHECK(positions.sizes() == x.sizes().slice(0, x.dim() - 2), who, ": positions must have the shape of x without heads and features");
    TORCH_CHECK(frequencies.scalar_type() == at::kDouble && frequencies.dim() == 1 && !frequencies.requires_grad(), who,
                ": frequencies must be one float64 for each pair, without gradient");
    TORCH_CHECK(2 * frequencies.size(0) <= x.size(-1), who, ": more frequencies than pairs of features");
    return rotary_op(x, positions, frequencies, interleaved, magnitude, false);
}

// ---- linear attention -----------------------------------------------------------------------------------

struct Attention {
    Tensor q, k, v, log_decay, state, reset;
    double scale = 1.0;
    const char *who = nullptr;
};

void strides_of(int64_t (&dst)[3], const Tensor &t, int64_t lead)
{
    // (without steps: one of them)
    for (int i = 0; i < 3; ++i) dst[i] = 0;
    if (t.size(0) > 1) dst[0] = t.stride(0);
    if (lead == 2 && t.size(1) > 1) dst[1] = t.stride(1);
    if (t.size(lead) > 1) dst[2] = t.stride(lead);
}

// q, k, v as the kernels read them: features adjacent
void lay_out(Attention &o)
{
    o.q = adjacent(o.q);
    o.k = adjacent(o.k);
    o.v = adjacent(o.v);
    o.log_decay = plain(o.log_decay);
    o.state = dense(o.state);
}

bf_linear_attention describe(const Attention &o)
{
    const int64_t lead = o.v.dim() - 2;
    bf_linear_attention d = {};
    d.dtype = dtype_code(o.v, false, o.who);
    d.batch = o.v.size(0);
    d.steps = lead == 2 ? o.v.size(1) : 1;
    d.heads = o.v.size(lead);
    d.groups = o.q.size(lead);
    d.features = o.q.size(lead + 1);
    d.values = o.v.size(lead + 1);
    strides_of(d.q_stride, o.q, lead);
    strides_of(d.k_stride, o.k, lead);
    strides_of(d.v_stride, o.v, lead);
    strides_of(d.decay_stride, o.log_decay, lead);
    if (o.reset.defined()) batch_steps(d.reset_stride, o.reset);
    d.scale = o.scale;
    return d;
}

void check_attention(const Attention &o, int64_t dims)
{
    const char *who = o.who, *lead = dims == 4 ? "(batch, steps, " : "(batch, ";
    require_device(o.v, who);
    require_beside(o.q, o.v, "q", who);
    require_beside(o.k, o.v, "k", who);
    require_beside(o.log_decay, o.v, "log_decay", who);
    TORCH_CHECK(o.v.dim() == dims, who, ": v must have shape ", lead, "heads, values)");
    TORCH_CHECK(o.q.dim() == dims && o.q.sizes() == o.k.sizes() && o.q.sizes().slice(0, dims - 2) == o.v.sizes().slice(0, dims - 2), who,
                ": q and k must have shape ", lead, "groups, features)");
    dtype_code(o.v, false, who);
    TORCH_CHECK(o.q.scalar_type() == o.v.scalar_type() && o.k.scalar_type() == o.v.scalar_type(), who, ": q, k and v must have the same dtype");
    const int64_t heads = o.v.size(dims - 2), groups = o.q.size(dims - 2);
    TORCH_CHECK(groups > 0 ? heads % groups == 0 : heads == 0, who, ": heads of v must be a multiple of those of q and k");
    TORCH_CHECK(o.q.size(-1) > 0 && o.v.size(-1) > 0 && o.q.size(-1) <= 128 && o.v.size(-1) <= 128, who,
                ": heads of 1 to 128 features and values are supported");
    TORCH_CHECK(o.log_decay.sizes() == o.v.sizes().slice(0, dims - 1), who, ": log_decay must have shape ", lead, "heads)");
    TORCH_CHECK(o.log_decay.scalar_type() == at::kFloat, who, ": log_decay must be float32");
    if (o.state.defined()) {
        require_beside(o.state, o.v, "state", who);
        TORCH_CHECK(o.state.dim() == 4 && o.state.size(0) == o.v.size(0) && o.state.size(1) == heads && o.state.size(2) == o.q.size(-1) &&
                        o.state.size(3) == o.v.size(-1),
                    who, ": state must have shape (batch, heads, features, values)");
        TORCH_CHECK(o.state.scalar_type() == at::kFloat, who, ": state must be float32");
    }
    if (o.reset.defined()) {
        require_beside(o.reset, o.v, "reset", who);
        TORCH_CHECK(o.reset.scalar_type() == at::kBool, who, ": reset must be bool");
        TORCH_CHECK(o.reset.dim() == 2 && o.reset.size(0) == o.v.size(0) && o.reset.size(1) == o.v.size(1), who,
                    ": reset must have shape (batch, steps)");
    }
}

// kept: filled where the caller asks for it
std::tuple<Tensor, Tensor> attention_fw(Attention o, Tensor *kept)
{
    const Guard guard(o.v.device());
    lay_out(o);
    const bf_linear_attention d = describe(o);
    const auto floats = o.v.options().dtype(at::kFloat);
    Tensor out = at::empty(o.v.sizes(), o.v.options());
    Tensor last = at::empty({d.batch, d.heads, d.features, d.values}, floats);
    const size_t bytes = valid_size(bf_linear_attention_fw_workspace_bytes(&d));
    const size_t kept_bytes = kept ? valid_size(bf_linear_attention_kept_bytes(&d)) : 0;
    const Tensor ws = workspace_like(o.v, bytes);
    if (kept) *kept = at::empty({(int64_t)kept_bytes}, o.v.options().dtype(at::kByte));
    check_rc(bf_linear_attention_fw(&d, o.q.data_ptr(), o.k.data_ptr(), o.v.data_ptr(), o.log_decay.data_ptr<float>(),
                                    static_cast<const float *>(ptr(o.state)), static_cast<const uint8_t *>(ptr(o.reset)), out.data_ptr(),
                                    last.data_ptr<float>(), kept_bytes > 0 ? kept->data_ptr() : nullptr, kept_bytes, ptr(ws), bytes,
                                    current_stream()),
             o.who);
    return {out, last};
}

struct AttentionNode : public torch::autograd::Node {
    SavedSlot q, k, v, log_decay, reset, kept;
    double scale = 1.0;
    bool with_state = false;
    const char *who = nullptr;

    // edges: q, k, v, log_decay, state
    variable_list apply(variable_list &&grads) override
    {
        variable_list out(num_outputs());
        if (!grads[0].defined() && !grads[1].defined()) return out;
        std::lock_guard<std::mutex> lock(mutex_);
        const auto self = getptr();
        Attention o;
        o.q = q.get(self);
        o.k = k.get(self);
        o.v = v.get(self);
        o.log_decay = log_decay.get(self);
        o.reset = reset.get(self);
        o.scale = scale;
        o.who = who;
        const Tensor states = kept.get(self);
        const bool want_state = task_should_compute_output(4);
        at::AutoDispatchBelowADInplaceOrView below;
        const Guard guard(o.v.device());
        lay_out(o);
        bf_linear_attention d = describe(o);
        const Tensor g = grads[0].defined() ? adjacent(grads[0]) : Tensor(), gl = dense(grads[1]);
        if (g.defined()) strides_of(d.grad_stride, g, 2);
        out[0] = at::empty(o.q.sizes(), o.q.options());
        out[1] = at::empty(o.k.sizes(), o.k.options());
        out[2] = at::empty(o.v.sizes(), o.v.options());
        out[3] = at::empty(o.log_decay.sizes(), o.log_decay.options());
        if (want_state) out[4] = at::empty({d.batch, d.heads, d.features, d.values}, o.log_decay.options());
        const size_t bytes = valid_size(bf_linear_attention_bw_workspace_bytes(&d));
        const Tensor ws = workspace_like(o.v, bytes);
        check_rc(bf_linear_attention_bw(&d, o.q.data_ptr(), o.k.data_ptr(), o.v.data_ptr(), o.log_decay.data_ptr<float>(),
                                        static_cast<const uint8_t *>(ptr(o.reset)), states.data_ptr(), (size_t)states.numel(), ptr(g),
                                        static_cast<const float *>(ptr(gl)), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(),
                                        out[3].data_ptr<float>(), static_cast<float *>(ptr(out[4])), ptr(ws), bytes, current_stream()),
                 who);
        refuse_second(out, *this, {grads[0], grads[1]}, who);
        return out;
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedSlot *s : {&q, &k, &v, &log_decay, &reset, &kept}) s->drop();
    }

    std::string name() const override { return "LinearAttentionBackward"; }
};

// (o, last)
std::tuple<Tensor, Tensor> linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, OptTensor state, OptTensor reset, double scale)
{
    Attention o;
    o.q = q;
    o.k = k;
    o.v = v;
    o.log_decay = log_decay;
    o.state = opt(state);
    o.reset = opt(reset);
    o.scale = scale;
    o.who = "linear_attention";
    check_attention(o, 4);
    refuse_tangents({o.q, o.k, o.v, o.log_decay, o.state}, o.who);
    if (!any_wants_grad({o.q, o.k, o.v, o.log_decay, o.state})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return attention_fw(o, nullptr);
    }
    std::shared_ptr<AttentionNode> node(new AttentionNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(o.q, o.k, o.v, o.log_decay, o.state));
    Tensor out, last, kept;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(out, last) = attention_fw(o, &kept);
    }
    node->q.set(o.q);
    node->k.set(o.k);
    node->v.set(o.v);
    node->log_decay.set(o.log_decay);
    node->reset.set(o.reset);
    node->kept.set(kept);
    node->scale = scale;
    node->who = o.who;
    torch::autograd::set_history(std::vector<Tensor>{out, last}, node);
    return {out, last};
}

// One new step of every sequence; state is updated in place.
Tensor linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor state, double scale)
{
    Attention o;
    o.q = q;
    o.k = k;
    o.v = v;
    o.log_decay = log_decay;
    o.state = state;
    o.scale = scale;
    o.who = "linear_attention_step";
    check_attention(o, 3);
    refuse_tangents({o.q, o.k, o.v, o.log_decay, o.state}, o.who);
    TORCH_CHECK(!any_wants_grad({o.q, o.k, o.v, o.log_decay, o.state}), o.who, ": has no gradient (use linear_attention, or torch.no_grad)");
    TORCH_CHECK(state.is_contiguous() && !state.is_neg(), o.who, ": state must be contiguous, it is updated in place");
    at::AutoDispatchBelowADInplaceOrView below;
    const Guard guard(v.device());
    lay_out(o);
    const bf_linear_attention d = describe(o);
    Tensor out = at::empty(o.v.sizes(), o.v.options());
    check_rc(bf_linear_attention_step(&d, o.q.data_ptr(), o.k.data_ptr(), o.v.data_ptr(), o.log_decay.data_ptr<float>(),
                                      state.data_ptr<float>(), out.data_ptr(), current_stream()),
             o.who);
    state.unsafeGetTensorImpl()->bump_version();
    return out;
}

// ---- sampling -------------------------------------------------------------------------------------------

// A setting: one a row, or (undefined) the number for all rows.
Tensor setting(const OptTensor &t, const Tensor &logits, at::ScalarType type, const char *name)
{
    const char *who = "sample";
    if (!t.has_value() || !t->defined()) return Tensor();
    require_beside(*t, logits, name, who);
    TORCH_CHECK(t->scalar_type() == type, who, ": ", name, " must be ", type, " or a number");
    TORCH_CHECK(t->sizes() == logits.sizes().slice(0, logits.dim() - 1), who, ": ", name, " must have the shape of logits without entries");
    return dense(*t);
}

Tensor sample(Tensor logits, Tensor uniform, OptTensor temperature, double temperature_all, OptTensor top_k, int64_t top_k_all,
              OptTensor top_p, double top_p_all, OptTensor min_p, double min_p_all)
{
    const char *who = "sample";
    require_device(logits, who);
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0, who, ": logits must have shape (*, entries)");
    at::AutoDispatchBelowADInplaceOrView below;
    const Guard guard(logits.device());
    bf_sample d = {};
    d.dtype = dtype_code(logits, false, who);
    TORCH_CHECK(uniform.defined(), who, ": uniform is missing");
    const Tensor u = setting(uniform, logits, at::kFloat, "uniform"), t = setting(temperature, logits, at::kFloat, "temperature"),
                 k = setting(top_k, logits, at::kLong, "top_k"), p = setting(top_p, logits, at::kFloat, "top_p"),
                 m = setting(min_p, logits, at::kFloat, "min_p");
    const Tensor rows = rows_of(logits);
    d.rows = rows.size(0);
    d.vocab = rows.size(1);
    d.logits_stride = row_stride(rows);
    d.temperature = temperature_all;
    d.top_k = top_k_all;
    d.top_p = top_p_all;
    d.min_p = min_p_all;
    Tensor token = at::empty(logits.sizes().slice(0, logits.dim() - 1), logits.options().dtype(at::kLong));
    check_rc(bf_sample_tokens(&d, rows.data_ptr(), u.data_ptr<float>(), static_cast<const float *>(ptr(t)),
                              static_cast<const int64_t *>(ptr(k)), static_cast<const float *>(ptr(p)), static_cast<const float *>(ptr(m)),
                              token.data_ptr<int64_t>(), current_stream()),
             who);
    return token;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torch_butterfly, m)
{
    m.def("rotary", rotary);
    m.def("linear_attention", linear_attention);
    m.def("linear_attention_step", linear_attention_step);
    m.def("sample", sample);
}
