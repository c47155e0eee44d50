// torch-library shim of the operators beside the multiply: rows (dropout, residual, layer norm), the gated
// recurrence, the linear layer with cross entropy.  Checks, allocation and autograd; the kernels are
// behind the C ABI of libbutterfly_hip.so.  Device tensors only: the Python functions of the same names
// compose them from tensor operations for host tensors.

#include "shim.hpp"

namespace {

// ---- rows: dropout, residual, layer norm ---------------------------------------------------------------

struct Rows {
    Tensor x, rng, residual, weight, bias;   // undefined: none
    double p = 0.0, eps = 0.0;
    bool norm = false;
    const char *who = nullptr;
};

bf_rowwise describe(const Rows &o, const Tensor &x)
{
    bf_rowwise d = {};
    d.dtype = dtype_code(x, false, o.who);
    d.param_dtype = d.dtype;
    for (const Tensor *t : {&o.weight, &o.bias})
        if (t->defined()) d.param_dtype = dtype_code(*t, false, o.who);
    d.rows = row_count(x);
    d.cols = x.size(-1);
    d.drop_probability = o.rng.defined() ? o.p : 0.0;
    d.eps = o.eps;
    return d;
}

void check_rows(const Rows &o)
{
    const char *who = o.who;
    require_device(o.x, who);
    TORCH_CHECK(o.x.dim() >= 1, who, ": the input must have at least one dimension");
    dtype_code(o.x, false, who);
    TORCH_CHECK(o.p >= 0.0 && o.p <= 1.0, who, ": p must be between 0 and 1, got ", o.p);
    if (o.rng.defined()) {
        require_beside(o.rng, o.x, "rng", who);
        TORCH_CHECK(o.rng.scalar_type() == at::kLong && o.rng.dim() == 1 && o.rng.size(0) == 2, who,
                    ": rng must hold two int64 (seed, call)");
    } else {
        TORCH_CHECK(o.p == 0.0, who, ": p > 0 needs rng");
    }
    if (o.residual.defined()) {
        require_beside(o.residual, o.x, "residual", who);
        TORCH_CHECK(o.residual.sizes() == o.x.sizes() && o.residual.scalar_type() == o.x.scalar_type(), who,
                    ": residual must have the shape and dtype of x");
    }
    for (const Tensor *t : {&o.weight, &o.bias}) {
        if (!t->defined()) continue;
        const char *name = t == &o.weight ? "weight" : "bias";
        require_beside(*t, o.x, name, who);
        TORCH_CHECK(t->dim() == 1 && t->size(0) == o.x.size(-1), who, ": ", name, " must have one entry per column");
        TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == o.x.scalar_type(), who, ": ", name,
                    " must be float32 or have the dtype of x");
    }
    TORCH_CHECK(!o.weight.defined() || !o.bias.defined() || o.weight.scalar_type() == o.bias.scalar_type(), who,
                ": weight and bias must have the same dtype");
    TORCH_CHECK(o.eps >= 0.0, who, ": eps must not be negative");
}

// sum and stats: filled where the caller asks for them (sum also where it is the only result)
Tensor rows_fw(const Rows &o, bool want_sum, Tensor *sum, Tensor *stats)
{
    const Guard guard(o.x.device());
    const Tensor x = rows_of(o.x), residual = o.residual.defined() ? rows_of(o.residual) : Tensor();
    bf_rowwise d = describe(o, o.x);
    d.x_stride = row_stride(x);
    if (residual.defined()) d.residual_stride = row_stride(residual);
    const Tensor weight = dense(o.weight), bias = dense(o.bias), rng = dense(o.rng);
    Tensor y, total;
    const auto options = o.x.options();
    if (o.norm) y = at::empty(o.x.sizes(), options);
    if (!o.norm || want_sum) total = at::empty(o.x.sizes(), options);
    if (stats) *stats = at::empty({d.rows, 2}, options.dtype(at::kFloat));
    if (x.numel() > 0)
        check_rc(bf_rowwise_fw(&d, x.data_ptr(), ptr(residual), static_cast<const int64_t *>(ptr(rng)), ptr(weight), ptr(bias),
                               ptr(total), ptr(y), stats ? stats->data_ptr<float>() : nullptr, current_stream()),
                 o.who);
    if (sum) *sum = total;
    return o.norm ? y : total;
}

std::tuple<Tensor, Tensor> rows_op(const Rows &o, bool two);

struct RowsNode : public torch::autograd::Node {
    SavedSlot total, stats, weight, rng;
    c10::SmallVector<int64_t, 6> shape;
    at::TensorOptions options;
    double p = 0.0, eps = 0.0;
    at::ScalarType param_type = at::kFloat;
    bool norm = false, two = false;
    const char *who = nullptr;

    // edges: x, residual, weight, bias
    variable_list apply(variable_list &&grads) override
    {
        variable_list out(num_outputs());
        const Tensor gy = grads[0], gs = two ? grads[1] : Tensor();
        if (!gy.defined() && !gs.defined()) return out;
        std::lock_guard<std::mutex> lock(mutex_);
        const auto self = getptr();
        const bool want_x = task_should_compute_output(0), want_residual = task_should_compute_output(1);
        Rows o;
        o.rng = rng.get(self);
        o.p = p;
        o.eps = eps;
        o.who = who;
        if (!norm || !gy.defined()) {
            // the gradient itself, through the mask for x: the operator itself, with derivatives of its own
            const Tensor g = gy.defined() ? gy : gs;
            if (want_residual) out[1] = g;
            if (want_x) {
                o.x = g;
                out[0] = o.rng.defined() ? std::get<0>(rows_op(o, false)) : g;
            }
            return out;
        }
        o.weight = weight.get(self);
        const Tensor sum = total.get(self), st = stats.get(self);
        apply_norm(o, gy, gs, sum, st, out);
        refuse_second(out, *this, {gy, gs}, who);
        return out;
    }

    void apply_norm(const Rows &o, const Tensor &gy, const Tensor &gs, const Tensor &sum, const Tensor &st, variable_list &out)
    {
        const bool want_x = task_should_compute_output(0), want_residual = task_should_compute_output(1);
        at::AutoDispatchBelowADInplaceOrView below;
        const bool want_weight = task_should_compute_output(2), want_bias = task_should_compute_output(3);
        const Guard guard(sum.device());
        bf_rowwise d = describe(o, sum);
        d.param_dtype = param_type == at::kFloat ? BF_F32 : BF_BF16;
        const Tensor x = rows_of(sum), g = rows_of(gy), more = gs.defined() ? rows_of(gs) : Tensor();
        d.x_stride = row_stride(x);
        d.grad_y_stride = row_stride(g);
        if (more.defined()) d.grad_sum_stride = row_stride(more);
        const Tensor w = dense(o.weight), state = dense(o.rng);
        // (without dropout the gradients of x and of the residual are one tensor)
        Tensor dx, dr;
        if (want_x && o.rng.defined()) dx = at::empty(shape, options);
        if (want_residual || (want_x && !o.rng.defined())) dr = at::empty(shape, options);
        if (want_weight) out[2] = at::empty({d.cols}, options.dtype(param_type));
        if (want_bias) out[3] = at::empty({d.cols}, options.dtype(param_type));
        const size_t bytes = want_weight || want_bias ? valid_size(bf_rowwise_bw_workspace_bytes(&d)) : 0;
        const Tensor ws = workspace_like(x, bytes);
        check_rc(bf_rowwise_bw(&d, x.data_ptr(), g.data_ptr(), ptr(more), static_cast<const int64_t *>(ptr(state)), ptr(w),
                               st.data_ptr<float>(), ptr(dx), ptr(dr), ptr(out[2]), ptr(out[3]), ptr(ws), bytes, current_stream()),
                 who);
        if (want_x) out[0] = dx.defined() ? dx : dr;
        if (want_residual) out[1] = dr;
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedSlot *s : {&total, &stats, &weight, &rng}) s->drop();
    }

    std::string name() const override { return norm ? "DropoutAddLayerNormBackward" : "DropoutAddBackward"; }
};

// two: the sum is a result beside y
std::tuple<Tensor, Tensor> rows_op(const Rows &o, bool two)
{
    check_rows(o);
    refuse_tangents({o.x, o.residual, o.weight, o.bias}, o.who);
    // what a norm's backward starts from: x itself where nothing is dropped or added
    const bool plain = !o.rng.defined() && !o.residual.defined();
    Tensor sum, stats, y;
    if (!any_wants_grad({o.x, o.residual, o.weight, o.bias})) {
        at::AutoDispatchBelowADInplaceOrView below;
        y = rows_fw(o, two, &sum, nullptr);
        return {y, sum};
    }
    std::shared_ptr<RowsNode> node(new RowsNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(o.x, o.residual, o.weight, o.bias));
    Tensor rng;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = rows_fw(o, two || !plain, &sum, o.norm ? &stats : nullptr);
    }
    node->shape = o.x.sizes();
    node->options = o.x.options();
    node->p = o.p;
    node->eps = o.eps;
    node->norm = o.norm;
    node->two = two;
    node->who = o.who;
    node->rng.set(o.rng);
    if (o.norm) {
        for (const Tensor *t : {&o.weight, &o.bias})
            if (t->defined()) node->param_type = t->scalar_type();
        if (!o.weight.defined() && !o.bias.defined()) node->param_type = o.x.scalar_type();
        node->weight.set(o.weight);
        node->stats.set(stats);
    }
    if (two) {
        torch::autograd::set_history(std::vector<Tensor>{y, sum}, node);
        if (o.norm) node->total.set(sum, true);
    } else {
        torch::autograd::set_history(y, node);
        if (o.norm) node->total.set(plain ? o.x : sum);
    }
    return {y, sum};
}

Tensor layer_norm(Tensor x, OptTensor weight, OptTensor bias, double eps)
{
    Rows o;
    o.x = x;
    o.weight = opt(weight);
    o.bias = opt(bias);
    o.eps = eps;
    o.norm = true;
    o.who = "layer_norm";
    return std::get<0>(rows_op(o, false));
}

Tensor dropout_add(Tensor x, OptTensor rng, double p, OptTensor residual)
{
    Rows o;
    o.x = x;
    o.rng = p > 0.0 ? opt(rng) : Tensor();
    o.p = p;
    o.residual = opt(residual);
    o.who = "dropout_add";
    return std::get<0>(rows_op(o, false));
}

// (y, sum)
std::tuple<Tensor, Tensor> dropout_add_layer_norm(Tensor x, OptTensor rng, double p, OptTensor residual, OptTensor weight,
                                                  OptTensor bias, double eps)
{
    Rows o;
    o.x = x;
    o.rng = p > 0.0 ? opt(rng) : Tensor();
    o.p = p;
    o.residual = opt(residual);
    o.weight = opt(weight);
    o.bias = opt(bias);
    o.eps = eps;
    o.norm = true;
    o.who = "dropout_add_layer_norm";
    return rows_op(o, true);
}

// The generator's present (seed of the replica, call), whose call number then goes up by one, in stream order.
Tensor rng_next(Tensor rng, int64_t replica)
{
    const char *who = "rng_next";
    require_device(rng, who);
    TORCH_CHECK(rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2 && rng.is_contiguous(), who,
                ": rng must be two adjacent int64 (seed, call)");
    at::AutoDispatchBelowADInplaceOrView below;
    const Guard guard(rng.device());
    Tensor taken = at::empty_like(rng);
    check_rc(bf_rng_next_of(rng.data_ptr<int64_t>(), taken.data_ptr<int64_t>(), replica, current_stream()), who);
    rng.unsafeGetTensorImpl()->bump_version();
    return taken;
}

// ---- gated recurrence ------------------------------------------------------------------------------------

struct Recurrence {
    Tensor gate, x, state, reset;
    bool sigmoid = true;
    const char *who = nullptr;
};

at::ScalarType state_type(const Tensor &x) { return x.is_complex() ? x.scalar_type() : at::kFloat; }

bf_recurrence describe(const Recurrence &o, const Tensor &gate, const Tensor &x)
{
    bf_recurrence d = {};
    d.dtype = dtype_code(x, true, o.who);
    d.sigmoid = o.sigmoid;
    d.batch = x.size(0);
    d.steps = x.size(1);
    d.channels = x.size(2);
    batch_steps(d.gate_stride, gate);
    batch_steps(d.x_stride, x);
    if (o.reset.defined()) batch_steps(d.reset_stride, o.reset);
    return d;
}

void check_recurrence(const Recurrence &o, int64_t dims)
{
    const char *who = o.who;
    require_device(o.x, who);
    require_beside(o.gate, o.x, "gate", who);
    TORCH_CHECK(o.x.dim() == dims, who, ": x must have shape ", dims == 3 ? "(batch, steps, channels)" : "(batch, channels)");
    TORCH_CHECK(o.gate.sizes() == o.x.sizes() && o.gate.scalar_type() == o.x.scalar_type(), who,
                ": gate must have the shape and dtype of x");
    dtype_code(o.x, true, who);
    TORCH_CHECK(!o.sigmoid || !o.x.is_complex(), who, ": sigmoid gates are real");
    if (o.state.defined()) {
        require_beside(o.state, o.x, "state", who);
        TORCH_CHECK(o.state.dim() == 2 && o.state.size(0) == o.x.size(0) && o.state.size(1) == o.x.size(dims - 1), who,
                    ": state must have shape (batch, channels)");
        TORCH_CHECK(o.state.scalar_type() == state_type(o.x), who, ": state must be ", state_type(o.x));
    }
    if (o.reset.defined()) {
        require_beside(o.reset, o.x, "reset", who);
        TORCH_CHECK(o.reset.scalar_type() == at::kBool, who, ": reset must be bool");
        TORCH_CHECK(o.reset.dim() == 2 && o.reset.size(0) == o.x.size(0) && o.reset.size(1) == o.x.size(1), who,
                    ": reset must have shape (batch, steps)");
    }
}

std::tuple<Tensor, Tensor> recurrence_fw(const Recurrence &o)
{
    const Guard guard(o.x.device());
    const Tensor gate = adjacent(o.gate), x = adjacent(o.x);
    const Tensor state = dense(o.state);
    bf_recurrence d = describe(o, gate, x);
    Tensor h = at::empty(x.sizes(), x.options());
    Tensor last = at::empty({d.batch, d.channels}, x.options().dtype(state_type(x)));
    const size_t bytes = valid_size(bf_recurrence_workspace_bytes(&d));
    const Tensor ws = workspace_like(x, bytes);
    check_rc(bf_recurrence_fw(&d, gate.data_ptr(), x.data_ptr(), ptr(state), static_cast<const uint8_t *>(ptr(o.reset)),
                              h.data_ptr(), last.data_ptr(), ptr(ws), bytes, current_stream()),
             o.who);
    return {h, last};
}

struct RecurrenceNode : public torch::autograd::Node {
    SavedSlot gate, x, state, reset, h;
    bool sigmoid = true;
    const char *who = nullptr;

    // edges: gate, x, state
    variable_list apply(variable_list &&grads) override
    {
        variable_list out(num_outputs());
        if (!grads[0].defined() && !grads[1].defined()) return out;
        std::lock_guard<std::mutex> lock(mutex_);
        const auto self = getptr();
        Recurrence o;
        o.gate = gate.get(self);
        o.x = x.get(self);
        o.state = state.get(self);
        o.reset = reset.get(self);
        o.sigmoid = sigmoid;
        o.who = who;
        const Tensor out_h = h.get(self);
        const bool want_state = task_should_compute_output(2);
        at::AutoDispatchBelowADInplaceOrView below;
        const Guard guard(o.x.device());
        const Tensor z = adjacent(o.gate), v = adjacent(o.x), before = out_h.contiguous();
        const Tensor first = dense(o.state);
        const Tensor g = grads[0].defined() ? adjacent(grads[0]) : Tensor();
        const Tensor gl = dense(grads[1]);
        bf_recurrence d = describe(o, z, v);
        if (g.defined()) batch_steps(d.grad_stride, g);
        out[0] = at::empty(v.sizes(), v.options());
        out[1] = at::empty(v.sizes(), v.options());
        if (want_state) out[2] = at::empty({d.batch, d.channels}, v.options().dtype(state_type(v)));
        const size_t bytes = valid_size(bf_recurrence_workspace_bytes(&d));
        const Tensor ws = workspace_like(v, bytes);
        check_rc(bf_recurrence_bw(&d, z.data_ptr(), v.data_ptr(), ptr(first), static_cast<const uint8_t *>(ptr(o.reset)),
                                  before.data_ptr(), ptr(g), ptr(gl), out[0].data_ptr(), out[1].data_ptr(), ptr(out[2]), ptr(ws),
                                  bytes, current_stream()),
                 who);
        refuse_second(out, *this, {grads[0], grads[1]}, who);
        return out;
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedSlot *s : {&gate, &x, &state, &reset, &h}) s->drop();
    }

    std::string name() const override { return "GatedRecurrenceBackward"; }
};

// (h, last)
std::tuple<Tensor, Tensor> gated_recurrence(Tensor gate, Tensor x, OptTensor state, OptTensor reset, bool sigmoid)
{
    Recurrence o;
    o.gate = gate;
    o.x = x;
    o.state = opt(state);
    o.reset = opt(reset);
    o.sigmoid = sigmoid;
    o.who = "gated_recurrence";
    check_recurrence(o, 3);
    refuse_tangents({o.gate, o.x, o.state}, o.who);
    if (!any_wants_grad({o.gate, o.x, o.state})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return recurrence_fw(o);
    }
    std::shared_ptr<RecurrenceNode> node(new RecurrenceNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(o.gate, o.x, o.state));
    Tensor h, last;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(h, last) = recurrence_fw(o);
    }
    node->gate.set(o.gate);
    node->x.set(o.x);
    node->state.set(o.state);
    node->reset.set(o.reset);
    node->sigmoid = sigmoid;
    node->who = o.who;
    torch::autograd::set_history(std::vector<Tensor>{h, last}, node);
    node->h.set(h, true);
    return {h, last};
}

// One new step of every sequence; state is updated in place.
Tensor gated_recurrence_step(Tensor gate, Tensor x, Tensor state, bool sigmoid)
{
    Recurrence o;
    o.gate = gate;
    o.x = x;
    o.state = state;
    o.sigmoid = sigmoid;
    o.who = "gated_recurrence_step";
    check_recurrence(o, 2);
    refuse_tangents({o.gate, o.x, o.state}, o.who);
    TORCH_CHECK(!any_wants_grad({o.gate, o.x, o.state}), o.who, ": has no gradient (use gated_recurrence, or torch.no_grad)");
    TORCH_CHECK(state.is_contiguous() && !state.is_conj() && !state.is_neg(), o.who, ": state must be contiguous, it is updated in place");
    at::AutoDispatchBelowADInplaceOrView below;
    const Guard guard(x.device());
    const Tensor z = adjacent(gate), v = adjacent(x);
    bf_recurrence d = {};
    d.dtype = dtype_code(v, true, o.who);
    d.sigmoid = sigmoid;
    d.batch = v.size(0);
    d.steps = 1;
    d.channels = v.size(1);
    d.gate_stride[0] = row_stride(z);
    d.x_stride[0] = row_stride(v);
    Tensor h = at::empty(v.sizes(), v.options());
    check_rc(bf_recurrence_step(&d, z.data_ptr(), v.data_ptr(), state.data_ptr(), h.data_ptr(), current_stream()), o.who);
    state.unsafeGetTensorImpl()->bump_version();
    return h;
}

// ---- linear layer and cross entropy ---------------------------------------------------------------------------

struct Xent {
    Tensor hidden, weight, target;
    int64_t ignore_index = -100, reduction = BF_XENT_MEAN;
    const char *who = "linear_cross_entropy";
};

bf_linear_xent describe(const Xent &o, const Tensor &hidden, const Tensor &weight)
{
    bf_linear_xent d = {};
    d.dtype = dtype_code(hidden, false, o.who);
    d.reduction = (int32_t)o.reduction;
    d.rows = hidden.size(0);
    d.features = hidden.size(1);
    d.vocab = weight.size(0);
    d.hidden_stride = row_stride(hidden);
    d.weight_stride = row_stride(weight);
    d.ignore_index = o.ignore_index;
    return d;
}

// (loss, kept operands); what the call was, for its backward one, in *desc
std::tuple<Tensor, Tensor> xent_fw(const Xent &o, bf_linear_xent *desc)
{
    const Guard guard(o.hidden.device());
    const Tensor hidden = rows_of(o.hidden), weight = aligned_rows_of(o.weight), target = o.target.contiguous();
    const bf_linear_xent d = describe(o, hidden, weight);
    if (desc) *desc = d;
    const auto options = hidden.options().dtype(at::kFloat);
    Tensor loss = o.reduction == BF_XENT_NONE ? at::empty(o.target.sizes(), options) : at::empty({}, options);
    const size_t bytes = valid_size(bf_linear_xent_fw_workspace_bytes(&d));
    const size_t kept_bytes = valid_size(bf_linear_xent_kept_bytes(&d));
    const Tensor ws = workspace_like(hidden, bytes), kept = workspace_like(hidden, kept_bytes);
    check_rc(bf_linear_xent_fw(&d, hidden.data_ptr(), weight.data_ptr(), target.data_ptr<int64_t>(), loss.data_ptr<float>(),
                               ptr(kept), kept_bytes, ptr(ws), bytes, current_stream()),
             o.who);
    return {loss, kept};
}

struct XentNode : public torch::autograd::Node {
    SavedSlot weight, kept;
    c10::SmallVector<int64_t, 6> hidden_shape;
    bf_linear_xent desc = {};

    // edges: hidden, weight
    variable_list apply(variable_list &&grads) override
    {
        variable_list out(num_outputs());
        if (!grads[0].defined()) return out;
        std::lock_guard<std::mutex> lock(mutex_);
        const auto self = getptr();
        const Tensor saved = weight.get(self), operands = kept.get(self);
        const bool want_hidden = task_should_compute_output(0), want_weight = task_should_compute_output(1);
        at::AutoDispatchBelowADInplaceOrView below;
        const Guard guard(saved.device());
        const Tensor w = aligned_rows_of(saved), g = dense(grads[0]);
        bf_linear_xent d = desc;
        d.weight_stride = row_stride(w);
        if (want_hidden) out[0] = at::empty(hidden_shape, w.options());
        if (want_weight) out[1] = at::empty(saved.sizes(), w.options());
        const size_t bytes = valid_size(bf_linear_xent_bw_workspace_bytes(&d));
        const Tensor ws = workspace_like(w, bytes);
        check_rc(bf_linear_xent_bw(&d, w.data_ptr(), g.data_ptr<float>(), operands.data_ptr(),
                                   (size_t)operands.numel(), ptr(out[0]), ptr(out[1]), ptr(ws), bytes, current_stream()),
                 "linear_cross_entropy");
        refuse_second(out, *this, {grads[0]}, "linear_cross_entropy");
        return out;
    }

    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        for (SavedSlot *s : {&weight, &kept}) s->drop();
    }

    std::string name() const override { return "LinearCrossEntropyBackward"; }
};

// reduction: 0 none, 1 mean, 2 sum
Tensor linear_cross_entropy(Tensor hidden, Tensor weight, Tensor target, int64_t ignore_index, int64_t reduction)
{
    Xent o;
    o.hidden = hidden;
    o.weight = weight;
    o.target = target;
    o.ignore_index = ignore_index;
    o.reduction = reduction;
    const char *who = o.who;
    require_device(hidden, who);
    require_beside(weight, hidden, "weight", who);
    require_beside(target, hidden, "target", who);
    TORCH_CHECK(hidden.dim() >= 1 && weight.dim() == 2 && weight.size(1) == hidden.size(-1), who,
                ": hidden must have shape (*, features) and weight (vocab, features)");
    dtype_code(hidden, false, who);
    TORCH_CHECK(weight.scalar_type() == hidden.scalar_type(), who, ": weight and hidden must have the same dtype");
    TORCH_CHECK(target.scalar_type() == at::kLong, who, ": target must be int64");
    TORCH_CHECK(target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), who, ": target must have the shape of hidden without features");
    TORCH_CHECK(weight.size(0) > 0 && weight.size(1) > 0, who, ": vocabulary and features must not be empty");
    TORCH_CHECK(reduction >= BF_XENT_NONE && reduction <= BF_XENT_SUM, who, ": reduction must be none, mean or sum");
    refuse_tangents({hidden, weight}, who);
    if (!any_wants_grad({hidden, weight})) {
        at::AutoDispatchBelowADInplaceOrView below;
        return std::get<0>(xent_fw(o, nullptr));
    }
    std::shared_ptr<XentNode> node(new XentNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(hidden, weight));
    Tensor loss, kept;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(loss, kept) = xent_fw(o, &node->desc);
    }
    node->hidden_shape = hidden.sizes();
    node->weight.set(weight);
    node->kept.set(kept);
    torch::autograd::set_history(loss, node);
    return loss;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torch_butterfly, m)
{
    m.def("layer_norm", layer_norm);
    m.def("dropout_add", dropout_add);
    m.def("dropout_add_layer_norm", dropout_add_layer_norm);
    m.def("rng_next(Tensor rng, int replica=0) -> Tensor", rng_next);
    m.def("gated_recurrence", gated_recurrence);
    m.def("gated_recurrence_step", gated_recurrence_step);
    m.def("linear_cross_entropy", linear_cross_entropy);
}
