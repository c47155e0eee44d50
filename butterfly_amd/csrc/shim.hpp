// What the torch-library shims of the operators beside the multiply share: checks, views, workspaces, saved tensors.  (Everything has
// internal linkage: each shim has its own.)
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/butterfly_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;
using OptTensor = c10::optional<Tensor>;

Tensor opt(const OptTensor &t) { return t.has_value() ? t.value() : Tensor(); }

void *current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

void check_rc(int rc, const char *who) { TORCH_CHECK(rc == BF_OK, who, ": ", bf_last_error()); }

size_t valid_size(size_t bytes)
{
    TORCH_CHECK(bytes != BF_SIZE_INVALID, "torch_butterfly: ", bf_last_error());
    return bytes;
}

Tensor workspace_like(const Tensor &t, size_t bytes)
{
    return bytes > 0 ? at::empty({(int64_t)bytes}, t.options().dtype(at::kByte)) : Tensor();
}

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

void require_device(const Tensor &t, const char *who)
{
    TORCH_CHECK(t.is_cuda(), who, ": tensors must live on a HIP device; this operator has no CPU path");
}

void require_beside(const Tensor &t, const Tensor &like, const char *name, const char *who)
{
    TORCH_CHECK(t.device() == like.device(), who, ": ", name, " must be on the device of the input");
}

void refuse_tangents(std::initializer_list<Tensor> tensors, const char *who)
{
    for (const Tensor &t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), who, ": no forward-mode derivative");
}

bool any_wants_grad(std::initializer_list<Tensor> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : tensors)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// Gradients that are to be differentiated again (create_graph) come with a history that says, once it is followed, that there
// is no second derivative; without one they would count as constants.
void refuse_second(variable_list &out, const torch::autograd::Node &node, std::initializer_list<Tensor> grads, const char *who)
{
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges;
    for (const auto &edge : node.next_edges())
        if (edge.is_valid()) edges.push_back(edge);
    for (const Tensor &t : grads)
        if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
    std::shared_ptr<torch::autograd::Node> error(
        new torch::autograd::Error(std::string(who) + ": no second derivative", std::move(edges)), torch::autograd::deleteNode);
    for (Tensor &t : out)
        if (t.defined()) torch::autograd::set_history(t, error);
}

int dtype_code(const Tensor &t, bool complex_too, const char *who)
{
    if (t.scalar_type() == at::kFloat) return BF_F32;
    if (t.scalar_type() == at::kBFloat16) return BF_BF16;
    if (complex_too && t.scalar_type() == at::kComplexFloat) return BF_C64;
    TORCH_CHECK(false, who, ": device kernels support float32", complex_too ? ", bfloat16 and complex64" : " and bfloat16",
                ", got ", t.scalar_type());
}

int64_t row_count(const Tensor &t)
{
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
    return n;
}

// What the memory holds is what the tensor is (views of conjugates may say otherwise).
Tensor plain(const Tensor &t) { return t.resolve_conj().resolve_neg(); }

Tensor dense(const Tensor &t) { return t.defined() ? plain(t).contiguous() : Tensor(); }

// A 2-d view (rows, columns) of a tensor with adjacent columns, or a copy.
Tensor rows_of(const Tensor &t)
{
    Tensor r = plain(t);
    if (r.dim() != 2) r = r.reshape({row_count(r), r.size(-1)});
    return r.size(1) > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

int64_t row_stride(const Tensor &rows) { return rows.size(0) > 1 ? rows.stride(0) : 0; }

// The same at a 16-byte aligned address.
Tensor aligned_rows_of(const Tensor &t)
{
    const Tensor r = rows_of(t);
    return (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) != 0 ? r.clone(at::MemoryFormat::Contiguous) : r;
}

// Last dimension adjacent.
Tensor adjacent(const Tensor &t)
{
    const Tensor r = plain(t);
    return r.size(-1) > 1 && r.stride(-1) != 1 ? r.contiguous() : r;
}

void batch_steps(int64_t (&dst)[2], const Tensor &t)
{
    for (int i = 0; i < 2; ++i) dst[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

struct SavedSlot {
    SavedVariable v;
    bool there = false;

    void set(const Tensor &t, bool is_output = false)
    {
        if (!t.defined()) return;
        v = SavedVariable(t, is_output);
        there = true;
    }
    Tensor get(const std::shared_ptr<torch::autograd::Node> &self) { return there ? v.unpack(self) : Tensor(); }
    void drop() { v.reset_data(); }
};

}  // namespace
