// Entry points of the linear attention (linear_attention.hpp): argument checks, cut into segments, launches.

#include "../../include/butterfly_hip.h"

#include <algorithm>

#include "error.hpp"
#include "linear_attention.hpp"

namespace {

using namespace bf;

constexpr int kWidest = 128;   // features, values: a state of 128 x 128 floats is half of a compute unit's registers

int check_attention(const bf_linear_attention *p)
{
    if (!p) return fail(BF_ERR_INVALID, "linear attention descriptor is NULL");
    if (p->dtype != BF_F32 && p->dtype != BF_BF16) return fail(BF_ERR_INVALID, "dtype must be BF_F32 or BF_BF16");
    if (p->batch < 0 || p->steps < 0 || p->heads < 0 || p->groups < 0 || p->features < 0 || p->values < 0)
        return fail(BF_ERR_INVALID, "sizes must be non-negative");
    if (p->heads > 0 && (p->groups == 0 || p->heads % p->groups != 0)) return fail(BF_ERR_INVALID, "heads must be a multiple of groups");
    if (p->features > kWidest || p->values > kWidest)
        return fail(BF_ERR_UNSUPPORTED, "heads of more than %d features or values are not supported", kWidest);
    if (p->features == 0 || p->values == 0) return fail(BF_ERR_INVALID, "features and values must be positive");
    // (one workgroup of up to 512 threads each: a grid has less than 2^32 of them)
    if (p->batch > ((int64_t)1 << 22) || p->heads > ((int64_t)1 << 22) || p->groups > ((int64_t)1 << 22) || p->batch * p->heads > ((int64_t)1 << 22))
        return fail(BF_ERR_UNSUPPORTED, "more than 2^22 sequences and heads are not supported");
    if (p->steps > ((int64_t)1 << 31)) return fail(BF_ERR_UNSUPPORTED, "more than 2^31 steps are not supported");
    // (a chunk's rows of a result lie within 2^31 bytes of each other)
    if (p->heads * std::max(p->features, p->values) > ((int64_t)1 << 22))
        return fail(BF_ERR_UNSUPPORTED, "steps of more than 2^22 features or values are not supported");
    for (int i = 0; i < 3; ++i)
        if (p->q_stride[i] < 0 || p->k_stride[i] < 0 || p->v_stride[i] < 0 || p->grad_stride[i] < 0 || p->decay_stride[i] < 0)
            return fail(BF_ERR_INVALID, "strides must be non-negative");
    if (p->reset_stride[0] < 0 || p->reset_stride[1] < 0) return fail(BF_ERR_INVALID, "strides must be non-negative");
    return BF_OK;
}

bool nothing(const bf_linear_attention *p) { return p->batch == 0 || p->heads == 0; }

int64_t square(const bf_linear_attention *p) { return p->features * p->values; }

bool small(const bf_linear_attention *p) { return p->features <= 64 && p->values <= 64; }

int chunk_steps(const bf_linear_attention *p) { return p->dtype == BF_F32 && !small(p) ? 32 : 64; }

int64_t chunk_count(const bf_linear_attention *p) { return (p->steps + chunk_steps(p) - 1) / chunk_steps(p); }

struct AttentionPlan {
    int64_t chunks = 0, segment_chunks = 0;
    int segments = 1;
    size_t states = 0, decays = 0, wide = 0;   // bytes

    size_t workspace() const { return states + 2 * decays + 2 * wide; }
};

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Sequences times heads are one workgroup each, a compute unit's: the registers of the launches with outputs or gradients (160 to 256 a
// lane, eight wavefronts) hold no second one.  (Those of the sums alone, 112 a lane for 64-wide heads, would; they share the cut.)  Fewer than half of the 256
// are cut into as many segments as fill them, no more: 10 heads of 65537 steps in 26 segments leave four workgroups for
// a second round and took twice the time of 25.  Segments of two chunks at least: 16 heads of 256 steps forward and backward 73 us in two
// segments, 86 in one (float; bfloat16 57 and 58); of 1024 steps 80 in eight, 303 in one.
AttentionPlan plan(const bf_linear_attention *p, bool back)
{
    AttentionPlan r;
    const int64_t heads = p->batch * p->heads;
    r.chunks = r.segment_chunks = chunk_count(p);
    if (heads <= 128 && r.chunks > 2) {
        const int64_t wanted = std::min<int64_t>(256 / heads, (r.chunks + 1) / 2);
        r.segment_chunks = (r.chunks + wanted - 1) / wanted;
        r.segments = (int)((r.chunks + r.segment_chunks - 1) / r.segment_chunks);
    }
    if (r.segments > 1) {
        r.states = rounded((size_t)r.segments * (size_t)heads * (size_t)square(p) * sizeof(float));
        r.decays = rounded((size_t)r.segments * (size_t)heads * sizeof(float));
    }
    if (back && p->heads != p->groups) r.wide = rounded((size_t)p->batch * p->steps * p->heads * p->features * sizeof(float));
    return r;
}

LaArgs fill(const bf_linear_attention *p)
{
    LaArgs a = {};
    for (int i = 0; i < 3; ++i) {
        a.q_stride[i] = p->q_stride[i];
        a.k_stride[i] = p->k_stride[i];
        a.v_stride[i] = p->v_stride[i];
        a.grad_stride[i] = p->grad_stride[i];
        a.decay_stride[i] = p->decay_stride[i];
    }
    for (int i = 0; i < 2; ++i) a.reset_stride[i] = p->reset_stride[i];
    a.batch = p->batch;
    a.steps = p->steps;
    a.heads = (int)p->heads;
    a.shared = (int)(p->heads / p->groups);
    a.features = (int)p->features;
    a.values = (int)p->values;
    a.scale = (float)p->scale;
    return a;
}

int place(LaArgs &a, const AttentionPlan &r, void *workspace, size_t bytes)
{
    a.chunks = r.chunks;
    a.segment_chunks = r.segment_chunks;
    a.segments = r.segments;
    const size_t need = r.workspace();
    if (need == 0) return BF_OK;
    if (!workspace || bytes < need)
        return fail(BF_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? bytes : 0);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BF_ERR_WORKSPACE, "workspace must be 16-byte aligned");
    char *w = static_cast<char *>(workspace);
    a.segment_state = reinterpret_cast<float *>(w);
    a.segment_decay = reinterpret_cast<float *>(w + r.states);
    a.segment_cut = reinterpret_cast<int *>(w + r.states + r.decays);
    return BF_OK;
}

int check_kept(const bf_linear_attention *p, const void *kept, size_t bytes)
{
    const size_t need = bf_linear_attention_kept_bytes(p);
    if (!kept || bytes < need) return fail(BF_ERR_WORKSPACE, "kept states of %zu bytes needed, %zu given", need, kept ? bytes : 0);
    if (reinterpret_cast<uintptr_t>(kept) & 15) return fail(BF_ERR_WORKSPACE, "kept states must be 16-byte aligned");
    return BF_OK;
}

// f(type, widest operand)
template <typename Fn>
void with_shape(const bf_linear_attention *p, Fn &&f)
{
    using Small = std::integral_constant<int, 64>;
    using Large = std::integral_constant<int, 128>;
    if (p->dtype == BF_F32) small(p) ? f(float(), Small()) : f(float(), Large());
    else small(p) ? f(bf16(), Small()) : f(bf16(), Large());
}

dim3 walk_grid(const LaArgs &a) { return dim3((unsigned)((a.batch * a.heads * a.segments + 7) / 8 * 8)); }

dim3 enter_grid(const LaArgs &a) { return dim3((unsigned)std::min<int64_t>((a.batch * a.heads * a.features * a.values + 255) / 256, 1 << 16)); }

// d_q or d_k from the gradients of each head, or of no heads: zeros (from: not read).
template <typename T>
void add_shared(const bf_linear_attention *p, const void *from, void *to, hipStream_t s)
{
    const int64_t rows = p->batch * p->steps, count = rows * p->groups * p->features;
    const dim3 grid((unsigned)std::min<int64_t>((count + 255) / 256, 1 << 16));
    la_shared_kernel<T><<<grid, dim3(256), 0, s>>>(static_cast<const float *>(from), static_cast<T *>(to), rows, (int)p->groups,
                                                   (int)(p->heads / p->groups), (int)p->features);
}

int copy_state(const bf_linear_attention *p, const float *from, float *to, hipStream_t s)
{
    if (!to) return BF_OK;
    const LaArgs a = fill(p);
    la_copy_kernel<<<enter_grid(a), dim3(256), 0, s>>>(from, to, a.batch * a.heads * square(p));
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

}  // namespace

extern "C" {

size_t bf_linear_attention_kept_bytes(const bf_linear_attention *p)
{
    if (check_attention(p)) return BF_SIZE_INVALID;
    return (size_t)p->batch * (size_t)p->heads * (size_t)chunk_count(p) * (size_t)p->features * (size_t)la_line((int)p->values) * sizeof(float);
}

size_t bf_linear_attention_fw_workspace_bytes(const bf_linear_attention *p)
{
    if (check_attention(p)) return BF_SIZE_INVALID;
    return nothing(p) ? 0 : plan(p, false).workspace();
}

size_t bf_linear_attention_bw_workspace_bytes(const bf_linear_attention *p)
{
    if (check_attention(p)) return BF_SIZE_INVALID;
    return nothing(p) ? 0 : plan(p, true).workspace();
}

int bf_linear_attention_fw(const bf_linear_attention *p, const void *q, const void *k, const void *v, const float *log_decay,
                           const float *state, const uint8_t *reset, void *o, float *last, void *kept, size_t kept_bytes,
                           void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_attention(p);
    if (rc) return rc;
    if (nothing(p)) return BF_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->steps == 0) return copy_state(p, state, last, s);
    if (!q || !k || !v || !log_decay || !o) return fail(BF_ERR_INVALID, "q, k, v, log_decay or o is NULL");
    if (kept && (rc = check_kept(p, kept, kept_bytes))) return rc;
    LaArgs a = fill(p);
    if ((rc = place(a, plan(p, false), workspace, workspace_bytes))) return rc;
    a.q = q;
    a.k = k;
    a.v = v;
    a.log_decay = log_decay;
    a.state = state;
    a.reset = reset;
    a.o = o;
    a.last = last;
    a.kept = static_cast<float *>(kept);
    with_shape(p, [&](auto type, auto widest) {
        using T = decltype(type);
        constexpr int D = decltype(widest)::value;
        if (a.segments > 1) {
            la_walk_kernel<T, D, false, false><<<walk_grid(a), dim3(LaShape<T, D>::THREADS), 0, s>>>(a);
            la_enter_kernel<false><<<enter_grid(a), dim3(256), 0, s>>>(a);
        }
        la_walk_kernel<T, D, true, false><<<walk_grid(a), dim3(LaShape<T, D>::THREADS), 0, s>>>(a);
    });
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

int bf_linear_attention_bw(const bf_linear_attention *p, const void *q, const void *k, const void *v, const float *log_decay,
                           const uint8_t *reset, const void *kept, size_t kept_bytes, const void *grad, const float *grad_last,
                           void *d_q, void *d_k, void *d_v, float *d_log_decay, float *d_state, void *workspace,
                           size_t workspace_bytes, void *stream)
{
    int rc = check_attention(p);
    if (rc) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (nothing(p)) {
        // (queries and keys of groups without heads)
        if (p->batch == 0 || p->steps == 0 || p->groups == 0) return BF_OK;
        if (!d_q || !d_k) return fail(BF_ERR_INVALID, "d_q or d_k is NULL");
        for (void *to : {d_q, d_k}) p->dtype == BF_F32 ? add_shared<float>(p, nullptr, to, s) : add_shared<bf16>(p, nullptr, to, s);
        BF_HIP_CHECK(hipGetLastError());
        return BF_OK;
    }
    if (p->steps == 0) return copy_state(p, grad_last, d_state, s);
    if (!q || !k || !v || !log_decay) return fail(BF_ERR_INVALID, "q, k, v or log_decay is NULL");
    if (!d_q || !d_k || !d_v || !d_log_decay) return fail(BF_ERR_INVALID, "d_q, d_k, d_v or d_log_decay is NULL");
    if ((rc = check_kept(p, kept, kept_bytes))) return rc;
    const AttentionPlan r = plan(p, true);
    LaArgs a = fill(p);
    if ((rc = place(a, r, workspace, workspace_bytes))) return rc;
    char *wide = static_cast<char *>(workspace) + r.states + 2 * r.decays;
    a.q = q;
    a.k = k;
    a.v = v;
    a.log_decay = log_decay;
    a.reset = reset;
    a.kept = static_cast<float *>(const_cast<void *>(kept));
    a.grad = grad;
    a.grad_last = grad_last;
    a.wide = r.wide > 0;
    a.d_q = a.wide ? wide : d_q;
    a.d_k = a.wide ? wide + r.wide : d_k;
    a.d_v = d_v;
    a.d_log_decay = d_log_decay;
    a.d_state = d_state;
    with_shape(p, [&](auto type, auto widest) {
        using T = decltype(type);
        constexpr int D = decltype(widest)::value;
        if (a.segments > 1) {
            la_walk_kernel<T, D, false, true><<<walk_grid(a), dim3(LaShape<T, D>::THREADS), 0, s>>>(a);
            la_enter_kernel<true><<<enter_grid(a), dim3(256), 0, s>>>(a);
        }
        la_back_kernel<T, D><<<walk_grid(a), dim3(LaShape<T, D>::THREADS), 0, s>>>(a);
        if (a.wide) {
            add_shared<T>(p, a.d_q, d_q, s);
            add_shared<T>(p, a.d_k, d_k, s);
        }
    });
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

int bf_linear_attention_step(const bf_linear_attention *p, const void *q, const void *k, const void *v, const float *log_decay,
                             float *state, void *o, void *stream)
{
    const int rc = check_attention(p);
    if (rc) return rc;
    if (nothing(p)) return BF_OK;
    if (!q || !k || !v || !log_decay || !state || !o) return fail(BF_ERR_INVALID, "q, k, v, log_decay, state or o is NULL");
    LaArgs a = fill(p);
    a.q = q;
    a.k = k;
    a.v = v;
    a.log_decay = log_decay;
    const bool quads = p->values % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
    int lanes_log = 0;
    while (((quads ? 4 : 1) << lanes_log) < p->values) ++lanes_log;
    const dim3 grid((unsigned)(p->batch * p->heads));
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_shape(p, [&](auto type, auto) {
        using T = decltype(type);
        if (quads) la_step_kernel<T, 4><<<grid, dim3(256), 0, s>>>(a, state, static_cast<T *>(o), lanes_log);
        else la_step_kernel<T, 1><<<grid, dim3(256), 0, s>>>(a, state, static_cast<T *>(o), lanes_log);
    });
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

}  // extern "C"
