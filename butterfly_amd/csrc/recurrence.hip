// Entry points of the gated linear recurrence (recurrence.hpp): argument checks, cut into chunks, launches.

#include "../../include/butterfly_hip.h"

#include <algorithm>

#include "error.hpp"
#include "recurrence.hpp"

namespace {

using namespace bf;

int check_recurrence(const bf_recurrence *p)
{
    if (!p) return fail(BF_ERR_INVALID, "recurrence descriptor is NULL");
    if (p->dtype != BF_F32 && p->dtype != BF_C64 && p->dtype != BF_BF16)
        return fail(BF_ERR_INVALID, "dtype must be BF_F32, BF_C64 or BF_BF16");
    if (p->sigmoid && p->dtype == BF_C64) return fail(BF_ERR_INVALID, "sigmoid gates are real: BF_C64 takes linear ones");
    if (p->batch < 0 || p->steps < 0 || p->channels < 0) return fail(BF_ERR_INVALID, "sizes must be non-negative");
    if (p->channels > ((int64_t)1 << 28)) return fail(BF_ERR_UNSUPPORTED, "more than 2^28 channels are not supported");
    if (p->steps > ((int64_t)1 << 40) || p->batch > ((int64_t)1 << 30)) return fail(BF_ERR_UNSUPPORTED, "too many steps or sequences");
    for (int i = 0; i < 2; ++i)
        if (p->gate_stride[i] < 0 || p->x_stride[i] < 0 || p->grad_stride[i] < 0 || p->reset_stride[i] < 0)
            return fail(BF_ERR_INVALID, "strides must be non-negative");
    return BF_OK;
}

bool nothing(const bf_recurrence *p) { return p->batch == 0 || p->channels == 0; }

struct RecurrencePlan {
    int64_t groups = 1, chunk = 0, chunks = 1;
    int waves = 1, waves_bw = 1;
    size_t state_bytes = 0, chunk_bytes = 0, run_bytes = 0, workspace = 0;   // of one of chunk_a, chunk_b; run_a, run_b
};

// Channels times batch make `groups * batch` workgroups.  A whole sequence is read once, at some 25 ns a step however few
// of them there are; cut into chunks of 16 runs of whole blocks of S steps, until some 512 are at work, the gates
// and inputs are read twice and two launches more are made.  A multiple of eight chunks is wanted, one XCD's each in turn
// (whole tiles of steps make them a few more or less: 65537 steps, 65 chunks, the last one of a single step):
// 88 workgroups of 4096 steps, float, forward and backward in 6 chunks 267 us, in 8 246.  Measured in float, forward and
// backward, whole and cut: 72 workgroups of 4096 steps 301 and 209 us, 96 313 and 276, 104 320 and 325, 128 338 and 403;
// 96 of 16384 1226 and 1119, 112 1251 and 1330; 64 of 512 62 and 79, 72 of 1024 71 and 68, 40 70 and 50.  In bfloat16 pairs
// 112 of 4096 455 and 361; 8 of 16384 1605 and 110.  So below 100 (128) of more than four tiles.
RecurrencePlan plan(const bf_recurrence *p)
{
    RecurrencePlan r;
    const bool pairs = p->dtype == BF_BF16 && p->channels > 1;
    const int v = pairs ? RecBF16::V : 1, s = p->dtype == BF_C64 ? RecC64::S : pairs ? RecBF16::S : RecF32::S;
    r.groups = (p->channels + 64 * v - 1) / (64 * v);
    const int64_t whole = r.groups * p->batch, tile = (int64_t)kRecWaves * s;
    r.chunk = std::max<int64_t>(p->steps, 1);
    if (whole < (pairs ? 128 : 100) && p->steps > 4 * tile) {
        const int64_t wanted = std::min<int64_t>(((512 + whole - 1) / whole + 7) / 8 * 8, (p->steps + tile - 1) / tile);
        r.chunk = std::max<int64_t>((p->steps / wanted + tile / 2) / tile, 1) * tile;
        r.chunks = (p->steps + r.chunk - 1) / r.chunk;
    }
    r.waves = (int)std::min<int64_t>((r.chunk + s - 1) / s, kRecWaves);
    const int sb = p->dtype == BF_C64 ? RecC64::SB : pairs ? RecBF16::SB : RecF32::SB;
    r.waves_bw = (int)std::min<int64_t>((r.chunk + sb - 1) / sb, kRecWaves);
    r.state_bytes = (size_t)p->batch * (size_t)p->channels * (p->dtype == BF_C64 ? 8 : 4);
    if (r.chunks > 1) {
        r.chunk_bytes = ((size_t)r.chunks * r.state_bytes + 255) / 256 * 256;
        r.run_bytes = ((size_t)r.chunks * kRecWaves * r.state_bytes + 255) / 256 * 256;
        r.workspace = 2 * (r.chunk_bytes + r.run_bytes) + (size_t)r.chunks * (1 + kRecWaves) * (size_t)p->batch * sizeof(int);
    }
    return r;
}

void fill(RecurrenceArgs &a, const bf_recurrence *p, const RecurrencePlan &r, void *workspace)
{
    a.gate_b = p->gate_stride[0];
    a.gate_t = p->gate_stride[1];
    a.x_b = p->x_stride[0];
    a.x_t = p->x_stride[1];
    a.grad_b = p->grad_stride[0];
    a.grad_t = p->grad_stride[1];
    a.reset_b = p->reset_stride[0];
    a.reset_t = p->reset_stride[1];
    a.batch = p->batch;
    a.steps = p->steps;
    a.channels = (int)p->channels;
    a.groups = (int)r.groups;
    a.chunk = r.chunk;
    a.chunks = (int)r.chunks;
    if (r.chunks > 1) {
        char *w = static_cast<char *>(workspace);
        a.run_a = w;
        a.run_b = w + r.run_bytes;
        a.chunk_a = w + 2 * r.run_bytes;
        a.chunk_b = w + 2 * r.run_bytes + r.chunk_bytes;
        a.chunk_cut = reinterpret_cast<int *>(w + 2 * (r.run_bytes + r.chunk_bytes));
        a.run_cut = a.chunk_cut + r.chunks * p->batch;
    }
}

int check_workspace(const RecurrencePlan &r, const void *workspace, size_t bytes)
{
    if (r.workspace == 0) return BF_OK;
    if (!workspace || bytes < r.workspace)
        return fail(BF_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", r.workspace, workspace ? bytes : 0);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BF_ERR_WORKSPACE, "workspace must be 16-byte aligned");
    return BF_OK;
}

int check_grid(const bf_recurrence *p, const RecurrencePlan &r)
{
    if (r.groups * p->batch > 0x7fffffff) return fail(BF_ERR_UNSUPPORTED, "too many sequences and channels for one launch");
    return BF_OK;
}

// Workgroups of sequences that stay whole, of up to 2^10 threads each: a dimension of a grid has less than 2^32 threads.
dim3 whole_grid(const bf_recurrence *p, const RecurrencePlan &r)
{
    const int64_t total = r.groups * p->batch, x = std::min<int64_t>(total, 1 << 21);
    return dim3((unsigned)x, (unsigned)((total + x - 1) / x));
}

// f(traits, sigmoid as a type)
template <typename F>
void with_kind(const bf_recurrence *p, F &&f)
{
    if (p->dtype == BF_C64) f(RecC64(), std::false_type());
    else if (p->dtype == BF_BF16 && p->channels == 1 && p->sigmoid) f(RecBF16One(), std::true_type());
    else if (p->dtype == BF_BF16 && p->channels == 1) f(RecBF16One(), std::false_type());
    else if (p->dtype == BF_BF16 && p->sigmoid) f(RecBF16(), std::true_type());
    else if (p->dtype == BF_BF16) f(RecBF16(), std::false_type());
    else if (p->sigmoid) f(RecF32(), std::true_type());
    else f(RecF32(), std::false_type());
}

int pass_on(const bf_recurrence *p, const void *in, void *out, hipStream_t s)
{
    if (!out) return BF_OK;
    const int64_t count = p->batch * p->channels;
    const dim3 grid((unsigned)std::min<int64_t>((count + 255) / 256, 4096));
    if (p->dtype == BF_C64)
        recurrence_pass_kernel<<<grid, dim3(256), 0, s>>>(static_cast<const float2 *>(in), static_cast<float2 *>(out), count);
    else
        recurrence_pass_kernel<<<grid, dim3(256), 0, s>>>(static_cast<const float *>(in), static_cast<float *>(out), count);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

}  // namespace

extern "C" {

size_t bf_recurrence_workspace_bytes(const bf_recurrence *p)
{
    if (check_recurrence(p)) return BF_SIZE_INVALID;
    return nothing(p) ? 0 : plan(p).workspace;
}

int bf_recurrence_fw(const bf_recurrence *p, const void *gate, const void *x, const void *state, const uint8_t *reset,
                     void *h, void *last, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_recurrence(p);
    if (rc) return rc;
    if (nothing(p)) return BF_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->steps == 0) return pass_on(p, state, last, s);
    if (!gate || !x || !h) return fail(BF_ERR_INVALID, "gate, x or h is NULL");
    const RecurrencePlan r = plan(p);
    if ((rc = check_grid(p, r)) || (rc = check_workspace(r, workspace, workspace_bytes))) return rc;
    RecurrenceArgs a = {};
    fill(a, p, r, workspace);
    a.gate = gate;
    a.x = x;
    a.state = state;
    a.reset = reset;
    a.h = h;
    a.last = last;
    with_kind(p, [&](auto kind, auto sigmoid) {
        using Tr = decltype(kind);
        constexpr bool SIG = decltype(sigmoid)::value;
        const unsigned x_blocks = (unsigned)(r.groups * p->batch);
        const dim3 enter((unsigned)((p->batch * p->channels + 63) / 64));
        if (r.chunks > 1) {
            const dim3 grid(x_blocks, ((unsigned)r.chunks + 7) / 8 * 8), threads(64 * kRecWaves);
            recurrence_runs_kernel<Tr, SIG, false><<<grid, threads, 0, s>>>(a);
            recurrence_enter_kernel<Tr, false><<<enter, dim3(64), 0, s>>>(a);
            recurrence_chunk_fw_kernel<Tr, SIG><<<grid, threads, 0, s>>>(a);
        } else {
            recurrence_fw_kernel<Tr, SIG><<<whole_grid(p, r), dim3(64 * r.waves), 0, s>>>(a);
        }
    });
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

int bf_recurrence_bw(const bf_recurrence *p, const void *gate, const void *x, const void *state, const uint8_t *reset,
                     const void *h, const void *grad, const void *grad_last, void *d_gate, void *d_x, void *d_state,
                     void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_recurrence(p);
    if (rc) return rc;
    if (nothing(p)) return BF_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->steps == 0) return pass_on(p, grad_last, d_state, s);
    if (!gate || !h || !d_gate || !d_x || (p->sigmoid && !x)) return fail(BF_ERR_INVALID, "gate, x, h, d_gate or d_x is NULL");
    const RecurrencePlan r = plan(p);
    if ((rc = check_grid(p, r)) || (rc = check_workspace(r, workspace, workspace_bytes))) return rc;
    RecurrenceArgs a = {};
    fill(a, p, r, workspace);
    a.gate = gate;
    a.x = x;
    a.state = state;
    a.reset = reset;
    a.h = const_cast<void *>(h);
    a.grad = grad;
    a.grad_last = grad_last;
    a.d_gate = d_gate;
    a.d_x = d_x;
    a.d_state = d_state;
    with_kind(p, [&](auto kind, auto sigmoid) {
        using Tr = decltype(kind);
        constexpr bool SIG = decltype(sigmoid)::value;
        const unsigned x_blocks = (unsigned)(r.groups * p->batch);
        const dim3 enter((unsigned)((p->batch * p->channels + 63) / 64));
        if (r.chunks > 1) {
            const dim3 grid(x_blocks, ((unsigned)r.chunks + 7) / 8 * 8), threads(64 * kRecWaves);
            recurrence_runs_kernel<Tr, SIG, true><<<grid, threads, 0, s>>>(a);
            recurrence_enter_kernel<Tr, true><<<enter, dim3(64), 0, s>>>(a);
            recurrence_chunk_bw_kernel<Tr, SIG><<<grid, threads, 0, s>>>(a);
        } else {
            recurrence_bw_kernel<Tr, SIG><<<whole_grid(p, r), dim3(64 * r.waves_bw), 0, s>>>(a);
        }
    });
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

int bf_recurrence_step(const bf_recurrence *p, const void *gate, const void *x, void *state, void *h, void *stream)
{
    const int rc = check_recurrence(p);
    if (rc) return rc;
    if (nothing(p)) return BF_OK;
    if (!gate || !x || !state || !h) return fail(BF_ERR_INVALID, "gate, x, state or h is NULL");
    RecurrenceArgs a = {};
    a.gate = gate;
    a.x = x;
    a.last = state;
    a.h = h;
    a.gate_b = p->gate_stride[0];
    a.x_b = p->x_stride[0];
    a.batch = p->batch;
    a.channels = (int)p->channels;
    with_kind(p, [&](auto kind, auto sigmoid) {
        using Tr = decltype(kind);
        const dim3 grid((unsigned)((p->channels + 256 * Tr::V - 1) / (256 * Tr::V)), (unsigned)std::min<int64_t>(p->batch, 65535));
        recurrence_step_kernel<Tr, decltype(sigmoid)::value><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a);
    });
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

}  // extern "C"
