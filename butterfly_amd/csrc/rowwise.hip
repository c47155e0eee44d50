// Entry points of the row operators (rowwise.hpp): argument checks, choice of the kernel, launches.

#include "../../include/butterfly_hip.h"

#include <algorithm>
#include <cmath>

#include "error.hpp"
#include "rowwise.hpp"

namespace {

using namespace bf;

constexpr int kRegisterCols = 8192;              // widest row that the register kernels hold
constexpr int64_t kMaxCols = (int64_t)1 << 28;   // column numbers and slices stay inside 32 bits

int check_rows(const bf_rowwise *p)
{
    if (!p) return fail(BF_ERR_INVALID, "row descriptor is NULL");
    if (p->dtype != BF_F32 && p->dtype != BF_BF16) return fail(BF_ERR_INVALID, "dtype must be BF_F32 or BF_BF16");
    if (p->param_dtype != BF_F32 && p->param_dtype != p->dtype)
        return fail(BF_ERR_INVALID, "param_dtype must be BF_F32 or the rows' dtype");
    if (p->rows < 0 || p->cols < 0) return fail(BF_ERR_INVALID, "sizes must be non-negative");
    if (p->cols > kMaxCols) return fail(BF_ERR_UNSUPPORTED, "rows of more than 2^28 columns are not supported");
    if (p->rows > ((int64_t)1 << 40)) return fail(BF_ERR_UNSUPPORTED, "too many rows");
    if (p->x_stride < 0 || p->residual_stride < 0 || p->grad_y_stride < 0 || p->grad_sum_stride < 0)
        return fail(BF_ERR_INVALID, "strides must be non-negative");
    if (!(p->drop_probability >= 0.0 && p->drop_probability <= 1.0))
        return fail(BF_ERR_INVALID, "drop_probability must be in [0, 1]");
    // (the generator's counter takes a row's number in 32 bits)
    if (p->drop_probability > 0.0 && p->rows > ((int64_t)1 << 32)) return fail(BF_ERR_UNSUPPORTED, "dropout of more than 2^32 rows is not supported");
    if (!(p->eps >= 0.0)) return fail(BF_ERR_INVALID, "eps must be non-negative");
    return BF_OK;
}

void fill_common(RowArgs &a, const bf_rowwise *p, const void *rng)
{
    // (ties to even, as Python's round)
    const uint32_t threshold = (uint32_t)std::nearbyint(65536.0 * p->drop_probability);
    a.rows = p->rows;
    a.cols = (int)p->cols;
    a.slice = (a.cols + 7) / 8 * 8;
    a.x_stride = p->x_stride;
    a.residual_stride = p->residual_stride;
    a.grad_y_stride = p->grad_y_stride;
    a.grad_sum_stride = p->grad_sum_stride;
    a.rng = threshold > 0 ? static_cast<const int64_t *>(rng) : nullptr;
    a.threshold = threshold;
    a.scale = threshold < 65536 ? (float)(65536.0 / (65536 - threshold)) : 0.0f;
    a.eps = (float)p->eps;
    a.wide_params = p->param_dtype == BF_F32;
}

// Lanes that share a row (L) and chunks of 8 columns each of them holds (K).  Measured (forward, forward with backward):
// 65536 x 512 float by 32 lanes 41.7 and 128 us, by 64 44.3 and 139; 32768 x 1000 by 64 43.4 and 134, by 128 46.8 and 168;
// 16384 x 2048 bfloat16 by 256 36.3 and 99, by 64 (K = 4) 40.3 and 97, float 45.5 and 132 beside 47.7 and 146; 8192 x
// 4096 by 256 44 and 138, by 512 52 and 142; 4096 x 8192 bfloat16 by 512 37 and 108, by 256 43 and 115, by 1024 74 and 134.
// Wider rows are read again, out of the L2: 2048 x 9000 float 45 and 118, by 512 lanes (K = 4) 60 and 133; 2048 x 16384
// bfloat16 47 and 120 beside 55 and 139 (float 71 and 223 beside 70 and 199).
template <typename F>
void with_row_shape(int cols, F &&f)
{
#define BF_SHAPE(L, K) f(std::integral_constant<int, L>(), std::integral_constant<int, K>())
    if (cols <= 64) BF_SHAPE(8, 1);
    else if (cols <= 128) BF_SHAPE(16, 1);
    else if (cols <= 256) BF_SHAPE(32, 1);
    else if (cols <= 512) BF_SHAPE(32, 2);
    else if (cols <= 1024) BF_SHAPE(64, 2);
    else if (cols <= 2048) BF_SHAPE(256, 1);
    else if (cols <= 4096) BF_SHAPE(256, 2);
    else BF_SHAPE(512, 2);
#undef BF_SHAPE
}

int row_groups(int cols)
{
    int g = 1;
    with_row_shape(cols, [&](auto l, auto) { g = row_threads<decltype(l)::value>() / decltype(l)::value; });
    return g;
}

// Workgroups of the backward call: each ends with a slice of column sums that is written and read back, so as few as
// fill the chip: 32768 x 4096 float by 512 290 us, by 256 333, by 1024 308.
int64_t backward_groups(const bf_rowwise *p)
{
    if (p->cols > kRegisterCols) return std::max<int64_t>(1, std::min<int64_t>((p->rows + 15) / 16, 64));
    const int64_t g = row_groups((int)p->cols);
    return std::max<int64_t>(1, std::min<int64_t>((p->rows + g - 1) / g, 512));
}

size_t slice_bytes(const bf_rowwise *p)
{
    return (size_t)backward_groups(p) * 2 * (size_t)((p->cols + 7) / 8 * 8) * sizeof(float);
}

template <typename T>
void launch_fw(const RowArgs &a, hipStream_t stream)
{
    if (!a.y) {
        int lanes_log = 3;
        while (lanes_log < 8 && (8 << lanes_log) < a.cols) ++lanes_log;
        const int64_t groups = 256 >> lanes_log;
        dropout_kernel<T><<<dim3((unsigned)std::min<int64_t>((a.rows + groups - 1) / groups, 4096)), dim3(256), 0, stream>>>(a, lanes_log);
    } else if (a.cols > kRegisterCols) {
        norm_fw_wide_kernel<T><<<dim3((unsigned)std::min<int64_t>(a.rows, 512)), dim3(kWideThreads), 0, stream>>>(a);
    } else {
        with_row_shape(a.cols, [&](auto l, auto k) {
            constexpr int L = decltype(l)::value, K = decltype(k)::value, B = row_threads<L>();
            const int64_t blocks = std::min<int64_t>((a.rows + B / L - 1) / (B / L), 2048);
            norm_fw_kernel<T, L, K><<<dim3((unsigned)blocks), dim3(B), 0, stream>>>(a);
        });
    }
}

template <typename T>
void launch_bw(const RowArgs &a, int64_t blocks, hipStream_t stream)
{
    if (a.cols > kRegisterCols) {
        norm_bw_wide_kernel<T><<<dim3((unsigned)std::min<int64_t>(a.rows, 512)), dim3(kWideThreads), 0, stream>>>(a);
        if (a.partial)
            norm_param_partial_kernel<T><<<dim3((unsigned)((a.cols + 511) / 512), (unsigned)blocks), dim3(256), 0, stream>>>(a);
    } else {
        with_row_shape(a.cols, [&](auto l, auto k) {
            constexpr int L = decltype(l)::value, K = decltype(k)::value;
            norm_bw_kernel<T, L, K><<<dim3((unsigned)blocks), dim3(row_threads<L>()), 0, stream>>>(a);
        });
    }
}

template <typename P>
void launch_sums(const ColumnSumArgs &c, hipStream_t s)
{
    const int entries = 2 * c.slice;
    if (entries >= 4096) column_sums_kernel<P, 16><<<dim3((unsigned)((entries + 63) / 64)), dim3(1024), 0, s>>>(c);
    else column_sums_kernel<P, 4><<<dim3((unsigned)((entries + 15) / 16)), dim3(1024), 0, s>>>(c);
}

__global__ void rng_next_kernel(int64_t *state, int64_t *taken, uint64_t add)
{
    const int64_t seed = state[0], call = state[1];
    taken[0] = (int64_t)((uint64_t)seed + add);
    taken[1] = call;
    state[1] = (int64_t)((uint64_t)call + 1);
}

}  // namespace

extern "C" {

int bf_rng_next(int64_t *state, int64_t *taken, void *stream) { return bf_rng_next_of(state, taken, 0, stream); }

int bf_rng_next_of(int64_t *state, int64_t *taken, int64_t replica, void *stream)
{
    if (!state || !taken) return fail(BF_ERR_INVALID, "state or taken is NULL");
    // (2^64 over the golden ratio, odd: seeds of neighbouring replicas lie far apart)
    rng_next_kernel<<<dim3(1), dim3(1), 0, static_cast<hipStream_t>(stream)>>>(state, taken, (uint64_t)replica * 0x9E3779B97F4A7C15ull);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

int bf_rowwise_fw(const bf_rowwise *p, const void *x, const void *residual, const int64_t *rng, const void *weight,
                  const void *bias, void *sum, void *y, float *stats, void *stream)
{
    const int rc = check_rows(p);
    if (rc) return rc;
    if (p->rows == 0 || p->cols == 0) return BF_OK;
    if (!x) return fail(BF_ERR_INVALID, "x is NULL");
    if (!sum && !y) return fail(BF_ERR_INVALID, "neither sum nor y is wanted");
    if (!y && (weight || bias || stats)) return fail(BF_ERR_INVALID, "weight, bias and stats belong to a norm: y is NULL");
    if (p->drop_probability > 0.0 && !rng) return fail(BF_ERR_INVALID, "a drop_probability needs a generator: rng is NULL");
    RowArgs a = {};
    fill_common(a, p, rng);
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.bias = bias;
    a.sum = sum;
    a.y = y;
    a.stats = reinterpret_cast<float2 *>(stats);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->dtype == BF_F32) launch_fw<float>(a, s);
    else launch_fw<bf16>(a, s);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

size_t bf_rowwise_bw_workspace_bytes(const bf_rowwise *p)
{
    if (check_rows(p)) return BF_SIZE_INVALID;
    if (p->rows == 0 || p->cols == 0) return 0;
    // the slices of column sums; rows that are read again: what each one's u is off by
    return slice_bytes(p) + (p->cols > kRegisterCols ? (size_t)p->rows * sizeof(float) : 0);
}

int bf_rowwise_bw(const bf_rowwise *p, const void *sum, const void *grad_y, const void *grad_sum, const int64_t *rng,
                  const void *weight, const float *stats, void *d_x, void *d_residual, void *d_weight, void *d_bias,
                  void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check_rows(p);
    if (rc) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->cols == 0) return BF_OK;
    if (p->rows > 0) {
        if (!sum || !grad_y || !stats) return fail(BF_ERR_INVALID, "sum, grad_y or stats is NULL");
        if (p->drop_probability > 0.0 && !rng) return fail(BF_ERR_INVALID, "a drop_probability needs a generator: rng is NULL");
    }
    const bool params = d_weight || d_bias;
    RowArgs a = {};
    fill_common(a, p, rng);
    const int64_t blocks = p->rows > 0 ? backward_groups(p) : 0;
    if (params && p->rows > 0) {
        const size_t need = bf_rowwise_bw_workspace_bytes(p);
        if (!workspace || workspace_bytes < need)
            return fail(BF_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : 0);
        if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(BF_ERR_WORKSPACE, "workspace must be 16-byte aligned");
        a.partial = static_cast<float *>(workspace);
        if (p->cols > kRegisterCols) a.shift = reinterpret_cast<float *>(static_cast<char *>(workspace) + slice_bytes(p));
    }
    a.x = sum;
    a.grad_y = grad_y;
    a.grad_sum = grad_sum;
    a.weight = weight;
    a.stats = reinterpret_cast<float2 *>(const_cast<float *>(stats));
    a.d_x = d_x;
    a.d_residual = d_residual;
    if (p->rows > 0 && (params || d_x || d_residual)) {
        if (p->dtype == BF_F32) launch_bw<float>(a, blocks, s);
        else launch_bw<bf16>(a, blocks, s);
        BF_HIP_CHECK(hipGetLastError());
    }
    if (params) {
        const ColumnSumArgs c = {a.partial, d_weight, d_bias, (int)blocks, a.slice, a.cols};
        if (p->param_dtype == BF_F32) launch_sums<float>(c, s);
        else launch_sums<bf16>(c, s);
        BF_HIP_CHECK(hipGetLastError());
    }
    return BF_OK;
}

}  // extern "C"
