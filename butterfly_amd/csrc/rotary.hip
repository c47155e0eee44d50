// Entry point of the rotary positions (rotary.hpp): argument checks, a workgroup's share, launch.

#include "../../include/butterfly_hip.h"

#include <algorithm>

#include "error.hpp"
#include "rotary.hpp"

namespace {

using namespace bf;

int check_rotary(const bf_rotary *p)
{
    if (!p) return fail(BF_ERR_INVALID, "rotary descriptor is NULL");
    if (p->dtype != BF_F32 && p->dtype != BF_BF16) return fail(BF_ERR_INVALID, "dtype must be BF_F32 or BF_BF16");
    if (p->batch < 0 || p->steps < 0 || p->heads < 0 || p->features < 0) return fail(BF_ERR_INVALID, "sizes must be non-negative");
    if (p->rotated < 0 || p->rotated > p->features || p->rotated % 2 != 0)
        return fail(BF_ERR_INVALID, "rotated must be even and at most features");
    if (p->rotated > 2 * kRotaryTable) return fail(BF_ERR_UNSUPPORTED, "more than %d rotated features are not supported", 2 * kRotaryTable);
    if (p->features > ((int64_t)1 << 20) || p->heads > ((int64_t)1 << 20) || p->batch > ((int64_t)1 << 40) || p->steps > ((int64_t)1 << 40))
        return fail(BF_ERR_UNSUPPORTED, "too many tokens, heads or features");
    // (their product counts items and workgroups)
    if ((double)p->batch * (double)p->steps * (double)p->heads * (double)p->features > 0x1p48)
        return fail(BF_ERR_UNSUPPORTED, "too many tokens, heads or features");
    for (int i = 0; i < 3; ++i)
        if (p->x_stride[i] < 0) return fail(BF_ERR_INVALID, "strides must be non-negative");
    if (p->position_stride[0] < 0 || p->position_stride[1] < 0) return fail(BF_ERR_INVALID, "strides must be non-negative");
    return BF_OK;
}

}  // namespace

extern "C" int bf_rotary_apply(const bf_rotary *p, const void *x, const int64_t *positions, const double *frequencies, void *y,
                               int32_t back, void *stream)
{
    const int rc = check_rotary(p);
    if (rc) return rc;
    if (p->batch == 0 || p->steps == 0 || p->heads == 0 || p->features == 0) return BF_OK;
    if (!x || !y) return fail(BF_ERR_INVALID, "x or y is NULL");
    if (p->rotated > 0 && (!positions || !frequencies)) return fail(BF_ERR_INVALID, "positions or frequencies is NULL");
    RotaryArgs a = {};
    a.x = x;
    a.y = y;
    a.positions = positions;
    a.frequencies = frequencies;
    for (int i = 0; i < 3; ++i) a.x_stride[i] = p->x_stride[i];
    for (int i = 0; i < 2; ++i) a.position_stride[i] = p->position_stride[i];
    a.steps = p->steps;
    a.tokens = p->batch * p->steps;
    a.heads = (int)p->heads;
    a.features = (int)p->features;
    a.rotated = (int)p->rotated;
    a.magnitude = (float)p->magnitude;
    a.back = back != 0;
    // Two items a thread where there are enough for 1024 workgroups, one otherwise.  The two large cases of rotary.hpp: 23.8 and 107 us;
    // with four 29.2 and 126, with one 24.2 and 130 (a token of 130 items leaves half of the threads idle); 64 tokens x 32 heads
    // with one 3.5, with four 6.0.
    const int pairs = a.rotated / 2, rest = a.features - a.rotated;
    const int64_t items = p->interleaved ? (a.features + 7) / 8 : (pairs + 7) / 8 + (rest + 7) / 8;
    const int64_t each = std::max<int64_t>(256, std::min<int64_t>(512, a.tokens * a.heads * items / 1024));
    a.heads_each = (int)std::max<int64_t>(1, std::min<int64_t>(a.heads, each / items));
    a.head_parts = (a.heads + a.heads_each - 1) / a.heads_each;
    a.tokens_each = (int)std::max<int64_t>(1, std::min<int64_t>(each / (items * a.heads_each), pairs > 0 ? kRotaryTable / pairs : each));
    const int64_t blocks = (a.tokens + a.tokens_each - 1) / a.tokens_each * a.head_parts;
    if (blocks >= ((int64_t)1 << 24)) return fail(BF_ERR_UNSUPPORTED, "too many tokens and heads for one launch");
    const dim3 grid((unsigned)blocks);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->dtype == BF_F32) p->interleaved ? rotary_kernel<float, true><<<grid, dim3(256), 0, s>>>(a) : rotary_kernel<float, false><<<grid, dim3(256), 0, s>>>(a);
    else p->interleaved ? rotary_kernel<bf16, true><<<grid, dim3(256), 0, s>>>(a) : rotary_kernel<bf16, false><<<grid, dim3(256), 0, s>>>(a);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}
