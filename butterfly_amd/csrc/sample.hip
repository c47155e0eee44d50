// Entry point of the sampling from logits (sample.hpp): argument checks, choice of the kernel, launch.

#include "../../include/butterfly_hip.h"

#include "error.hpp"
#include "sample.hpp"

namespace {

using namespace bf;

// (weights of up to 2^44 that sum to less than 2^63)
constexpr int64_t kMostTokens = (int64_t)1 << 19;

int check_sample(const bf_sample *p)
{
    if (!p) return fail(BF_ERR_INVALID, "sample descriptor is NULL");
    if (p->dtype != BF_F32 && p->dtype != BF_BF16) return fail(BF_ERR_INVALID, "dtype must be BF_F32 or BF_BF16");
    if (p->rows < 0 || p->vocab < 0) return fail(BF_ERR_INVALID, "sizes must be non-negative");
    if (p->rows > 0 && p->vocab == 0) return fail(BF_ERR_INVALID, "vocab must be positive");
    if (p->vocab > kMostTokens) return fail(BF_ERR_UNSUPPORTED, "vocabularies of more than 2^19 entries are not supported");
    // (1024 threads a row: a grid has less than 2^32 of them)
    if (p->rows >= ((int64_t)1 << 22)) return fail(BF_ERR_UNSUPPORTED, "2^22 rows and more are not supported");
    if (p->logits_stride < 0) return fail(BF_ERR_INVALID, "strides must be non-negative");
    return BF_OK;
}

template <typename T>
void launch(const SampleArgs &a, int64_t rows, hipStream_t s)
{
    const dim3 grid((unsigned)rows), threads(kSampleThreads);
    const int64_t held = (int64_t)kSampleThreads * (16 / sizeof(T));   // entries that one piece a thread holds
    // The fewest pieces that hold the row: a pass goes through all of them, whether the row fills them or not (64 rows of 30001 floats in
    // 8 pieces 34.6 us, in 16 of them 45.7).
    if (a.vocab <= held) sample_kernel<T, 1><<<grid, threads, 0, s>>>(a);
    else if (a.vocab <= 2 * held) sample_kernel<T, 2><<<grid, threads, 0, s>>>(a);
    else if (a.vocab <= 4 * held) sample_kernel<T, 4><<<grid, threads, 0, s>>>(a);
    else if (a.vocab <= 8 * held) sample_kernel<T, 8><<<grid, threads, 0, s>>>(a);
    else if (a.vocab <= 16 * held) sample_kernel<T, 16><<<grid, threads, 0, s>>>(a);
    else sample_kernel<T, 0><<<grid, threads, 0, s>>>(a);
}

}  // namespace

extern "C" int bf_sample_tokens(const bf_sample *p, const void *logits, const float *uniform, const float *temperature,
                                const int64_t *top_k, const float *top_p, const float *min_p, int64_t *token, void *stream)
{
    const int rc = check_sample(p);
    if (rc) return rc;
    if (p->rows == 0) return BF_OK;
    if (!logits || !uniform || !token) return fail(BF_ERR_INVALID, "logits, uniform or token is NULL");
    SampleArgs a = {};
    a.logits = logits;
    a.uniform = uniform;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.temperature_all = p->temperature;
    a.top_k_all = p->top_k;
    a.top_p_all = p->top_p;
    a.min_p_all = p->min_p;
    a.token = token;
    a.stride = p->logits_stride;
    a.vocab = (int)p->vocab;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->dtype == BF_F32) launch<float>(a, p->rows, s);
    else launch<bf16>(a, p->rows, s);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}
