// Rotary positions: of every head's first `rotated` features, pair p (features p and p + rotated / 2, or 2 p and 2 p + 1) is
// turned by position * frequency[p] and scaled:  (a, b) -> m (a cos - b sin, a sin + b cos);  the others are copied.  The gradient
// is turned back by the same angles.
//
// A workgroup takes some tokens and heads: it forms the tokens' cosines and sines once, in LDS, for all of its heads.  The angle
// is formed in double and reduced to a turn there (a float would have lost it at a position of a few thousand); what is left
// of it, at most half a turn, goes through the float functions.
//
// Bound by memory: 16 x 2048 x 16 x 64 bfloat16 in 23.2 us, 134 MB at 5.8 TB/s; 65537 x 10 x 100 floats, neighbours, 50 of them
// turned, in 107 us, 524 MB at 4.9 TB/s; 64 tokens x 32 heads in 3.4 us, a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vec8.hpp"

namespace bf {

struct RotaryArgs {
    const void *x;
    void *y;
    const int64_t *positions;
    const double *frequencies;
    int64_t x_stride[3], position_stride[2];   // batch, step, head
    int64_t steps, tokens;                     // tokens: batch * steps
    int heads, features, rotated;
    int tokens_each, heads_each, head_parts;   // of a workgroup; workgroups side by side over the heads
    float magnitude;
    bool back;
};

constexpr int kRotaryTable = 2048;   // cosines and sines a workgroup holds

template <typename T, bool NEIGHBOURS>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a)
{
    __shared__ float2 table[kRotaryTable];
    const int64_t first = (int64_t)(blockIdx.x / a.head_parts) * a.tokens_each;
    const int head0 = (int)(blockIdx.x % a.head_parts) * a.heads_each;
    const int tokens = (int)min((int64_t)a.tokens_each, a.tokens - first), heads = min(a.heads_each, a.heads - head0);
    const int pairs = a.rotated / 2, rest = a.features - a.rotated;
    for (int at = threadIdx.x; at < tokens * pairs; at += 256) {
        const int64_t token = first + at / pairs;
        const int64_t position = a.positions[token / a.steps * a.position_stride[0] + token % a.steps * a.position_stride[1]];
        const double turns = (double)position * (a.frequencies[at % pairs] * 0.15915494309189535);
        float sine, cosine;
        sincospif(2.0f * (float)(turns - rint(turns)), &sine, &cosine);
        table[at] = make_float2(a.magnitude * cosine, a.back ? -a.magnitude * sine : a.magnitude * sine);
    }
    __syncthreads();
    // Eight pairs at a time, then eight of the features that are copied; or eight neighbours of all of them.
    const int turned = NEIGHBOURS ? (a.features + 7) / 8 : (pairs + 7) / 8, items = NEIGHBOURS ? turned : turned + (rest + 7) / 8;
    for (int at = threadIdx.x; at < tokens * heads * items; at += 256) {
        const int item = at % items, n = at / items, head = head0 + n % heads, t = n / heads;
        const int64_t token = first + t;
        const T *x = static_cast<const T *>(a.x) + token / a.steps * a.x_stride[0] + token % a.steps * a.x_stride[1] + head * a.x_stride[2];
        T *y = static_cast<T *>(a.y) + (token * a.heads + head) * a.features;
        const float2 *turn = table + t * pairs;
        float u[8], v[8];
        if (!NEIGHBOURS && item >= turned) {
            const int col = (item - turned) * 8;
            load8(x + a.rotated, col, rest, 0.0f, u);
            store8(y + a.rotated, col, rest, u);
        } else if (NEIGHBOURS) {
            load8(x, item * 8, a.features, 0.0f, u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool turns = item * 4 + i < pairs;
                const float2 z = turn[turns ? item * 4 + i : 0];
                const float one = u[2 * i] * z.x - u[2 * i + 1] * z.y, two = u[2 * i] * z.y + u[2 * i + 1] * z.x;
                v[2 * i] = turns ? one : u[2 * i];
                v[2 * i + 1] = turns ? two : u[2 * i + 1];
            }
            store8(y, item * 8, a.features, v);
        } else {
            load8(x, item * 8, pairs, 0.0f, u);
            load8(x + pairs, item * 8, pairs, 0.0f, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 z = turn[min(item * 8 + i, pairs - 1)];
                const float one = u[i] * z.x - v[i] * z.y;
                v[i] = u[i] * z.y + v[i] * z.x;
                u[i] = one;
            }
            store8(y, item * 8, pairs, u);
            store8(y + pairs, item * 8, pairs, v);
        }
    }
}

}  // namespace bf
