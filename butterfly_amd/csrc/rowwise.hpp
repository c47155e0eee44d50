// What stands between two layers of a block, row by row:
//
//   sum = residual + drop(x)           drop(x) = keep ? x * scale : 0
//   y   = (sum - mean) * rstd * weight + bias,  rstd = 1 / sqrt(var + eps)
//
// each part optional (no generator: nothing is dropped; no residual; no y: the sum alone).  Backward, with
// u = (sum - mean) * rstd and gw = grad_y * weight:
//
//   d_sum = rstd * (gw - mean(gw) - u * mean(gw * u)) + grad_sum;  d_residual = d_sum;
//   d_x = keep ? d_sum * scale : 0;  d_weight = column sums of grad_y * u;  d_bias = those of grad_y
//
// Some twenty operations an element against 4 to 20 bytes: memory bounds every kernel here, so each reads a
// row once and keeps it in registers between the statistics and the result.  L lanes share a row and
// hold K chunks of 8 columns each; the column sums stay in the registers of the lanes that own the
// columns while a workgroup walks its rows, and leave it once (partial slices, added by
// column_sums_kernel in a fixed order: no atomics, the same bits every time).
//
// The generator is Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// 2011): one block of four words gives the 16-bit numbers of a chunk of 8 columns, so forward and
// backward make the same mask from (seed, call, row, chunk) and none is stored.  16 bits an element
// resolve p to 1/65536 at half the generator's work of 32.
#pragma once

#include "vec8.hpp"

namespace bf {

struct RowArgs {
    const void *x, *residual;           // forward; backward: x is the sum
    const void *weight, *bias;          // NULL: ones, zeros
    const void *grad_y, *grad_sum;      // backward; grad_sum may be NULL
    void *sum, *y;                      // NULL: not wanted
    void *d_x, *d_residual;             // d_residual NULL: not wanted
    float2 *stats;                      // (mean, rstd) of each row; NULL forward: not wanted
    float *partial;                     // backward: (workgroups, 2, slice) column sums; NULL: not wanted
    float *shift;                       // backward, rows read again, with partial: what each row's u is off by
    const int64_t *rng;                 // (seed, call); NULL: nothing is dropped
    int64_t rows;
    int64_t x_stride, residual_stride, grad_y_stride, grad_sum_stride;
    int cols;
    int slice;                          // cols rounded up to 8
    uint32_t threshold;                 // 16-bit numbers below it drop
    float scale, eps;
    int wide_params;                    // weight and bias are float whatever T is
};

// ---- the generator -----------------------------------------------------------------------

__device__ __forceinline__ uint4 philox(uint4 c, uint2 k)
{
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)0xD2511F53u * c.x, b = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.y, (uint32_t)a);
        k.x += 0x9E3779B9u;
        k.y += 0xBB67AE85u;
    }
    return c;
}

struct Dropper {
    bool on;
    uint2 key, call;
    uint32_t threshold;
    float scale;

    __device__ __forceinline__ explicit Dropper(const RowArgs &a)
        : on(a.rng != nullptr), key(make_uint2(0, 0)), call(make_uint2(0, 0)), threshold(a.threshold), scale(a.scale)
    {
        if (!on) return;
        const uint64_t s = (uint64_t)a.rng[0], c = (uint64_t)a.rng[1];
        key = make_uint2((uint32_t)s, (uint32_t)(s >> 32));
        call = make_uint2((uint32_t)c, (uint32_t)(c >> 32));
    }

    // (a dropped element is zero whatever it was, infinite or NaN too)
    __device__ __forceinline__ void apply(int64_t row, int col, float (&v)[8]) const
    {
        if (!on) return;
        const uint4 r = philox(make_uint4((uint32_t)col >> 3, (uint32_t)row, call.x, call.y), key);
        const uint32_t words[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = (words[i] & 0xffffu) >= threshold ? v[2 * i] * scale : 0.0f;
            v[2 * i + 1] = (words[i] >> 16) >= threshold ? v[2 * i + 1] * scale : 0.0f;
        }
    }
};

// residual + drop(x), zeros past the row's end
template <typename T>
__device__ __forceinline__ void total8(const RowArgs &a, const Dropper &drop, int64_t row, int col, float (&v)[8])
{
    load8(reinterpret_cast<const T *>(a.x) + row * a.x_stride, col, a.cols, 0.0f, v);
    if (a.residual) {
        float r[8];
        load8(reinterpret_cast<const T *>(a.residual) + row * a.residual_stride, col, a.cols, 0.0f, r);
        drop.apply(row, col, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    } else {
        drop.apply(row, col, v);
    }
}

template <typename T>
__device__ __forceinline__ void param8(const void *p, int wide, int col, int cols, float fill, float (&v)[8])
{
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fill;
    } else if (wide) {
        load8(reinterpret_cast<const float *>(p), col, cols, 0.0f, v);
    } else {
        load8(reinterpret_cast<const T *>(p), col, cols, 0.0f, v);
    }
}

// ---- without a norm: sum = residual + drop(x) ------------------------------------------------
// lanes: a power of two up to 256, lanes that share a row.  16384 x 1024 bfloat16 with a residual: 16 us (100 MB, 6.3 TB/s, part
// of it out of caches), the same backward; 50 x 784 float 3.2 (a launch).
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(RowArgs a, int lanes_log)
{
    const Dropper drop(a);
    const int lanes = 1 << lanes_log, groups = 256 >> lanes_log;
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log;
    for (int64_t row = (int64_t)blockIdx.x * groups + group; row < a.rows; row += (int64_t)gridDim.x * groups) {
        T *out = reinterpret_cast<T *>(a.sum) + row * a.cols;
        for (int col = lane * 8; col < a.cols; col += lanes * 8) {
            float v[8];
            total8<T>(a, drop, row, col, v);
            store8(out, col, a.cols, v);
        }
    }
}

// ---- rows held in registers ---------------------------------------------------------------------

template <int L>
constexpr int row_threads() { return L < 256 ? 256 : L; }

// Columns of a row that wave w of its L / 64 holds.
template <int L, int K>
__device__ __forceinline__ int wave_cols(int w, int cols)
{
    int n = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int left = cols - 8 * (k * L + 64 * w);
        n += left < 0 ? 0 : left > 512 ? 512 : left;
    }
    return n;
}

// A row's mean as base + shift and its sum of squared deviations.  The shift is what a float mean is off by (an
// offset of 1000 in front of deviations of 1 costs 2^-15 of them otherwise): the mean of the deviations from base.
// Rows of several wavefronts: each wavefront's deviations from its own mean, joined with their sums s_w as
// M2_w + 2 e_w s_w + n_w e_w^2, e_w from the row's mean to the wavefront's; one barrier.
struct Moments {
    float base, shift, m2;
    __device__ __forceinline__ float mean() const { return base + shift; }
    __device__ __forceinline__ float from(float v) const { return (v - base) - shift; }
};

template <int L, int K>
__device__ __forceinline__ Moments row_moments(const float (&v)[K][8], int lane, int cols, float4 (*lds)[16], int turn)
{
    constexpr int W = L < 64 ? L : 64;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[k][i];   // (zeros past the row's end)
    s = lanes_sum<W>(s);
    const int n = L <= 64 ? cols : wave_cols<L, K>(lane >> 6, cols);
    Moments m;
    m.base = n > 0 ? s / (float)n : 0.0f;
    float off = 0.0f, q = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = 8 * (k * L + lane) + i < cols ? v[k][i] - m.base : 0.0f;
            off += d;
            q = fmaf(d, d, q);
        }
    off = lanes_sum<W>(off);
    q = lanes_sum<W>(q);
    if constexpr (L <= 64) {
        m.shift = off / (float)cols;
        m.m2 = q - off * m.shift;
        if (m.m2 < 0.0f) m.m2 = 0.0f;
    } else {
        if ((lane & 63) == 0) lds[turn][lane >> 6] = make_float4(m.base, off, q, 0.0f);
        __syncthreads();
        m.base = lds[turn][0].x;
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) {
            const float4 p = lds[turn][w];
            const int nw = wave_cols<L, K>(w, cols);
            total += nw > 0 ? fmaf((float)nw, p.x - m.base, p.y) : 0.0f;
        }
        m.shift = total / (float)cols;
        m.m2 = 0.0f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) {
            const float4 p = lds[turn][w];
            const int nw = wave_cols<L, K>(w, cols);
            const float e = (p.x - m.base) - m.shift;
            m.m2 += nw > 0 ? fmaf(e, fmaf((float)nw, e, 2.0f * p.y), p.z) : 0.0f;
        }
        if (m.m2 < 0.0f) m.m2 = 0.0f;
    }
    return m;
}

// 32768 x 4096 float 217 us (1.07 GB, 5.0 TB/s); 8192 x 2048 float with dropout, residual and their sum written 56 (268 MB, 4.8
// TB/s); 3001 x 1000 bfloat16 7.2; 16 x 512 float 3.7.
template <typename T, int L, int K>
__global__ __launch_bounds__(row_threads<L>()) void norm_fw_kernel(RowArgs a)
{
    constexpr int G = row_threads<L>() / L;
    __shared__ float4 lds[2][16];
    const Dropper drop(a);
    const int lane = threadIdx.x % L;
    float w[K][8], b[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        param8<T>(a.weight, a.wide_params, 8 * (k * L + lane), a.cols, 1.0f, w[k]);
        param8<T>(a.bias, a.wide_params, 8 * (k * L + lane), a.cols, 0.0f, b[k]);
    }
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L; row < a.rows; row += (int64_t)gridDim.x * G) {
        float v[K][8];
#pragma unroll
        for (int k = 0; k < K; ++k) total8<T>(a, drop, row, 8 * (k * L + lane), v[k]);
        if (a.sum) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                store8(reinterpret_cast<T *>(a.sum) + row * a.cols, 8 * (k * L + lane), a.cols, v[k]);
        }
        const Moments m = row_moments<L, K>(v, lane, a.cols, lds, turn);
        turn ^= 1;
        const float rstd = 1.0f / sqrtf(m.m2 / (float)a.cols + a.eps);
        if (a.stats && lane == 0) a.stats[row] = make_float2(m.mean(), rstd);
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = fmaf(m.from(v[k][i]) * rstd, w[k][i], b[k][i]);
            store8(reinterpret_cast<T *>(a.y) + row * a.cols, 8 * (k * L + lane), a.cols, v[k]);
        }
    }
}

// A workgroup's column sums, those of its row groups joined in ascending order.
template <int L, int K>
__device__ __forceinline__ void store_sums(const float (&v)[K][8], float *joined, float *out, int slice)
{
    constexpr int B = row_threads<L>(), G = B / L;
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    if constexpr (G > 1) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) joined[group * (L * K * 8) + (k * 8 + i) * L + lane] = v[k][i];
        __syncthreads();
        for (int at = threadIdx.x; at < L * K * 8; at += B) {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < G; ++j) s += joined[j * (L * K * 8) + at];
            const int col = 8 * (at / (8 * L) * L + at % L) + at / L % 8;
            if (col < slice) out[col] = (float)s;
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = 8 * (k * L + lane);
            if (col < slice) store8_whole(out + col, v[k]);
        }
    }
}

// u is formed from the row's float mean, which is off by its rounding (2^-24 of an offset in front of the deviations): by
// delta = mean(u), since the true u have none.  So the row's sums are those of gw, gw u and u, and u, and mean(gw u) by
// delta mean(gw), are put right behind them, before the columns take their share.  (The sum behind a dropout in bfloat16 is
// its rounded self here, the statistics those of the unrounded one: 2^-9 of a gradient that has no more bits.)
// 32768 x 4096 float 292 us (1.61 GB, 5.5 TB/s); 8192 x 2048 float with dropout and three gradients 64 (336 MB, 5.2 TB/s); 3001 x
// 1000 bfloat16 12.3.
template <typename T, int L, int K>
__global__ __launch_bounds__(row_threads<L>()) void norm_bw_kernel(RowArgs a)
{
    constexpr int B = row_threads<L>(), G = B / L, W = L < 64 ? L : 64;
    __shared__ float4 lds[2][16];
    __shared__ float joined[G > 1 ? B * K * 8 : 1];
    const Dropper drop(a);
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const float inv = 1.0f / (float)a.cols;
    float w[K][8], dw[K][8] = {}, db[K][8] = {};
#pragma unroll
    for (int k = 0; k < K; ++k) param8<T>(a.weight, a.wide_params, 8 * (k * L + lane), a.cols, 1.0f, w[k]);
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * G + group; row < a.rows; row += (int64_t)gridDim.x * G) {
        float u[K][8], g[K][8];
        const float2 st = a.stats[row];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = 8 * (k * L + lane);
            // (past the row's end u and g are zero)
            load8(reinterpret_cast<const T *>(a.x) + row * a.x_stride, col, a.cols, st.x, u[k]);
            load8(reinterpret_cast<const T *>(a.grad_y) + row * a.grad_y_stride, col, a.cols, 0.0f, g[k]);
        }
        float c1 = 0.0f, c2 = 0.0f, delta = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                u[k][i] = (u[k][i] - st.x) * st.y;
                const float gw = g[k][i] * w[k][i];
                c1 += gw;
                c2 = fmaf(gw, u[k][i], c2);
                delta += u[k][i];
            }
        c1 = lanes_sum<W>(c1);
        c2 = lanes_sum<W>(c2);
        delta = lanes_sum<W>(delta);
        if constexpr (L > 64) {
            if ((lane & 63) == 0) lds[turn][lane >> 6] = make_float4(c1, c2, delta, 0.0f);
            __syncthreads();
            c1 = c2 = delta = 0.0f;
#pragma unroll
            for (int i = 0; i < L / 64; ++i) {
                const float4 p = lds[turn][i];
                c1 += p.x;
                c2 += p.y;
                delta += p.z;
            }
            turn ^= 1;
        }
        c1 *= inv;
        delta *= inv;
        c2 = fmaf(-delta, c1, c2 * inv);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = 8 * (k * L + lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = u[k][i] - delta;
                dw[k][i] = fmaf(g[k][i], v, dw[k][i]);
                db[k][i] += g[k][i];
                g[k][i] = st.y * (g[k][i] * w[k][i] - c1 - v * c2);
            }
            if (a.grad_sum) {
                float more[8];
                load8(reinterpret_cast<const T *>(a.grad_sum) + row * a.grad_sum_stride, col, a.cols, 0.0f, more);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[k][i] += more[i];
            }
            if (a.d_residual) store8(reinterpret_cast<T *>(a.d_residual) + row * a.cols, col, a.cols, g[k]);
            if (a.d_x) {
                drop.apply(row, col, g[k]);
                store8(reinterpret_cast<T *>(a.d_x) + row * a.cols, col, a.cols, g[k]);
            }
        }
    }
    if (!a.partial) return;
    float *out = a.partial + (int64_t)blockIdx.x * 2 * a.slice;
    store_sums<L, K>(dw, joined, out, a.slice);
    store_sums<L, K>(db, joined, out + a.slice, a.slice);
}

// ---- rows too wide for the registers of a workgroup: read again instead -----------------------------
// 2048 x 9000 float: 47 us forward, 123 with backward; 2048 x 16384 71 and 225 (the second read out of the L2).

constexpr int kWideThreads = 1024;

__device__ __forceinline__ float2 block_sum(float2 v, float2 (*lds)[16], int turn)
{
    v = make_float2(lanes_sum<64>(v.x), lanes_sum<64>(v.y));
    if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    v = make_float2(0.0f, 0.0f);
    for (int i = 0; i < kWideThreads / 64; ++i) v = make_float2(v.x + lds[turn][i].x, v.y + lds[turn][i].y);
    return v;
}

// (three sums; the fourth is nothing)
__device__ __forceinline__ float4 block_sum(float4 v, float4 (*lds)[16], int turn)
{
    v = make_float4(lanes_sum<64>(v.x), lanes_sum<64>(v.y), lanes_sum<64>(v.z), 0.0f);
    if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < kWideThreads / 64; ++i) {
        const float4 p = lds[turn][i];
        v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, 0.0f);
    }
    return v;
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void norm_fw_wide_kernel(RowArgs a)
{
    __shared__ float2 lds[2][16];
    const Dropper drop(a);
    const float inv = 1.0f / (float)a.cols;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float v[8];
        float2 s = make_float2(0.0f, 0.0f);
        for (int col = threadIdx.x * 8; col < a.cols; col += kWideThreads * 8) {
            total8<T>(a, drop, row, col, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s.x += v[i];
        }
        Moments m;
        m.base = block_sum(s, lds, 0).x * inv;
        s = make_float2(0.0f, 0.0f);
        for (int col = threadIdx.x * 8; col < a.cols; col += kWideThreads * 8) {
            total8<T>(a, drop, row, col, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = col + i < a.cols ? v[i] - m.base : 0.0f;
                s.x += d;
                s.y = fmaf(d, d, s.y);
            }
        }
        s = block_sum(s, lds, 1);
        m.shift = s.x * inv;
        m.m2 = s.y - s.x * m.shift;
        if (m.m2 < 0.0f) m.m2 = 0.0f;
        const float rstd = 1.0f / sqrtf(m.m2 * inv + a.eps);
        if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(m.mean(), rstd);
        for (int col = threadIdx.x * 8; col < a.cols; col += kWideThreads * 8) {
            float w[8], b[8];
            total8<T>(a, drop, row, col, v);
            if (a.sum) store8(reinterpret_cast<T *>(a.sum) + row * a.cols, col, a.cols, v);
            param8<T>(a.weight, a.wide_params, col, a.cols, 1.0f, w);
            param8<T>(a.bias, a.wide_params, col, a.cols, 0.0f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(m.from(v[i]) * rstd, w[i], b[i]);
            store8(reinterpret_cast<T *>(a.y) + row * a.cols, col, a.cols, v);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void norm_bw_wide_kernel(RowArgs a)
{
    __shared__ float4 lds[2][16];
    const Dropper drop(a);
    const float inv = 1.0f / (float)a.cols;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = reinterpret_cast<const T *>(a.x) + row * a.x_stride;
        const T *gy = reinterpret_cast<const T *>(a.grad_y) + row * a.grad_y_stride;
        const float2 st = a.stats[row];
        float u[8], g[8], w[8];
        float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // of gw, gw u and u
        for (int col = threadIdx.x * 8; col < a.cols; col += kWideThreads * 8) {
            load8(x, col, a.cols, st.x, u);
            load8(gy, col, a.cols, 0.0f, g);
            param8<T>(a.weight, a.wide_params, col, a.cols, 1.0f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                g[i] *= w[i];
                u[i] = (u[i] - st.x) * st.y;
                c.x += g[i];
                c.y = fmaf(g[i], u[i], c.y);
                c.z += u[i];
            }
        }
        c = block_sum(c, lds, turn);
        turn ^= 1;
        const float c1 = c.x * inv, delta = c.z * inv, c2 = fmaf(-delta, c1, c.y * inv);
        if (a.shift && threadIdx.x == 0) a.shift[row] = delta;
        if (!a.d_x && !a.d_residual) continue;
        for (int col = threadIdx.x * 8; col < a.cols; col += kWideThreads * 8) {
            load8(x, col, a.cols, 0.0f, u);
            load8(gy, col, a.cols, 0.0f, g);
            param8<T>(a.weight, a.wide_params, col, a.cols, 1.0f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = st.y * (g[i] * w[i] - c1 - fmaf(u[i] - st.x, st.y, -delta) * c2);
            if (a.grad_sum) {
                load8(reinterpret_cast<const T *>(a.grad_sum) + row * a.grad_sum_stride, col, a.cols, 0.0f, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] += u[i];
            }
            if (a.d_residual) store8(reinterpret_cast<T *>(a.d_residual) + row * a.cols, col, a.cols, g);
            if (a.d_x) {
                drop.apply(row, col, g);
                store8(reinterpret_cast<T *>(a.d_x) + row * a.cols, col, a.cols, g);
            }
        }
    }
}

// The column sums of such rows: grid (chunks of 512 columns, row partitions), four row groups a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void norm_param_partial_kernel(RowArgs a)
{
    __shared__ float joined[256 * 8];
    const int lane = threadIdx.x & 63, group = threadIdx.x >> 6, col = (blockIdx.x * 64 + lane) * 8;
    float dw[8] = {}, db[8] = {};
    if (col < a.cols) {
        for (int64_t row = (int64_t)blockIdx.y * 4 + group; row < a.rows; row += (int64_t)gridDim.y * 4) {
            const float2 st = a.stats[row];
            const float delta = a.shift[row];
            float u[8], g[8];
            load8(reinterpret_cast<const T *>(a.x) + row * a.x_stride, col, a.cols, 0.0f, u);
            load8(reinterpret_cast<const T *>(a.grad_y) + row * a.grad_y_stride, col, a.cols, 0.0f, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dw[i] = fmaf(g[i], fmaf(u[i] - st.x, st.y, -delta), dw[i]);
                db[i] += g[i];
            }
        }
    }
    float *out = a.partial + (int64_t)blockIdx.y * 2 * a.slice + blockIdx.x * 512;
#pragma unroll
    for (int which = 0; which < 2; ++which, out += a.slice) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) joined[group * 512 + lane * 8 + i] = which ? db[i] : dw[i];
        __syncthreads();
        for (int at = threadIdx.x; at < 512; at += 256)
            if (blockIdx.x * 512 + at < a.slice)
                out[at] = (joined[at] + joined[512 + at]) + (joined[1024 + at] + joined[1536 + at]);
    }
}

// out[c] = sum of the slices' entry c, for d_weight and d_bias side by side: Q times four neighbouring entries and
// 1024 / Q runs of slices a workgroup, each run ascending, the runs joined pairwise (in double: a sum over many rows
// that nearly cancels keeps what the slices hold).  Q = 16 reads 256 bytes of a slice at a time, 4 makes four times as
// many workgroups for narrow rows: 512 slices of 4096 columns 5.7 us, of 1000 4.0.
struct ColumnSumArgs {
    const float *partial;     // (parts, 2, slice)
    void *d_weight, *d_bias;  // NULL: not wanted
    int parts, slice, cols;
};

template <typename P, int Q>
__global__ __launch_bounds__(1024) void column_sums_kernel(ColumnSumArgs a)
{
    constexpr int kRuns = 1024 / Q;
    __shared__ double lds[kRuns][4 * Q];
    const int at = (blockIdx.x * Q + threadIdx.x % Q) * 4, run = threadIdx.x / Q;
    double s[4] = {};
    if (at < 2 * a.slice) {
#pragma unroll 4
        for (int p = run; p < a.parts; p += kRuns) {
            const quad_at_4 v = *reinterpret_cast<const quad_at_4 *>(a.partial + (int64_t)p * 2 * a.slice + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[run][threadIdx.x % Q * 4 + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int half = kRuns / 2; half >= 1; half /= 2) {
        if (run < half) {
#pragma unroll
            for (int i = 0; i < 4; ++i) lds[run][threadIdx.x % Q * 4 + i] += lds[run + half][threadIdx.x % Q * 4 + i];
        }
        __syncthreads();
    }
    if (threadIdx.x >= 4 * Q) return;
    const int entry = blockIdx.x * Q * 4 + threadIdx.x;
    if (entry >= 2 * a.slice) return;
    const int col = entry < a.slice ? entry : entry - a.slice;
    void *out = entry < a.slice ? a.d_weight : a.d_bias;
    if (out && col < a.cols) reinterpret_cast<P *>(out)[col] = (P)(float)lds[0][threadIdx.x];
}

}  // namespace bf
