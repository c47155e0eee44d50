// Linear attention with a decay for each head:  S_t = a_t S_{t-1} + k_t^T v_t,  o_t = scale q_t S_t,  a = exp(log_decay), S a
// (features, values) matrix of floats for each sequence and head; where a reset is set, S_{t-1} counts as zero.
//
// In chunks of C steps, with L_i the sum of a chunk's log decays up to step i (from the last reset on), S the state in front of
// the chunk and D_ij = scale exp(L_i - L_j) for j <= i of one document, else 0, b_i = scale exp(L_i) and w_j = exp(L_C - L_j) for
// steps that no reset parts from the chunk's start and end, else 0:
//   O  = (Q K^T . D) V + b Q S          S' = exp(L_C) S + K^T w V
// and backward, E the gradient of the state behind the chunk, G = (Q K^T . D) . (dO V^T) below the diagonal:
//   dV = (Q K^T . D)^T dO + w K E       dK = (dO V^T . D)^T Q + w V E^T       dQ = (dO V^T . D) K + b dO S^T
//   E' = exp(L_C) E + Q^T b dO
//   d log a_t = sum_{i >= t > j} G_ij + sum_{i >= t} q_i (b dO S^T)_i + sum_{j < t} k_j (w V E^T)_j + exp(L_C) <E, S>
// where the first sum is formed as sum_{i >= t} (row sum - column sum of G), within a document.
//
// A workgroup walks the chunks of one head of one sequence (or of a segment of it) with the state in the sums of the matrix
// units, so that q, k, v are read and o is written once.  For sequences and heads that do not fill the chip, segments of
// a sequence run side by side: a first launch forms what each adds to the state (la_walk_kernel without outputs), a second one the
// states between them, a third one the outputs.
//
// Products run on the matrix units, 16 x 16 tiles, float sums.  float operands: the float instruction, all bits.  bfloat16:
// inputs as they are; float factors as several bfloat16 numbers that add up to them: three (24 bits) for what is added
// to a state, two (16 bits) for states and for the products' inner factors Q K^T . D, dO V^T . D (the results are rounded to
// 8 bits; one number would leave errors of the size of that rounding).  An operand of a product over 32 steps or features
// is two pieces of 4 elements in a lane, of steps 4 g .. 4 g + 3 (g: lane / 16) of two neighbouring tiles: the layout that
// sums have, so that sums become operands without leaving their lane.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vec8.hpp"

namespace bf {

struct LaArgs {
    const void *q, *k, *v, *grad;            // grad: of o, may be NULL (zeros)
    const float *log_decay, *state, *grad_last;   // states may be NULL (zeros)
    const uint8_t *reset;                    // may be NULL
    void *o;
    float *last, *kept;                      // may be NULL
    void *d_q, *d_k, *d_v;
    float *d_log_decay, *d_state;            // d_state may be NULL
    int64_t q_stride[3], k_stride[3], v_stride[3], grad_stride[3], decay_stride[3], reset_stride[2];  // batch, step, head
    int64_t batch, steps, chunks;            // chunks: of a whole sequence
    int heads, shared;                       // shared: heads that share queries and keys
    int features, values;
    int64_t segment_chunks;                  // chunks of a segment
    int segments;
    float scale;
    bool wide;                               // d_q and d_k are floats of each head, to be added up over the heads that share them
    float *segment_state;                    // (segments, batch * heads, features, values)
    float *segment_decay;                    // (segments, batch * heads)
    int *segment_cut;
};

typedef float LaAcc __attribute__((ext_vector_type(4)));
typedef bf16 LaHalf4 __attribute__((ext_vector_type(4)));
typedef bf16 LaHalf8 __attribute__((ext_vector_type(8)));

template <typename T> struct LaFrag;
template <> struct LaFrag<bf16> { using type = LaHalf4; };
template <> struct LaFrag<float> { using type = LaAcc; };

// Chunks of 64 steps; float rows of 128 features: 32, four operands and the state's gradient are all that LDS holds.
template <typename T, int D>
struct LaShape {
    static constexpr int C = sizeof(T) == 4 && D == 128 ? 32 : 64;
    static constexpr int W = D / 16;                 // wavefronts: each owns 16 columns of a state
    static constexpr int TT = C / 16, DT = D / 16;   // tiles
    static constexpr int E = 16 / sizeof(T);         // elements of a load
    static constexpr int LD = D + E, LDC = C + E;    // rows in LDS: 16 bytes more, so that sixteen of them start in different banks
    static constexpr int LOADS = C * D / E / (64 * W);
    // pairs of tiles (i, j) with j <= i, and those above the diagonal that a product of 32 steps reads
    static constexpr int PAIRS = TT == 4 ? 12 : 4;
    static constexpr int INNER = sizeof(T) == 4 ? 1 : 2;   // numbers that an inner factor or a state is split into
    static constexpr int ADDED = sizeof(T) == 4 ? 1 : 3;   // and what is added to a state
    // the state's gradient in LDS (for dV): there is no room for a second number beside rows of 128
    static constexpr int HELD = sizeof(T) == 4 || D == 128 ? 1 : 2;
};

__device__ __forceinline__ LaAcc la_mma(LaHalf4 a0, LaHalf4 a1, LaHalf4 b0, LaHalf4 b1, LaAcc c)
{
    const LaHalf8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ LaAcc la_mma(LaAcc a0, LaAcc a1, LaAcc b0, LaAcc b1, LaAcc c)
{
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[s], b0[s], c, 0, 0, 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[s], b1[s], c, 0, 0, 0);
    return c;
}

// Element s is [row0 + lane % 16][col0 + 4 g + s]: the sum runs over neighbours in memory.
template <typename F, typename T>
__device__ __forceinline__ F la_rows(const T *lds, int stride, int row0, int col0)
{
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const F *>(lds + (row0 + (lane & 15)) * stride + col0 + 4 * (lane >> 4));
}
// Element s is [row0 + 4 g + s][col0 + lane % 16]: the sum runs over rows.
__device__ __forceinline__ LaHalf4 la_cols(const bf16 *lds, int stride, int row0, int col0)
{
    typedef short Quad16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) Quad16 LdsQuad;
    const int lane = threadIdx.x & 63, i = lane & 15;
    // (16 lanes hand in 4 rows of 16 columns and get them by columns)
    const bf16 *p = lds + (row0 + 4 * (lane >> 4) + (i >> 2)) * stride + col0 + 4 * (i & 3);
    return __builtin_bit_cast(LaHalf4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad *)p));
}
__device__ __forceinline__ LaAcc la_cols(const float *lds, int stride, int row0, int col0)
{
    const int lane = threadIdx.x & 63;
    const float *p = lds + (row0 + 4 * (lane >> 4)) * stride + col0 + (lane & 15);
    return LaAcc{p[0], p[stride], p[2 * stride], p[3 * stride]};
}

// x as N numbers of the operands' type, each the rounded rest of those before it.
template <int N>
__device__ __forceinline__ void la_split(LaAcc x, LaHalf4 (&out)[N])
{
#pragma unroll
    for (int n = 0; n < N; ++n) {
        out[n] = __builtin_convertvector(x, LaHalf4);
        if (n + 1 < N) x -= __builtin_convertvector(out[n], LaAcc);
    }
}
template <int N>
__device__ __forceinline__ void la_split(LaAcc x, LaAcc (&out)[N]) { out[0] = x; }

__device__ __forceinline__ LaAcc la_float(LaHalf4 v) { return __builtin_convertvector(v, LaAcc); }
__device__ __forceinline__ LaAcc la_float(LaAcc v) { return v; }

template <int CTRL>
__device__ __forceinline__ float la_dpp(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Sum over the 16 lanes of a row, the same in each (exchanges: neighbours, pairs, mirrored halves, mirrored rows).
__device__ __forceinline__ float la_sum16(float v)
{
    v += la_dpp<0xB1>(v);
    v += la_dpp<0x4E>(v);
    v += la_dpp<0x141>(v);
    v += la_dpp<0x140>(v);
    return v;
}

// 16 bytes of a row; what lies behind its end is zero.
template <typename T>
__device__ __forceinline__ uint4 la_load(const T *row, int col, int cols)
{
    constexpr int E = 16 / sizeof(T);
    using Quad = std::conditional_t<sizeof(T) == 4, quad_at_4, quad_at_2>;
    if (col + E <= cols) {
        const Quad v = *reinterpret_cast<const Quad *>(row + col);
        return __builtin_bit_cast(uint4, v);
    }
    T part[E];
#pragma unroll
    for (int i = 0; i < E; ++i) part[i] = col + i < cols ? row[col + i] : (T)0.0f;
    return __builtin_bit_cast(uint4, part);
}

// The largest magnitude among the numbers of v, as bits; at least la_infinite<T> where one is not finite.
typedef uint16_t LaShort2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ void la_magnitude(uint4 v, uint32_t &m)
{
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            m = max(m, words[i] & 0x7fffffffu);
        } else {
            m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(LaShort2, m),
                                                                       __builtin_bit_cast(LaShort2, words[i] & 0x7fff7fffu)));
        }
    }
}
template <typename T>
__device__ __forceinline__ bool la_not_finite(uint32_t m)
{
    if constexpr (sizeof(T) == 4) return m >= 0x7f800000u;
    else return (m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u;
}

// The steps of a chunk that a lane brings into LDS, on their way in registers.
template <typename T, int D>
struct LaPiece {
    using S = LaShape<T, D>;
    uint4 v[S::LOADS];

    __device__ __forceinline__ void fetch(const T *base, int64_t stride, int rows, int cols)
    {
#pragma unroll
        for (int n = 0; n < S::LOADS; ++n) {
            const int at = threadIdx.x + n * 64 * S::W, row = at / (D / S::E), col = at % (D / S::E) * S::E;
            v[n] = base && row < rows && col < cols ? la_load(base + row * stride, col, cols) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(T *lds, uint32_t &m) const
    {
#pragma unroll
        for (int n = 0; n < S::LOADS; ++n) {
            const int at = threadIdx.x + n * 64 * S::W, row = at / (D / S::E), col = at % (D / S::E) * S::E;
            *reinterpret_cast<uint4 *>(lds + row * S::LD + col) = v[n];
            la_magnitude<T>(v[n], m);
        }
    }
};

// Sums of a chunk's log decays, to the base 2, as two floats of together 48 bits: their differences keep the bits of the
// decays between two steps, whatever the steps in front have summed up to.  part: resets so far.
template <int C>
struct LaLevels {
    float hi[C], lo[C];
    int part[C];

    __device__ __forceinline__ float from_start(int i) const { return __builtin_amdgcn_exp2f(hi[i] + lo[i]); }
    __device__ __forceinline__ float between(int i, int j) const { return __builtin_amdgcn_exp2f((hi[i] - hi[j]) + (lo[i] - lo[j])); }
};

// One step a lane.  A decay below 2^-160 is zero beside anything in 32 bits and counts as that.
template <int C>
__device__ __forceinline__ void la_levels(LaLevels<C> &out, float log_decay, bool reset)
{
    const int lane = threadIdx.x & 63;
    const double x = (double)log_decay * 1.4426950408889634;
    double level = reset ? 0.0 : x < -160.0 ? -160.0 : x;
    int part = reset;
#pragma unroll
    for (int d = 1; d < C; d *= 2) {
        const double before = __shfl_up(level, d, 64);
        const int resets = __shfl_up(part, d, 64);
        if (lane >= d) {
            if (part == 0) level += before;
            part += resets;
        }
    }
    if (lane < C) {
        const float hi = (float)level;
        out.hi[lane] = hi;
        // (not finite: the difference of two of them is what it is)
        out.lo[lane] = (float)(level - (double)hi);
        out.part[lane] = part;
    }
}

struct LaDecay {
    float log_decay = 0.0f;
    bool reset = false;

    __device__ __forceinline__ void fetch(const LaArgs &a, const float *log_decay_row, const uint8_t *reset_row, int64_t t0, int rows)
    {
        const int lane = threadIdx.x & 63;
        log_decay = lane < rows ? log_decay_row[(t0 + lane) * a.decay_stride[1]] : 0.0f;
        reset = reset_row && lane < rows && reset_row[(t0 + lane) * a.reset_stride[1]] != 0;
    }
};

// (ti, tj) of pair n
template <int TT>
__device__ __forceinline__ void la_pair(int n, int &ti, int &tj)
{
    if (n < 4) {
        ti = n >> 1;
        tj = n & 1;
    } else {
        ti = 2 + ((n - 4) >> 2);
        tj = (n - 4) & 3;
    }
}

// The pieces of step t alone: the others count as zero whatever they are.
template <typename F>
__device__ __forceinline__ F la_only(F f, int t)
{
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < 4; ++s)
        if (4 * g + s != (t & 15)) f[s] = 0.0f;
    return f;
}

// Sum over the steps of tiles first .. last of a(part, tile) x b(tile), onto c (rows: steps row0 + 4 g + r of the chunk).
// bad: something is not finite.  Then step by step, and only onto the rows that `meets(row, step)`: what a factor of
// zero stands for must not turn into NaN.
template <int N, int TT, typename F, typename A, typename B, typename M>
__device__ __forceinline__ void la_over_steps(LaAcc &c, int first, int last, bool bad, A &&a, B &&b, M &&meets)
{
    if (!bad) {
#pragma unroll
        for (int p = 0; p < TT; p += 2)
            if (p + 1 >= first && p <= last) {
#pragma unroll
                for (int n = 0; n < N; ++n) c = la_mma(a(n, p), a(n, p + 1), b(p), b(p + 1), c);
            }
        return;
    }
    const F zero = {};
    for (int tile = first; tile <= last; ++tile)
        for (int t = 16 * tile; t < 16 * tile + 16; ++t) {
            LaAcc d = {};
            for (int n = 0; n < N; ++n) d = la_mma(la_only(a(n, tile), t), zero, la_only(b(tile), t), zero, d);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (meets(r, t)) c[r] += d[r];
        }
}

__device__ __forceinline__ int64_t la_offset(const int64_t (&stride)[3], int64_t b, int64_t t, int64_t h)
{
    return b * stride[0] + t * stride[1] + h * stride[2];
}

// Neighbouring heads lie next to each other in memory, and those of a group read the same rows: an XCD (workgroups go round
// them in turn) takes a run of them.
__device__ __forceinline__ int64_t la_unit(int64_t units)
{
    const int64_t per = (units + 7) / 8;
    const int64_t u = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    return (blockIdx.x >> 3) < per ? u : units;
}

// A head's walk over its chunks.  OUT: outputs, and the states in front of the chunks where they are kept; otherwise
// what a segment adds to the state: of k^T w v forward, of q^T b grad with BACK (from the end).
template <typename T, int D, bool OUT, bool BACK>
__global__ __launch_bounds__(4 * D) void la_walk_kernel(const LaArgs a)
{
    using S = LaShape<T, D>;
    using F = typename LaFrag<T>::type;
    constexpr int C = S::C, W = S::W, TT = S::TT, DT = S::DT, LD = S::LD, LDC = S::LDC;
    __shared__ __align__(16) T ks[C * LD];
    __shared__ __align__(16) T vs[C * LD];
    __shared__ __align__(16) T qs[OUT ? C * LD : 16];
    __shared__ __align__(16) T ps[OUT ? S::INNER * C * LDC : 16];
    __shared__ __align__(16) LaLevels<C> levels;
    __shared__ int bad_chunk[2];

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const int64_t heads = a.batch * a.heads, unit = la_unit(heads * a.segments);
    if (unit >= heads * a.segments) return;
    const int64_t segment = unit / heads, bh = unit % heads, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t first = segment * a.segment_chunks, end = min(first + a.segment_chunks, a.chunks);
    const int count = (int)(end - first), features = a.features, values = a.values;
    const T *q = static_cast<const T *>(a.q) + (OUT ? la_offset(a.q_stride, b, 0, h / a.shared) : 0);
    const T *k = BACK ? static_cast<const T *>(a.q) + la_offset(a.q_stride, b, 0, h / a.shared)
                      : static_cast<const T *>(a.k) + la_offset(a.k_stride, b, 0, h / a.shared);
    const T *v = BACK ? (a.grad ? static_cast<const T *>(a.grad) + la_offset(a.grad_stride, b, 0, h) : nullptr)
                      : static_cast<const T *>(a.v) + la_offset(a.v_stride, b, 0, h);
    const int64_t k_step = BACK ? a.q_stride[1] : a.k_stride[1], v_step = BACK ? a.grad_stride[1] : a.v_stride[1];
    const float *decay_row = a.log_decay + la_offset(a.decay_stride, b, 0, h);
    const uint8_t *reset_row = a.reset ? a.reset + b * a.reset_stride[0] : nullptr;

    // rows: features 16 t + 4 g + r, column: value 16 wave + lane % 16
    LaAcc s[DT];
    const int col = 16 * wave + i16;
    const float *start = !OUT ? nullptr : a.segments > 1 ? a.segment_state + (segment * heads + bh) * features * values
                                       : a.state ? a.state + bh * features * values : nullptr;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * t + 4 * g + r;
            s[t][r] = start && row < features && col < values ? start[row * values + col] : 0.0f;
        }

    LaPiece<T, D> nk, nv, nq;
    LaDecay nd;
    auto fetch = [&](int n) {
        const int64_t chunk = BACK ? end - 1 - n : first + n, t0 = chunk * C;
        const int rows = (int)min((int64_t)C, a.steps - t0);
        nk.fetch(k + t0 * k_step, k_step, rows, features);
        nv.fetch(v ? v + t0 * v_step : nullptr, v_step, rows, values);
        if constexpr (OUT) nq.fetch(q + t0 * a.q_stride[1], a.q_stride[1], rows, features);
        if (wave == 0) nd.fetch(a, decay_row, reset_row, t0, rows);
    };
    if (threadIdx.x < 2) bad_chunk[threadIdx.x] = 0;
    fetch(0);
    __syncthreads();
    double total = 0.0;
    int cuts = 0;
    for (int n = 0; n < count; ++n) {
        const int64_t chunk = BACK ? end - 1 - n : first + n, t0 = chunk * C;
        uint32_t magnitude = 0;
        nk.store(ks, magnitude);
        nv.store(vs, magnitude);
        if constexpr (OUT) nq.store(qs, magnitude);
        if (la_not_finite<T>(magnitude)) bad_chunk[n & 1] = 1;
        if (wave == 0) la_levels<C>(levels, nd.log_decay, nd.reset);
        __syncthreads();
        const bool bad = bad_chunk[n & 1] != 0;
        if (threadIdx.x == 0) bad_chunk[(n + 1) & 1] = 0;
        if (n + 1 < count) fetch(n + 1);

        if constexpr (OUT) {
            // Q K^T . D, transposed in the sums: rows are steps j
            for (int p = wave; p < S::PAIRS; p += W) {
                int ti, tj;
                la_pair<TT>(p, ti, tj);
                LaAcc c = {};
                if (tj <= ti) {
#pragma unroll
                    for (int x = 0; x < D; x += 32)
                        c = la_mma(la_rows<F>(ks, LD, 16 * tj, x), la_rows<F>(ks, LD, 16 * tj, x + 16), la_rows<F>(qs, LD, 16 * ti, x),
                                   la_rows<F>(qs, LD, 16 * ti, x + 16), c);
                }
                const int i = 16 * ti + i16;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * tj + 4 * g + r;
                    c[r] = j <= i && levels.part[j] == levels.part[i] ? c[r] * (a.scale * levels.between(i, j)) : 0.0f;
                }
                F f[S::INNER];
                la_split(c, f);
#pragma unroll
                for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ps + (m * C + i) * LDC + 16 * tj + 4 * g) = f[m];
            }
        }
        F vf[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) vf[t] = la_cols(vs, LD, 16 * t, 16 * wave);
        if constexpr (OUT) {
            if (a.kept) {
                float *to = a.kept + (bh * a.chunks + chunk) * features * values;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 16 * t + 4 * g + r;
                        if (row < features && col < values) to[row * values + col] = s[t][r];
                    }
            }
            LaAcc o[TT] = {};
#pragma unroll
            for (int x = 0; x < DT; x += 2) {
                F s0[S::INNER], s1[S::INNER];
                la_split(s[x], s0);
                la_split(s[x + 1], s1);
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const F q0 = la_rows<F>(qs, LD, 16 * t, 16 * x), q1 = la_rows<F>(qs, LD, 16 * t, 16 * x + 16);
#pragma unroll
                    for (int m = 0; m < S::INNER; ++m) o[t] = la_mma(q0, q1, s0[m], s1[m], o[t]);
                }
            }
            __syncthreads();
            T *out = static_cast<T *>(a.o) + ((b * a.steps + t0) * a.heads + h) * values;
            const int rows = (int)min((int64_t)C, a.steps - t0);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * t + 4 * g + r;
                    o[t][r] = levels.part[i] == 0 ? o[t][r] * (a.scale * levels.from_start(i)) : 0.0f;
                }
                la_over_steps<S::INNER, TT, F>(
                    o[t], 0, t, bad, [&](int m, int j) { return la_rows<F>(ps + m * C * LDC, LDC, 16 * t, 16 * j); },
                    [&](int j) { return la_cols(vs, LD, 16 * j, 16 * wave); },
                    [&](int r, int j) { const int i = 16 * t + 4 * g + r; return j <= i && levels.part[j] == levels.part[i]; });
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * t + 4 * g + r;
                    if (i < rows && col < values) out[(int64_t)i * a.heads * values + col] = (T)o[t][r];
                }
            }
        }
        // the state behind the chunk (BACK: its gradient in front of it)
        const int part = levels.part[C - 1];
        const float decay = levels.from_start(C - 1);
#pragma unroll
        for (int t = 0; t < DT; ++t) s[t] = part == 0 ? s[t] * decay : LaAcc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TT; t += 2) {
            F w[2][S::ADDED];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                LaAcc x = la_float(vf[t + u]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * (t + u) + 4 * g + r;
                    x[r] = levels.part[j] != (BACK ? 0 : part) ? 0.0f : x[r] * (BACK ? a.scale * levels.from_start(j) : levels.between(C - 1, j));
                }
                la_split(x, w[u]);
            }
#pragma unroll
            for (int x = 0; x < DT; ++x) {
                F k0 = la_cols(ks, LD, 16 * t, 16 * x), k1 = la_cols(ks, LD, 16 * t + 16, 16 * x);
                if (bad) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (levels.part[16 * t + 4 * g + r] != (BACK ? 0 : part)) k0[r] = 0.0f;
                        if (levels.part[16 * t + 16 + 4 * g + r] != (BACK ? 0 : part)) k1[r] = 0.0f;
                    }
                }
#pragma unroll
                for (int m = 0; m < S::ADDED; ++m) s[x] = la_mma(k0, k1, w[0][m], w[1][m], s[x]);
            }
        }
        if constexpr (!OUT) {
            total += (double)levels.hi[C - 1] + (double)levels.lo[C - 1];
            cuts |= part;
        }
        __syncthreads();
    }
    float *to = OUT ? (segment == a.segments - 1 && a.last ? a.last + bh * features * values : nullptr)
                    : a.segment_state + (segment * heads + bh) * features * values;
    if (to) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * t + 4 * g + r;
                if (row < features && col < values) to[row * values + col] = s[t][r];
            }
    }
    if (!OUT && threadIdx.x == 0) {
        a.segment_decay[segment * heads + bh] = (float)exp2(total);
        a.segment_cut[segment * heads + bh] = cuts;
    }
}

// What segments add to the state becomes the state each starts from (BACK: the gradient of the one it ends with).
template <bool BACK>
__global__ __launch_bounds__(256) void la_enter_kernel(const LaArgs a)
{
    const int64_t square = (int64_t)a.features * a.values, heads = a.batch * a.heads, count = heads * square;
    const float *from = BACK ? a.grad_last : a.state;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) {
        const int64_t bh = at / square;
        float s = from ? from[at] : 0.0f;
        for (int n = 0; n < a.segments; ++n) {
            const int64_t segment = BACK ? a.segments - 1 - n : n;
            float *p = a.segment_state + segment * count + at;
            const float added = *p, decay = a.segment_decay[segment * heads + bh];
            const bool cut = a.segment_cut[segment * heads + bh] != 0;
            *p = s;
            s = cut ? added : decay * s + added;
        }
    }
}

// (from: NULL for zeros)
__global__ __launch_bounds__(256) void la_copy_kernel(const float *from, float *to, int64_t count)
{
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) to[at] = from ? from[at] : 0.0f;
}

// The gradients, chunk by chunk from a segment's end, with the states that the forward call kept.
template <typename T, int D>
__global__ __launch_bounds__(4 * D) void la_back_kernel(const LaArgs a)
{
    using S = LaShape<T, D>;
    using F = typename LaFrag<T>::type;
    constexpr int C = S::C, W = S::W, TT = S::TT, DT = S::DT, LD = S::LD, LDC = S::LDC;
    __shared__ __align__(16) T qs[C * LD];
    __shared__ __align__(16) T ks[C * LD];
    __shared__ __align__(16) T vs[C * LD];
    __shared__ __align__(16) T gs[C * LD];
    __shared__ __align__(16) T es[S::HELD * D * LD];         // E, rows are features
    __shared__ __align__(16) T ps[S::INNER * C * LDC];       // (Q K^T . D)^T, rows are steps j
    __shared__ __align__(16) T ds[S::INNER * C * LDC];       // (dO V^T . D)^T
    __shared__ __align__(16) LaLevels<C> levels;
    __shared__ float row_sums[TT][C], col_sums[TT][C], start_sums[W][C], end_sums[W][C], through[W];
    __shared__ int bad_chunk[2];

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const int64_t heads = a.batch * a.heads, unit = la_unit(heads * a.segments);
    if (unit >= heads * a.segments) return;
    const int64_t segment = unit / heads, bh = unit % heads, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t first = segment * a.segment_chunks, end = min(first + a.segment_chunks, a.chunks);
    const int count = (int)(end - first), features = a.features, values = a.values;
    const T *q = static_cast<const T *>(a.q) + la_offset(a.q_stride, b, 0, h / a.shared);
    const T *k = static_cast<const T *>(a.k) + la_offset(a.k_stride, b, 0, h / a.shared);
    const T *v = static_cast<const T *>(a.v) + la_offset(a.v_stride, b, 0, h);
    const T *go = a.grad ? static_cast<const T *>(a.grad) + la_offset(a.grad_stride, b, 0, h) : nullptr;
    const float *decay_row = a.log_decay + la_offset(a.decay_stride, b, 0, h);
    const uint8_t *reset_row = a.reset ? a.reset + b * a.reset_stride[0] : nullptr;

    // E transposed: rows are values 16 t + 4 g + r, column: feature 16 wave + lane % 16; S likewise
    LaAcc e[DT], before[DT];
    const int col = 16 * wave + i16;
    auto fetch_square = [&](const float *from, LaAcc (&to)[DT]) {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const int row = 16 * t + 4 * g;
            if (from && col < features && row + 4 <= values) {
                const quad_at_4 x = *reinterpret_cast<const quad_at_4 *>(from + (int64_t)col * values + row);
                to[t] = LaAcc{x[0], x[1], x[2], x[3]};
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) to[t][r] = from && col < features && row + r < values ? from[(int64_t)col * values + row + r] : 0.0f;
            }
        }
    };
    fetch_square(a.segments > 1 ? a.segment_state + (segment * heads + bh) * features * values
                                : a.grad_last ? a.grad_last + bh * features * values : nullptr, e);

    LaPiece<T, D> nq, nk, nv, ng;
    LaDecay nd;
    auto fetch = [&](int n) {
        const int64_t chunk = end - 1 - n, t0 = chunk * C;
        const int rows = (int)min((int64_t)C, a.steps - t0);
        nq.fetch(q + t0 * a.q_stride[1], a.q_stride[1], rows, features);
        nk.fetch(k + t0 * a.k_stride[1], a.k_stride[1], rows, features);
        nv.fetch(v + t0 * a.v_stride[1], a.v_stride[1], rows, values);
        ng.fetch(go ? go + t0 * a.grad_stride[1] : nullptr, a.grad_stride[1], rows, values);
        if (wave == 0) nd.fetch(a, decay_row, reset_row, t0, rows);
    };
    if (threadIdx.x < 2) bad_chunk[threadIdx.x] = 0;
    fetch(0);
    __syncthreads();
    for (int n = 0; n < count; ++n) {
        const int64_t chunk = end - 1 - n, t0 = chunk * C;
        const int rows = (int)min((int64_t)C, a.steps - t0);
        uint32_t magnitude = 0;
        nq.store(qs, magnitude);
        nk.store(ks, magnitude);
        nv.store(vs, magnitude);
        ng.store(gs, magnitude);
        if (la_not_finite<T>(magnitude)) bad_chunk[n & 1] = 1;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            F f[S::HELD];
            la_split(e[t], f);
#pragma unroll
            for (int m = 0; m < S::HELD; ++m) *reinterpret_cast<F *>(es + (m * D + col) * LD + 16 * t + 4 * g) = f[m];
        }
        if (wave == 0) la_levels<C>(levels, nd.log_decay, nd.reset);
        __syncthreads();
        const bool bad = bad_chunk[n & 1] != 0;
        if (threadIdx.x == 0) bad_chunk[(n + 1) & 1] = 0;
        fetch_square(a.kept + (bh * a.chunks + chunk) * features * values, before);
        if (n + 1 < count) fetch(n + 1);

        for (int p = wave; p < S::PAIRS; p += W) {
            int ti, tj;
            la_pair<TT>(p, ti, tj);
            LaAcc c = {}, d = {}, gg = {};
            if (tj <= ti) {
#pragma unroll
                for (int x = 0; x < D; x += 32) {
                    c = la_mma(la_rows<F>(qs, LD, 16 * ti, x), la_rows<F>(qs, LD, 16 * ti, x + 16), la_rows<F>(ks, LD, 16 * tj, x),
                               la_rows<F>(ks, LD, 16 * tj, x + 16), c);
                    d = la_mma(la_rows<F>(gs, LD, 16 * ti, x), la_rows<F>(gs, LD, 16 * ti, x + 16), la_rows<F>(vs, LD, 16 * tj, x),
                               la_rows<F>(vs, LD, 16 * tj, x + 16), d);
                }
            }
            const int j = 16 * tj + i16;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * ti + 4 * g + r;
                const bool there = j <= i && levels.part[j] == levels.part[i];
                const float f = a.scale * levels.between(i, j);
                c[r] = there ? c[r] * f : 0.0f;
                gg[r] = there && j < i ? c[r] * d[r] : 0.0f;
                d[r] = there ? d[r] * f : 0.0f;
            }
            F f[S::INNER];
            la_split(c, f);
#pragma unroll
            for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ps + (m * C + j) * LDC + 16 * ti + 4 * g) = f[m];
            la_split(d, f);
#pragma unroll
            for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ds + (m * C + j) * LDC + 16 * ti + 4 * g) = f[m];
            float column = (gg[0] + gg[1]) + (gg[2] + gg[3]);
            column += __shfl_xor(column, 16, 64);
            column += __shfl_xor(column, 32, 64);
            if (g == 0) col_sums[ti][j] = column;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float sum = la_sum16(gg[r]);
                if (i16 == 0) row_sums[tj][16 * ti + 4 * g + r] = sum;
            }
        }
        __syncthreads();

        const int part = levels.part[C - 1];
        const float decay = levels.from_start(C - 1);
        auto to_end = [&](int j, float x) { return levels.part[j] == part ? x * levels.between(C - 1, j) : 0.0f; };
        auto to_start = [&](int i, float x) { return levels.part[i] == 0 ? x * (a.scale * levels.from_start(i)) : 0.0f; };
        auto meets = [&](int i, int j) { return j <= i && levels.part[j] == levels.part[i]; };
        const int64_t row0 = (b * a.steps + t0) * a.heads + h, row_step = a.heads;

        // dV: rows are steps j, columns this wavefront's values
        {
            LaAcc c[TT] = {};
#pragma unroll
            for (int x = 0; x < D; x += 32)
#pragma unroll
                for (int m = 0; m < S::HELD; ++m) {
                    const F e0 = la_cols(es + m * D * LD, LD, x, 16 * wave), e1 = la_cols(es + m * D * LD, LD, x + 16, 16 * wave);
#pragma unroll
                    for (int t = 0; t < TT; ++t) c[t] = la_mma(la_rows<F>(ks, LD, 16 * t, x), la_rows<F>(ks, LD, 16 * t, x + 16), e0, e1, c[t]);
                }
            T *out = static_cast<T *>(a.d_v) + row0 * values + col;
#pragma unroll
            for (int t = 0; t < TT; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) c[t][r] = to_end(16 * t + 4 * g + r, c[t][r]);
                la_over_steps<S::INNER, TT, F>(
                    c[t], t, TT - 1, bad, [&](int m, int i) { return la_rows<F>(ps + m * C * LDC, LDC, 16 * t, 16 * i); },
                    [&](int i) { return la_cols(gs, LD, 16 * i, 16 * wave); },
                    [&](int r, int i) { return meets(i, 16 * t + 4 * g + r); });
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * t + 4 * g + r;
                    if (j < rows && col < values) out[j * row_step * values] = (T)c[t][r];
                }
            }
        }
        F qf[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) qf[t] = la_cols(qs, LD, 16 * t, 16 * wave);
        auto store = [&](void *to, int step, float x) {
            if (step >= rows || col >= features) return;
            const int64_t at = (row0 + step * row_step) * features + col;
            if (a.wide) static_cast<float *>(to)[at] = x;
            else static_cast<T *>(to)[at] = (T)x;
        };
        // dK: rows are steps j, columns this wavefront's features
        {
            F kf[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) kf[t] = la_cols(ks, LD, 16 * t, 16 * wave);
            LaAcc c[TT] = {}, d[TT] = {};
#pragma unroll
            for (int x = 0; x < DT; x += 2) {
                F e0[S::INNER], e1[S::INNER], s0[S::INNER], s1[S::INNER];
                la_split(e[x], e0);
                la_split(e[x + 1], e1);
                la_split(before[x], s0);
                la_split(before[x + 1], s1);
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const F v0 = la_rows<F>(vs, LD, 16 * t, 16 * x), v1 = la_rows<F>(vs, LD, 16 * t, 16 * x + 16);
                    const F g0 = la_rows<F>(gs, LD, 16 * t, 16 * x), g1 = la_rows<F>(gs, LD, 16 * t, 16 * x + 16);
#pragma unroll
                    for (int m = 0; m < S::INNER; ++m) {
                        c[t] = la_mma(v0, v1, e0[m], e1[m], c[t]);
                        d[t] = la_mma(g0, g1, s0[m], s1[m], d[t]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const LaAcc kx = la_float(kf[t]), qx = la_float(qf[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * t + 4 * g + r;
                    c[t][r] = to_end(j, c[t][r]);
                    d[t][r] = to_start(j, d[t][r]);
                    const float at_end = la_sum16(levels.part[j] == part ? c[t][r] * kx[r] : 0.0f);
                    const float at_start = la_sum16(levels.part[j] == 0 ? d[t][r] * qx[r] : 0.0f);
                    if (i16 == 0) end_sums[wave][j] = at_end;
                    if (i16 == 1) start_sums[wave][j] = at_start;
                }
                la_over_steps<S::INNER, TT, F>(
                    c[t], t, TT - 1, bad, [&](int m, int i) { return la_rows<F>(ds + m * C * LDC, LDC, 16 * t, 16 * i); },
                    [&](int i) { return la_cols(qs, LD, 16 * i, 16 * wave); },
                    [&](int r, int i) { return meets(i, 16 * t + 4 * g + r); });
                // dQ: rows are steps i
                la_over_steps<S::INNER, TT, F>(
                    d[t], 0, t, bad, [&](int m, int j) { return la_cols(ds + m * C * LDC, LDC, 16 * j, 16 * t); },
                    [&](int j) { return la_cols(ks, LD, 16 * j, 16 * wave); },
                    [&](int r, int j) { return meets(16 * t + 4 * g + r, j); });
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    store(a.d_k, 16 * t + 4 * g + r, c[t][r]);
                    store(a.d_q, 16 * t + 4 * g + r, d[t][r]);
                }
            }
        }
        // <E, S>, and E in front of the chunk
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += e[t][r] * before[t][r];
            e[t] = part == 0 ? e[t] * decay : LaAcc{0.f, 0.f, 0.f, 0.f};
        }
        sum = la_sum16(sum);
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lane == 0) through[wave] = sum;
#pragma unroll
        for (int t = 0; t < TT; t += 2) {
            F w[2][S::ADDED];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                LaAcc x = la_float(qf[t + u]);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = to_start(16 * (t + u) + 4 * g + r, x[r]);
                la_split(x, w[u]);
            }
#pragma unroll
            for (int x = 0; x < DT; ++x) {
                F g0 = la_cols(gs, LD, 16 * t, 16 * x), g1 = la_cols(gs, LD, 16 * t + 16, 16 * x);
                if (bad) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (levels.part[16 * t + 4 * g + r] != 0) g0[r] = 0.0f;
                        if (levels.part[16 * t + 16 + 4 * g + r] != 0) g1[r] = 0.0f;
                    }
                }
#pragma unroll
                for (int m = 0; m < S::ADDED; ++m) e[x] = la_mma(g0, g1, w[0][m], w[1][m], e[x]);
            }
        }
        __syncthreads();
        if (wave == 0) {
            // one step a lane: sums over the later steps of its document, sums over the earlier ones
            const int t = min(lane, C - 1);
            float later = 0.0f, earlier = 0.0f;
            for (int x = 0; x <= ((t >> 4) | 1); ++x) later += row_sums[x][t];
            for (int x = (t >> 4) & ~1; x < TT; ++x) later -= col_sums[x][t];
            for (int x = 0; x < W; ++x) {
                later += start_sums[x][t];
                earlier += end_sums[x][t];
            }
            const int mine = levels.part[t];
            float crossing = 0.0f;
            if (part == 0)
                for (int x = 0; x < W; ++x) crossing += decay * through[x];
#pragma unroll
            for (int d = 1; d < C; d *= 2) {
                const float down = __shfl_down(later, d, 64), up = __shfl_up(earlier, d, 64);
                const int part_down = __shfl_down(mine, d, 64), part_up = __shfl_up(mine, d, 64);
                if (lane + d < C && part_down == mine) later += down;
                if (lane >= d && part_up == mine) earlier += up;
            }
            float before_t = __shfl_up(earlier, 1, 64);
            const int part_before = __shfl_up(mine, 1, 64);
            if (lane == 0 || part_before != mine) before_t = 0.0f;
            // (the decay of a reset step meets nothing)
            const bool starts = mine != (lane == 0 ? 0 : part_before);
            if (lane < rows) a.d_log_decay[row0 + lane * row_step] = starts ? 0.0f : later + before_t + crossing;
        }
    }
    if (segment == 0 && a.d_state) {
        float *to = a.d_state + bh * features * values;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * t + 4 * g + r;
                if (col < features && row < values) to[(int64_t)col * values + row] = e[t][r];
            }
    }
}

// Gradients of queries or keys that heads share: the sum over those heads, in order.
template <typename T>
__global__ __launch_bounds__(256) void la_shared_kernel(const float *from, T *to, int64_t rows, int groups, int shared, int features)
{
    const int64_t count = rows * groups * features;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / features;
        const float *p = from + row * shared * features + at % features;
        float sum = p[0];
        for (int n = 1; n < shared; ++n) sum += p[(int64_t)n * features];
        to[at] = (T)sum;
    }
}

// One step of every head: the state is read and written once, which is all that this costs.  LANES lanes take V neighbouring
// values of a feature's row each, the others of 256 its further features; 64 x 16 heads of 64 x 64: 33.5 MB.
template <typename T, int V>
__global__ __launch_bounds__(256) void la_step_kernel(const LaArgs a, float *state, T *o, int lanes_log)
{
    __shared__ float sums[256 * V];
    const int64_t bh = blockIdx.x, b = bh / a.heads;
    const int h = (int)(bh % a.heads), features = a.features, values = a.values;
    const T *q = static_cast<const T *>(a.q) + la_offset(a.q_stride, b, 0, h / a.shared);
    const T *k = static_cast<const T *>(a.k) + la_offset(a.k_stride, b, 0, h / a.shared);
    const T *v = static_cast<const T *>(a.v) + la_offset(a.v_stride, b, 0, h);
    const float decay = expf(a.log_decay[la_offset(a.decay_stride, b, 0, h)]);
    const int lanes = 1 << lanes_log, lane = threadIdx.x & (lanes - 1), first = threadIdx.x >> lanes_log, every = 256 >> lanes_log;
    const int col = lane * V;
    float *s = state + bh * features * values + col;
    float vx[V], sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        vx[i] = col + i < values ? to_float(v[col + i]) : 0.0f;
        sum[i] = 0.0f;
    }
    if (col < values) {
#pragma unroll 4
        for (int d = first; d < features; d += every) {
            using Vec = float __attribute__((ext_vector_type(V)));
            Vec *p = reinterpret_cast<Vec *>(s + (int64_t)d * values);
            Vec x = *p;
            const float kx = to_float(k[d]), qx = to_float(q[d]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[i] = decay * x[i] + kx * vx[i];
                sum[i] += qx * x[i];
            }
            *p = x;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sums[threadIdx.x * V + i] = sum[i];
    __syncthreads();
    for (int at = threadIdx.x; at < values; at += 256) {
        float total = 0.0f;
        for (int n = 0; n < every; ++n) total += sums[((n << lanes_log) + at / V) * V + at % V];
        o[bh * values + at] = (T)(a.scale * total);
    }
}

}  // namespace bf
