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
// 8 bits; one number would leave errors of the size of that rounding).  The decays' gradients are floats: what they are summed
// from, b dO S^T and w V E^T, takes S and E as three numbers as well (two: 4% off the backward kernels' time, and decays'
// gradients off by 2e-6 instead of 3e-7).  An operand of a product over 32 steps or features is two
// pieces of 4 elements in a lane (LaPair); a state that is taken from sums keeps their order, 4 g .. 4 g + 3 (g: lane / 16)
// of two neighbouring tiles, and so does what it meets, so that sums become operands without leaving their lane.
//
// Measured, one workgroup a compute unit, 64 x 64 states and 128 x 128 ones:
//   16 x 2048 steps, 16 heads, bfloat16       forward 116 us                          backward 244
//    8 x 1001 steps, 16 heads, float          forward 26 + 6 + 56                     backward 26 + 5 + 110
//    1 x 65537 steps, 10 heads of 100         forward 132 + 7 + 350                   backward 134 + 8 + 656
// (sums of a segment, states between segments, outputs).  The first one moves 403 MB forward, 3.5 TB/s, and 604 MB backward, 2.5: it
// is bound by the chunk's own chain of products (LDS moves data for 37% of the cycles both ways, the vector unit issues for 50%
// and 57%, the matrix unit for 12% and 13%; three or four barriers a chunk between them), with two wavefronts a SIMD to hide each
// other.  The backward kernel of 128-wide bfloat16 heads has 38 registers and 156 bytes a lane in scratch memory.
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
typedef int LaParts __attribute__((ext_vector_type(4)));
typedef bf16 LaHalf4 __attribute__((ext_vector_type(4)));
typedef bf16 LaHalf8 __attribute__((ext_vector_type(8)));

template <typename T> struct LaFrag;
template <> struct LaFrag<bf16> { using type = LaHalf4; };
template <> struct LaFrag<float> { using type = LaAcc; };

// Chunks of 64 steps; float rows of 128 features: 32, four operands and the state's gradient are all that LDS holds.
template <typename T, int D>
struct LaShape {
    static constexpr int C = sizeof(T) == 4 && D == 128 ? 32 : 64;
    static constexpr int SLICES = D / 16;            // of 16 columns of a state or a result
    // wavefronts of a slice: two of 64 columns share the steps and the rows of the state (two wavefronts on each SIMD), the
    // state's operands then go through LDS.  Those of 128 columns stay in the sums: the backward kernel has no room for them (152 of
    // 160 KB without), the forward one of bfloat16 would (74 and 70)
    static constexpr int HALVES = D == 64 ? 2 : 1;
    static constexpr int W = SLICES * HALVES, THREADS = 64 * W;
    static constexpr int TT = C / 16, DT = D / 16;   // tiles of a chunk, of a state
    static constexpr int OWN_T = TT / HALVES, OWN_D = DT / HALVES;
    static constexpr int E = 16 / sizeof(T);         // elements of a load
    static constexpr int LD = D + E, LDC = C + E;    // rows in LDS: 16 bytes more, so that sixteen of them start in different banks
    static constexpr int LOADS = C * D / E / THREADS;
    // pairs of tiles (i, j) with j <= i, and those above the diagonal that a product of 32 steps reads
    static constexpr int PAIRS = TT == 4 ? 12 : 4, EACH = (PAIRS + W - 1) / W;
    static constexpr int INNER = sizeof(T) == 4 ? 1 : 2;   // numbers that an inner factor or a state is split into
    static constexpr int ADDED = sizeof(T) == 4 ? 1 : 3;   // and what is added to a state

    // A wavefront's tiles of steps: all, or the first and last or the two in between, which meet equally many others.
    static __device__ __forceinline__ int tile(int half, int u) { return HALVES == 1 ? u : u == 0 ? half : 3 - half; }
    // The pair of tiles that holds it: pairs of earlier steps are those up to it, of later ones those from it on.
    static constexpr int pair_of(int u) { return HALVES == 1 ? u / 2 : u; }
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

template <typename P>
__device__ __forceinline__ LaAcc la_mma(P a, P b, LaAcc c) { return la_mma(a.a, a.b, b.a, b.b, c); }

// The lane's number, of TIGHT kernels as something that the compiler knows nothing of: what is computed from it is computed where
// it is needed.  (Left to itself it forms every address of a chunk in front of the loop and keeps them all, in scratch memory
// where registers end.)
template <bool TIGHT>
__device__ __forceinline__ int la_lane()
{
    int lane = threadIdx.x & 63;
    if constexpr (TIGHT) asm volatile("" : "+v"(lane));
    return lane;
}

// Element s is [row0 + lane % 16][col0 + 4 g + s]: the sum runs over neighbours in memory.
template <typename F, typename T>
__device__ __forceinline__ F la_rows(int lane, const T *lds, int stride, int row0, int col0)
{
    return *reinterpret_cast<const F *>(lds + (row0 + (lane & 15)) * stride + col0 + 4 * (lane >> 4));
}
// Element s is [row0 + 4 g + s][col0 + lane % 16]: the sum runs over rows.
__device__ __forceinline__ LaHalf4 la_cols(int lane, const bf16 *lds, int stride, int row0, int col0)
{
    typedef short Quad16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) Quad16 LdsQuad;
    const int i = lane & 15;
    // (16 lanes hand in 4 rows of 16 columns and get them by columns)
    const bf16 *p = lds + (row0 + 4 * (lane >> 4) + (i >> 2)) * stride + col0 + 4 * (i & 3);
    return __builtin_bit_cast(LaHalf4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad *)p));
}
__device__ __forceinline__ LaAcc la_cols(int lane, const float *lds, int stride, int row0, int col0)
{
    const float *p = lds + (row0 + 4 * (lane >> 4)) * stride + col0 + (lane & 15);
    return LaAcc{p[0], p[stride], p[2 * stride], p[3 * stride]};
}

// An operand of 32 steps or features, in two pieces.  bfloat16: eight neighbours 8 g .. 8 g + 7 in a lane, so that rows are read 16
// bytes at a time (LDS moves 128 bytes a cycle then, 64 in pieces of 8, and was busy for two thirds of the time); float: 4 g ..
// 4 g + 3 of both halves, whose rows start in different banks.
template <typename F>
struct LaPair {
    F a, b;
};
template <typename T>
constexpr int la_first(int g) { return sizeof(T) == 2 ? 8 * g : 4 * g; }            // where a lane's first piece starts
template <typename T>
constexpr int la_second(int g) { return sizeof(T) == 2 ? 8 * g + 4 : 16 + 4 * g; }  // and its second

__device__ __forceinline__ LaPair<LaHalf4> la_rows2(int lane, const bf16 *lds, int stride, int row0, int col0)
{
    const LaHalf8 v = *reinterpret_cast<const LaHalf8 *>(lds + (row0 + (lane & 15)) * stride + col0 + 8 * (lane >> 4));
    return {__builtin_shufflevector(v, v, 0, 1, 2, 3), __builtin_shufflevector(v, v, 4, 5, 6, 7)};
}
__device__ __forceinline__ LaPair<LaAcc> la_rows2(int lane, const float *lds, int stride, int row0, int col0)
{
    return {la_rows<LaAcc>(lane, lds, stride, row0, col0), la_rows<LaAcc>(lane, lds, stride, row0, col0 + 16)};
}
__device__ __forceinline__ LaPair<LaHalf4> la_cols2(int lane, const bf16 *lds, int stride, int row0, int col0)
{
    // (rows 8 g instead of 4 g)
    const int more = row0 + 4 * (lane >> 4);
    return {la_cols(lane, lds, stride, more, col0), la_cols(lane, lds, stride, more + 4, col0)};
}
__device__ __forceinline__ LaPair<LaAcc> la_cols2(int lane, const float *lds, int stride, int row0, int col0)
{
    return {la_cols(lane, lds, stride, row0, col0), la_cols(lane, lds, stride, row0 + 16, col0)};
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

// The steps of a chunk that a lane brings into LDS, on their way in registers: 16 bytes of a row each, always the same columns.
// Nothing depends on what is loaded until it is stored, and nothing branches: rows behind the last step read that one, columns
// behind a row's end its first ones, and the 16 bytes that a row's end cuts are read as the row's last 16 and moved down.
// What does not exist is zero in LDS.
template <typename T, int D>
struct LaPiece {
    using S = LaShape<T, D>;
    using Quad = std::conditional_t<sizeof(T) == 4, quad_at_4, quad_at_2>;
    static constexpr int ROWS = S::THREADS / (D / S::E);   // between a lane's rows
    Quad v[S::LOADS];
    const T *base;
    int64_t stride, offset;   // offset: of the lane's first 16 bytes from a chunk's first row
    int cols, col, row, from; // col: where the 16 bytes go; from: and come from
    int shift;                // bits that they move down

    __device__ __forceinline__ void init(const T *start, int64_t step, int columns)
    {
        base = start;
        stride = step;
        cols = columns;
        col = (int)threadIdx.x % (D / S::E) * S::E;
        row = (int)threadIdx.x / (D / S::E);
        const bool cut = col < cols && col + S::E > cols && cols >= S::E;
        from = col >= cols ? 0 : cut ? cols - S::E : col;
        shift = cut ? (col - from) * 8 * (int)sizeof(T) : 0;
        offset = row * stride + from;
    }
    // whole chunks of rows of at least 16 bytes
    __device__ __forceinline__ void fetch_whole(int64_t t0)
    {
        const T *start = base + t0 * stride;
#pragma unroll
        for (int n = 0; n < S::LOADS; ++n) v[n] = *reinterpret_cast<const Quad *>(start + n * ROWS * stride + offset);
    }
    __device__ __forceinline__ void fetch_any(int64_t t0, int rows)
    {
        const T *start = base + t0 * stride;
#pragma unroll
        for (int n = 0; n < S::LOADS; ++n) {
            const T *at = start + min(row + n * ROWS, rows - 1) * stride;
            if (cols >= S::E) {
                v[n] = *reinterpret_cast<const Quad *>(at + from);
            } else {
                // (narrower than 16 bytes: one by one)
                T x[S::E];
#pragma unroll
                for (int i = 0; i < S::E; ++i) x[i] = i < cols ? at[i] : (T)0.0f;
                v[n] = __builtin_bit_cast(Quad, x);
            }
        }
    }
    // magnitude: of what is stored, see la_magnitude
    template <bool EVEN>
    __device__ __forceinline__ void store(T *lds, int rows, uint32_t &magnitude) const
    {
#pragma unroll
        for (int n = 0; n < S::LOADS; ++n) {
            uint4 x = __builtin_bit_cast(uint4, v[n]);
            if constexpr (!EVEN) {
                uint64_t low = (uint64_t)x.y << 32 | x.x, high = (uint64_t)x.w << 32 | x.z;
                low = shift >= 64 ? high >> (shift - 64) : low >> shift | (high << 1) << (63 - shift);
                high = shift >= 64 ? 0 : high >> shift;
                x = make_uint4((uint32_t)low, (uint32_t)(low >> 32), (uint32_t)high, (uint32_t)(high >> 32));
            }
            const bool there = (row + n * ROWS < rows) & (col < cols);
            x.x = there ? x.x : 0;
            x.y = there ? x.y : 0;
            x.z = there ? x.z : 0;
            x.w = there ? x.w : 0;
            *reinterpret_cast<uint4 *>(lds + (row + n * ROWS) * S::LD + col) = x;
            la_magnitude<T>(x, magnitude);
        }
    }
};

// What the products take from a chunk's decays.  Sums of log decays, to the base 2, as two floats of together 48 bits: their
// differences keep the bits of the decays between two steps, whatever the steps in front have summed up to.  part: resets
// so far.  start, end: what steps meet of the states in front of and behind the chunk (scale exp(L_i), exp(L_C - L_j)),
// kNothing where a reset lies between.  group: decays so far that are infinite (less than 256), and 256 times those that are NaN.  They
// are left out of the sums, which start behind them as behind a reset, so that steps on one side keep their factors, and
// steps that are parted by one get it.
constexpr float kNothing = -0.0f;
__device__ __forceinline__ bool la_nothing(float factor) { return __builtin_bit_cast(int, factor) == INT32_MIN; }

// The factor f between steps of two groups.
__device__ __forceinline__ float la_crossed(float f, int one, int other)
{
    return one == other ? f : (one ^ other) >> 8 ? NAN : INFINITY;
}

// (a multiple of 16 bytes: several lie one behind the other, and four neighbouring steps are read at once)
template <int C>
struct __align__(16) LaLevels {
    float hi[C], lo[C], start[C], end[C];
    int part[C], group[C];
    float decay;   // over the whole chunk; kNothing: a reset lies within
    bool broken;   // not all groups are 0

    __device__ __forceinline__ LaAcc quad(const float (&v)[C], int at) const { return *reinterpret_cast<const LaAcc *>(v + at); }
    // scale exp(L_i - L_j) for four neighbouring steps i or j and one other one
    __device__ __forceinline__ LaAcc between(LaAcc hi0, LaAcc lo0, float hi1, float lo1, float sign) const
    {
        LaAcc f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = __builtin_amdgcn_exp2f(sign * ((hi0[r] - hi1) + (lo0[r] - lo1)));
        return f;
    }
    // the same of a broken chunk
    __device__ __forceinline__ LaAcc crossed(LaAcc f, int at, int other) const
    {
        const LaParts groups = *reinterpret_cast<const LaParts *>(group + at);
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = la_crossed(f[r], groups[r], other);
        return f;
    }
};

static_assert(sizeof(LaLevels<32>) % 16 == 0 && sizeof(LaLevels<64>) % 16 == 0);

// (kNothing: zero, whatever x is)
__device__ __forceinline__ LaAcc la_times(LaAcc x, LaAcc factor)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = la_nothing(factor[r]) ? 0.0f : x[r] * factor[r];
    return x;
}
__device__ __forceinline__ LaAcc la_times(LaAcc x, float factor) { return la_times(x, LaAcc{factor, factor, factor, factor}); }

// Lanes' values moved up: by 1, 2, 4, 8 within rows of 16, then the last of a row to the next one, the last of two rows to the
// next two.  Lanes that get nothing keep `none`.
template <int STEP>
__device__ __forceinline__ int la_up(int none, int v)
{
    constexpr int ctrl = STEP < 16 ? 0x110 + STEP : STEP == 16 ? 0x142 : 0x143;
    return __builtin_amdgcn_update_dpp(none, v, ctrl, STEP == 16 ? 0xa : STEP == 32 ? 0xc : 0xf, 0xf, false);
}
template <int STEP>
__device__ __forceinline__ float la_up(float none, float v)
{
    return __builtin_bit_cast(float, la_up<STEP>(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v)));
}
template <int STEP>
__device__ __forceinline__ double la_up(double none, double v)
{
    typedef int Two __attribute__((ext_vector_type(2)));
    const Two n = __builtin_bit_cast(Two, none), x = __builtin_bit_cast(Two, v);
    return __builtin_bit_cast(double, Two{la_up<STEP>(n[0], x[0]), la_up<STEP>(n[1], x[1])});
}

// One round of a sum over the lanes up to this one that lie in its part (parts grow with the lanes; -1: no lane).
template <int STEP, typename V>
__device__ __forceinline__ void la_scan_round(V &sum, int part)
{
    const V before = la_up<STEP>((V)0, sum);
    if (la_up<STEP>(-1, part) == part) sum += before;
}
template <typename V>
__device__ __forceinline__ void la_scan(V &sum, int part)
{
    la_scan_round<1>(sum, part);
    la_scan_round<2>(sum, part);
    la_scan_round<4>(sum, part);
    la_scan_round<8>(sum, part);
    la_scan_round<16>(sum, part);
    la_scan_round<32>(sum, part);
}

template <typename V>
__device__ __forceinline__ void la_scan(V &sum)
{
    sum += la_up<1>((V)0, sum);
    sum += la_up<2>((V)0, sum);
    sum += la_up<4>((V)0, sum);
    sum += la_up<8>((V)0, sum);
    sum += la_up<16>((V)0, sum);
    sum += la_up<32>((V)0, sum);
}

// One step a lane.  A decay below 2^-160 is zero beside anything in 32 bits and counts as that, one of 2^128 or more as infinite.
template <int C>
__device__ __forceinline__ void la_levels(LaLevels<C> &out, float log_decay, bool reset, float scale)
{
    const int lane = threadIdx.x & 63;
    const double x = (double)log_decay * 1.4426950408889634;
    const bool infinite = !reset && x >= 128.0, nan = !reset && x != x;
    double level = reset | infinite | nan ? 0.0 : x < -160.0 ? -160.0 : x;
    const uint64_t resets = __ballot(reset), infinities = __ballot(infinite), nans = __ballot(nan), below = ((uint64_t)2 << lane) - 1;
    const int part = __popcll(resets & below), parts = __popcll(resets);
    const bool broken = (infinities | nans) != 0;
    int group = 0, groups = 0;
    if (broken) {
        group = __popcll(infinities & below) + 256 * __popcll(nans & below);
        groups = __popcll(infinities) + 256 * __popcll(nans);
    }
    if ((resets | infinities | nans) == 0) la_scan(level);
    else la_scan(level, part + __popcll((infinities | nans) & below));
    const float hi = (float)level, from_start = __builtin_amdgcn_exp2f(hi);
    const double last = __shfl(level, C - 1, 64);
    const float to_end = __builtin_amdgcn_exp2f((float)(last - level));
    if (lane < C) {
        out.hi[lane] = hi;
        out.lo[lane] = (float)(level - (double)hi);
        out.start[lane] = part == 0 ? scale * la_crossed(from_start, group, 0) : kNothing;
        out.end[lane] = part == parts ? la_crossed(to_end, group, groups) : kNothing;
        out.part[lane] = part;
        out.group[lane] = group;
        if (lane == C - 1) {
            out.decay = part == 0 ? la_crossed(from_start, group, 0) : kNothing;
            out.broken = broken;
        }
    }
}

// A chunk's decays and resets, one step a lane, on their way in registers.
template <int C>
struct LaDecay {
    const float *log_decay;
    const uint8_t *reset;
    int64_t stride, reset_stride;
    float x;
    uint8_t flag = 0;
    bool inside, resets;

    __device__ __forceinline__ void init(const LaArgs &a, int64_t b, int h)
    {
        log_decay = a.log_decay + b * a.decay_stride[0] + h * a.decay_stride[2];
        stride = a.decay_stride[1];
        resets = a.reset != nullptr;
        reset = resets ? a.reset + b * a.reset_stride[0] : nullptr;
        reset_stride = a.reset_stride[1];
    }
    __device__ __forceinline__ void fetch(int64_t t0, int rows)
    {
        const int lane = threadIdx.x & 63, at = min(lane, rows - 1);
        x = log_decay[(t0 + at) * stride];
        if (resets) flag = reset[(t0 + at) * reset_stride];
        inside = lane < rows && lane < C;
    }
    __device__ __forceinline__ void levels(LaLevels<C> &out, float scale) const
    {
        la_levels<C>(out, inside ? x : 0.0f, inside && resets && flag != 0, scale);
    }
};

// Values of a row of the kept states: whole quads (those behind the last value are zero)
__host__ __device__ __forceinline__ int la_line(int values) { return (values + 3) / 4 * 4; }

// (ti, tj) of pair n: those with j <= i of two rows of tiles, then of the next two, out of a number for each (two bits a pair)
__device__ __forceinline__ void la_pair(int n, int &ti, int &tj)
{
    ti = 0xffaa50 >> 2 * n & 3;
    tj = 0xe4e444 >> 2 * n & 3;
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

// Sum over the steps of the pairs of tiles first .. last of a2(part, pair) x b2(pair), onto c (rows: steps of the chunk).
// BAD: something in the chunk, or one of its decays, is not finite.  Then step by step (a, b: of a tile), and only onto the rows that `meets(row, step)`: what a factor of
// zero stands for must not turn into NaN.
template <bool BAD, int N, int TT, typename F, typename A2, typename B2, typename A, typename B, typename M>
__device__ __forceinline__ void la_over_steps(LaAcc &c, int first, int last, A2 &&a2, B2 &&b2, A &&a, B &&b, M &&meets)
{
    if constexpr (!BAD) {
#pragma unroll
        for (int p = 0; p < TT / 2; ++p)
            if (p >= first && p <= last) {
#pragma unroll
                for (int n = 0; n < N; ++n) c = la_mma(a2(n, p), b2(p), c);
            }
    } else {
        const F zero = {};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
        for (int t = 32 * first; t < 32 * last + 32; ++t) {
            const int lane = la_lane<true>();
            LaAcc d = {};
#pragma unroll 1
            for (int n = 0; n < N; ++n) d = la_mma(la_only(a(lane, n, t >> 4), t), zero, la_only(b(lane, t >> 4), t), zero, d);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (meets(r, t)) c[r] += d[r];
        }
    }
}

// A chunk's rows of a dense result: 16-bit or 32-bit stores of a tile, whose range check drops rows behind the last step and
// columns behind the last one, so that nothing branches.  Each tile has a descriptor of its own (scalars), for one descriptor the
// lanes' offsets of all tiles would be kept in registers from chunk to chunk.  (What the check is to see is in the lane's
// register.)
template <typename T>
struct LaOut {
    T *row0;
    int rows;
    unsigned at, row_bytes;

    __device__ __forceinline__ LaOut(T *to, int count, int row_elements, int g, int col, int cols)
    {
        row0 = to;
        rows = count;
        row_bytes = (unsigned)(row_elements * (int)sizeof(T));
        at = col < cols ? 4 * g * row_bytes + col * (unsigned)sizeof(T) : 0x80000000u;
    }
    __device__ __forceinline__ void store(int tile, LaAcc x) const
    {
        char *base = reinterpret_cast<char *>(row0) + (int64_t)(16 * tile) * row_bytes;
        const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(base, 0, max(rows - 16 * tile, 0) * (int)row_bytes, 0x00020000);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float y = x[r];
            const int offset = (int)(at + r * row_bytes);
            if constexpr (sizeof(T) == 4) {
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, y), to, offset, 0, 0);
            } else {
                const bf16 z = (bf16)y;
                __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, z), to, offset, 0, 0);
            }
        }
    }
};

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

// A head's walk over its chunks: the next chunk's rows are on their way while this one's products run, so that a chunk's 24 KiB
// (64 x 64 bfloat16) cost no time of their own.  OUT: outputs, and the states in front of the chunks where they are kept; otherwise
// what a segment adds to the state: of k^T w v forward, of q^T b grad with BACK (from the end).
template <typename T, int D, bool OUT, bool BACK>
__global__ __launch_bounds__((LaShape<T, D>::THREADS)) void la_walk_kernel(const LaArgs a)
{
    using S = LaShape<T, D>;
    using F = typename LaFrag<T>::type;
    constexpr int C = S::C, W = S::W, TT = S::TT, DT = S::DT, OT = S::OWN_T, OD = S::OWN_D, LD = S::LD, LDC = S::LDC;
    constexpr bool SHARED = OUT && S::HALVES > 1;   // the state's operands in LDS
    __shared__ __align__(16) T ks[C * LD];
    __shared__ __align__(16) T vs[C * LD];
    __shared__ __align__(16) T qs[OUT ? C * LD : 16];
    __shared__ __align__(16) T ps[OUT ? S::INNER * C * LDC : 16];
    __shared__ __align__(16) T ss[SHARED ? S::INNER * D * LD : 16];   // S, rows are values
    __shared__ __align__(16) LaLevels<C> both_levels[2];
    __shared__ int bad_chunk[2];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const int slice = wave % S::SLICES, half = wave / S::SLICES;
    const int64_t heads = a.batch * a.heads, unit = la_unit(heads * a.segments);
    if (unit >= heads * a.segments) return;
    const int64_t segment = unit / heads, bh = unit % heads, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t first = segment * a.segment_chunks, end = min(first + a.segment_chunks, a.chunks);
    const int count = (int)(end - first), features = a.features, values = a.values;
    const bool nothing = BACK && !a.grad;   // (no gradient of o: zeros, whatever is read)

    // rows: features 16 (half OD + t) + 4 g + r, column: value 16 slice + lane % 16
    LaAcc s[OD];
    const int col = 16 * slice + i16, row0 = 16 * half * OD + 4 * g;
    const float *start = !OUT ? nullptr : a.segments > 1 ? a.segment_state + (segment * heads + bh) * features * values
                                       : a.state ? a.state + bh * features * values : nullptr;
#pragma unroll
    for (int t = 0; t < OD; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + 16 * t + r;
            s[t][r] = start && row < features && col < values ? start[row * values + col] : 0.0f;
        }

    LaPiece<T, D> nk, nv, nq;
    if constexpr (BACK) {
        nk.init(static_cast<const T *>(a.q) + la_offset(a.q_stride, b, 0, h / a.shared), a.q_stride[1], features);
        nv.init(static_cast<const T *>(nothing ? a.v : a.grad) + la_offset(nothing ? a.v_stride : a.grad_stride, b, 0, h),
                nothing ? a.v_stride[1] : a.grad_stride[1], values);
    } else {
        nk.init(static_cast<const T *>(a.k) + la_offset(a.k_stride, b, 0, h / a.shared), a.k_stride[1], features);
        nv.init(static_cast<const T *>(a.v) + la_offset(a.v_stride, b, 0, h), a.v_stride[1], values);
    }
    if constexpr (OUT) nq.init(static_cast<const T *>(a.q) + la_offset(a.q_stride, b, 0, h / a.shared), a.q_stride[1], features);
    LaDecay<C> nd;
    nd.init(a, b, h);
    auto chunk_of = [&](int n) { return BACK ? end - 1 - n : first + n; };
    auto rows_of = [&](int n) { return (int)min((int64_t)C, a.steps - chunk_of(n) * C); };
    const bool wide = features >= S::E && values >= S::E, even = features % S::E == 0 && values % S::E == 0;
    auto fetch = [&](int n) {
        const int64_t t0 = chunk_of(n) * C;
        const int rows = rows_of(n);
        if (__builtin_expect(wide && rows == C, 1)) {
            nk.fetch_whole(t0);
            nv.fetch_whole(t0);
            if constexpr (OUT) nq.fetch_whole(t0);
        } else {
            nk.fetch_any(t0, rows);
            nv.fetch_any(t0, rows);
            if constexpr (OUT) nq.fetch_any(t0, rows);
        }
    };
    if (threadIdx.x < 2) bad_chunk[threadIdx.x] = 0;
    // The decays are fetched two chunks ahead, in front of the next chunk's rows: once those have arrived, they have, too.
    auto fetch_decays = [&](int n) { nd.fetch(chunk_of(min(n, count - 1)) * C, rows_of(min(n, count - 1))); };
    if (wave == W - 1) {
        fetch_decays(0);
        nd.levels(both_levels[0], a.scale);
        fetch_decays(1);
    }
    fetch(0);
    __syncthreads();
    double total = 0.0;
    int cuts = 0;
    for (int n = 0; n < count; ++n) {
        const int lane = la_lane<(D > 64)>(), i16 = lane & 15, g = lane >> 4, col = 16 * slice + i16;
        const int64_t chunk = chunk_of(n), t0 = chunk * C;
        const int rows = rows_of(n);
        const LaLevels<C> &levels = both_levels[n & 1];
        uint32_t magnitude = 0;
        auto store = [&](auto even_type) {
            constexpr bool EVEN = decltype(even_type)::value;
            nk.template store<EVEN>(ks, rows, magnitude);
            nv.template store<EVEN>(vs, nothing ? 0 : rows, magnitude);
            if constexpr (OUT) nq.template store<EVEN>(qs, rows, magnitude);
        };
        if (__builtin_expect(even, 1)) store(std::true_type());
        else store(std::false_type());
        if constexpr (SHARED) {
#pragma unroll
            for (int t = 0; t < OD; ++t) {
                F f[S::INNER];
                la_split(s[t], f);
#pragma unroll
                for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ss + (m * D + col) * LD + 16 * half * OD + 4 * g + 16 * t) = f[m];
            }
        }
        if (la_not_finite<T>(magnitude)) bad_chunk[n & 1] = 1;
        __syncthreads();
        const bool bad = (bad_chunk[n & 1] != 0) | levels.broken;
        if (threadIdx.x == 0) bad_chunk[(n + 1) & 1] = 0;
        if (wave == W - 1) {
            if (n + 1 < count) nd.levels(both_levels[(n + 1) & 1], a.scale);
            fetch_decays(n + 2);
        }
        // (behind the last chunk: that one once more)
        fetch(min(n + 1, count - 1));

        auto products = [&](auto bad_type) {
            constexpr bool BAD = decltype(bad_type)::value;
            if constexpr (OUT) {
                // Q K^T . D, transposed in the sums: rows are steps j
#pragma unroll
                for (int u = 0; u < S::EACH; ++u) {
                    const int p = wave + u * W;
                    if (S::PAIRS % W != 0 && p >= S::PAIRS) break;
                    int ti, tj;
                    la_pair(p, ti, tj);
                    LaAcc c = {};
#pragma unroll
                    for (int x = 0; x < D; x += 32)
                        c = la_mma(la_rows2(lane, ks, LD, 16 * tj, x), la_rows2(lane, qs, LD, 16 * ti, x), c);
                    const int i = 16 * ti + i16, j = 16 * tj + 4 * g, part = levels.part[i];
                    LaAcc f_ij = levels.between(levels.quad(levels.hi, j), levels.quad(levels.lo, j), levels.hi[i], levels.lo[i], -1.0f);
                    if constexpr (BAD) f_ij = levels.crossed(f_ij, j, levels.group[i]);
                    const LaParts parts = *reinterpret_cast<const LaParts *>(levels.part + j);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = c[r] * (a.scale * f_ij[r]);
                        c[r] = (j + r <= i) & (parts[r] == part) ? x : 0.0f;
                    }
                    F f[S::INNER];
                    la_split(c, f);
#pragma unroll
                    for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ps + (m * C + i) * LDC + j) = f[m];
                }
            }
            LaPair<F> vf[TT / 2];
#pragma unroll
            for (int p = 0; p < TT / 2; ++p) vf[p] = la_cols2(lane, vs, LD, 32 * p, 16 * slice);
            if constexpr (OUT) {
                if (a.kept) {
                    const LaOut<float> to(a.kept + (bh * a.chunks + chunk) * features * la_line(values), features, la_line(values), g, col, la_line(values));
#pragma unroll
                    for (int t = 0; t < OD; ++t) to.store(half * OD + t, s[t]);
                }
                LaAcc o[OT] = {};
#pragma unroll
                for (int x = 0; x < D; x += 32) {
                    // (a state from its sums has their order: 4 g .. 4 g + 3 of two tiles)
                    LaPair<F> sx[S::INNER];
                    if constexpr (SHARED) {
#pragma unroll
                        for (int m = 0; m < S::INNER; ++m) sx[m] = la_rows2(lane, ss + m * D * LD, LD, 16 * slice, x);
                    } else {
                        F s0[S::INNER], s1[S::INNER];
                        la_split(s[x / 16], s0);
                        la_split(s[x / 16 + 1], s1);
#pragma unroll
                        for (int m = 0; m < S::INNER; ++m) sx[m] = {s0[m], s1[m]};
                    }
#pragma unroll
                    for (int u = 0; u < OT; ++u) {
                        const int t = S::tile(half, u);
                        LaPair<F> qx;
                        if constexpr (SHARED) qx = la_rows2(lane, qs, LD, 16 * t, x);
                        else qx = {la_rows<F>(lane, qs, LD, 16 * t, x), la_rows<F>(lane, qs, LD, 16 * t, x + 16)};
#pragma unroll
                        for (int m = 0; m < S::INNER; ++m) o[u] = la_mma(qx, sx[m], o[u]);
                    }
                }
                __syncthreads();
                const LaOut<T> to(static_cast<T *>(a.o) + ((b * a.steps + t0) * a.heads + h) * values, rows, a.heads * values, g, col, values);
#pragma unroll
                for (int u = 0; u < OT; ++u) {
                    const int t = S::tile(half, u);
                    o[u] = la_times(o[u], levels.quad(levels.start, 16 * t + 4 * g));
                    la_over_steps<BAD, S::INNER, TT, F>(
                        o[u], 0, S::pair_of(u), [&](int m, int p) { return la_rows2(lane, ps + m * C * LDC, LDC, 16 * t, 32 * p); },
                        [&](int p) { return vf[p]; }, [&](int lane, int m, int j) { return la_rows<F>(lane, ps + m * C * LDC, LDC, 16 * t, 16 * j); },
                        [&](int lane, int j) { return la_cols(lane, vs, LD, 16 * j, 16 * slice); },
                        [&](int r, int j) { const int i = 16 * t + 4 * g + r; return j <= i && levels.part[j] == levels.part[i]; });
                }
#pragma unroll
                for (int u = 0; u < OT; ++u) to.store(S::tile(half, u), o[u]);
            }
            // the state behind the chunk (BACK: its gradient in front of it)
            const float decay = levels.decay;
#pragma unroll
            for (int t = 0; t < OD; ++t) s[t] = la_times(s[t], decay);
#pragma unroll
            for (int p = 0; p < TT / 2; ++p) {
                const LaAcc one = levels.quad(BACK ? levels.start : levels.end, 32 * p + la_first<T>(g));
                const LaAcc two = levels.quad(BACK ? levels.start : levels.end, 32 * p + la_second<T>(g));
                F w1[S::ADDED], w2[S::ADDED];
                la_split(la_times(la_float(vf[p].a), one), w1);
                la_split(la_times(la_float(vf[p].b), two), w2);
#pragma unroll
                for (int x = 0; x < OD; ++x) {
                    LaPair<F> kx = la_cols2(lane, ks, LD, 32 * p, 16 * (half * OD + x));
                    if constexpr (BAD) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (la_nothing(one[r])) kx.a[r] = 0.0f;
                            if (la_nothing(two[r])) kx.b[r] = 0.0f;
                        }
                    }
#pragma unroll
                    for (int m = 0; m < S::ADDED; ++m) s[x] = la_mma(kx, LaPair<F>{w1[m], w2[m]}, s[x]);
                }
            }
        };
        if (__builtin_expect(bad, 0)) products(std::true_type());
        else products(std::false_type());
        if constexpr (!OUT) {
            total += levels.broken ? (double)levels.decay : (double)levels.hi[C - 1] + (double)levels.lo[C - 1];
            cuts |= levels.part[C - 1];
        }
        __syncthreads();
    }
    float *to = OUT ? (segment == a.segments - 1 && a.last ? a.last + bh * features * values : nullptr)
                    : a.segment_state + (segment * heads + bh) * features * values;
    if (to) {
#pragma unroll
        for (int t = 0; t < OD; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = row0 + 16 * t + r;
                if (row < features && col < values) to[row * values + col] = s[t][r];
            }
    }
    if (!OUT && threadIdx.x == 0) {
        a.segment_decay[segment * heads + bh] = (float)exp2(total);
        a.segment_cut[segment * heads + bh] = cuts;
    }
}

// (25 segments of 10 heads of 100 x 100: 8 us for 20 MB, bound by the few workgroups that they make)
// What segments add to the state becomes the state each starts from (BACK: the gradient of the one it ends with).
template <bool BACK>
__global__ __launch_bounds__(256) void la_enter_kernel(const LaArgs a)
{
    const int64_t square = (int64_t)a.features * a.values, heads = a.batch * a.heads, count = heads * square;
    const float *from = BACK ? a.grad_last : a.state;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) {
        const int64_t bh = at / square;
        float s = from ? from[at] : 0.0f;
        // (eight segments on their way at once: none waits for the state of the one in front)
        for (int n = 0; n < a.segments; n += 8) {
            float added[8] = {}, decay[8] = {};
            int cut[8] = {};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (n + i >= a.segments) break;
                const int64_t segment = BACK ? a.segments - 1 - (n + i) : n + i;
                added[i] = a.segment_state[segment * count + at];
                decay[i] = a.segment_decay[segment * heads + bh];
                cut[i] = a.segment_cut[segment * heads + bh];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (n + i >= a.segments) break;
                const int64_t segment = BACK ? a.segments - 1 - (n + i) : n + i;
                a.segment_state[segment * count + at] = s;
                s = cut[i] != 0 ? added[i] : decay[i] * s + added[i];
            }
        }
    }
}

// (from: NULL for zeros)
__global__ __launch_bounds__(256) void la_copy_kernel(const float *from, float *to, int64_t count)
{
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) to[at] = from ? from[at] : 0.0f;
}

// The gradients, chunk by chunk from a segment's end, with the states that the forward call kept (formed again they would cost the
// walk once more, 116 us of the first case above; kept, 268 MB to write and read, 56 us).
template <typename T, int D>
__global__ __launch_bounds__((LaShape<T, D>::THREADS)) void la_back_kernel(const LaArgs a)
{
    using S = LaShape<T, D>;
    using F = typename LaFrag<T>::type;
    constexpr int C = S::C, W = S::W, TT = S::TT, DT = S::DT, OT = S::OWN_T, OD = S::OWN_D, LD = S::LD, LDC = S::LDC;
    constexpr bool SHARED = S::HALVES > 1;             // E's operands for dK in LDS too, to the chunk's end
    constexpr int EP = SHARED ? S::ADDED : S::INNER;   // numbers of E in LDS
    constexpr int HELD = EP * D * LD, FACTORS = 2 * S::INNER * C * LDC;
    __shared__ __align__(16) T qs[C * LD];
    __shared__ __align__(16) T ks[C * LD];
    __shared__ __align__(16) T vs[C * LD];
    __shared__ __align__(16) T gs[C * LD];
    // E, rows are features; (Q K^T . D)^T and (dO V^T . D)^T, rows are steps j, in its place where it is not needed any more
    __shared__ __align__(16) T room[SHARED ? HELD + FACTORS : HELD > FACTORS ? HELD : FACTORS];
    T *const es = room, *const ps = room + (SHARED ? HELD : 0), *const ds = ps + S::INNER * C * LDC;
    __shared__ __align__(16) LaLevels<C> three_levels[3];   // of the chunk, the next one, and the last one's for its decays' gradients
    struct Sums {
        // (of two chunks: the next one's are written while the decays' gradients of this one are formed)
        float row[2][TT][C], col[2][TT][C];
        float start[S::SLICES][C], end[S::SLICES][C], through[S::SLICES];
    };
    __shared__ __align__(16) Sums sums;
    __shared__ int bad_chunk[2];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const int slice = wave % S::SLICES, half = wave / S::SLICES;
    const int64_t heads = a.batch * a.heads, unit = la_unit(heads * a.segments);
    if (unit >= heads * a.segments) return;
    const int64_t segment = unit / heads, bh = unit % heads, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t first = segment * a.segment_chunks, end = min(first + a.segment_chunks, a.chunks);
    const int count = (int)(end - first), features = a.features, values = a.values;

    // E transposed: rows are values 16 (half OD + t) + 4 g + r, column: feature 16 slice + lane % 16
    LaAcc e[OD];
    const int col = 16 * slice + i16, value0 = 16 * half * OD + 4 * g;
    const float *behind = a.segments > 1 ? a.segment_state + (segment * heads + bh) * features * values
                          : a.grad_last ? a.grad_last + bh * features * values : nullptr;
#pragma unroll
    for (int t = 0; t < OD; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = value0 + 16 * t + r;
            e[t][r] = behind && col < features && row < values ? behind[col * values + row] : 0.0f;
        }

    // (nothing is moved ahead of it: with 128 columns the operands of later products would push others out of the registers)
    auto hold = [] { if constexpr (D > 64) __builtin_amdgcn_sched_barrier(0); };
    const bool nothing = !a.grad;   // (no gradient of o: zeros, whatever is read)
    LaPiece<T, D> nq, nk, nv, ng;
    nq.init(static_cast<const T *>(a.q) + la_offset(a.q_stride, b, 0, h / a.shared), a.q_stride[1], features);
    nk.init(static_cast<const T *>(a.k) + la_offset(a.k_stride, b, 0, h / a.shared), a.k_stride[1], features);
    nv.init(static_cast<const T *>(a.v) + la_offset(a.v_stride, b, 0, h), a.v_stride[1], values);
    ng.init(static_cast<const T *>(nothing ? a.v : a.grad) + la_offset(nothing ? a.v_stride : a.grad_stride, b, 0, h),
            nothing ? a.v_stride[1] : a.grad_stride[1], values);
    LaDecay<C> nd;
    nd.init(a, b, h);
    auto chunk_of = [&](int n) { return end - 1 - n; };
    auto rows_of = [&](int n) { return (int)min((int64_t)C, a.steps - chunk_of(n) * C); };
    const bool wide = features >= S::E && values >= S::E, even = features % S::E == 0 && values % S::E == 0;
    auto fetch = [&](int n) {
        const int64_t t0 = chunk_of(n) * C;
        const int rows = rows_of(n);
        if (__builtin_expect(wide && rows == C, 1)) {
            nq.fetch_whole(t0);
            nk.fetch_whole(t0);
            nv.fetch_whole(t0);
            ng.fetch_whole(t0);
        } else {
            nq.fetch_any(t0, rows);
            nk.fetch_any(t0, rows);
            nv.fetch_any(t0, rows);
            ng.fetch_any(t0, rows);
        }
    };
    const int line = la_line(values);

    // The decays' gradients of a chunk, one step a lane: sums over the later steps of its document, sums over the earlier ones.
    auto decays = [&](int n) {
        const LaLevels<C> &levels = three_levels[n % 3];
        const int mine = levels.part[min(lane, C - 1)], parts = levels.part[C - 1], part_before = __shfl_up(mine, 1, 64);
        // later steps: lanes reversed, so that they are the earlier ones
        const int t = C - 1 - min(lane, C - 1), reversed = parts - levels.part[t];
        float later = 0.0f, earlier = 0.0f;
#pragma unroll
        for (int x = 0; x < TT; ++x) {
            later += x <= ((t >> 4) | 1) ? sums.row[n & 1][x][t] : 0.0f;
            later -= x >= ((t >> 4) & ~1) ? sums.col[n & 1][x][t] : 0.0f;
        }
#pragma unroll
        for (int x = 0; x < S::SLICES; ++x) {
            later += sums.start[x][t];
            earlier += sums.end[x][min(lane, C - 1)];
        }
        la_scan(later, reversed);
        la_scan(earlier, mine);
        later = __shfl(later, C - 1 - min(lane, C - 1), 64);
        float ahead = __shfl_up(earlier, 1, 64);
        if (lane == 0 || part_before != mine) ahead = 0.0f;
        float crossing = 0.0f;
        if (parts == 0) {
#pragma unroll
            for (int x = 0; x < S::SLICES; ++x) crossing += sums.through[x];
            crossing *= levels.decay;
        }
        // (the decay of a reset step meets nothing)
        const bool starts = mine != (lane == 0 ? 0 : part_before);
        if (lane < rows_of(n)) a.d_log_decay[((b * a.steps + chunk_of(n) * C + lane) * a.heads) + h] = starts ? 0.0f : later + ahead + crossing;
    };

    if (threadIdx.x < 2) bad_chunk[threadIdx.x] = 0;
    // The decays are fetched two chunks ahead, in front of the next chunk's rows: once those have arrived, they have, too.
    auto fetch_decays = [&](int n) { nd.fetch(chunk_of(min(n, count - 1)) * C, rows_of(min(n, count - 1))); };
    if (wave == W - 1) {
        fetch_decays(0);
        nd.levels(three_levels[0], a.scale);
        fetch_decays(1);
    }
    fetch(0);
    __syncthreads();
    for (int n = 0; n < count; ++n) {
        const int lane = la_lane<(D > 64)>(), i16 = lane & 15, g = lane >> 4, col = 16 * slice + i16;
        const int64_t chunk = chunk_of(n), t0 = chunk * C;
        const int rows = rows_of(n);
        const LaLevels<C> &levels = three_levels[n % 3];
        LaLevels<C> &next_levels = three_levels[(n + 1) % 3];
        uint32_t magnitude = 0;
        auto store_all = [&](auto even_type) {
            constexpr bool EVEN = decltype(even_type)::value;
            nq.template store<EVEN>(qs, rows, magnitude);
            nk.template store<EVEN>(ks, rows, magnitude);
            nv.template store<EVEN>(vs, rows, magnitude);
            ng.template store<EVEN>(gs, nothing ? 0 : rows, magnitude);
        };
        if (__builtin_expect(even, 1)) store_all(std::true_type());
        else store_all(std::false_type());
        if (la_not_finite<T>(magnitude)) bad_chunk[n & 1] = 1;
#pragma unroll
        for (int t = 0; t < OD; ++t) {
            F f[EP];
            la_split(e[t], f);
#pragma unroll
            for (int m = 0; m < EP; ++m) *reinterpret_cast<F *>(es + (m * D + col) * LD + 16 * half * OD + 4 * g + 16 * t) = f[m];
        }
        __syncthreads();
        const bool bad = (bad_chunk[n & 1] != 0) | levels.broken;
        if (threadIdx.x == 0) bad_chunk[(n + 1) & 1] = 0;
        // the state in front of the chunk (what lies outside of it: some address inside, zero when it is used)
        // before[t]: values value_of(t) .. + 3, in the order of the operands that it meets: those in LDS, or E's sums
        LaAcc before[DT] = {};
        auto value_of = [](int t, int g) { return SHARED ? 32 * (t / 2) + (t % 2 ? la_second<T>(g) : la_first<T>(g)) : 16 * t + 4 * g; };
        auto fetch_state = [&] {
            const float *from = a.kept + (bh * a.chunks + chunk) * features * line + (col < features ? col * line : 0);
#pragma unroll
            for (int t = 0; t < DT; ++t) before[t] = *reinterpret_cast<const LaAcc *>(from + (value_of(t, g) < line ? value_of(t, g) : 0));
        };
        // (behind the last chunk: that one once more)
        auto fetch_next = [&] {
            if (wave == W - 1) fetch_decays(n + 2);
            fetch(min(n + 1, count - 1));
        };
        if (wave == W - 1 && n + 1 < count) nd.levels(next_levels, a.scale);
        // (128 columns leave no registers for what is not needed yet)
        if constexpr (SHARED) {
            fetch_state();
            fetch_next();
        }
        if (n > 0 && wave == W - 2) decays(n - 1);

        // dV, rows are steps j, columns this wavefront's values: w K E
        LaAcc dv[OT] = {};
#pragma unroll
        for (int x = 0; x < D; x += 32) {
            LaPair<F> ex[S::INNER];
#pragma unroll
            for (int m = 0; m < S::INNER; ++m) ex[m] = la_cols2(lane, es + m * D * LD, LD, x, 16 * slice);
#pragma unroll
            for (int u = 0; u < OT; ++u) {
                const LaPair<F> kx = la_rows2(lane, ks, LD, 16 * S::tile(half, u), x);
#pragma unroll
                for (int m = 0; m < S::INNER; ++m) dv[u] = la_mma(kx, ex[m], dv[u]);
            }
            hold();
        }
        // the inner factors and G
        constexpr int EACH = S::EACH;
        LaAcc cs[EACH] = {}, dds[EACH] = {}, gg[EACH] = {};
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            const int p = wave + u * W;
            if (S::PAIRS % W != 0 && p >= S::PAIRS) break;
            int ti, tj;
            la_pair(p, ti, tj);
            LaAcc c = {}, d = {};
#pragma unroll
            for (int x = 0; x < D; x += 32) {
                c = la_mma(la_rows2(lane, qs, LD, 16 * ti, x), la_rows2(lane, ks, LD, 16 * tj, x), c);
                d = la_mma(la_rows2(lane, gs, LD, 16 * ti, x), la_rows2(lane, vs, LD, 16 * tj, x), d);
                hold();
            }
            const int j = 16 * tj + i16, i = 16 * ti + 4 * g, part = levels.part[j];
            LaAcc f_ij = levels.between(levels.quad(levels.hi, i), levels.quad(levels.lo, i), levels.hi[j], levels.lo[j], 1.0f);
            if (__builtin_expect(bad, 0)) f_ij = levels.crossed(f_ij, i, levels.group[j]);
            const LaParts parts = *reinterpret_cast<const LaParts *>(levels.part + i);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool there = (j <= i + r) & (parts[r] == part);
                const float f = a.scale * f_ij[r], x = c[r] * f, y = d[r] * f, z = x * d[r];
                c[r] = there ? x : 0.0f;
                gg[u][r] = there & (j < i + r) ? z : 0.0f;
                d[r] = there ? y : 0.0f;
            }
            hold();
            cs[u] = c;
            dds[u] = d;
        }
        if constexpr (!SHARED) __syncthreads();
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
            if (S::PAIRS % W != 0 && wave + u * W >= S::PAIRS) break;
            int ti, tj;
            la_pair(wave + u * W, ti, tj);
            const int j = 16 * tj + i16, i = 16 * ti + 4 * g;
            F f[S::INNER];
            la_split(cs[u], f);
#pragma unroll
            for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ps + (m * C + j) * LDC + i) = f[m];
            la_split(dds[u], f);
#pragma unroll
            for (int m = 0; m < S::INNER; ++m) *reinterpret_cast<F *>(ds + (m * C + j) * LDC + i) = f[m];
            float column = (gg[u][0] + gg[u][1]) + (gg[u][2] + gg[u][3]);
            column += __shfl_xor(column, 16, 64);
            column += __shfl_xor(column, 32, 64);
            sums.col[n & 1][ti][j] = column;   // (the same from four lanes)
            LaAcc row;
#pragma unroll
            for (int r = 0; r < 4; ++r) row[r] = la_sum16(gg[u][r]);
            *reinterpret_cast<LaAcc *>(&sums.row[n & 1][tj][i]) = row;   // (from sixteen)
        }
        __syncthreads();
        if constexpr (!SHARED) fetch_state();

        const float decay = levels.decay;
        const int64_t row0 = (b * a.steps + t0) * a.heads + h;
        auto products = [&](auto bad_type) {
            constexpr bool BAD = decltype(bad_type)::value;
            auto meets = [&](int i, int j) { return j <= i && levels.part[j] == levels.part[i]; };
            auto store = [&](void *rows_of_all, const LaAcc (&x)[OT]) {
                if (a.wide) {
                    const LaOut<float> to(static_cast<float *>(rows_of_all) + row0 * features, rows, a.heads * features, g, col, features);
#pragma unroll
                    for (int u = 0; u < OT; ++u) to.store(S::tile(half, u), x[u]);
                } else {
                    const LaOut<T> to(static_cast<T *>(rows_of_all) + row0 * features, rows, a.heads * features, g, col, features);
#pragma unroll
                    for (int u = 0; u < OT; ++u) to.store(S::tile(half, u), x[u]);
                }
            };
#pragma unroll
            for (int u = 0; u < OT; ++u) {
                const int t = S::tile(half, u);
                dv[u] = la_times(dv[u], levels.quad(levels.end, 16 * t + 4 * g));
                la_over_steps<BAD, S::INNER, TT, F>(
                    dv[u], S::pair_of(u), TT / 2 - 1, [&](int m, int p) { return la_rows2(lane, ps + m * C * LDC, LDC, 16 * t, 32 * p); },
                    [&](int p) { return la_cols2(lane, gs, LD, 32 * p, 16 * slice); },
                    [&](int lane, int m, int i) { return la_rows<F>(lane, ps + m * C * LDC, LDC, 16 * t, 16 * i); },
                    [&](int lane, int i) { return la_cols(lane, gs, LD, 16 * i, 16 * slice); },
                    [&](int r, int i) { return meets(i, 16 * t + 4 * g + r); });
            }
            {
                const LaOut<T> to(static_cast<T *>(a.d_v) + row0 * values, rows, a.heads * values, g, col, values);
#pragma unroll
                for (int u = 0; u < OT; ++u) to.store(S::tile(half, u), dv[u]);
            }
            hold();
            // dQ, rows are steps i, columns this wavefront's features: b dO S^T
            LaAcc d[OT] = {};
#pragma unroll
            for (int x = 0; x < DT; ++x) {
                const bool there = (col < features) & (value_of(x, g) < line);
#pragma unroll
                for (int r = 0; r < 4; ++r) before[x][r] = there ? before[x][r] : 0.0f;
            }
#pragma unroll
            for (int x = 0; x < DT; x += 2) {
                F s0[S::ADDED], s1[S::ADDED];
                la_split(before[x], s0);
                la_split(before[x + 1], s1);
#pragma unroll
                for (int u = 0; u < OT; ++u) {
                    const int t = S::tile(half, u);
                    LaPair<F> gx;
                    if constexpr (SHARED) gx = la_rows2(lane, gs, LD, 16 * t, 16 * x);
                    else gx = {la_rows<F>(lane, gs, LD, 16 * t, 16 * x), la_rows<F>(lane, gs, LD, 16 * t, 16 * x + 16)};
#pragma unroll
                    for (int m = 0; m < S::ADDED; ++m) d[u] = la_mma(gx, LaPair<F>{s0[m], s1[m]}, d[u]);
                }
                hold();
            }
            LaPair<F> qf[TT / 2], kf[TT / 2];
#pragma unroll
            for (int p = 0; p < TT / 2; ++p) {
                qf[p] = la_cols2(lane, qs, LD, 32 * p, 16 * slice);
                kf[p] = la_cols2(lane, ks, LD, 32 * p, 16 * slice);
            }
            // <E, S>, where E is in registers
            float sum = 0.0f;
            if constexpr (!SHARED) {
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum += e[t][r] * before[t][r];
            }
#pragma unroll
            for (int u = 0; u < OT; ++u) {
                const int t = S::tile(half, u), i = 16 * t + 4 * g;
                const LaAcc to_start = levels.quad(levels.start, i);
                d[u] = la_times(d[u], to_start);
                // (a step that a reset parts from the state: zero times what may not be finite)
                LaAcc at_start = d[u] * la_float(la_cols(lane, qs, LD, 16 * t, 16 * slice));
#pragma unroll
                for (int r = 0; r < 4; ++r) at_start[r] = la_sum16(la_nothing(to_start[r]) ? 0.0f : at_start[r]);
                *reinterpret_cast<LaAcc *>(&sums.start[slice][i]) = at_start;
                la_over_steps<BAD, S::INNER, TT, F>(
                    d[u], 0, S::pair_of(u), [&](int m, int p) { return la_cols2(lane, ds + m * C * LDC, LDC, 32 * p, 16 * t); },
                    [&](int p) { return kf[p]; }, [&](int lane, int m, int j) { return la_cols(lane, ds + m * C * LDC, LDC, 16 * j, 16 * t); },
                    [&](int lane, int j) { return la_cols(lane, ks, LD, 16 * j, 16 * slice); },
                    [&](int r, int j) { return meets(16 * t + 4 * g + r, j); });
            }
            store(a.d_q, d);
            hold();
            if constexpr (!SHARED) fetch_next();
            // dK, rows are steps j: w V E^T
            LaAcc c[OT] = {};
#pragma unroll
            for (int x = 0; x < DT; x += 2) {
                LaPair<F> ex[S::ADDED];
                if constexpr (SHARED) {
                    LaAcc one = {}, two = {};
#pragma unroll
                    for (int m = 0; m < S::ADDED; ++m) {
                        ex[m] = la_rows2(lane, es + m * D * LD, LD, 16 * slice, 16 * x);
                        one += la_float(ex[m].a);
                        two += la_float(ex[m].b);
                    }
                    // (both halves read all of it: <E, S> of the first one)
                    one *= before[x];
                    two *= before[x + 1];
                    sum += ((one[0] + one[1]) + (one[2] + one[3])) + ((two[0] + two[1]) + (two[2] + two[3]));
                } else {
                    // (as something new: the numbers split off for dV would be kept for this in registers that there are not)
                    LaAcc here = e[x], next = e[x + 1];
                    asm volatile("" : "+v"(here), "+v"(next));
                    F e0[S::ADDED], e1[S::ADDED];
                    la_split(here, e0);
                    la_split(next, e1);
#pragma unroll
                    for (int m = 0; m < S::ADDED; ++m) ex[m] = {e0[m], e1[m]};
                }
#pragma unroll
                for (int u = 0; u < OT; ++u) {
                    const int t = S::tile(half, u);
                    LaPair<F> vx;
                    if constexpr (SHARED) vx = la_rows2(lane, vs, LD, 16 * t, 16 * x);
                    else vx = {la_rows<F>(lane, vs, LD, 16 * t, 16 * x), la_rows<F>(lane, vs, LD, 16 * t, 16 * x + 16)};
#pragma unroll
                    for (int m = 0; m < S::ADDED; ++m) c[u] = la_mma(vx, ex[m], c[u]);
                }
                hold();
            }
#pragma unroll
            for (int u = 0; u < OT; ++u) {
                const int t = S::tile(half, u), j = 16 * t + 4 * g;
                const LaAcc to_end = levels.quad(levels.end, j);
                c[u] = la_times(c[u], to_end);
                LaAcc at_end = c[u] * la_float(la_cols(lane, ks, LD, 16 * t, 16 * slice));
#pragma unroll
                for (int r = 0; r < 4; ++r) at_end[r] = la_sum16(la_nothing(to_end[r]) ? 0.0f : at_end[r]);
                *reinterpret_cast<LaAcc *>(&sums.end[slice][j]) = at_end;
                la_over_steps<BAD, S::INNER, TT, F>(
                    c[u], S::pair_of(u), TT / 2 - 1, [&](int m, int p) { return la_rows2(lane, ds + m * C * LDC, LDC, 16 * t, 32 * p); },
                    [&](int p) { return qf[p]; }, [&](int lane, int m, int i) { return la_rows<F>(lane, ds + m * C * LDC, LDC, 16 * t, 16 * i); },
                    [&](int lane, int i) { return la_cols(lane, qs, LD, 16 * i, 16 * slice); },
                    [&](int r, int i) { return meets(i, 16 * t + 4 * g + r); });
            }
            store(a.d_k, c);
            sum = la_sum16(sum);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (half == 0) sums.through[slice] = sum;
            hold();
            // E in front of the chunk
#pragma unroll
            for (int t = 0; t < OD; ++t) e[t] = la_times(e[t], decay);
#pragma unroll
            for (int p = 0; p < TT / 2; ++p) {
                const LaAcc one = levels.quad(levels.start, 32 * p + la_first<T>(g)), two = levels.quad(levels.start, 32 * p + la_second<T>(g));
                F w1[S::ADDED], w2[S::ADDED];
                la_split(la_times(la_float(qf[p].a), one), w1);
                la_split(la_times(la_float(qf[p].b), two), w2);
#pragma unroll
                for (int x = 0; x < OD; ++x) {
                    LaPair<F> gx = la_cols2(lane, gs, LD, 32 * p, 16 * (half * OD + x));
                    if constexpr (BAD) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (la_nothing(one[r])) gx.a[r] = 0.0f;
                            if (la_nothing(two[r])) gx.b[r] = 0.0f;
                        }
                    }
#pragma unroll
                    for (int m = 0; m < S::ADDED; ++m) e[x] = la_mma(gx, LaPair<F>{w1[m], w2[m]}, e[x]);
                }
                hold();
            }
        };
        if (__builtin_expect(bad, 0)) products(std::true_type());
        else products(std::false_type());
        __syncthreads();
    }
    if (wave == W - 2) decays(count - 1);
    if (segment == 0 && a.d_state) {
        float *to = a.d_state + bh * features * values;
#pragma unroll
        for (int t = 0; t < OD; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = value0 + 16 * t + r;
                if (col < features && row < values) to[col * values + row] = e[t][r];
            }
    }
}

// Gradients of queries or keys that heads share: the sum over those heads, in order (zero over none).
template <typename T>
__global__ __launch_bounds__(256) void la_shared_kernel(const float *from, T *to, int64_t rows, int groups, int shared, int features)
{
    const int64_t count = rows * groups * features;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (int64_t)gridDim.x * 256) {
        const int64_t row = at / features;
        const float *p = from + row * shared * features + at % features;
        float sum = shared > 0 ? p[0] : 0.0f;
        for (int n = 1; n < shared; ++n) sum += p[(int64_t)n * features];
        to[at] = (T)sum;
    }
}

// One step of every head: the state is read and written once, which is all that this costs.  LANES lanes take V neighbouring
// values of a feature's row each, the others of 256 its further features.  64 x 16 heads of 64 x 64: 33.5 MB in 7.4 us, 4.5 TB/s; one sequence: 4.1 us, a launch.
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
