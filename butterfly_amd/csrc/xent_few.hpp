// The loss of xent.hpp for few rows (1 .. 64): the bytes of the weights bound it, not the matrix units, so
// they are read as they lie (any alignment, no copy in another form), once forward and once backward, and d_weight is
// written once.  The logits of so few rows take no more room than the weights and stay in memory for
// the backward call, which a tile of 128 or 256 rows would form again out of weights read again.
//
// All three products are MFMA tiles (16 x 16, K = 32) whose operands come straight into registers: 16-byte loads
// of weight in the lanes that multiply them, and the small operands (hidden, d_l) from an array in the order
// of the lanes, "fragments" of 64 x 16 bytes, that the L2 holds.
//
//   logits    A = weight: lane (i, g) holds 8 features of vocabulary entry i, B = hidden.  K in any order, as long as
//             both have the same: float's two loads of 4 features are 16 apart, so each takes 64 neighbouring
//             bytes of a row.
//   d_hidden  contraction over the vocabulary: lane (i, g) loads its columns E i .. E i + E - 1 (E = 4 floats or 8
//             bfloat16 numbers) of entries 8 g + j, j = 0 .. 7, and column E i + t of them is tile t's operand: the
//             transposition is a choice of registers.
//   d_weight  A = d_l^T, B = hidden^T in the same order of columns, so a lane's results are 16 neighbouring bytes.
//
// Number formats.  bfloat16 as in xent.hpp.  float: x = x1 + x2 + x3 in three bfloat16 numbers of 8 bits each, which is
// exact and needs no power of two (nor a pass over the weights to find it); of the nine products the six of
// 2^-16 and above are taken, sums in float: what is left out is below 2^-21 of a product.
//
// Measured, forward and backward beside the tiles of xent.hpp: 33 rows, 1843 features, 67371 entries, float 508 us beside 1438;
// 7 x 2109 x 43964 324 beside 934; 1 x 172 x 81752 84 beside 340; bfloat16 1 x 1056 x 23742 84 beside 137; forward alone 21 x 3444 x
// 54104 bfloat16 124 beside 278.
#pragma once

#include "xent.hpp"

namespace bf {

typedef uint32_t Quad __attribute__((ext_vector_type(4)));

constexpr int kFewRows = 64;
constexpr int kFewThreads = 256;

template <typename T>
struct Few {
    static constexpr bool kFloat = sizeof(T) == 4;
    static constexpr int kPlanes = kFloat ? 3 : 1;
    static constexpr int kEach = 16 / sizeof(T);            // elements of a 16-byte load
    static constexpr int kChunk = 128 / sizeof(T);          // features of a chunk of the logits' k
    static constexpr int kChunkFrags = kFloat ? 3 : 2;      // of 16 hidden rows: planes, or halves of the chunk
    static constexpr int kCols = 16 * kEach;                // columns of a wavefront's part of the gradients
};

__device__ __forceinline__ Acc4 mfma_few(Frag a, Frag b, Acc4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight numbers in three planes of bfloat16, each the upper half of what the ones before leave (of a NaN or an
// infinity: NaN in the second).
__device__ __forceinline__ void split_bf16(const float (&x)[8], Frag (&f)[3])
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f[p][i] = (int)__builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);
        if (p < 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] -= __uint_as_float(__float_as_uint(v[i]) & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void planes_of(const float (&x)[8], Frag (&f)[3]) { split_bf16(x, f); }
__device__ __forceinline__ void planes_of(const float (&x)[8], Frag (&f)[1])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) f[0][i] = (int)pack_bf16(x[2 * i], x[2 * i + 1]);
}

// a b over the planes, the small products first
__device__ __forceinline__ Acc4 product_of(const Frag (&a)[3], const Frag (&b)[3], Acc4 c)
{
    c = mfma_few(a[2], b[0], c);
    c = mfma_few(a[0], b[2], c);
    c = mfma_few(a[1], b[1], c);
    c = mfma_few(a[1], b[0], c);
    c = mfma_few(a[0], b[1], c);
    return mfma_few(a[0], b[0], c);
}
__device__ __forceinline__ Acc4 product_of(const Frag (&a)[1], const Frag (&b)[1], Acc4 c) { return mfma_few(a[0], b[0], c); }

// 16 bytes from element col on of a row; past the row's `cols` elements zeros
template <typename T>
__device__ __forceinline__ Quad load_cut(const T *row, int col, int cols)
{
    Quad q = {0, 0, 0, 0};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < cols) q[i] = reinterpret_cast<const uint32_t *>(row)[col + i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) q[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(row)[col + i] << (i & 1) * 16;
    }
    return q;
}

// ---- which rows count, and hidden in fragments -------------------------------------------------------------------

struct XentFewPackArgs {
    const void *hidden;
    const int64_t *target;
    int64_t hidden_stride;
    int rows, tiles, features;      // tiles of 16 rows
    int64_t vocab, ignore;
    XentScalars *scalars;
    int *index, *position, *label;
    char *by_feature;               // [chunk][plane or half][tile]: the logits' operand
    char *by_row;                   // [part of the columns][32 rows][plane][column within a load]: d_weight's
};

// Every workgroup finds the counted rows by itself (one load of a wavefront).
template <typename T>
__global__ __launch_bounds__(kFewThreads) void xent_few_pack_kernel(XentFewPackArgs a)
{
    using F = Few<T>;
    __shared__ int index[kFewRows];
    __shared__ int counted_at;
    if (threadIdx.x < 64) {
        const int row = threadIdx.x;
        const int64_t t = row < a.rows ? a.target[row] : a.ignore;
        const uint64_t counts = __ballot(t != a.ignore);
        const bool in = counts >> row & 1;
        const int place = __popcll(counts & ((1ull << row) - 1)), n = __popcll(counts);
        if (in) index[place] = row;
        if (row == 0) counted_at = n;
        if (blockIdx.x == 0) {
            if (row < a.rows) a.position[row] = in ? place : -1;
            if (in) {
                a.index[place] = row;
                a.label[place] = t >= 0 && t < a.vocab ? (int)t : -1;
            }
            if (row == 0) {
                a.scalars->counted = n;
                a.scalars->hidden_scale = a.scalars->weight_scale = a.scalars->grad_scale = 1.0f;
            }
        }
    }
    __syncthreads();
    const int counted = counted_at;
    const T *hidden = reinterpret_cast<const T *>(a.hidden);
    auto at = [&](int n, int k) { return n < counted && k < a.features ? to_float(hidden[index[n] * a.hidden_stride + k]) : 0.0f; };
    constexpr int kHalves = F::kFloat ? 1 : 2;
    const int chunks = (a.features + F::kChunk - 1) / F::kChunk, parts = (a.features + F::kCols - 1) / F::kCols;
    const int steps = (a.tiles + 1) / 2;
    const int64_t first = (int64_t)chunks * kHalves * a.tiles * 64, total = first + (int64_t)parts * steps * F::kEach * 64;
    for (int64_t id = (int64_t)blockIdx.x * kFewThreads + threadIdx.x; id < total; id += (int64_t)gridDim.x * kFewThreads) {
        const int lane = (int)(id & 63), i = lane & 15, g = lane >> 4;
        float x[8];
        char *out;
        int64_t stride;      // between planes
        if (id < first) {
            const int tile = (int)(id / 64 % a.tiles), piece = (int)(id / 64 / a.tiles);   // (chunk, half)
            const int c = piece / kHalves, half = piece % kHalves;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = at(tile * 16 + i, c * F::kChunk + (F::kFloat ? (j >> 2) * 16 + 4 * g + (j & 3) : half * 32 + 8 * g + j));
            out = a.by_feature + ((int64_t)(c * F::kChunkFrags + half) * a.tiles + tile) * 1024 + lane * 16;
            stride = (int64_t)a.tiles * 1024;
        } else {
            const int64_t rest = (id - first) / 64;
            const int t = (int)(rest % F::kEach), step = (int)(rest / F::kEach % steps), part = (int)(rest / F::kEach / steps);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = at(step * 32 + 8 * g + j, part * F::kCols + F::kEach * i + t);
            out = a.by_row + (((int64_t)part * steps + step) * F::kPlanes * F::kEach + t) * 1024 + lane * 16;
            stride = F::kEach * 1024;
        }
        Frag f[F::kPlanes];
        planes_of(x, f);
#pragma unroll
        for (int p = 0; p < F::kPlanes; ++p) *reinterpret_cast<Frag *>(out + p * stride) = f[p];
    }
}

// ---- logits ----------------------------------------------------------------------------------------------------

struct XentFewLogitsArgs {
    const void *weight;
    int64_t weight_stride, vocab;
    int features, parts, wide;      // parts: workgroups, the first `wide` of them of 64 entries
    const XentScalars *scalars;
    const char *by_feature;
    float *logits;                  // (rows by place, stride)
    int64_t stride;
    float2 *partial;                // (rows by place, parts): maximum, sum
};

// LDS of a workgroup of 16 MT entries
template <int NT, int MT>
struct FewLds {
    union {
        Quad staged[4][16 * MT][8];
        Acc4 sums[4][MT * NT][64];
    };
    float2 tops[MT][NT * 16];
};

// 16 MT entries from `first` on by a workgroup; its four wavefronts take every fourth chunk of the features, and join their sums in
// LDS.  Eight lanes load a row's 128 bytes; the lanes that multiply them get them through the wavefront's own part of LDS
// (unit u of row r at u ^ (r & 7), so that neither way meets its own banks; 6 rows, 3185 features, 32906 entries,
// bfloat16 81 us, straight into those lanes, 16 bytes of 16 rows a load, 111).
template <typename T, int NT, int MT>
__device__ __forceinline__ void few_logits(const XentFewLogitsArgs &a, int64_t first, int part, FewLds<NT, MT> &lds)
{
    using F = Few<T>;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int counted = a.scalars->counted, full = a.features / F::kChunk;
    const T *row[2 * MT];
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) {
        const int64_t v = first + 8 * j + (lane >> 3);
        row[j] = reinterpret_cast<const T *>(a.weight) + (v < a.vocab ? v : a.vocab - 1) * a.weight_stride;
    }
    Acc4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
    auto load = [&](int c, Quad (&w)[2 * MT]) {
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) w[j] = *reinterpret_cast<const quad_at_2 *>(row[j] + c * F::kChunk + F::kEach * (lane & 7));
    };
    // (a wavefront's LDS accesses are done in their order)
    auto settle = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    };
    auto stage = [&](const Quad (&w)[2 * MT]) {
        settle();
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) lds.staged[wave][8 * j + (lane >> 3)][(lane & 7) ^ (lane >> 3)] = w[j];
        settle();
    };
    auto multiply = [&](int c) {
        const Frag *h = reinterpret_cast<const Frag *>(a.by_feature + (int64_t)c * (F::kChunkFrags * NT * 1024)) + lane;
        Frag b[NT][F::kChunkFrags];
#pragma unroll
        for (int s = 0; s < F::kChunkFrags; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n) b[n][s] = h[(s * NT + n) * 64];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const Quad w[2] = {lds.staged[wave][16 * t + i][g ^ (i & 7)], lds.staged[wave][16 * t + i][(4 + g) ^ (i & 7)]};
            if constexpr (F::kFloat) {
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(w[k >> 2][k & 3]);
                Frag f[3];
                split_bf16(x, f);
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[t][n] = product_of(f, b[n], acc[t][n]);
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int s = 0; s < 2; ++s) acc[t][n] = mfma_few(__builtin_bit_cast(Frag, w[s]), b[n][s], acc[t][n]);
            }
        }
    };
    Quad now[2 * MT], then[2 * MT];
    int c = wave;
    if (c < full) load(c, now);
    if (c + 4 < full) load(c + 4, then);
    for (; c < full; c += 8) {
        stage(now);
        if (c + 8 < full) load(c + 8, now);
        multiply(c);
        if (c + 4 >= full) break;
        stage(then);
        if (c + 12 < full) load(c + 12, then);
        multiply(c + 4);
    }
    if (full * F::kChunk < a.features && (full & 3) == wave) {
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) now[j] = load_cut(row[j], full * F::kChunk + F::kEach * (lane & 7), a.features);
        stage(now);
        multiply(full);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) lds.sums[wave][t * NT + n][lane] = acc[t][n];
    __syncthreads();
    for (int k = wave; k < MT * NT; k += 4) {
        const int tile = k / NT, n = k % NT;
        Acc4 l = lds.sums[0][k][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) l += lds.sums[w][k][lane];
        const int place = n * 16 + i;
        const int64_t v = first + 16 * tile + 4 * g;
        if (place < counted) *reinterpret_cast<Acc4 *>(a.logits + place * a.stride + v) = l;
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (v + r >= a.vocab) l[r] = -INFINITY;
            top = fmaxf(top, l[r]);
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        float at = top == -INFINITY ? 0.0f : top;
        if (is_far(at)) {
            l = l - at;
            at = 0.0f;
        }
        const float from = -at * kLog2e;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(fmaf(l[r], kLog2e, from));
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lane < 16) lds.tops[tile][place] = make_float2(top, sum * rounded_off(at, from));
    }
    __syncthreads();
    if ((int)threadIdx.x >= counted) return;
    Joined all;
#pragma unroll
    for (int t = 0; t < MT; ++t) all.join(lds.tops[t][threadIdx.x]);
    a.partial[(int64_t)threadIdx.x * a.parts + part] = make_float2(all.top, all.sum);
}

// Workgroups of 64 entries, and behind them of 16 entries for those that would not fill the chip once more.  The weights' bytes
// bound it: 60 x 4096 x 65536 bfloat16 in 118 us (4.6 TB/s; without the narrow ones 162), 33 x 1843 x 67371 float in 171 (2.9
// TB/s; without 210; its split and six products leave the loads two workgroups a compute unit).
template <typename T, int NT>
__global__ __launch_bounds__(kFewThreads, 2) void xent_few_logits_kernel(XentFewLogitsArgs a)
{
    __shared__ FewLds<NT, 4> lds;
    const int id = blockIdx.x;
    if (id < a.wide) few_logits<T, NT, 4>(a, (int64_t)id * 64, id, lds);
    else few_logits<T, NT, 1>(a, (int64_t)a.wide * 64 + (int64_t)(id - a.wide) * 16, id, reinterpret_cast<FewLds<NT, 1> &>(lds));
}

template <typename T, int NT>
__global__ __launch_bounds__(kFewThreads, 2) void xent_few_narrow_logits_kernel(XentFewLogitsArgs a)
{
    __shared__ FewLds<NT, 1> lds;
    few_logits<T, NT, 1>(a, (int64_t)blockIdx.x * 16, blockIdx.x, lds);
}

struct XentFewJoinArgs {
    const float2 *partial;
    const float *logits;
    int64_t stride;
    const int *index, *position, *label;
    const XentScalars *scalars;
    int parts;
    float *lse, *losses;
};

// One workgroup a row.
__global__ __launch_bounds__(kFewThreads) void xent_few_join_kernel(XentFewJoinArgs a)
{
    __shared__ float2 waves[kFewThreads / 64];
    const int place = blockIdx.x;
    if (threadIdx.x == 0 && a.position[place] < 0) a.losses[place] = 0.0f;
    if (place >= a.scalars->counted) return;
    const float2 *partial = a.partial + (int64_t)place * a.parts;
    Joined all;
#pragma unroll 4
    for (int p = threadIdx.x; p < a.parts; p += kFewThreads) all.join(partial[p]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const float2 other = make_float2(__shfl_xor(all.top, d, 64), __shfl_xor(all.sum, d, 64));
        all.join(other);
    }
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = make_float2(all.top, all.sum);
    __syncthreads();
    if (threadIdx.x != 0) return;
    Joined row;
    for (int w = 0; w < kFewThreads / 64; ++w) row.join(waves[w]);
    const int label = a.label[place];
    const float lse = label < 0 ? __builtin_nanf("") : row.lse();
    a.lse[place] = lse;
    a.losses[a.index[place]] = label < 0 ? lse : lse - a.logits[place * a.stride + label];
}

// ---- d_l -------------------------------------------------------------------------------------------------------

struct XentFewDlArgs {
    const float *logits;
    int64_t stride, vocab;
    const float *lse;
    const int *index, *label;
    const XentScalars *scalars;
    XentGrad grad;
    char *by_entry;      // [32 entries][plane][tile]: d_hidden's operand
    char *by_row;        // [16 entries][32 rows][plane]: d_weight's
};

// 32 entries a workgroup, a wavefront a tile of 16 rows.  One gradient a row goes into d_l, a common one onto the sums.
// 33 rows of 67371 float entries: 10 us.
template <typename T, int NT>
__global__ __launch_bounds__(64 * NT) void xent_few_dl_kernel(XentFewDlArgs a)
{
    using F = Few<T>;
    constexpr int kSteps = (NT + 1) / 2;
    __shared__ uint16_t lds[F::kPlanes][NT * 16][32 + 2];
    const int tile = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, place = tile * 16 + i;
    const int64_t v = (int64_t)blockIdx.x * 32 + 8 * g;
    float x[8] = {};
    if (place < a.scalars->counted) {
        const float share = a.grad.each ? a.grad.grad[a.index[place]] : 1.0f;
        if (share != 0.0f) {
            const float far = is_far(a.lse[place]) ? a.lse[place] : 0.0f;
            const float lse = a.lse[place] - far, from = -lse * kLog2e, exact = rounded_off(lse, from);
            const int64_t label = a.label[place] - v;
            const Acc4 *l = reinterpret_cast<const Acc4 *>(a.logits + place * a.stride + v);
            const Acc4 lo = l[0] - far, hi = l[1] - far;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(fmaf(j < 4 ? lo[j & 3] : hi[j & 3], kLog2e, from)) * exact;
                x[j] = v + j < a.vocab ? (label == j ? p - 1.0f : p) * share : 0.0f;
            }
        }
    }
    Frag f[F::kPlanes];
    planes_of(x, f);
#pragma unroll
    for (int p = 0; p < F::kPlanes; ++p) {
        if (a.by_entry) *reinterpret_cast<Frag *>(a.by_entry + (((int64_t)blockIdx.x * F::kPlanes + p) * NT + tile) * 1024 + lane * 16) = f[p];
#pragma unroll
        for (int j = 0; j < 8; ++j) lds[p][place][8 * g + j] = (uint16_t)((uint32_t)f[p][j >> 1] >> (j & 1) * 16);
    }
    if (!a.by_row) return;
    __syncthreads();
    for (int k = tile; k < 2 * kSteps * F::kPlanes; k += NT) {
        const int p = k % F::kPlanes, step = k / F::kPlanes % kSteps, half = k / F::kPlanes / kSteps;
        Frag t = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int n = step * 32 + 8 * g + j;
            if (n < NT * 16) t[j >> 1] |= (int)((uint32_t)lds[p][n][16 * half + i] << (j & 1) * 16);
        }
        *reinterpret_cast<Frag *>(a.by_row + ((((int64_t)blockIdx.x * 2 + half) * kSteps + step) * F::kPlanes + p) * 1024 + lane * 16) = t;
    }
}

// ---- gradients -------------------------------------------------------------------------------------------------

struct XentFewGradArgs {
    const void *weight;
    int64_t weight_stride, vocab;
    int features, rows;
    const XentScalars *scalars;
    XentGrad grad;
    const char *by_entry, *by_row, *hidden;   // fragments of d_l, of d_l^T, of hidden^T
    int parts;                                // of the columns
    int splits_hidden, blocks_hidden;         // workgroups from 0 on make d_hidden's sums, the others d_weight
    int splits_weight;
    float *partial;                           // (splits_hidden, rows, features)
    void *d_weight;
};

// Sums over a run of entries (32 a step) of d_hidden's columns kCols part .. .
template <typename T, int NT>
__device__ __forceinline__ void few_d_hidden(const XentFewGradArgs &a, int part, int split)
{
    using F = Few<T>;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, col = part * F::kCols + F::kEach * i;
    const int64_t steps = (a.vocab + 31) / 32, begin = steps * split / a.splits_hidden, end = steps * (split + 1) / a.splits_hidden;
    // A load past its row's end reads the next row (those columns go nowhere); the last step's rows have none, and
    // rows shorter than a load or on top of each other not enough.  Lanes with no column at all read the first ones.
    const int64_t careful = a.features < F::kEach || a.weight_stride < a.features ? begin : steps - 1;
    const T *base = reinterpret_cast<const T *>(a.weight) + (col < a.features ? col : 0);
    Acc4 acc[F::kEach][NT];
#pragma unroll
    for (int t = 0; t < F::kEach; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
    auto load = [&](int64_t s, Quad (&w)[8]) {
        const T *p = base + (s * 32 + 8 * g) * a.weight_stride;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const quad_at_2 *>(p + j * a.weight_stride);
    };
    auto multiply = [&](int64_t s, const Quad (&w)[8]) {
        const Frag *d = reinterpret_cast<const Frag *>(a.by_entry + s * (F::kPlanes * NT * 1024)) + lane;
        Frag b[NT][F::kPlanes];
#pragma unroll
        for (int p = 0; p < F::kPlanes; ++p)
#pragma unroll
            for (int n = 0; n < NT; ++n) b[n][p] = d[(p * NT + n) * 64];
#pragma unroll
        for (int t = 0; t < F::kEach; ++t) {
            Frag f[F::kPlanes];
            if constexpr (F::kFloat) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j][t]);
                split_bf16(x, f);
            } else {
                // column t of two entries: their lower or their upper halves
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    f[0][j] = (int)__builtin_amdgcn_perm(w[2 * j + 1][t >> 1], w[2 * j][t >> 1], t & 1 ? 0x07060302u : 0x05040100u);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = product_of(b[n], f, acc[t][n]);
        }
    };
    Quad now[8], then[8];
    const int64_t whole = end < careful ? end : careful;
    int64_t s = begin;
    if (s < whole) load(s, now);
    for (; s < whole; s += 2) {
        if (s + 1 < whole) load(s + 1, then);
        multiply(s, now);
        if (s + 1 >= whole) break;
        if (s + 2 < whole) load(s + 2, now);
        multiply(s + 1, then);
    }
    for (s = whole; s < end; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t v = s * 32 + 8 * g + j;
            now[j] = load_cut(reinterpret_cast<const T *>(a.weight) + (v < a.vocab ? v : a.vocab - 1) * a.weight_stride, col, a.features);
        }
        multiply(s, now);
    }
    const int counted = a.scalars->counted;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int place = n * 16 + 4 * g + r;
            if (place >= counted) continue;
            float *out = a.partial + ((int64_t)split * a.rows + place) * a.features + col;
#pragma unroll
            for (int t = 0; t < F::kEach; t += 4) {
                const quad_at_4 q = {acc[t][n][r], acc[t + 1][n][r], acc[t + 2][n][r], acc[t + 3][n][r]};
                if (col + t + 4 <= a.features) {
                    *reinterpret_cast<quad_at_4 *>(out + t) = q;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + t + k < a.features) out[t + k] = q[k];
                }
            }
        }
}

// Columns kCols part .. of a run of d_weight's rows.
template <typename T, int NT>
__device__ __forceinline__ void few_d_weight(const XentFewGradArgs &a, int part, int split)
{
    using F = Few<T>;
    constexpr int kSteps = (NT + 1) / 2;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, col = part * F::kCols + F::kEach * i;
    const int64_t tiles = (a.vocab + 15) / 16, begin = tiles * split / a.splits_weight, end = tiles * (split + 1) / a.splits_weight;
    const float scale = a.grad.scale(a.scalars);
    const Frag *hidden = reinterpret_cast<const Frag *>(a.hidden) + (int64_t)part * (kSteps * F::kPlanes * F::kEach * 64) + lane;
    const Frag *d_l = reinterpret_cast<const Frag *>(a.by_row) + lane;
    Frag h[kSteps][F::kEach][F::kPlanes];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int t = 0; t < F::kEach; ++t)
#pragma unroll
            for (int p = 0; p < F::kPlanes; ++p) h[s][t][p] = hidden[((s * F::kPlanes + p) * F::kEach + t) * 64];
    Frag next[kSteps][F::kPlanes];
    auto load = [&](int64_t v) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int p = 0; p < F::kPlanes; ++p) next[s][p] = d_l[((v * kSteps + s) * F::kPlanes + p) * 64];
    };
    if (begin < end) load(begin);
    for (int64_t v = begin; v < end; ++v) {
        Frag d[kSteps][F::kPlanes];
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int p = 0; p < F::kPlanes; ++p) d[s][p] = next[s][p];
        if (v + 1 < end) load(v + 1);
        Acc4 acc[F::kEach];
#pragma unroll
        for (int t = 0; t < F::kEach; ++t) {
            acc[t] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) acc[t] = product_of(d[s], h[s][t], acc[t]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t row = v * 16 + 4 * g + r;
            if (row >= a.vocab) continue;
            T *out = reinterpret_cast<T *>(a.d_weight) + row * a.features + col;
            float x[F::kEach];
#pragma unroll
            for (int t = 0; t < F::kEach; ++t) x[t] = acc[t][r] * scale;
            if (col + F::kEach <= a.features) {
                if constexpr (F::kFloat) *reinterpret_cast<quad_at_4 *>(out) = quad_at_4{x[0], x[1], x[2], x[3]};
                else store8_whole(out, x);
            } else {
#pragma unroll
                for (int t = 0; t < F::kEach; ++t)
                    if (col + t < a.features) out[t] = (T)x[t];
            }
        }
    }
}

// Both gradients in one launch: neither needs the other, one reads while the other one writes.  The weights' bytes bound it,
// read and written once: 7 rows, 2109 features, 43964 entries, float 154 us (4.8 TB/s), 6 x 3185 x 32906 bfloat16 77 (5.4),
// 33 x 1843 x 67371 float 280 to 309 (3.2 .. 3.6); the sums behind them 9.
template <typename T, int NT>
__global__ __launch_bounds__(kFewThreads, 2) void xent_few_grad_kernel(XentFewGradArgs a)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x < a.blocks_hidden) {
        const int unit = blockIdx.x * 4 + wave;
        if (unit < a.parts * a.splits_hidden) few_d_hidden<T, NT>(a, unit % a.parts, unit / a.parts);
    } else {
        const int unit = ((int)blockIdx.x - a.blocks_hidden) * 4 + wave;
        if (unit < a.parts * a.splits_weight) few_d_weight<T, NT>(a, unit % a.parts, unit / a.parts);
    }
}

}  // namespace bf
