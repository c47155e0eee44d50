// Softmax cross entropy of logits = hidden weight^T over a large vocabulary, without the logits in memory:
//
//   loss_i = log sum_v exp(l_iv) - l_i,target(i),   l_iv = hidden_i . weight_v
//   d_l_iv = g_i (exp(l_iv - lse_i) - [v = target(i)]);  d_hidden = d_l weight;  d_weight = d_l^T hidden
//
// Forward: a matrix product whose workgroups keep their tile of logits in registers and leave, for each row,
// the maximum and the sum of exponentials over the tile's vocabulary; those are joined in ascending
// order.  Backward, vocabulary piece by piece: the tile again, its d_l in 16 bits to a piece-sized buffer, then
// two products with that buffer, d_hidden's partial sums over the pieces and d_weight's rows of the piece.
// 2 rows x vocabulary x features operations forward and 6 backward, all on the matrix units (matmul.hpp),
// which bound every call but those of a few rows (there the weights' bytes do).
//
// Rows whose target is ignored are left out before anything else: the others' hidden rows are gathered, so
// ignored ones cost nothing and what they hold (NaN too) reaches nothing.
//
// Number formats.  bfloat16 operands multiply as they are; d_l is rounded to bfloat16 (2^-9), like every gradient
// of such a model.  float operands are split, x 2^e = hi + lo in two float16 numbers of together 22 bits,
// e the power of two that brings the operand's largest number to 2^14 .. 2^15 (one for hidden, one for
// weight; d_l is at most one times the largest g, e = 15), and a product is hi lo + lo hi + hi hi with sums in float: three
// products at the 16-bit rate, 16 times that of float ones on this card, for a relative error of 2^-22 a factor, as long as
// numbers are within 2^-17 of the largest (below that an absolute error of 2^-39 of it).
#pragma once

#include "matmul.hpp"

namespace bf {

constexpr int kXentThreads = 1024;   // of the single-workgroup kernels

struct XentScalars {
    float hidden_scale, weight_scale;   // the powers of two
    float grad_scale;                   // largest |g_i| (d_l is kept over it)
    unsigned hidden_max, weight_max;    // bits of the largest magnitudes
    int counted;                        // rows whose target is not ignored
};

// ---- which rows count -----------------------------------------------------------------------------------

struct XentRowsArgs {
    const int64_t *target;
    int64_t rows, vocab, ignore;
    XentScalars *scalars;
    int *index;          // (rows) the counted rows in ascending order
    int *position;       // (rows) a row's place among them, -1: ignored
    int *label;          // (rows) by place: the target, -1 where it is no entry of the vocabulary
    float *picked;       // (rows) by place: NaN, for the target's logit; NULL: not wanted
};

__global__ __launch_bounds__(kXentThreads) void xent_rows_kernel(XentRowsArgs a)
{
    __shared__ int sums[kXentThreads / 64];
    const int64_t per = (a.rows + kXentThreads - 1) / kXentThreads, begin = threadIdx.x * per;
    const int64_t end = begin + per < a.rows ? begin + per : a.rows;
    int n = 0;
    for (int64_t i = begin; i < end; ++i) n += a.target[i] != a.ignore;
    int at = n;   // inclusive sum over the wavefront
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(at, d, 64);
        if ((int)(threadIdx.x & 63) >= d) at += v;
    }
    if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = at;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kXentThreads / 64; ++w) {
        if (w < (int)(threadIdx.x >> 6)) before += sums[w];
        total += sums[w];
    }
    at += before - n;
    for (int64_t i = begin; i < end; ++i) {
        const int64_t t = a.target[i];
        const bool in = t != a.ignore;
        a.position[i] = in ? at : -1;
        if (!in) continue;
        a.index[at] = (int)i;
        a.label[at] = t >= 0 && t < a.vocab ? (int)t : -1;
        if (a.picked) a.picked[at] = __builtin_nanf("");
        ++at;
    }
    if (threadIdx.x == 0) {
        a.scalars->counted = total;
        a.scalars->hidden_max = a.scalars->weight_max = 0;
        a.scalars->hidden_scale = a.scalars->weight_scale = a.scalars->grad_scale = 1.0f;
    }
}

// ---- operands in the form the products read ----------------------------------------------------------------

// Largest magnitude, as bits (any order of the additions gives the same).  index: the rows to look at.
__global__ __launch_bounds__(256) void xent_largest_kernel(const float *x, int64_t rows, int64_t cols, int64_t stride,
                                                           const int *index, const XentScalars *scalars, unsigned *largest)
{
    const int64_t n = index ? scalars->counted : rows;
    unsigned m = 0;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const float *row = x + (index ? index[r] : r) * stride;
        for (int64_t c = threadIdx.x; c < cols; c += 256) {
            const unsigned v = __float_as_uint(row[c]) & 0x7fffffffu;
            m = v > m ? v : m;
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned v = (unsigned)__shfl_xor((int)m, d, 64);
        m = v > m ? v : m;
    }
    if ((threadIdx.x & 63) == 0 && m > 0) atomicMax(largest, m);
}

// 2^e that brings the number to 2^14 .. 2^15 (infinite, NaN or zero: 1)
__device__ __forceinline__ float scale_of(unsigned bits)
{
    const int e = (int)(bits >> 23);
    if (bits == 0 || e == 255) return 1.0f;
    const int up = 14 - (e - 127);
    return __uint_as_float((unsigned)((up > 100 ? 100 : up) + 127) << 23);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float rest_f16(float v) { return v - (float)(_Float16)v; }

struct XentPackArgs {
    const void *x;
    char *out;              // rows of `stride` bytes, in F16 two planes
    int64_t rows, cols, x_stride, stride, plane;
    const int *index;       // rows to gather (the rest of the `rows` rows zeros); NULL: all
    XentScalars *scalars;
    int which;              // 0: hidden, 1: weight
};

// Rows gathered and padded with zeros up to the stride; float ones split in two.
template <typename T>
__global__ __launch_bounds__(256) void xent_pack_kernel(XentPackArgs a)
{
    constexpr bool F16 = sizeof(T) == 4;
    const int units = (int)(a.stride / 16);
    const int64_t n = a.index ? a.scalars->counted : a.rows;
    float scale = 1.0f;
    if constexpr (F16) {
        scale = scale_of(a.which ? a.scalars->weight_max : a.scalars->hidden_max);
        if (blockIdx.x == 0 && threadIdx.x == 0) (a.which ? a.scalars->weight_scale : a.scalars->hidden_scale) = scale;
    }
    const int64_t total = a.rows * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / units;
        const int col = (int)(i - r * units) * 8;
        float v[8];
        const T *row = reinterpret_cast<const T *>(a.x) + (a.index && r < n ? a.index[r] : r) * a.x_stride;
        load8(row, col, r < n ? (int)a.cols : 0, 0.0f, v);
        uint32_t w[4], low[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (F16) {
                w[k] = pack_f16(v[2 * k] * scale, v[2 * k + 1] * scale);
                low[k] = pack_f16(rest_f16(v[2 * k] * scale), rest_f16(v[2 * k + 1] * scale));
            } else {
                w[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
            }
        }
        char *out = a.out + r * a.stride + col * 2;
        *reinterpret_cast<uint4 *>(out) = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (F16) *reinterpret_cast<uint4 *>(out + a.plane) = make_uint4(low[0], low[1], low[2], low[3]);
    }
}

// ---- the logits' tiles --------------------------------------------------------------------------------------

struct XentTileArgs {
    MatOperand weight, hidden;
    const XentScalars *scalars;
    const int *label;
    int64_t rows;               // as laid out (an upper bound of the counted ones)
    int64_t vocab;              // entries from the operand's first on
    int64_t first;              // number of that one
    int features_steps;
    int tiles_m, tiles_n;
    // forward
    float2 *partial;            // (2 tiles_m, rows): maximum, sum
    float *picked;
    // backward
    const float *lse, *share;   // by place; share: g_i over the largest
    char *d_l;                  // (rows, stride bytes), in F16 two planes
    int64_t stride, plane;
};

// Tile of workgroup `id`: the XCDs (workgroups go to them in turn) get runs of neighbouring tiles, so that those
// that share rows of an operand share an L2.
__device__ __forceinline__ int xcd_order(int id, int total)
{
    const int per = total / 8, over = total % 8, xcd = id % 8, at = id / 8;
    return xcd * per + (xcd < over ? xcd : over) + at;
}

// Tiles in bands of `band` rows of the grid, each band walked column by column.
__device__ __forceinline__ void tile_at(int id, int tiles_m, int tiles_n, int band, int &tm, int &tn)
{
    const int per = band * tiles_n, b = id / per, in = id - b * per;
    const int height = tiles_m - b * band < band ? tiles_m - b * band : band;
    tm = b * band + in % height;
    tn = in / height;
}

template <bool F16, int BM, int BN, bool BACKWARD>
__global__ __launch_bounds__(kMatThreads, 1) void xent_logits_kernel(XentTileArgs a)
{
    using Tile = MatTile<kRows, kRows, F16, BM, BN, true>;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int counted = a.scalars->counted;
    int tm, tn;
    tile_at(xcd_order(blockIdx.x, a.tiles_m * a.tiles_n), a.tiles_m, a.tiles_n, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    if (n0 >= counted) return;
    Acc4 acc[Tile::kMT][Tile::kNT];
    Tile::run(a.weight, a.hidden, m0, n0, 0, a.features_steps, lds, acc);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = wave >> 1;
    // (powers of two, each within the range of float)
    const float scale_h = F16 ? 1.0f / a.scalars->hidden_scale : 1.0f, scale_w = F16 ? 1.0f / a.scalars->weight_scale : 1.0f;
    const int mw = m0 + part * (BM / 2);
#pragma unroll
    for (int j = 0; j < Tile::kNT; ++j) {
        const int row = n0 + (wave & 1) * (BN / 2) + j * 16 + (lane & 15);
        const bool there = row < counted;
        const int label = there ? a.label[row] - (int)a.first : -1;
        if constexpr (!BACKWARD) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int v = mw + Tile::tile_row(i) + r;
                    if constexpr (F16) acc[i][j][r] = acc[i][j][r] * scale_h * scale_w;
                    if (v == label && there) a.picked[row] = acc[i][j][r];
                    if (v < a.vocab) top = fmaxf(top, acc[i][j][r]);
                }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            // (NaN is no maximum, and an infinite one would make NaN of its own term: both show in the sum)
            const float from = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (mw + Tile::tile_row(i) + r < a.vocab) sum += __expf(acc[i][j][r] - from);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (lane < 16 && there) a.partial[(int64_t)(2 * tm + part) * a.rows + row] = make_float2(top, sum);
        } else {
            const float lse = there ? a.lse[row] : 0.0f, share = there ? a.share[row] : 0.0f;
#pragma unroll
            for (int i = 0; i < Tile::kMT; ++i) {
                const int v0 = mw + Tile::tile_row(i);
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float l = (F16 ? acc[i][j][r] * scale_h * scale_w : acc[i][j][r]) - lse;
                    p[r] = F16 ? expf(l) : __expf(l);
                    if (v0 + r == label) p[r] -= 1.0f;
                    p[r] = v0 + r < a.vocab && share != 0.0f ? p[r] * share : 0.0f;
                    if constexpr (F16) p[r] *= 32768.0f;
                }
                char *out = a.d_l + (int64_t)row * a.stride + v0 * 2;
                if constexpr (F16) {
                    *reinterpret_cast<uint2 *>(out) = make_uint2(pack_f16(p[0], p[1]), pack_f16(p[2], p[3]));
                    *reinterpret_cast<uint2 *>(out + a.plane) =
                        make_uint2(pack_f16(rest_f16(p[0]), rest_f16(p[1])), pack_f16(rest_f16(p[2]), rest_f16(p[3])));
                } else {
                    *reinterpret_cast<uint2 *>(out) = make_uint2(pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]));
                }
            }
        }
    }
}

// ---- a row's log-sum-exp and loss ------------------------------------------------------------------------------

struct XentJoinArgs {
    const float2 *partial;
    const float *picked;
    const int *position;
    int64_t rows;
    int parts;
    float *lse, *losses;    // (rows), as the caller numbers them; zero where ignored
};

// 16 rows and 16 runs of partials a workgroup
__global__ __launch_bounds__(256) void xent_join_kernel(XentJoinArgs a)
{
    __shared__ float2 lds[16][17];
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
    const int run = threadIdx.x >> 4, at = row < a.rows ? a.position[row] : -1;
    const int per = (a.parts + 15) / 16, end = (run + 1) * per < a.parts ? (run + 1) * per : a.parts;
    float top = -INFINITY, sum = 0.0f;
    auto join = [&](float2 p) {
        if (p.x > top) {
            sum = sum * __expf(top - p.x) + p.y;
            top = p.x;
        } else {
            // (all of them minus infinity, or NaN: their sums say so)
            sum += p.x == top || p.x == -INFINITY ? p.y : p.y * __expf(p.x - top);
        }
    };
    if (at >= 0)
        for (int p = run * per; p < end; ++p) join(a.partial[(int64_t)p * a.rows + at]);
    lds[run][threadIdx.x & 15] = make_float2(top, sum);
    __syncthreads();
    if (run != 0 || row >= a.rows) return;
    top = -INFINITY;
    sum = 0.0f;
    for (int i = 0; i < 16; ++i) join(lds[i][threadIdx.x]);
    const float lse = (top == -INFINITY ? 0.0f : top) + logf(sum);
    a.lse[row] = at >= 0 ? lse : 0.0f;
    a.losses[row] = at >= 0 ? lse - a.picked[at] : 0.0f;
}

// loss = the sum of the rows' (over the counted ones, `mean`), in a fixed order
__global__ __launch_bounds__(kXentThreads) void xent_total_kernel(const float *losses, int64_t rows, const XentScalars *scalars,
                                                                  int mean, float *loss)
{
    __shared__ float sums[kXentThreads / 64];
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < rows; i += kXentThreads) s += losses[i];
    s = lanes_sum<64>(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = 0.0f;
    for (int w = 0; w < kXentThreads / 64; ++w) s += sums[w];
    *loss = mean ? s / (float)scalars->counted : s;
}

// ---- backward: what each row's d_l is multiplied by ---------------------------------------------------------------

struct XentShareArgs {
    const float *grad;      // one number, or one a row (each)
    const float *lse;       // (rows), as the caller numbers them
    const int *index, *label;
    XentScalars *scalars;
    int each, mean;
    float *share, *lse_at;  // by place
};

__global__ __launch_bounds__(kXentThreads) void xent_share_kernel(XentShareArgs a)
{
    __shared__ float sums[kXentThreads / 64];
    const int n = a.scalars->counted;
    float most = 0.0f;
    if (a.each) {
        for (int i = threadIdx.x; i < n; i += kXentThreads) most = fmaxf(most, fabsf(a.grad[a.index[i]]));
#pragma unroll
        for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = most;
        __syncthreads();
        for (int w = 0; w < kXentThreads / 64; ++w) most = fmaxf(most, sums[w]);
    } else {
        most = n == 0 ? 0.0f : a.mean ? *a.grad / (float)n : *a.grad;
    }
    if (threadIdx.x == 0) a.scalars->grad_scale = most;
    for (int i = threadIdx.x; i < n; i += kXentThreads) {
        float s = 1.0f;
        if (a.each) s = most == 0.0f ? a.grad[a.index[i]] : a.grad[a.index[i]] / most;   // (zeros and NaN only)
        a.share[i] = a.label[i] < 0 ? __builtin_nanf("") : s;
        a.lse_at[i] = a.lse[a.index[i]];
    }
}

// ---- backward: the gradients' products -----------------------------------------------------------------------------

struct XentGradArgs {
    MatOperand a, b;            // a: what is multiplied with d_l, along m; b: d_l
    const XentScalars *scalars;
    int64_t m, n;               // sizes of the result (n rows of m)
    int tiles_m, tiles_n;
    int steps, splits;          // k steps in all (d_weight: an upper bound), parts they are cut into
    int add;                    // sums are added to what is there
    float *partial;             // (splits, n, m), or
    void *out;                  // (n, m) dense in T
};

// d_hidden: n are rows, k the vocabulary (d_l row by row); d_weight: n the vocabulary, k the counted rows
template <typename T, MatLayout LB, int BM, int BN>
__global__ __launch_bounds__(kMatThreads, 1) void xent_grad_kernel(XentGradArgs a)
{
    constexpr bool F16 = sizeof(T) == 4, OF_WEIGHT = LB == kCols;
    using Tile = MatTile<kCols, LB, F16, BM, BN, false>;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int counted = a.scalars->counted;
    const int tiles = a.tiles_m * a.tiles_n, split = blockIdx.x / tiles;
    int tm, tn;
    tile_at(xcd_order(blockIdx.x % tiles, tiles), a.tiles_m, a.tiles_n, 8, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    if (!OF_WEIGHT && n0 >= counted) return;
    const int steps = OF_WEIGHT ? (counted + kMatK - 1) / kMatK : a.steps;
    const int per = (steps + a.splits - 1) / a.splits, first = split * per;
    const int count = steps - first < per ? steps - first : per;
    Acc4 acc[Tile::kMT][Tile::kNT];
    Tile::run(a.a, a.b, m0, n0, first, count, lds, acc);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float scale = a.scalars->grad_scale;
    if constexpr (F16) scale *= 1.0f / 32768.0f / (OF_WEIGHT ? a.scalars->hidden_scale : a.scalars->weight_scale);
#pragma unroll
    for (int j = 0; j < Tile::kNT; ++j) {
        const int64_t row = n0 + (wave & 1) * (BN / 2) + j * 16 + (lane & 15);
        if (row >= (OF_WEIGHT ? a.n : (int64_t)counted)) continue;
#pragma unroll
        for (int i = 0; i < Tile::kMT; ++i) {
            const int64_t m = m0 + (wave >> 1) * (BM / 2) + Tile::tile_row(i);
            if (m >= a.m) continue;
            if (a.out) {
                T *out = reinterpret_cast<T *>(a.out) + row * a.m + m;
                const Acc4 v = acc[i][j] * scale;
                if (m + 4 <= a.m) {
                    if constexpr (F16) {
                        *reinterpret_cast<quad_at_4 *>(out) = quad_at_4{v[0], v[1], v[2], v[3]};
                    } else {
                        typedef uint32_t pair_at_2 __attribute__((ext_vector_type(2), aligned(2)));
                        *reinterpret_cast<pair_at_2 *>(out) = pair_at_2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (m + r < a.m) out[r] = (T)v[r];
                }
            } else {
                float *out = a.partial + ((int64_t)split * a.n + row) * a.m + m;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < a.m) out[r] = (a.add ? out[r] : 0.0f) + acc[i][j][r];
            }
        }
    }
}

struct XentGatherArgs {
    const float *partial;       // (splits, n, m)
    const int *position;        // rows of the result come from these places (-1: zeros); NULL: as they are
    const XentScalars *scalars;
    void *out;
    int64_t rows, n, m;         // rows of the result, of a split
    int splits, of_weight;
};

// The splits' sums in ascending order, scaled and rounded once.
template <typename T>
__global__ __launch_bounds__(256) void xent_gather_kernel(XentGatherArgs a)
{
    constexpr bool F16 = sizeof(T) == 4;
    float scale = a.scalars->grad_scale;
    if constexpr (F16) scale *= 1.0f / 32768.0f / (a.of_weight ? a.scalars->hidden_scale : a.scalars->weight_scale);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = a.position ? a.position[row] : row;
        T *out = reinterpret_cast<T *>(a.out) + row * a.m;
        for (int64_t m = threadIdx.x; m < a.m; m += 256) {
            float s = 0.0f;
            if (at >= 0) {
                for (int p = 0; p < a.splits; ++p) s += a.partial[((int64_t)p * a.n + at) * a.m + m];
                s *= scale;
            }
            out[m] = (T)s;
        }
    }
}

}  // namespace bf
