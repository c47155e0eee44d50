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
// which bound every call but those of a few rows (there the weights' bytes do: xent_few.hpp).
// Measured at 8192 rows (7370 of them counted), 1024 features, 32768 entries, bfloat16: 1890 us forward and backward, of which
// the logits take 499 (0.99 PFLOP/s), d_l 2 x 258 (two pieces; the same product and 2 x 241 MB written), d_hidden 2 x
// 244, d_weight 2 x 220, everything else 50.  At 2000 (1800) x 1000 x 30001, float: 1452 us: 367, 402, 331, 347 (three products
// each: 0.81 to 0.98 PFLOP/s), the largest numbers and the copies in two planes 88.
//
// Rows whose target is ignored are left out before anything else: the others' hidden rows are gathered, so
// what ignored ones hold (NaN too) reaches nothing, and they cost nothing but the tiles that the counted ones leave unfilled.
//
// Number formats.  bfloat16 operands multiply as they are; d_l is rounded to bfloat16 (2^-9), like every gradient
// of such a model.  float operands are split, x 2^e = hi + lo in two float16 numbers of together 22 bits,
// e the power of two that brings the operand's largest number to 2^14 .. 2^15 (one for hidden, one for
// weight; d_l is at most one, e = 15), and a product is hi lo + lo hi + hi hi with sums in float: three
// products at the 16-bit rate, 16 times that of float ones on this card, for a relative error of 2^-22 a factor.  The lower
// halves are kept times 2^11: numbers from 2^-28 of the largest up have their 22 bits, from 2^-40 eleven, below 2^-51 none.
// With one gradient a row d_l is without it in float (rows of small ones would lose their bits): d_hidden's rows are multiplied
// at the end, and d_weight's product takes hidden's rows times their share of the largest.
#pragma once

#include "matmul.hpp"

namespace bf {

constexpr int kXentThreads = 1024;   // of the single-workgroup kernels

struct XentScalars {
    float hidden_scale, weight_scale;   // the powers of two
    float grad_scale;                   // one gradient a row: the largest finite |g_i| (shares are kept over it)
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
    float *picked;       // (rows) by place: NaN, for the target's logit
};

// 8192 rows a round, eight times 64 neighbours a wavefront: 5.3 us for 8192 rows (latencies; one workgroup).
__global__ __launch_bounds__(kXentThreads) void xent_rows_kernel(XentRowsArgs a)
{
    constexpr int kEach = 8, kWaves = kXentThreads / 64;
    __shared__ int sums[2][kWaves];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int done = 0, turn = 0;
    for (int64_t from = 0; from < a.rows; from += kXentThreads * kEach, turn ^= 1) {
        const int64_t begin = from + wave * (64 * kEach) + lane;
        int64_t t[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) t[k] = begin + 64 * k < a.rows ? a.target[begin + 64 * k] : a.ignore;
        uint64_t counts[kEach];
        int n = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            counts[k] = __ballot(t[k] != a.ignore);
            n += __popcll(counts[k]);
        }
        if (lane == 0) sums[turn][wave] = n;
        __syncthreads();
        int at = done;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int v = sums[turn][w];
            if (w < wave) at += v;
            done += v;
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int64_t row = begin + 64 * k;
            const bool in = counts[k] >> lane & 1;
            const int place = at + __popcll(counts[k] & ((1ull << lane) - 1));
            if (row < a.rows) a.position[row] = in ? place : -1;
            if (in) {
                a.index[place] = (int)row;
                a.label[place] = t[k] >= 0 && t[k] < a.vocab ? (int)t[k] : -1;
                a.picked[place] = __builtin_nanf("");
            }
            at += __popcll(counts[k]);
        }
    }
    if (threadIdx.x == 0) {
        a.scalars->counted = done;
        a.scalars->hidden_max = a.scalars->weight_max = 0;
        a.scalars->hidden_scale = a.scalars->weight_scale = a.scalars->grad_scale = 1.0f;
    }
}

// ---- operands in the form the products read ----------------------------------------------------------------

// Largest magnitude of the finite numbers, as bits (any order gives the same): what is not finite stays so under any scale,
// and the others keep theirs.  index: the rows to look at.  Memory bounds it: 35 us for 120 MB (3.4 TB/s).
__global__ __launch_bounds__(256) void xent_largest_kernel(const float *x, int64_t rows, int64_t cols, int64_t stride,
                                                           const int *index, const XentScalars *scalars, unsigned *largest)
{
    __shared__ unsigned lds[4];
    const int units = (int)((cols + 7) / 8);
    const int64_t total = (index ? scalars->counted : rows) * units;
    unsigned m = 0;
#pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / units;
        float v[8];
        load8(x + (index ? index[r] : r) * stride, (int)(i - r * units) * 8, (int)cols, 0.0f, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const unsigned b = __float_as_uint(v[k]) & 0x7fffffffu;
            m = b > m && b < 0x7f800000u ? b : m;
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned v = (unsigned)__shfl_xor((int)m, d, 64);
        m = v > m ? v : m;
    }
    // (all of them go to one address, one after another: one a workgroup, and none where a larger number is there)
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 4; ++w) m = lds[w] > m ? lds[w] : m;
    if (m > __hip_atomic_load(largest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(largest, m);
}

// 2^e that brings the number to 2^14 .. 2^15 (zero: 1)
__device__ __forceinline__ float scale_of(unsigned bits)
{
    const int e = (int)(bits >> 23);
    if (bits == 0) return 1.0f;
    const int up = 14 - (e - 127);
    return __uint_as_float((unsigned)((up > 100 ? 100 : up) + 127) << 23);
}

// Two numbers' upper and lower float16 halves, the lower ones times 2^kRaised.  The numbers are hidden from the compiler: rounded from the
// product that made one of them, not from the number itself, an upper half could be another one than
// the lower half is the rest to.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &high, uint32_t &low)
{
    constexpr float kFactor = 1 << kRaised;
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    asm("" : "+v"(a), "+v"(b));
    const f16x2 h = {(_Float16)a, (_Float16)b};
    const f16x2 l = {(_Float16)((a - (float)h[0]) * kFactor), (_Float16)((b - (float)h[1]) * kFactor)};
    high = __builtin_bit_cast(uint32_t, h);
    low = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ float whole(_Float16 high, _Float16 low) { return fmaf((float)low, 1.0f / (1 << kRaised), (float)high); }

struct XentPackArgs {
    const void *x;
    char *out;              // rows of `stride` bytes, in F16 two planes
    int64_t rows, cols, x_stride, stride, plane;
    const int *index;       // rows to gather (the rest of the `rows` rows zeros); NULL: all
    XentScalars *scalars;
    int which;              // 0: hidden, 1: weight
};

// Rows gathered and padded with zeros up to the stride; float ones split in two.  Memory bounds it: 258 MB of float read and
// as many written in 82 us (6.3 TB/s).
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
                split_f16(v[2 * k] * scale, v[2 * k + 1] * scale, w[k], low[k]);
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

struct XentGrad {
    const float *grad;      // one number, or one a row (each)
    int each, mean;

    __device__ __forceinline__ float scale(const XentScalars *s) const
    {
        if (each) return s->grad_scale;
        return s->counted == 0 ? 0.0f : mean ? *grad / (float)s->counted : *grad;
    }
};

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
    const float *lse, *share;   // by place; share NULL: ones; float: only whether it is zero
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

constexpr float kLog2e = 1.44269504088896340736f;

// exp(l - v) is formed as exp2(l log2(e) + from), from = -v log2(e) rounded; the factor that undoes the rounding.
__device__ __forceinline__ float rounded_off(float v, float from) { return __builtin_amdgcn_exp2f(-fmaf(v, kLog2e, from)); }

// Beyond it that factor, 2^(half a unit of v log2(e)), would itself pass the range (from 2^31 on): there v is taken off first.
__device__ __forceinline__ bool is_far(float v) { return fabsf(v) > 0x1p24f && fabsf(v) < INFINITY; }

// Workgroups stay for tile after tile (grid: as many as the chip holds at a time), so that a tile's exponentials and
// stores run while the next one's operands arrive: 512 rows (461 counted), 4096 features, 65536 entries, bfloat16 in 230 us
// (1.08 PFLOP/s; 1.20 with the rows that only fill up a tile), 572 (515) x 2659 x 24269 float by small tiles in 271.
template <bool F16, int BM, int BN, int BUFFERS, bool BACKWARD>
__global__ __launch_bounds__(mat_threads(BM, BN, BUFFERS), 1) void xent_logits_kernel(XentTileArgs a)
{
    using Tile = MatTiles<kRows, kRows, F16, BM, BN, BUFFERS, true>;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int counted = a.scalars->counted;
    const int tiles_n = (counted + BN - 1) / BN, total = a.tiles_m * tiles_n;
    const int lane = threadIdx.x & 63, part = Tile::wave_m();
    // (powers of two, each within the range of float, and their product where the logits are)
    const float scale = F16 ? 1.0f / a.scalars->hidden_scale * (1.0f / a.scalars->weight_scale) : 1.0f;
    if ((int)blockIdx.x >= total) return;
    Tile tiles(a.weight, a.hidden, lds);
    int ahead = blockIdx.x;
    auto next = [&](int &m, int &n, int &first, int &count) {
        if (ahead >= total) return false;
        int tm, tn;
        tile_at(xcd_order(ahead, total), a.tiles_m, tiles_n, 8, tm, tn);
        m = tm * BM;
        n = tn * BN;
        first = 0;
        count = a.features_steps;
        ahead += gridDim.x;
        return true;
    };
    tiles.begin(next);
    for (int id = blockIdx.x; id < total; id += gridDim.x) {
        Acc4 acc[Tile::kMT][Tile::kNT];
        tiles.run(a.features_steps, next, acc);
        int tm, tn;
        tile_at(xcd_order(id, total), a.tiles_m, tiles_n, 8, tm, tn);
        const int n0 = tn * BN, mw = tm * BM + part * Tile::kPartM, of = Tile::kWavesM * tm + part;
        const bool whole = mw + Tile::kPartM <= a.vocab;   // no entry past the vocabulary's end
#pragma unroll
        for (int j = 0; j < Tile::kNT; ++j) {
            const int row = n0 + Tile::wave_n() * Tile::kPartN + j * 16 + (lane & 15);
            const bool there = row < counted;
            // the label's place among the wavefront's entries, if it is one of them
            const int label = there ? a.label[row] - (int)a.first - mw : -1;
            const bool labelled = __any(label >= 0 && label < Tile::kPartM);
            if constexpr (F16) {
#pragma unroll
                for (int i = 0; i < Tile::kMT; ++i) acc[i][j] = acc[i][j] * scale;
            }
            if constexpr (!BACKWARD) {
                if (labelled) {
#pragma unroll
                    for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (Tile::tile_row(i) + r == label) a.picked[row] = acc[i][j][r];
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (mw + Tile::tile_row(i) + r >= a.vocab) acc[i][j][r] = -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < Tile::kMT; ++i)
                    top = fmaxf(fmaxf(fmaxf(top, acc[i][j][0]), fmaxf(acc[i][j][1], acc[i][j][2])), acc[i][j][3]);
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                // (NaN is no maximum, and an infinite one would make NaN of its own term: both show in the sum)
                float at = top == -INFINITY ? 0.0f : top;
                if (__any(is_far(at))) {
#pragma unroll
                    for (int i = 0; i < Tile::kMT; ++i) acc[i][j] = acc[i][j] - at;
                    at = 0.0f;
                }
                const float from = -at * kLog2e;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], kLog2e, from));
                sum += __shfl_xor(sum, 16, 64);
                sum += __shfl_xor(sum, 32, 64);
                if (lane < 16 && there) a.partial[(int64_t)of * a.rows + row] = make_float2(top, sum * rounded_off(at, from));
            } else {
                const float share = there ? a.share ? a.share[row] : 1.0f : 0.0f;
                // (no share: the exponentials of minus infinity, zeros)
                float lse = share != 0.0f ? a.lse[row] : INFINITY;
                if (__any(is_far(lse))) {
                    const float off = is_far(lse) ? lse : 0.0f;
#pragma unroll
                    for (int i = 0; i < Tile::kMT; ++i) acc[i][j] = acc[i][j] - off;
                    lse -= off;
                }
                const float from = -lse * kLog2e;
                const float exact = share != 0.0f ? rounded_off(lse, from) : 1.0f;
#pragma unroll
                for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], kLog2e, from));
                if (labelled) {
#pragma unroll
                    for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (Tile::tile_row(i) + r == label && share != 0.0f) acc[i][j][r] -= 1.0f / exact;
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < Tile::kMT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (mw + Tile::tile_row(i) + r >= a.vocab) acc[i][j][r] = 0.0f;
                }
                const float factor = F16 ? share != 0.0f ? 32768.0f * exact : 0.0f : share * exact;
                char *out = a.d_l + (int64_t)row * a.stride + (mw + Tile::tile_row(0)) * 2;
                // sixteen neighbouring entries from four tiles
#pragma unroll
                for (int i = 0; i < Tile::kMT; i += 4) {
                    uint32_t w[8], low[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const Acc4 p = acc[i + k][j] * factor;
                        if constexpr (F16) {
                            split_f16(p[0], p[1], w[2 * k], low[2 * k]);
                            split_f16(p[2], p[3], w[2 * k + 1], low[2 * k + 1]);
                        } else {
                            w[2 * k] = pack_bf16(p[0], p[1]);
                            w[2 * k + 1] = pack_bf16(p[2], p[3]);
                        }
                    }
                    uint4 *to = reinterpret_cast<uint4 *>(out + i / 4 * 128);
                    to[0] = make_uint4(w[0], w[1], w[2], w[3]);
                    to[1] = make_uint4(w[4], w[5], w[6], w[7]);
                    if constexpr (F16) {
                        uint4 *below = reinterpret_cast<uint4 *>(out + a.plane + i / 4 * 128);
                        below[0] = make_uint4(low[0], low[1], low[2], low[3]);
                        below[1] = make_uint4(low[4], low[5], low[6], low[7]);
                    }
                }
            }
        }
    }
    Tile::end();
}

// ---- a row's log-sum-exp and loss ------------------------------------------------------------------------------

// The maximum of parts of a row and the sum of exponentials over it.
struct Joined {
    float top = -INFINITY, sum = 0.0f;

    __device__ __forceinline__ void join(float2 p)
    {
        if (p.x > top) {
            sum = sum * __expf(top - p.x) + p.y;
            top = p.x;
        } else {
            // (all of them minus infinity, or NaN: their sums say so)
            sum += p.x == top || p.x == -INFINITY ? p.y : p.y * __expf(p.x - top);
        }
    }
    __device__ __forceinline__ float lse() const { return (top == -INFINITY ? 0.0f : top) + logf(sum); }
};

struct XentJoinArgs {
    const float2 *partial;
    const float *picked;
    const int *position, *label;
    int64_t rows;
    int parts;
    float *lse;             // (rows) by place; NaN where the target is no entry of the vocabulary, so all that follows is
    float *losses;          // (rows), as the caller numbers them; zero where ignored
};

// 8 rows and 128 runs of their parts a workgroup (rows are neighbours in memory): 13 us for 8192 rows in 256 parts, by runs
// of a sixteenth of the parts 65 rows in 1924 parts took 27, now 11.
__global__ __launch_bounds__(1024) void xent_join_kernel(XentJoinArgs a)
{
    __shared__ float2 lds[16][8];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 3;
    const int64_t row = (int64_t)blockIdx.x * 8 + (lane & 7);
    const int at = row < a.rows ? a.position[row] : -1;
    Joined all;
    if (at >= 0) {
        const int end = (int)((int64_t)a.parts * (run + 1) / 128);
#pragma unroll 4
        for (int p = (int)((int64_t)a.parts * run / 128); p < end; ++p) all.join(a.partial[(int64_t)p * a.rows + at]);
    }
#pragma unroll
    for (int d = 8; d < 64; d *= 2) all.join(make_float2(__shfl_down(all.top, d, 64), __shfl_down(all.sum, d, 64)));
    if (lane < 8) lds[threadIdx.x >> 6][lane] = make_float2(all.top, all.sum);
    __syncthreads();
    if (threadIdx.x >= 8 || row >= a.rows) return;
    Joined whole;
    for (int i = 0; i < 16; ++i) whole.join(lds[i][threadIdx.x]);
    const float lse = whole.lse();
    if (at >= 0) a.lse[at] = a.label[at] < 0 ? __builtin_nanf("") : lse;
    a.losses[row] = at >= 0 ? lse - a.picked[at] : 0.0f;
}

// loss = the sum of the rows' (over the counted ones, `mean`), in a fixed order
__global__ __launch_bounds__(kXentThreads) void xent_total_kernel(const float *losses, int64_t rows, const XentScalars *scalars,
                                                                  int mean, float *loss)
{
    __shared__ float sums[kXentThreads / 64];
    float s = 0.0f;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < rows; i += kXentThreads) s += losses[i];
    s = lanes_sum<64>(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = 0.0f;
    for (int w = 0; w < kXentThreads / 64; ++w) s += sums[w];
    *loss = mean ? s / (float)scalars->counted : s;
}

// ---- backward: what the rows' d_l are multiplied by ---------------------------------------------------------------
// g_i = scale share_i.  One gradient for all: shares of one.  One a row: scale is the largest finite |g_i| (one that is not
// finite stays its row's own).
__global__ __launch_bounds__(kXentThreads) void xent_share_kernel(XentGrad g, const int *index, XentScalars *scalars, float *share)
{
    __shared__ float sums[kXentThreads / 64];
    const int n = scalars->counted;
    float most = 0.0f;
    for (int i = threadIdx.x; i < n; i += kXentThreads) {
        const float v = fabsf(g.grad[index[i]]);
        most = v < INFINITY ? fmaxf(most, v) : most;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = most;
    __syncthreads();
    for (int w = 0; w < kXentThreads / 64; ++w) most = fmaxf(most, sums[w]);
    if (threadIdx.x == 0) scalars->grad_scale = most;
    // (none but zeros: the numbers themselves)
    for (int i = threadIdx.x; i < n; i += kXentThreads) share[i] = most == 0.0f ? g.grad[index[i]] : g.grad[index[i]] / most;
}

// Hidden's two planes times the rows' shares, zeros behind the counted rows (float).
struct XentSharedArgs {
    const char *hidden;
    char *out;
    int64_t rows, stride, plane;
    const float *share;
    const XentScalars *scalars;
};

__global__ __launch_bounds__(256) void xent_shared_kernel(XentSharedArgs a)
{
    const int units = (int)(a.stride / 16), counted = a.scalars->counted;
    const int64_t total = a.rows * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / units, at = i * 16;
        uint32_t w[4] = {}, low[4] = {};
        if (r < counted) {
            const float share = a.share[r];
            const f16x8 h = *reinterpret_cast<const f16x8 *>(a.hidden + at), l = *reinterpret_cast<const f16x8 *>(a.hidden + a.plane + at);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                split_f16(whole(h[2 * k], l[2 * k]) * share, whole(h[2 * k + 1], l[2 * k + 1]) * share, w[k], low[k]);
        }
        *reinterpret_cast<uint4 *>(a.out + at) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4 *>(a.out + a.plane + at) = make_uint4(low[0], low[1], low[2], low[3]);
    }
}

// ---- backward: the gradients' products -----------------------------------------------------------------------------

struct XentGradArgs {
    MatOperand a, b;            // a: what is multiplied with d_l, along m; b: d_l
    const XentScalars *scalars;
    XentGrad grad;
    int64_t m, n;               // sizes of the result (n rows of m)
    int tiles_m, tiles_n;
    int steps, splits;          // k steps in all (d_weight: an upper bound), parts they are cut into
    int add;                    // sums are added to what is there
    float *partial;             // (splits, n, m), or
    void *out;                  // (n, m) dense in T
};

// Parts of at least one step.
__device__ __forceinline__ int xent_splits(int splits, int steps) { return splits < steps ? splits : steps > 1 ? steps : 1; }

// d_hidden: n are rows, k the vocabulary (d_l row by row); d_weight: n the vocabulary, k the counted rows.  Where the
// result has few tiles its k steps are cut into parts whose sums the gather adds: 65 rows, 91 features, 123157 entries,
// float, d_hidden in one tile by 240 workgroups takes 31 us and 12 for the gather, by 32 it took 142 and 20.
template <typename T, MatLayout LB, int BM, int BN, int BUFFERS>
__global__ __launch_bounds__(mat_threads(BM, BN, BUFFERS), 1) void xent_grad_kernel(XentGradArgs a)
{
    constexpr bool F16 = sizeof(T) == 4, OF_WEIGHT = LB == kCols;
    using Tile = MatTiles<kCols, LB, F16, BM, BN, BUFFERS, false>;
    __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
    const int counted = a.scalars->counted;
    const int tiles_n = OF_WEIGHT ? a.tiles_n : (counted + BN - 1) / BN, tiles = a.tiles_m * tiles_n;
    const int steps = OF_WEIGHT ? (counted + kMatK - 1) / kMatK : a.steps;
    const int splits = xent_splits(a.splits, steps), total = tiles * splits;
    const int lane = threadIdx.x & 63;
    float scale = a.grad.scale(a.scalars);
    if constexpr (F16) scale *= 1.0f / 32768.0f / (OF_WEIGHT ? a.scalars->hidden_scale : a.scalars->weight_scale);
    if ((int)blockIdx.x >= total) return;
    Tile tile(a.a, a.b, lds);
    auto place = [&](int id, int &tm, int &tn, int &split, int &first, int &count) {
        const int at = xcd_order(id, total);
        split = at / tiles;
        tile_at(at - split * tiles, a.tiles_m, tiles_n, 8, tm, tn);
        first = (int)((int64_t)steps * split / splits);
        count = (int)((int64_t)steps * (split + 1) / splits) - first;
    };
    int ahead = blockIdx.x;
    auto next = [&](int &m, int &n, int &first, int &count) {
        if (ahead >= total || steps == 0) return false;
        int tm, tn, split;
        place(ahead, tm, tn, split, first, count);
        m = tm * BM;
        n = tn * BN;
        ahead += gridDim.x;
        return true;
    };
    tile.begin(next);
    for (int id = blockIdx.x; id < total; id += gridDim.x) {
        int tm, tn, split, first, count;
        place(id, tm, tn, split, first, count);
        Acc4 acc[Tile::kMT][Tile::kNT];
        tile.run(count, next, acc);
        const int m0 = tm * BM, n0 = tn * BN;
        float *partial = a.partial + (int64_t)split * a.n * a.m;
#pragma unroll
        for (int j = 0; j < Tile::kNT; ++j) {
            const int64_t row = n0 + Tile::wave_n() * Tile::kPartN + j * 16 + (lane & 15);
            if (row >= (OF_WEIGHT ? a.n : (int64_t)counted)) continue;
#pragma unroll
            for (int i = 0; i < Tile::kMT; ++i) {
                const int64_t m = m0 + Tile::wave_m() * Tile::kPartM + Tile::tile_row(i);
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
                    float *out = partial + row * a.m + m;
                    if (m + 4 <= a.m) {
                        quad_at_4 v = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                        if (a.add) v += *reinterpret_cast<quad_at_4 *>(out);
                        *reinterpret_cast<quad_at_4 *>(out) = v;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < a.m) out[r] = (a.add ? out[r] : 0.0f) + acc[i][j][r];
                    }
                }
            }
        }
    }
    Tile::end();
}

// d_weight of no rows at all
template <typename T>
__global__ __launch_bounds__(256) void xent_zero_kernel(T *out, int64_t count)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) out[i] = (T)0.0f;
}

struct XentGatherArgs {
    const float *partial;       // (splits, n, m)
    const int *position;        // rows of the result come from these places (-1: zeros); NULL: as they are
    const XentScalars *scalars;
    XentGrad grad;
    void *out;
    int64_t rows, n, m;         // rows of the result, of a split
    int splits, of_weight;
    const float *row_grad;      // what each row of the result is multiplied by instead of grad's; NULL: nothing
};

// The splits' sums in ascending order, scaled and rounded once: eight neighbours a thread.  Memory bounds it: 8 splits of
// 2000 x 1000 in 18 us (4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void xent_gather_kernel(XentGatherArgs a)
{
    constexpr bool F16 = sizeof(T) == 4;
    float scale = a.row_grad ? 1.0f : a.grad.scale(a.scalars);
    if constexpr (F16) scale *= 1.0f / 32768.0f / (a.of_weight ? a.scalars->hidden_scale : a.scalars->weight_scale);
    const int splits = a.of_weight ? xent_splits(a.splits, (a.scalars->counted + kMatK - 1) / kMatK) : a.splits;
    const int m = (int)a.m, units = (m + 7) / 8;
    const int64_t total = a.rows * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / units, at = a.position ? a.position[row] : row;
        const int col = (int)(i - row * units) * 8;
        float s[8] = {};
        if (at >= 0) {
            for (int p = 0; p < splits; ++p) {
                float v[8];
                load8(a.partial + ((int64_t)p * a.n + at) * m, col, m, 0.0f, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) s[k] += v[k];
            }
            const float row_grad = a.row_grad ? a.row_grad[row] : 1.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k] = s[k] * scale * row_grad;
        }
        store8(reinterpret_cast<T *>(a.out) + row * m, col, m, s);
    }
}

// The same for d_hidden's rows in many splits: 128 columns of a row a workgroup, 32 runs of the splits side by side, each and
// then all of them in ascending order.  SCALED: by the powers of two of the product's operands.
template <typename T, bool SCALED>
__global__ __launch_bounds__(1024) void xent_gather_runs_kernel(XentGatherArgs a)
{
    __shared__ Acc4 lds[32][32];
    const int m = (int)a.m, run = threadIdx.x >> 5, col = blockIdx.x * 128 + (threadIdx.x & 31) * 4;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const int at = a.position[row];
        Acc4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (at >= 0 && col < m) {
            const int begin = a.splits * run / 32, end = a.splits * (run + 1) / 32;
            const float *p = a.partial + (int64_t)at * m + col;
            const int64_t stride = a.n * m;
            if (col + 4 <= m) {
#pragma unroll 8
                for (int k = begin; k < end; ++k) s += Acc4(*reinterpret_cast<const quad_at_4 *>(p + k * stride));
            } else {
                for (int k = begin; k < end; ++k)
                    for (int c = 0; c < 4; ++c)
                        if (col + c < m) s[c] += p[k * stride + c];
            }
        }
        __syncthreads();
        lds[run][threadIdx.x & 31] = s;
        __syncthreads();
        if (run != 0 || col >= m) continue;
#pragma unroll 4
        for (int k = 1; k < 32; ++k) s += lds[k][threadIdx.x];
        float scale = a.row_grad ? 1.0f : a.grad.scale(a.scalars);
        if constexpr (SCALED) scale *= 1.0f / 32768.0f / a.scalars->weight_scale;
        s = s * scale * (a.row_grad ? a.row_grad[row] : 1.0f);
        T *out = reinterpret_cast<T *>(a.out) + row * m + col;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (col + c < m) out[c] = at >= 0 ? (T)s[c] : (T)0.0f;
    }
}

}  // namespace bf
