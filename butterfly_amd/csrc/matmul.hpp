// Matrix products on the matrix units, for the loss of xent.hpp: out[n][m] = sum over k of A[m][k] B[n][k], 16-bit
// operands, sums in float.  Each operand lies in memory either with k adjacent (kRows: its row m or n holds the k's)
// or with m / n adjacent (kCols: its row k holds them), so the three products of a loss (logits, gradients
// of the hidden rows and of the weights) take hidden, weight and the logits' gradient as they are, and
// none is transposed.
//
// A workgroup of four wavefronts makes a BM x BN tile, each wavefront a quarter of it as 16 x 16 MFMA tiles
// (K = 32), out of k steps of 64 that lie in LDS twice: while one is used the next one is on its way, by
// 16-byte loads straight into LDS that hold no registers.  LDS reads bound a wavefront's tile before the matrix
// units do unless it is large: at 128 x 128 a step takes 1024 clocks of LDS reads (four wavefronts,
// 128 bytes a clock) beside 2048 of MFMA, at 64 x 64 as many as of MFMA.
//
// 16-byte units are placed in LDS so that no read meets another one's banks: kRows, unit u of row r at u ^ (r & 7);
// kCols, at u ^ 2 s(r) with s(r) = (r & 3) + 4 ((r >> 3) & 1), read four k's at a time through the
// transposing LDS load (within 16 lanes, lane 4 k + q asks for four columns of row k and lane j receives
// column j of four rows).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vec8.hpp"

namespace bf {

typedef int MatDesc __attribute__((ext_vector_type(4)));
typedef int Frag __attribute__((ext_vector_type(4)));
typedef float Acc4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char LdsByte;

constexpr int kMatK = 64;          // k's of a step
constexpr int kMatThreads = 256;

enum MatLayout { kRows, kCols };

// Values in two f16 halves (hi + lo) are two planes; a product then runs over hi lo + lo hi + hi hi.
struct MatOperand {
    const char *base;      // element (0, 0) of the first plane
    int64_t plane;         // bytes between planes
    int64_t stride;        // bytes between rows
    int64_t bytes;         // of a plane from base on that may be read: loads beyond are zero
};

__device__ __forceinline__ void load_unit_to_lds(MatDesc desc, unsigned lds_addr, int voff, int soff)
{
    int keep_m0;
    asm volatile("s_mov_b32 %0, m0\n\t"
                 "s_mov_b32 m0, %1\n\t"
                 "s_nop 0\n\t"
                 "buffer_load_dwordx4 %2, %3, %4 offen lds\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(keep_m0)
                 : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(voff), "s"(desc), "s"(soff)
                 : "memory");
}

// One operand's way into LDS: SIZE rows or columns of it, k step by k step.
template <MatLayout LAYOUT, int SIZE, bool SPREAD>
struct MatFeed {
    static constexpr int kLoads = SIZE / 32;                 // of a wavefront a step
    static constexpr int kUnits = SIZE / 8;                  // kCols: 16-byte units of a k row
    static constexpr int kPerLoad = LAYOUT == kRows ? 8 : 64 / kUnits;   // rows that a load covers
    static constexpr int kVariants = LAYOUT == kRows ? 1 : 4;
    const char *at;
    int64_t left;
    int stride, wave;
    int voff[kVariants];

    __device__ __forceinline__ void init(const MatOperand &o, int first)
    {
        const int lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        stride = (int)o.stride;
        if constexpr (LAYOUT == kRows) {
            // SPREAD: LDS row 16 t + i holds row 64 (t / 4) + 16 (i / 4) + 4 (t % 4) + i % 4, so that the
            // four rows a lane gets of each of four tiles' results are sixteen neighbours
            const int row = SPREAD ? (lane >> 5) * 16 + ((lane >> 3) & 3) : lane >> 3;
            voff[0] = row * stride + ((lane & 7) ^ (lane >> 3)) * 16;
        } else {
            const int row = lane / kUnits, unit = lane % kUnits;
#pragma unroll
            for (int v = 0; v < 4; ++v) voff[v] = row * stride + ((unit ^ (place(v, row) << 1)) * 16);
        }
        start(o, first, 0);
    }

    // s(r) of the rows that load number j of a wavefront covers, as far as it depends on j (v) and the lane's row
    static __device__ __forceinline__ int place(int v, int row)
    {
        return kPerLoad == 2 ? ((v & 1) * 2 + row) | (v >> 1) << 2 : row | (v & 1) << 2;
    }
    static constexpr int variant(int j)
    {
        return LAYOUT == kRows ? 0 : kPerLoad == 2 ? (j & 1) | (j >> 2 & 1) << 1 : j >> 1 & 1;
    }

    // to k step `step`, SIZE rows or columns from `first` on
    __device__ __forceinline__ void start(const MatOperand &o, int first, int64_t step, int plane = 0)
    {
        const int64_t skip = LAYOUT == kRows ? first * o.stride + step * (kMatK * 2) : step * kMatK * o.stride + (int64_t)first * 2;
        at = o.base + plane * o.plane + skip;
        left = o.bytes - skip;
    }

    __device__ __forceinline__ void issue(unsigned lds)
    {
        const unsigned long long a = (unsigned long long)at;
        MatDesc d;
        d.x = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
        d.y = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff));
        d.z = __builtin_amdgcn_readfirstlane((int)(left < 0 ? 0 : left < 0x7fffff00 ? left : 0x7fffff00));
        d.w = 0x00020000;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int jj = wave * kLoads + j;
            const int row = LAYOUT == kRows && SPREAD ? (jj >> 3) * 64 + (jj & 1) * 32 + ((jj >> 1) & 3) * 4 : jj * kPerLoad;
            load_unit_to_lds(d, lds + jj * 1024, voff[variant(j)], row * stride);
        }
        const int64_t step = LAYOUT == kRows ? kMatK * 2 : (int64_t)kMatK * stride;
        at += step;
        left -= step;
    }
};

// One operand's way out of LDS: the wavefront's 16-wide tiles of a half step (32 k's).
template <MatLayout LAYOUT, int SIZE>
struct MatReader {
    static constexpr int kTiles = SIZE / 32;
    unsigned addr[LAYOUT == kRows ? 2 : kTiles];

    // offset: of the operand in a buffer
    __device__ __forceinline__ void init(unsigned offset, int part)
    {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
        if constexpr (LAYOUT == kRows) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                addr[half] = offset + (part * kTiles * 16 + i) * 128 + (((g + 4 * half) ^ (i & 7)) * 16);
        } else {
            const int kk = i >> 2, q = i & 3, s = kk | (g & 1) << 2;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                addr[t] = offset + (8 * g + kk) * (SIZE * 2) + (((part * kTiles + t) ^ s) * 32) + (q >> 1) * 16 + (q & 1) * 8;
        }
    }

    template <int HALF>
    __device__ __forceinline__ void read(LdsByte *buffer, Frag (&f)[kTiles]) const
    {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if constexpr (LAYOUT == kRows) {
                f[t] = *(__attribute__((address_space(3))) const Frag *)(buffer + addr[HALF] + t * 2048);
            } else {
                typedef short Quad16 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) Quad16 LdsQuad;
                LdsByte *a = buffer + addr[t] + HALF * 32 * SIZE * 2;
                const Quad16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad *)a);
                const Quad16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad *)(a + 4 * SIZE * 2));
                typedef short Oct16 __attribute__((ext_vector_type(8)));
                f[t] = __builtin_bit_cast(Frag, (Oct16)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        }
    }
};

template <bool F16>
__device__ __forceinline__ Acc4 mfma(Frag a, Frag b, Acc4 c)
{
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The tile at (m0, n0) over k steps first .. first + count - 1 (count may be zero).  acc[mt][nt][r] is element
// (m, n) with n = n0 + BN / 2 * (wave & 1) + 16 nt + lane % 16 and m = m0 + BM / 2 * (wave >> 1) + what
// tile_row() says.  F16: both operands in two planes.
template <MatLayout LA, MatLayout LB, bool F16, int BM, int BN, bool SPREAD>
struct MatTile {
    static constexpr int kMT = BM / 32, kNT = BN / 32;
    static constexpr int kBytesA = BM * kMatK * 2, kBytesB = BN * kMatK * 2, kBuffer = kBytesA + kBytesB;
    static constexpr int kLds = 2 * kBuffer;

    // m of result r of tile mt, from the wavefront's first
    static __device__ __forceinline__ int tile_row(int mt)
    {
        const int g = (threadIdx.x & 63) >> 4;
        return SPREAD ? (mt >> 2) * 64 + g * 16 + (mt & 3) * 4 : mt * 16 + g * 4;
    }

    static __device__ __forceinline__ void run(const MatOperand &a, const MatOperand &b, int m0, int n0, int64_t first,
                                               int count, char *lds_bytes, Acc4 (&acc)[kMT][kNT])
    {
        LdsByte *near = (LdsByte *)lds_bytes;
        const unsigned lds = (unsigned)(unsigned long long)near;
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int j = 0; j < kNT; ++j) acc[i][j] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
        const int steps = count * (F16 ? 3 : 1);
        if (steps <= 0) return;
        MatFeed<LA, BM, SPREAD> feed_a;
        MatFeed<LB, BN, false> feed_b;
        feed_a.init(a, m0);
        feed_b.init(b, n0);
        MatReader<LA, BM> read_a;
        MatReader<LB, BN> read_b;
        read_a.init(0, wave >> 1);
        read_b.init(kBytesA, wave & 1);
        int pass = 0, fed = 0;
        auto feed = [&](unsigned buffer) {
            if (fed == 0) {
                // (the small products first)
                feed_a.start(a, m0, first, F16 && pass == 1);
                feed_b.start(b, n0, first, F16 && pass == 0);
            }
            feed_a.issue(lds + buffer);
            feed_b.issue(lds + buffer + kBytesA);
            if (++fed == count) {
                fed = 0;
                ++pass;
            }
        };
        auto arrive = [&] {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        Frag fa[2][kMT], fb[2][kNT];
        feed(0);
        arrive();
        if (steps > 1) feed(kBuffer);
        read_a.template read<0>(near, fa[0]);
        read_b.template read<0>(near, fb[0]);
        for (int step = 0; step < steps; ++step) {
            const unsigned buffer = (unsigned)(step & 1) * kBuffer;
            read_a.template read<1>(near + buffer, fa[1]);
            read_b.template read<1>(near + buffer, fb[1]);
#pragma unroll
            for (int i = 0; i < kMT; ++i)
#pragma unroll
                for (int j = 0; j < kNT; ++j) acc[i][j] = mfma<F16>(fa[0][i], fb[0][j], acc[i][j]);
            // this buffer is read, the other one's loads have landed, for all four wavefronts
            __builtin_amdgcn_sched_barrier(0);
            arrive();
            if (step + 2 < steps) feed(buffer);
            if (step + 1 < steps) {
                read_a.template read<0>(near + kBuffer - buffer, fa[0]);
                read_b.template read<0>(near + kBuffer - buffer, fb[0]);
            }
#pragma unroll
            for (int i = 0; i < kMT; ++i)
#pragma unroll
                for (int j = 0; j < kNT; ++j) acc[i][j] = mfma<F16>(fa[1][i], fb[1][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

}  // namespace bf
