// Matrix products on the matrix units, for the loss of xent.hpp: out[n][m] = sum over k of A[m][k] B[n][k], 16-bit
// operands, sums in float.  Each operand lies in memory either with k adjacent (kRows: its row m or n holds the k's)
// or with m / n adjacent (kCols: its row k holds them), so the three products of a loss (logits, gradients
// of the hidden rows and of the weights) take hidden, weight and the logits' gradient as they are, and
// none is transposed.
//
// A workgroup makes a BM x BN tile, each wavefront a part of it as 16 x 16 MFMA tiles (K = 32), out of k steps of 64
// that lie in LDS in two to four buffers: while one is used the others are on their way, by 16-byte loads straight into LDS
// that hold no registers.  LDS reads bound a wavefront's part before the matrix units do unless it is large: a
// step of 256 x 256 tiles by eight wavefronts (128 x 64 each) takes 1536 clocks of LDS reads (128 bytes a clock) beside 2048
// of MFMA, of 128 x 128 by four (64 x 64) 512 beside 512, which is why large tiles are taken wherever
// there are enough of them.
//
// What bounds it: the matrix units at the clock that the card's power leaves them.  7370 x 1024 x 32768 in bfloat16 runs at
// 0.99 PFLOP/s (logits, exponentials included), 1.01 (d_hidden), 1.12 (d_weight), a library's products of 8192 rows
// at 1.05, 1.29 and 1.47, the same MFMAs without any load at 1.5.  Steps of 32 in four buffers, loads in clumps, other row
// orders and a stride off the powers of two changed nothing by more than 3%.
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

// Wavefronts of a workgroup, two along m: those of a large tile, or of a small one that has a compute unit to itself
// (four buffers), are two on each SIMD, so that one of them computes while the other one's loads and reads are
// taken; small tiles of two buffers leave room for two workgroups a compute unit instead.
constexpr int mat_waves(int bm, int bn, int buffers) { return bm * bn >= 256 * 256 || buffers > 2 ? 8 : 4; }
constexpr int mat_threads(int bm, int bn, int buffers) { return 64 * mat_waves(bm, bn, buffers); }

enum MatLayout { kRows, kCols };

// Values in two f16 halves (hi + lo) are two planes; a product then runs over hi lo + lo hi + hi hi.  The lower halves are kept
// times 2^kRaised, so that they reach further below the upper ones; the sums of the first two products are divided by it.
constexpr int kRaised = 11;

struct MatOperand {
    const char *base;      // element (0, 0) of the first plane
    int64_t plane;         // bytes between planes
    int64_t stride;        // bytes between rows
    int64_t bytes;         // of a plane from base on that may be read: loads beyond are zero
    int tail;              // kRows, the first operand: bytes of a row's last k step that are the row's, a multiple of 16; the
                           // others of 128 are zero
};

constexpr int kWholeTail = kMatK * 2;

// lds_addr: where the wavefront's 64 units go (wave-uniform); offset: from the descriptor's base, within 2^31, the sum of a
// lane's and of the load's own.  The sum is in the lane's register when the load is made: what an instruction adds from a
// scalar register itself takes no part in the range check.  It is formed in these lines, or the compiler keeps a register
// for every load's.
// (m0 is not saved: nothing else in these kernels uses it, and the compiler is told; its warning is that it
// will not keep it for anybody either; with the move of m0 and the sum five wait states, which a descriptor needs that a
// lane's read has just brought to scalar registers, and which the compiler does not count in front of these lines)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_unit_to_lds(MatDesc desc, unsigned lds_addr, int lane_offset, int load_offset)
{
    int offset;
    asm volatile("s_mov_b32 m0, %1\n\t"
                 "v_add_u32_e32 %0, %4, %2\n\t"
                 "s_nop 2\n\t"
                 "buffer_load_dwordx4 %0, %3, 0 offen lds"
                 : "=&v"(offset)
                 : "s"(lds_addr), "v"(lane_offset), "s"(desc), "s"(load_offset)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Where the loads of one operand read, SIZE rows or columns of it, k step by k step: numbers alone, which the host can go
// through as well.  From step to step only the lanes' offsets move (a wavefront that is alone on its SIMD has few
// instructions to spare between MFMAs); the base moves every steps() steps, before they pass 2^30.
template <MatLayout LAYOUT, int SIZE, bool SPREAD, int WAVES>
struct MatPath {
    static constexpr int kLoads = SIZE / 8 / WAVES;          // of a wavefront a step
    static constexpr int kUnits = SIZE / 8;                  // kCols: 16-byte units of a k row
    static constexpr int kPerLoad = LAYOUT == kRows ? 8 : 64 / kUnits;   // rows that a load covers
    static constexpr int kVariants = LAYOUT == kRows ? 1 : kLoads;
    int stride, first_offset[kVariants], lane_offset[kVariants], load_offset[kLoads];   // a load's: the same in all lanes

    __host__ __device__ __forceinline__ void init(int64_t stride_, int wave, int lane)
    {
        stride = (int)stride_;
        if constexpr (LAYOUT == kRows) {
            // SPREAD: LDS row 16 t + i holds row 64 (t / 4) + 16 (i / 4) + 4 (t % 4) + i % 4, so that the
            // four rows a lane gets of each of four tiles' results are sixteen neighbours
            const int row = SPREAD ? (lane >> 5) * 16 + ((lane >> 3) & 3) : lane >> 3;
            first_offset[0] = row * stride + ((lane & 7) ^ (lane >> 3)) * 16;
        } else {
            const int row = lane / kUnits;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int r = (wave * kLoads + j) * kPerLoad + row, s = (r & 3) | ((r >> 3) & 1) << 2;
                first_offset[j] = row * stride + (lane % kUnits ^ s << 1) * 16;
            }
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int jj = wave * kLoads + j;
            load_offset[j] = (LAYOUT == kRows && SPREAD ? (jj >> 3) * 64 + (jj & 1) * 32 + ((jj >> 1) & 3) * 4 : jj * kPerLoad) * stride;
        }
    }

    // steps that one base serves
    __host__ __device__ __forceinline__ int steps() const
    {
        const int n = LAYOUT == kRows ? 1 << 20 : (1 << 30) / (kMatK * stride) - 1;
        return n > 1 ? n : 1;
    }

    // To k step `step`, SIZE rows or columns from `first` on: the base's distance from the operand's, and in `left` the
    // bytes from there on that may be read (loads beyond are zeros; `nothing`: all of them).
    __host__ __device__ __forceinline__ int64_t start(const MatOperand &o, int first, int64_t step, bool nothing, int &left)
    {
        const int64_t skip = LAYOUT == kRows ? first * o.stride + step * (kMatK * 2) : step * kMatK * o.stride + (int64_t)first * 2;
        const int64_t rest = nothing ? 0 : o.bytes - skip;
        left = (int)(rest < 0 ? 0 : rest < 0x7fffff00 ? rest : 0x7fffff00);
#pragma unroll
        for (int v = 0; v < kVariants; ++v) lane_offset[v] = first_offset[v];
        return skip;
    }
    // In front of a row's last k step: the lanes whose unit lies behind the row's end read nothing (in rows that lie as a
    // caller has them there may be anything, NaN too, which the other operand's zeros would not undo).
    __host__ __device__ __forceinline__ void cut(const MatOperand &o, int lane)
    {
        if constexpr (LAYOUT == kRows) {
            if (((lane & 7) ^ (lane >> 3)) * 16 >= o.tail) lane_offset[0] = kRefused;
        }
    }
    static constexpr int kRefused = (int)0x80000000u;   // (as the range check takes it: behind everything, with a load's own offset too)
    static constexpr __host__ __device__ int variant(int j) { return LAYOUT == kRows ? 0 : j; }
    // of load j, as the range check sees it
    __host__ __device__ __forceinline__ int offset(int j) const { return lane_offset[variant(j)] + load_offset[j]; }
    __host__ __device__ __forceinline__ void advance()
    {
#pragma unroll
        for (int v = 0; v < kVariants; ++v) lane_offset[v] += LAYOUT == kRows ? kMatK * 2 : kMatK * stride;
    }
};

// One operand's way into LDS.
template <MatLayout LAYOUT, int SIZE, bool SPREAD, int WAVES>
struct MatFeed {
    MatPath<LAYOUT, SIZE, SPREAD, WAVES> path;
    int wave;
    MatDesc desc;

    __device__ __forceinline__ void init(const MatOperand &o)
    {
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        path.init(o.stride, wave, threadIdx.x & 63);
    }
    __device__ __forceinline__ int steps() const { return path.steps(); }
    __device__ __forceinline__ void start(const MatOperand &o, int first, int64_t step, int plane, bool nothing)
    {
        int left;
        const int64_t skip = path.start(o, first, step, nothing, left);
        const unsigned long long a = (unsigned long long)(o.base + plane * o.plane + skip);
        desc.x = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
        desc.y = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff));
        desc.z = __builtin_amdgcn_readfirstlane(left);
        desc.w = 0x00020000;
    }
    __device__ __forceinline__ void load(unsigned lds, int j) const
    {
        const unsigned to = lds + (wave * path.kLoads + j) * 1024;
        load_unit_to_lds(desc, to, path.lane_offset[path.variant(j)], path.load_offset[j]);
    }
    __device__ __forceinline__ void advance() { path.advance(); }
    // (the lane's number made anew: no register holds it until here)
    __device__ __forceinline__ void cut(const MatOperand &o)
    {
        if (LAYOUT == kRows && o.tail < kWholeTail) path.cut(o, __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)));
    }
};

// One operand's way out of LDS: the wavefront's 16-wide tiles of a half step (32 k's).
template <MatLayout LAYOUT, int SIZE, int PARTS>
struct MatReader {
    static constexpr int kTiles = SIZE / 16 / PARTS;
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
    __device__ __forceinline__ Frag read(LdsByte *buffer, int t) const
    {
        if constexpr (LAYOUT == kRows) {
            return *(__attribute__((address_space(3))) const Frag *)(buffer + addr[HALF] + t * 2048);
        } else {
            typedef short Quad16 __attribute__((ext_vector_type(4)));
            typedef short Oct16 __attribute__((ext_vector_type(8)));
            typedef __attribute__((address_space(3))) Quad16 LdsQuad;
            LdsByte *a = buffer + addr[t] + HALF * 32 * SIZE * 2;
            const Quad16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad *)a);
            const Quad16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad *)(a + 4 * SIZE * 2));
            return __builtin_bit_cast(Frag, (Oct16)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// c += a b, the sums in accumulation registers: as builtins the compiler moves every one of 256 of them
// to ordinary registers and back once a step.  What it then no longer sees: two wait states between a vector
// instruction that writes an operand and the MFMA that reads it (mfma_operand, behind which an operand is where
// its MFMAs read it), and those between the last MFMA and the first read of its sums (mfma_settle; a sum's next
// MFMA is kMT kNT of them away).
template <bool F16>
__device__ __forceinline__ void mfma(Frag a, Frag b, Acc4 &c)
{
    if constexpr (F16) asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

__device__ __forceinline__ void mfma_operand(Frag &f) { asm volatile("s_nop 1" : "+v"(f)); }

template <int MT, int NT>
__device__ __forceinline__ void mfma_settle(Acc4 (&acc)[MT][NT])
{
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    // (every sum passes through here: none is read in front of it)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// Tiles of BM x BN, one after another, as one stream of k steps: while a step is computed the one after the next is
// asked for, across the boundary between two tiles too, so the next tile's first steps arrive while the
// sums of the one before are dealt with.  acc[mt][nt][r] is element (m, n) with n = n0 + kPartN wave_n() + 16 nt +
// lane % 16 and m = m0 + kPartM wave_m() + what tile_row() says.  F16: both operands in two planes.
template <MatLayout LA, MatLayout LB, bool F16, int BM, int BN, int BUFFERS, bool SPREAD>
struct MatTiles {
    static constexpr int kWaves = mat_waves(BM, BN, BUFFERS), kWavesM = 2, kWavesN = kWaves / kWavesM;
    static constexpr int kPartM = BM / kWavesM, kPartN = BN / kWavesN;     // a wavefront's part
    static constexpr int kMT = kPartM / 16, kNT = kPartN / 16, kPasses = F16 ? 3 : 1;
    static constexpr int kBytesA = BM * kMatK * 2, kBytesB = BN * kMatK * 2, kBuffer = kBytesA + kBytesB;
    static constexpr int kLds = BUFFERS * kBuffer;
    static constexpr int kLoadsA = BM / 8 / kWaves, kLoads = (BM + BN) / 8 / kWaves;
    static_assert(kMT >= kNT && kLoads % kMT == 0, "reads and loads are dealt out to rows of MFMAs");

    // m of result r of tile mt, from the wavefront's first
    static __device__ __forceinline__ int tile_row(int mt)
    {
        const int g = (threadIdx.x & 63) >> 4;
        return SPREAD ? (mt >> 2) * 64 + g * 16 + (mt & 3) * 4 : mt * 16 + g * 4;
    }

    // The wavefront's part of a tile.
    static __device__ __forceinline__ int wave_m() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kWavesN; }
    static __device__ __forceinline__ int wave_n() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWavesN; }

    const MatOperand &a, &b;
    LdsByte *near;
    unsigned lds, buffer = 0;
    MatFeed<LA, BM, SPREAD, kWaves> feed_a;
    MatFeed<LB, BN, false, kWaves> feed_b;
    MatReader<LA, BM, kWavesM> read_a;
    MatReader<LB, BN, kWavesN> read_b;
    Frag fa[2][kMT], fb[2][kNT];
    // the tile that is asked for: its place, its first k step, their number; how far it is asked for
    int m0 = 0, n0 = 0, first = 0, count = 0, pass = kPasses - 1, fed = 0, until = 0;

    __device__ __forceinline__ MatTiles(const MatOperand &a_, const MatOperand &b_, char *lds_bytes)
        : a(a_), b(b_), near((LdsByte *)lds_bytes), lds((unsigned)(unsigned long long)(LdsByte *)lds_bytes)
    {
        feed_a.init(a);
        feed_b.init(b);
        read_a.init(0, wave_m());
        read_b.init(kBytesA, wave_n());
    }

    // next(m0, n0, first, count): the next tile (count >= 1), or false when there is none
    template <typename Next>
    __device__ __forceinline__ void feed_begin(Next &next)
    {
        if (fed == until) {
            if (fed == count) {
                fed = 0;
                if (++pass == kPasses) {
                    pass = 0;
                    if (!next(m0, n0, first, count)) count = 0x7fffffff;
                }
            }
            // (the small products first; behind the last tile loads of nothing)
            const bool nothing = count == 0x7fffffff;
            feed_a.start(a, m0, first + (nothing ? 0 : fed), F16 && pass == 1, nothing);
            feed_b.start(b, n0, first + (nothing ? 0 : fed), F16 && pass == 0, nothing);
            until = min(count - fed, min(feed_a.steps(), feed_b.steps())) + fed;
        }
        // (float operands and b have rows of whole steps)
        if (++fed == count && !F16) feed_a.cut(a);
    }
    __device__ __forceinline__ void feed_load(unsigned to, int i)
    {
        if (i < kLoadsA) feed_a.load(lds + to, i);
        else feed_b.load(lds + to + kBytesA, i - kLoadsA);
    }
    __device__ __forceinline__ void feed_end()
    {
        feed_a.advance();
        feed_b.advance();
    }

    template <typename Next>
    __device__ __forceinline__ void feed(unsigned to, Next &next)
    {
        feed_begin(next);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) feed_load(to, i);
        feed_end();
    }

    static __device__ __forceinline__ void barrier()
    {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    // Before the first step.
    template <typename Next>
    __device__ __forceinline__ void begin(Next &next)
    {
#pragma unroll
        for (int i = 0; i < BUFFERS; ++i) feed(i * kBuffer, next);
        // (the later steps' loads may still be on their way)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads *(BUFFERS - 1)) : "memory");
        barrier();
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
            fa[0][i] = read_a.template read<0>(near, i);
            if (i < kNT) fb[0][i] = read_b.template read<0>(near, i);
        }
    }

    // Behind the last step: no load may write LDS that is another workgroup's.
    static __device__ __forceinline__ void end() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

    // One k step.  Reads and loads are spread between the MFMAs, which take 16 clocks each and wait for nothing
    // but their operands: in front of each row of kNT of them one or two reads, and in the second half kLoads / kMT loads.
    template <typename Next>
    __device__ __forceinline__ void step(Next &next, Acc4 (&acc)[kMT][kNT])
    {
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
            fa[1][i] = read_a.template read<1>(near + buffer, i);
            if (i < kNT) fb[1][i] = read_b.template read<1>(near + buffer, i);
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < kNT; ++j) mfma_operand(fb[0][j]);
            }
            mfma_operand(fa[0][i]);
#pragma unroll
            for (int j = 0; j < kNT; ++j) mfma<F16>(fa[0][i], fb[0][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        // This buffer is read, the next one's loads have landed, for all wavefronts.  Memory operations complete in order here, so the
        // count stays right beside others that it does not know (stores of a tile's end, registers that the compiler keeps in
        // scratch memory): with them in front or behind, it waits for more.
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads *(BUFFERS - 2)) : "memory");
        barrier();
        feed_begin(next);
        const unsigned other = BUFFERS == 2 ? kBuffer - buffer : buffer + kBuffer == kLds ? 0 : buffer + kBuffer;
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
#pragma unroll
            for (int k = 0; k < kLoads / kMT; ++k) feed_load(buffer, i * (kLoads / kMT) + k);
            fa[0][i] = read_a.template read<0>(near + other, i);
            if (i < kNT) fb[0][i] = read_b.template read<0>(near + other, i);
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < kNT; ++j) mfma_operand(fb[1][j]);
            }
            mfma_operand(fa[1][i]);
#pragma unroll
            for (int j = 0; j < kNT; ++j) mfma<F16>(fa[1][i], fb[1][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        feed_end();
        buffer = other;
    }

    // A tile's sums, over `steps` steps.
    template <typename Next>
    __device__ __forceinline__ void run(int steps, Next &next, Acc4 (&acc)[kMT][kNT])
    {
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int j = 0; j < kNT; ++j) acc[i][j] = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
        mfma_settle(acc);
        for (int s = 0; s < steps * kPasses; ++s) {
            step(next, acc);
            if (F16 && s == 2 * steps - 1) {
                mfma_settle(acc);
#pragma unroll
                for (int i = 0; i < kMT; ++i)
#pragma unroll
                    for (int j = 0; j < kNT; ++j) {
                        // (one sum after the other, or they all wait in registers that there are not)
                        asm volatile("" : "+a"(acc[i][j]));
                        acc[i][j] = acc[i][j] * (1.0f / (1 << kRaised));
                        asm volatile("" : "+a"(acc[i][j]));
                    }
                mfma_settle(acc);
            }
        }
        mfma_settle(acc);
    }
};

}  // namespace bf
