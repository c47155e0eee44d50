// The gated linear recurrence over sequences, channel by channel:
//
//   h_t = a_t h_{t-1} + b_t      sigmoid gates: a = s(gate), b = (1 - a) x;  linear: a = gate, b = x
//
// with h_{-1} the state handed in, and h_{t-1} taken as zero where reset_t is set (the first step of a packed
// document).  Backward, from the last step: c_T = grad_state, e_t = grad_t + c_{t+1}, c_t = conj(a_t) e_t
// (zero at a reset), and with p_t = h_{t-1} (zero at a reset)
//
//   linear: d_gate = e conj(p), d_x = e;   sigmoid: d_gate = e (p - x) a (1 - a), d_x = e (1 - a).
//
// Forward moves 3 elements a step and channel, backward 6, against some 20 operations: memory bounds both,
// if enough of it is asked for at a time.  A step depends on the one before, but steps compose:
// a run of them is h -> A h + B.  So a workgroup takes 64 lanes of channels and up to 16 wavefronts
// side by side in time: each holds S steps in registers, works out its (A, B), the wavefronts
// exchange those through LDS (one barrier a tile of 16 S steps), and each then runs its steps again from its own h, the
// next tile's elements on their way meanwhile.  Everything is read and written once.
// Where channels times batch are too few workgroups to fill the chip the sequence is cut into chunks of 16 runs, a
// wavefront each: one launch forms the runs' and chunks' (A, B), the next one walks the chunks, the third one
// starts each run from there (a fixed order: the same sums at every call).
//
// h is kept in float (complex64: two) whatever the rows' type; 1 - a is s(-gate), not a difference,
// or decays close to one would lose it.  Backward h_{t-1} is what the forward call wrote, rounded where the rows
// are bfloat16: d_gate then has 2^-9 of h beside its own rounding, and no second copy of h in float is written and read.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "vec8.hpp"

namespace bf {

constexpr int kRecWaves = 16;

struct RecurrenceArgs {
    const void *gate, *x;               // (batch, steps, channels), channels adjacent
    const void *state;                  // (batch, channels) dense, NULL: zeros
    const uint8_t *reset;               // (batch, steps), NULL: none
    void *h;                            // (batch, steps, channels) dense
    void *last;                         // (batch, channels) dense
    const void *grad, *grad_last;       // backward; NULL: zeros
    void *d_gate, *d_x, *d_state;       // dense
    int64_t gate_b, gate_t, x_b, x_t, grad_b, grad_t, reset_b, reset_t;
    int64_t steps, chunk;               // chunk: steps of a chunk (the last one may be shorter)
    int64_t batch;
    int channels, groups, chunks;       // groups: workgroups across the channels
    void *chunk_a, *chunk_b;            // (chunks, batch, channels): what a chunk does
    void *run_a, *run_b;                // (chunks, kRecWaves, batch, channels): what stands in front of a run in its chunk
    int *chunk_cut, *run_cut;           // the same by sequence: a reset inside
};

// V channels a lane, in registers as V accumulators; S steps a wavefront forward, SB backward, SR where runs are formed (so
// that 64 registers do and two workgroups fit a compute unit).
struct RecF32 {
    using Elem = float;
    using Acc = float;
    static constexpr int V = 1, S = 8, SB = 8, SR = 8;
    static constexpr bool kExact = true;
};
struct RecBF16 {
    using Elem = bf16;
    using Acc = float;
    static constexpr int V = 2, S = 8, SB = 4, SR = 4;   // (eight steps of four tensors of two channels do not fit 128 registers)
    static constexpr bool kExact = false;   // (the gates have eight bits)
};
struct RecC64 {
    using Elem = float2;
    using Acc = float2;
    static constexpr int V = 1, S = 4, SB = 4, SR = 4;
    static constexpr bool kExact = true;
};

__device__ __forceinline__ float one_of(float) { return 1.0f; }
__device__ __forceinline__ float2 one_of(float2) { return make_float2(1.0f, 0.0f); }
__device__ __forceinline__ bool is_zero(float v) { return v == 0.0f; }
__device__ __forceinline__ bool is_zero(float2 v) { return v.x == 0.0f && v.y == 0.0f; }

// A single channel of bfloat16: no neighbour to load with it.
struct RecBF16One {
    using Elem = bf16;
    using Acc = float;
    static constexpr int V = 1, S = 8, SB = 8, SR = 8;
    static constexpr bool kExact = false;
};

// What a lane loads of one row, on its way until widen() looks at it.  Columns past the end repeat the row's last ones (every
// address is valid); nothing of theirs is stored.  A pair that the row's end cuts is loaded from one column
// before, and its first half is the upper one.
template <typename Tr>
struct RecLoad {
    static constexpr int V = Tr::V;
    using E = typename Tr::Elem;
    using Raw = std::conditional_t<V == 2, uint32_t, E>;
    uint32_t at;   // bytes: with a row's address in scalar registers a load needs no address arithmetic
    bool cut;

    __device__ __forceinline__ RecLoad(int c, int n) : at((uint32_t)(c + V <= n ? c : n - V) * (uint32_t)sizeof(E)), cut(V == 2 && c == n - 1) {}
    __device__ __forceinline__ Raw load(const E *row) const
    {
        typedef uint32_t word_at_2 __attribute__((aligned(2)));
        if constexpr (V == 2) return *reinterpret_cast<const word_at_2 *>(reinterpret_cast<const char *>(row) + at);
        else return *reinterpret_cast<const E *>(reinterpret_cast<const char *>(row) + at);
    }
    __device__ __forceinline__ void widen(Raw raw, typename Tr::Acc (&v)[V]) const
    {
        if constexpr (V == 2) {
            v[0] = __builtin_bit_cast(float, cut ? raw & 0xffff0000u : raw << 16);
            v[1] = __builtin_bit_cast(float, raw & 0xffff0000u);
        } else if constexpr (sizeof(E) == 2) {
            v[0] = (float)raw;
        } else {
            v[0] = raw;
        }
    }
};
__device__ __forceinline__ void put(bf16 *row, int c, int n, const float (&v)[1])
{
    if (c < n) row[c] = (bf16)v[0];
}
__device__ __forceinline__ void put(float *row, int c, int n, const float (&v)[1])
{
    if (c < n) row[c] = v[0];
}
__device__ __forceinline__ void put(float2 *row, int c, int n, const float2 (&v)[1])
{
    if (c < n) row[c] = v[0];
}
__device__ __forceinline__ void put(bf16 *row, int c, int n, const float (&v)[2])
{
    typedef uint32_t word_at_2 __attribute__((aligned(2)));
    if (c + 1 < n) *reinterpret_cast<word_at_2 *>(row + c) = pack_bf16(v[0], v[1]);
    else if (c < n) row[c] = (bf16)v[0];
}
template <int V, typename A>
__device__ __forceinline__ void get_state(const A *row, int c, int n, A (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = row && c + i < n ? row[c + i] : zero_of(A());
}
template <int V, typename A>
__device__ __forceinline__ void put_state(A *row, int c, int n, const A (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (c + i < n) row[c + i] = v[i];
}

// s(z) and s(-z) from one exponential, e = exp(-z): 1 / (1 + e) and e / (1 + e), neither a difference.  e stops at 2^126,
// where the first is as good as zero and the second still one.  EXACT: the exponent's rounding (2^-24 of it, so some 2^-21 of
// e at the ends) is put back.
template <bool EXACT>
__device__ __forceinline__ void sigmoids(float z, float &a, float &rest)
{
    constexpr float kLog2e = 1.44269504088896340736f;
    float t = -z * kLog2e;
    t = t > 126.0f ? 126.0f : t;   // (NaN stays NaN)
    float e = __builtin_amdgcn_exp2f(t);
    if constexpr (EXACT) {
        const float off = fmaf(-z, kLog2e, -t);
        e = fabsf(off) < 1.0f ? fmaf(e, off * 0.69314718f, e) : e;   // (not where t was cut or z is infinite)
    }
    a = __builtin_amdgcn_rcpf(1.0f + e);
    rest = e * a;
}

template <bool SIG, bool EXACT, typename A>
__device__ __forceinline__ void gate_of(A z, A &a, A &rest)
{
    if constexpr (SIG) sigmoids<EXACT>(z, a, rest);
    else { a = z; rest = one_of(z); }
}

template <typename A>
__device__ __forceinline__ A step_of(bool cut, A a, A h, A b)
{
    return cut ? b : mac(b, a, h);
}

// Runs and chunks compose by products of many gates, which may overflow where nothing is there to be multiplied (leading
// zeros under gates above one): zero through them is zero, as it is step by step.  (A number below one may be infinite
// behind a product that has passed 2^128 where step by step it is not yet.)
template <typename A>
__device__ __forceinline__ A chunk_of(bool cut, A a, A h, A b)
{
    return cut || is_zero(h) ? b : mac(b, a, h);
}
// the gates' product of two of them
template <typename A>
__device__ __forceinline__ A gates_of(bool cut, A a, A b)
{
    return cut || is_zero(a) || is_zero(b) ? zero_of(A()) : mul(a, b);
}

// carry behind the composition in a slot (columns past the end repeat the last one)
template <int V, typename A>
__device__ __forceinline__ void compose(const void *from_a, const void *from_b, const int *from_cut, int64_t slot, int c, int n, A (&carry)[V])
{
    const bool cut = from_cut[slot];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = c + v < n ? c + v : n - 1;
        const A ca = reinterpret_cast<const A *>(from_a)[slot * n + col], cb = reinterpret_cast<const A *>(from_b)[slot * n + col];
        carry[v] = chunk_of(cut, ca, carry[v], cb);
    }
}

// The runs of a tile's wavefronts, and what enters each.  Two buffers that alternate: one barrier a tile.
template <typename Tr>
struct Runs {
    typename Tr::Acc a[2][kRecWaves][Tr::V][64], b[2][kRecWaves][Tr::V][64];
    int cut[2][kRecWaves];
};

// FROM_LAST: the wavefronts compose from the last one back.
template <typename Tr, bool FROM_LAST>
__device__ __forceinline__ void exchange(Runs<Tr> &runs, int turn, int wave, int waves, int lane, bool cut,
                                         const typename Tr::Acc (&ra)[Tr::V], const typename Tr::Acc (&rb)[Tr::V],
                                         typename Tr::Acc (&carry)[Tr::V], typename Tr::Acc (&mine)[Tr::V])
{
    using A = typename Tr::Acc;
#pragma unroll
    for (int v = 0; v < Tr::V; ++v) {
        runs.a[turn][wave][v][lane] = ra[v];
        runs.b[turn][wave][v][lane] = rb[v];
    }
    if (lane == 0) runs.cut[turn][wave] = cut;
    __syncthreads();
    for (int i = 0; i < waves; ++i) {
        const int w = FROM_LAST ? waves - 1 - i : i;
        const bool cut_w = runs.cut[turn][w];
#pragma unroll
        for (int v = 0; v < Tr::V; ++v) {
            const A ca = runs.a[turn][w][v][lane], cb = runs.b[turn][w][v][lane];
            if (w == wave) mine[v] = carry[v];
            carry[v] = chunk_of(cut_w, ca, carry[v], cb);
        }
    }
}

// The resets of `steps` steps from t on as bits, steps past `end` unset.
__device__ __forceinline__ uint64_t reset_bits(const RecurrenceArgs &a, int64_t b, int64_t t, int64_t end, int steps, int lane)
{
    if (!a.reset) return 0;
    const bool in = lane < steps && t + lane < end;
    const uint8_t r = in ? a.reset[b * a.reset_b + (t + lane) * a.reset_t] : 0;
    return __ballot(r != 0);
}

// What a wavefront works on: 64 V channels of a sequence.
template <typename Tr>
struct RecPlace {
    using E = typename Tr::Elem;
    using A = typename Tr::Acc;
    int lane, wave, waves, chunk, c, n;
    int64_t b, begin, end;     // the workgroup's steps
    bool there;                // whether it has any (a grid in two dimensions may have more than there is work for)

    // Workgroups go to the eight XCDs in turn.  Rows seldom begin at a cache line, so the groups of channels of one
    // chunk belong on one XCD, behind each other, where a line that two of them share is in one L2: chunk k is XCD k % 8's
    // (grid: chunks up to a multiple of 8), and whole sequences are runs of neighbours for each XCD.
    __device__ __forceinline__ explicit RecPlace(const RecurrenceArgs &p)
        : lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), waves(blockDim.x >> 6), n(p.channels)
    {
        const uint64_t id = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x, xcd = id % 8;
        unsigned x;
        if (p.chunks > 1) {
            chunk = (int)(id / 8 / gridDim.x * 8 + xcd);
            x = (unsigned)(id / 8 % gridDim.x);
            there = chunk < p.chunks;
        } else {
            const uint64_t total = (uint64_t)p.batch * p.groups, per = total / 8, over = total % 8;
            chunk = 0;
            x = (unsigned)(xcd * per + (xcd < over ? xcd : over) + id / 8);
            there = id < total;
        }
        b = x / (unsigned)p.groups;
        c = ((int)(x % (unsigned)p.groups) * 64 + lane) * Tr::V;
        begin = (int64_t)chunk * p.chunk;
        end = begin + p.chunk < p.steps ? begin + p.chunk : p.steps;
    }
    __device__ __forceinline__ const E *rows(const void *p, int64_t stride) const { return reinterpret_cast<const E *>(p) + b * stride; }
    __device__ __forceinline__ const A *state(const void *p) const { return p ? reinterpret_cast<const A *>(p) + b * n : nullptr; }
    __device__ __forceinline__ A *state(void *p) const { return reinterpret_cast<A *>(p) + b * n; }
};

// S rows of one tensor from step t on (those past `end` repeat the last one).
template <int S, typename Tr>
__device__ __forceinline__ void load_steps(typename RecLoad<Tr>::Raw (&raw)[S], const RecLoad<Tr> &in, const typename Tr::Elem *rows,
                                           int64_t stride, int64_t t, int64_t end)
{
    const typename Tr::Elem *row = rows + (t < end ? t : end - 1) * stride;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        raw[s] = in.load(row);
        if (t + s + 1 < end) row += stride;
    }
}
// The h in front of each of S steps from t on (t = 0: the first step's own, to be replaced by the state).
template <int S, typename Tr>
__device__ __forceinline__ void load_before(typename RecLoad<Tr>::Raw (&raw)[S], const RecLoad<Tr> &in, const typename Tr::Elem *rows,
                                            int64_t stride, int64_t t, int64_t end)
{
    const int64_t first = (t < end ? t : end - 1) - 1;
    const typename Tr::Elem *row = rows + (first < 0 ? 0 : first) * stride;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        raw[s] = in.load(row);
        if (first + s >= 0 && t + s + 1 < end) row += stride;
    }
}

// f(std::true_type) where none of S steps is a reset and all of them exist, the rule; f(std::false_type) otherwise.
template <typename F>
__device__ __forceinline__ void by_kind(bool plain, F &&f)
{
    if (plain) f(std::true_type());
    else f(std::false_type());
}

// ---- sequences that stay whole ---------------------------------------------------------------------------
// grid: batch x groups workgroups in one or two dimensions; 64 x waves threads.  16 sequences of 2048 steps and 1024 channels, float: 83 us (402 MB, 4.8 TB/s),
// backward 155 (805 MB, 5.2 TB/s): memory bounds both.  As many steps of 512 channels, complex64 (the same bytes, half the
// workgroups): 147 and 213; of 1024 channels, bfloat16 (half the bytes, half the workgroups): 86 and 159.
template <typename Tr, bool SIG>
__global__ __launch_bounds__(64 * kRecWaves) void recurrence_fw_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    using E = typename Tr::Elem;
    constexpr int V = Tr::V, S = Tr::S;
    __shared__ Runs<Tr> runs;
    const RecPlace<Tr> at(p);
    if (!at.there) return;
    const int c = at.c, n = at.n;
    const int64_t end = at.end;
    const RecLoad<Tr> in(c, n);
    const E *gate = at.rows(p.gate, p.gate_b), *x = at.rows(p.x, p.x_b);
    A carry[V];
    get_state<V>(at.state(p.state), c, n, carry);
    typename RecLoad<Tr>::Raw next_z[S], next_x[S];
    uint64_t next_cut = 0;
    auto fetch = [&](int64_t t) {
        load_steps<S, Tr>(next_z, in, gate, p.gate_t, t, end);
        load_steps<S, Tr>(next_x, in, x, p.x_t, t, end);
        next_cut = reset_bits(p, at.b, t, end, S, at.lane);
    };
    fetch(at.wave * S);
    const int tile = at.waves * S;
    int turn = 0;
    for (int64_t t0 = 0; t0 < end; t0 += tile, turn ^= 1) {
        const int64_t t = t0 + at.wave * S;
        const int count = (int)(end - t < 0 ? 0 : end - t < S ? end - t : S);
        const uint64_t cuts = next_cut;
        A za[S][V], zb[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            in.widen(next_z[s], za[s]);
            in.widen(next_x[s], zb[s]);
        }
        if (t0 + tile < end) fetch(t + tile);
        A ra[V], rb[V], mine[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { ra[v] = one_of(A()); rb[v] = zero_of(A()); }
        by_kind(cuts == 0 && count == S, [&](auto plain) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool cut = !plain.value && (cuts >> s & 1);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A a, rest;
                    gate_of<SIG, Tr::kExact>(za[s][v], a, rest);
                    if constexpr (SIG) zb[s][v] = mul(rest, zb[s][v]);
                    za[s][v] = a;
                    if (!plain.value && s >= count) continue;   // steps past the end change nothing
                    rb[v] = step_of(cut, a, rb[v], zb[s][v]);
                    ra[v] = cut ? zero_of(A()) : mul(ra[v], a);
                }
            }
        });
        exchange<Tr, false>(runs, turn, at.wave, at.waves, at.lane, cuts != 0, ra, rb, carry, mine);
        E *out = reinterpret_cast<E *>(p.h) + (at.b * p.steps + t) * n;
        by_kind(cuts == 0 && count == S, [&](auto plain) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool cut = !plain.value && (cuts >> s & 1);
#pragma unroll
                for (int v = 0; v < V; ++v) mine[v] = step_of(cut, za[s][v], mine[v], zb[s][v]);
                if (plain.value || s < count) put(out, c, n, mine);
                out += n;
            }
        });
    }
    if (at.wave == 0 && p.last) put_state<V>(at.state(p.last), c, n, carry);
}

// Operands of S steps backward, in registers: a, grad, (p - x) a (1 - a) or p, 1 - a.
template <typename Tr, bool SIG>
struct RecBack {
    static constexpr int V = Tr::V, S = Tr::SB;
    using A = typename Tr::Acc;
    using E = typename Tr::Elem;
    typename RecLoad<Tr>::Raw next_z[S], next_g[S], next_x[S], next_p[S];
    uint64_t next_cut = 0;
    A a[S][V], g[S][V], u[S][V], r[S][V];

    __device__ __forceinline__ void fetch(const RecurrenceArgs &p, const RecPlace<Tr> &at, const RecLoad<Tr> &in, int64_t t, int64_t end)
    {
        load_steps<S, Tr>(next_z, in, at.rows(p.gate, p.gate_b), p.gate_t, t, end);
        // (without a gradient of h: something that is there, and not looked at)
        if (p.grad) load_steps<S, Tr>(next_g, in, at.rows(p.grad, p.grad_b), p.grad_t, t, end);
        if constexpr (SIG) load_steps<S, Tr>(next_x, in, at.rows(p.x, p.x_b), p.x_t, t, end);
        load_before<S, Tr>(next_p, in, at.rows(p.h, p.steps * at.n), at.n, t, end);
        next_cut = reset_bits(p, at.b, t, end, S, at.lane);
    }
    __device__ __forceinline__ void take(const RecurrenceArgs &p, const RecPlace<Tr> &at, const RecLoad<Tr> &in, int64_t t)
    {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            in.widen(next_z[s], a[s]);
            in.widen(next_p[s], u[s]);
            if constexpr (SIG) in.widen(next_x[s], r[s]);
        }
        if (p.grad) {
#pragma unroll
            for (int s = 0; s < S; ++s) in.widen(next_g[s], g[s]);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) g[s][v] = zero_of(A());
        }
        if (t == 0) get_state<V>(at.state(p.state), at.c, at.n, u[0]);
    }
    template <bool PLAIN>
    __device__ __forceinline__ void gates(uint64_t cuts)
    {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A gate, rest;
                gate_of<SIG, Tr::kExact>(a[s][v], gate, rest);
                if (!PLAIN && (cuts >> s & 1)) u[s][v] = zero_of(A());
                if constexpr (SIG) {
                    u[s][v] = (u[s][v] - r[s][v]) * (gate * rest);
                    r[s][v] = rest;
                }
                a[s][v] = conj_of(gate);
            }
    }
    // The steps from the last one back, c going through them; rows of the results from step t on.
    template <bool PLAIN>
    __device__ __forceinline__ void steps(const RecurrenceArgs &p, const RecPlace<Tr> &at, int64_t t, int count, uint64_t cuts, A (&c)[V])
    {
        const int64_t row = (at.b * p.steps + t + S - 1) * at.n;
        E *dz = reinterpret_cast<E *>(p.d_gate) + row, *dx = reinterpret_cast<E *>(p.d_x) + row;
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            if (PLAIN || s < count) {
                const bool cut = !PLAIN && (cuts >> s & 1);
                A out_z[V], out_x[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const A e = add(g[s][v], c[v]);
                    out_z[v] = mul(e, conj_of(u[s][v]));
                    if constexpr (SIG) out_x[v] = mul(e, r[s][v]);
                    else out_x[v] = e;
                    c[v] = cut ? zero_of(A()) : mul(a[s][v], e);
                }
                put(dz, at.c, at.n, out_z);
                put(dx, at.c, at.n, out_x);
            }
            dz -= at.n;
            dx -= at.n;
        }
    }
};

// The same from the last step back, on c: c -> conj(a) (grad + c).
template <typename Tr, bool SIG>
__global__ __launch_bounds__(64 * kRecWaves) void recurrence_bw_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    constexpr int V = Tr::V, S = Tr::SB;
    __shared__ Runs<Tr> runs;
    const RecPlace<Tr> at(p);
    if (!at.there) return;
    const int64_t end = at.end;
    const RecLoad<Tr> in(at.c, at.n);
    A carry[V];
    get_state<V>(at.state(p.grad_last), at.c, at.n, carry);
    RecBack<Tr, SIG> back;
    const int tile = at.waves * S;
    const int64_t first = (end - 1) / tile * tile;   // the last tile
    back.fetch(p, at, in, first + at.wave * S, end);
    int turn = 0;
    for (int64_t t0 = first; t0 >= 0; t0 -= tile, turn ^= 1) {
        const int64_t t = t0 + at.wave * S;
        const int count = (int)(end - t < 0 ? 0 : end - t < S ? end - t : S);
        const uint64_t cuts = back.next_cut;
        back.take(p, at, in, t);
        if (t0 - tile >= 0) back.fetch(p, at, in, t - tile, end);
        A ra[V], rb[V], mine[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { ra[v] = one_of(A()); rb[v] = zero_of(A()); }
        by_kind(cuts == 0 && count == S, [&](auto plain) {
            back.template gates<plain.value>(cuts);
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const bool cut = !plain.value && (cuts >> s & 1);
                if (!plain.value && s >= count) continue;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    rb[v] = cut ? zero_of(A()) : mul(back.a[s][v], add(back.g[s][v], rb[v]));
                    ra[v] = cut ? zero_of(A()) : mul(ra[v], back.a[s][v]);
                }
            }
        });
        exchange<Tr, true>(runs, turn, at.wave, at.waves, at.lane, cuts != 0, ra, rb, carry, mine);
        by_kind(cuts == 0 && count == S, [&](auto plain) { back.template steps<plain.value>(p, at, t, count, cuts, mine); });
    }
    if (at.wave == 0 && p.d_state) put_state<V>(at.state(p.d_state), at.c, at.n, carry);
}

// ---- sequences cut into chunks ------------------------------------------------------------------------------
// grid (batch x groups, chunks), kRecWaves wavefronts, each with a run of its own: len = chunk / kRecWaves steps.  The first
// launch forms every run's (A, B) as composed from the chunk's start (backward: end) up to the run, and the chunks';
// the second one walks those from chunk to chunk; the third one starts each run from there, and the wavefronts need
// nothing of each other.  65537 steps of 1000 channels, bfloat16: forward 70 + 10 + 75 us (3.7 TB/s, a chain of 65 chunks,
// 5.2 TB/s), backward 66 + 11 + 167 (4.0 and 4.7 TB/s): memory bounds it, though a copy runs at 4.8.  Of 500 channels,
// complex64 (twice the bytes): 140 + 12 + 153 and 133 + 12 + 271.  The first launch's half of
// the registers took 10 us off each direction; the third one in workgroups of four wavefronts, or the first one walking
// against the third one's direction (for the caches), gained nothing.  With every wavefront walking the chunks in front of its own,
// instead of a launch between, the third launches took 123 and 193.

template <typename Tr, bool SIG, bool BACKWARD>
__global__ __launch_bounds__(64 * kRecWaves, 8) void recurrence_runs_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    constexpr int V = Tr::V, S = Tr::SR;
    __shared__ Runs<Tr> runs;
    const RecPlace<Tr> at(p);
    if (!at.there) return;
    const RecLoad<Tr> in(at.c, at.n);
    const int64_t len = p.chunk / kRecWaves, begin = at.begin + at.wave * len;
    const int64_t end = begin + len < at.end ? begin + len : at.end;
    // forward (gates, inputs), backward (gates, gradients)
    const void *second = BACKWARD ? p.grad : p.x;
    const int64_t second_b = BACKWARD ? p.grad_b : p.x_b, second_t = BACKWARD ? p.grad_t : p.x_t;
    A ra[V], rb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { ra[v] = one_of(A()); rb[v] = zero_of(A()); }
    bool any_cut = false;
    if (begin < end) {
        typename RecLoad<Tr>::Raw next_z[S], next_x[S];
        uint64_t next_cut = 0;
        auto fetch = [&](int64_t t) {
            load_steps<S, Tr>(next_z, in, at.rows(p.gate, p.gate_b), p.gate_t, t, end);
            if (second) load_steps<S, Tr>(next_x, in, at.rows(second, second_b), second_t, t, end);
            next_cut = reset_bits(p, at.b, t, end, S, at.lane);
        };
        const int64_t blocks = (end - begin + S - 1) / S;
        fetch(BACKWARD ? begin + (blocks - 1) * S : begin);
        for (int64_t k = 0; k < blocks; ++k) {
            const int64_t t = begin + (BACKWARD ? blocks - 1 - k : k) * S;
            const int count = (int)(end - t < S ? end - t : S);
            const uint64_t cuts = next_cut;
            A za[S][V], zb[S][V];
#pragma unroll
            for (int s = 0; s < S; ++s) in.widen(next_z[s], za[s]);
            if (second) {
#pragma unroll
                for (int s = 0; s < S; ++s) in.widen(next_x[s], zb[s]);
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s)
#pragma unroll
                    for (int v = 0; v < V; ++v) zb[s][v] = zero_of(A());
            }
            if (k + 1 < blocks) fetch(BACKWARD ? t - S : t + S);
            any_cut |= cuts != 0;
            by_kind(cuts == 0 && count == S, [&](auto plain) {
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const int s = BACKWARD ? S - 1 - i : i;
                    const bool cut = !plain.value && (cuts >> s & 1);
                    if (!plain.value && s >= count) continue;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        A a, rest;
                        gate_of<SIG, Tr::kExact>(za[s][v], a, rest);
                        if constexpr (BACKWARD) {
                            a = conj_of(a);
                            rb[v] = cut ? zero_of(A()) : mul(a, add(zb[s][v], rb[v]));
                        } else {
                            rb[v] = step_of(cut, a, rb[v], SIG ? mul(rest, zb[s][v]) : zb[s][v]);
                        }
                        ra[v] = cut ? zero_of(A()) : mul(ra[v], a);
                    }
                }
            });
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        runs.a[0][at.wave][v][at.lane] = ra[v];
        runs.b[0][at.wave][v][at.lane] = rb[v];
    }
    if (at.lane == 0) runs.cut[0][at.wave] = any_cut;
    __syncthreads();
    // what stands in front of this wavefront's run, and (the last one's own wavefront) behind all of them
    const int turn = BACKWARD ? kRecWaves - 1 - at.wave : at.wave, last = turn == kRecWaves - 1;
    A pa[V], pb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { pa[v] = one_of(A()); pb[v] = zero_of(A()); }
    bool cut = false;
    auto write = [&](void *to_a, void *to_b, int *to_cut, int64_t slot) {
        put_state<V>(reinterpret_cast<A *>(to_a) + (slot * p.batch + at.b) * at.n, at.c, at.n, pa);
        put_state<V>(reinterpret_cast<A *>(to_b) + (slot * p.batch + at.b) * at.n, at.c, at.n, pb);
        if (at.lane == 0 && at.c == 0) to_cut[slot * p.batch + at.b] = cut;
    };
    auto add_run = [&](int i) {
        const int w = BACKWARD ? kRecWaves - 1 - i : i;
        const bool cut_w = runs.cut[0][w];
        cut |= cut_w;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const A ca = runs.a[0][w][v][at.lane], cb = runs.b[0][w][v][at.lane];
            pb[v] = chunk_of(cut_w, ca, pb[v], cb);
            pa[v] = gates_of(cut_w, pa[v], ca);
        }
    };
    for (int i = 0; i < turn; ++i) add_run(i);
    write(p.run_a, p.run_b, p.run_cut, (int64_t)at.chunk * kRecWaves + at.wave);
    if (last) {
        add_run(turn);
        write(p.chunk_a, p.chunk_b, p.chunk_cut, at.chunk);
    }
}

// What enters each chunk, in the place of its A: the state through the chunks in front of it, one after another.
template <typename Tr, bool BACKWARD>
__global__ __launch_bounds__(64) void recurrence_enter_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    const int64_t states = p.batch * p.channels, at = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (at >= states) return;
    const int64_t b = at / p.channels;
    const A *state = reinterpret_cast<const A *>(BACKWARD ? p.grad_last : p.state);
    A *a = reinterpret_cast<A *>(p.chunk_a) + at, carry = state ? state[at] : zero_of(A());
    const A *add_b = reinterpret_cast<const A *>(p.chunk_b) + at;
    constexpr int kAhead = 32;   // loads on their way at a time: the walk itself is short
    for (int from = 0; from < p.chunks; from += kAhead) {
        A ca[kAhead], cb[kAhead];
        bool cut[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int k = from + i < p.chunks ? from + i : p.chunks - 1;
            const int64_t slot = BACKWARD ? p.chunks - 1 - k : k;
            ca[i] = a[slot * states];
            cb[i] = add_b[slot * states];
            cut[i] = p.chunk_cut[slot * p.batch + b] != 0;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (from + i < p.chunks) {
                a[(int64_t)(BACKWARD ? p.chunks - 1 - from - i : from + i) * states] = carry;
                carry = chunk_of(cut[i], ca[i], carry, cb[i]);
            }
        }
    }
}

// What enters a wavefront's run.
template <typename Tr>
__device__ __forceinline__ void enter_run(const RecurrenceArgs &p, const RecPlace<Tr> &at, typename Tr::Acc (&carry)[Tr::V])
{
    using A = typename Tr::Acc;
    get_state<Tr::V>(reinterpret_cast<const A *>(p.chunk_a) + (at.chunk * p.batch + at.b) * at.n, at.c, at.n, carry);
    compose<Tr::V>(p.run_a, p.run_b, p.run_cut, ((int64_t)at.chunk * kRecWaves + at.wave) * p.batch + at.b, at.c, at.n, carry);
}

template <typename Tr, bool SIG>
__global__ __launch_bounds__(64 * kRecWaves) void recurrence_chunk_fw_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    using E = typename Tr::Elem;
    constexpr int V = Tr::V, S = Tr::S;
    const RecPlace<Tr> at(p);
    if (!at.there) return;
    const int c = at.c, n = at.n;
    const RecLoad<Tr> in(c, n);
    const int64_t len = p.chunk / kRecWaves, begin = at.begin + at.wave * len;
    const int64_t end = begin + len < at.end ? begin + len : at.end;
    if (begin >= end) return;
    typename RecLoad<Tr>::Raw next_z[S], next_x[S];
    uint64_t next_cut = 0;
    auto fetch = [&](int64_t t) {
        load_steps<S, Tr>(next_z, in, at.rows(p.gate, p.gate_b), p.gate_t, t, end);
        load_steps<S, Tr>(next_x, in, at.rows(p.x, p.x_b), p.x_t, t, end);
        next_cut = reset_bits(p, at.b, t, end, S, at.lane);
    };
    fetch(begin);
    A h[V];
    enter_run(p, at, h);
    E *out = reinterpret_cast<E *>(p.h) + (at.b * p.steps + begin) * n;
    for (int64_t t = begin; t < end; t += S) {
        const int count = (int)(end - t < S ? end - t : S);
        const uint64_t cuts = next_cut;
        A za[S][V], zb[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            in.widen(next_z[s], za[s]);
            in.widen(next_x[s], zb[s]);
        }
        if (t + S < end) fetch(t + S);
        by_kind(cuts == 0 && count == S, [&](auto plain) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool cut = !plain.value && (cuts >> s & 1);
                if (!plain.value && s >= count) continue;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A a, rest;
                    gate_of<SIG, Tr::kExact>(za[s][v], a, rest);
                    h[v] = step_of(cut, a, h[v], SIG ? mul(rest, zb[s][v]) : zb[s][v]);
                }
                put(out, c, n, h);
                out += n;
            }
        });
    }
    if (end == p.steps && p.last) put_state<V>(at.state(p.last), c, n, h);
}

template <typename Tr, bool SIG>
__global__ __launch_bounds__(64 * kRecWaves) void recurrence_chunk_bw_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    constexpr int V = Tr::V, S = Tr::SB;
    const RecPlace<Tr> at(p);
    if (!at.there) return;
    const RecLoad<Tr> in(at.c, at.n);
    const int64_t len = p.chunk / kRecWaves, begin = at.begin + at.wave * len;
    const int64_t end = begin + len < at.end ? begin + len : at.end;
    if (begin >= end) return;
    RecBack<Tr, SIG> back;
    const int64_t first = begin + (end - begin - 1) / S * S;
    back.fetch(p, at, in, first, end);
    A carry[V];
    enter_run(p, at, carry);
    for (int64_t t = first; t >= begin; t -= S) {
        const int count = (int)(end - t < S ? end - t : S);
        const uint64_t cuts = back.next_cut;
        back.take(p, at, in, t);
        if (t > begin) back.fetch(p, at, in, t - S, end);
        by_kind(cuts == 0 && count == S, [&](auto plain) {
            back.template gates<plain.value>(cuts);
            back.template steps<plain.value>(p, at, t, count, cuts, carry);
        });
    }
    if (begin == 0 && p.d_state) put_state<V>(at.state(p.d_state), at.c, at.n, carry);
}

// One step of every sequence, the state updated in place.  grid (channels / 256 rounded up, batch).  64 sequences of 1024
// channels, float: 3.1 us, a launch's; the call's 6.7 are the host's.
template <typename Tr, bool SIG>
__global__ __launch_bounds__(256) void recurrence_step_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    using E = typename Tr::Elem;
    constexpr int V = Tr::V;
    const int c = (blockIdx.x * 256 + threadIdx.x) * V, n = p.channels;
    if (c >= n) return;
    const RecLoad<Tr> in(c, n);
    for (int64_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
        A z[V], x[V], h[V];
        in.widen(in.load(reinterpret_cast<const E *>(p.gate) + b * p.gate_b), z);
        in.widen(in.load(reinterpret_cast<const E *>(p.x) + b * p.x_b), x);
        A *state = reinterpret_cast<A *>(p.last) + b * n;
        get_state<V>(state, c, n, h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            A a, rest;
            gate_of<SIG, Tr::kExact>(z[v], a, rest);
            h[v] = mac(SIG ? mul(rest, x[v]) : x[v], a, h[v]);
        }
        put_state<V>(state, c, n, h);
        put(reinterpret_cast<E *>(p.h) + b * n, c, n, h);
    }
}

// No steps at all: what comes in goes out.
template <typename A>
__global__ __launch_bounds__(256) void recurrence_pass_kernel(const A *in, A *out, int64_t count)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        out[i] = in ? in[i] : zero_of(A());
}

}  // namespace bf
