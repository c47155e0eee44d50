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
// Where channels times batch are too few workgroups to fill the chip the sequence is cut into chunks: one
// launch forms the chunks' (A, B), the next one starts each chunk from their composition in
// ascending order (the same sums at every call).
//
// h is kept in float (complex64: two) whatever the rows' type; 1 - a is s(-gate), not a difference,
// or decays close to one would lose it.
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
    int channels, groups;               // groups: workgroups across the channels
    void *chunk_a, *chunk_b;            // (chunks, batch, channels)
    int *chunk_cut;                     // (chunks, batch): a reset inside
};

// V channels a lane, in registers as V accumulators; S steps a wavefront forward, SB backward.
struct RecF32 {
    using Elem = float;
    using Acc = float;
    static constexpr int V = 1, S = 8, SB = 8;
};
struct RecBF16 {
    using Elem = bf16;
    using Acc = float;
    static constexpr int V = 2, S = 8, SB = 4;   // (eight steps of four tensors of two channels do not fit 128 registers)
};
struct RecC64 {
    using Elem = float2;
    using Acc = float2;
    static constexpr int V = 1, S = 4, SB = 4;
};

__device__ __forceinline__ float one_of(float) { return 1.0f; }
__device__ __forceinline__ float2 one_of(float2) { return make_float2(1.0f, 0.0f); }
__device__ __forceinline__ bool is_zero(float v) { return v == 0.0f; }
__device__ __forceinline__ bool is_zero(float2 v) { return v.x == 0.0f && v.y == 0.0f; }

// A single channel of bfloat16: no neighbour to load with it.
struct RecBF16One {
    using Elem = bf16;
    using Acc = float;
    static constexpr int V = 1, S = 8, SB = 8;
};

// What a lane loads of one row, on its way until widen() looks at it.  Columns past the end repeat the row's last ones (every
// address is valid); nothing of theirs is stored.  A pair that the row's end cuts is loaded from one column
// before, and its first half is the upper one.
template <typename Tr>
struct RecLoad {
    static constexpr int V = Tr::V;
    using E = typename Tr::Elem;
    using Raw = std::conditional_t<V == 2, uint32_t, E>;
    int at;
    bool cut;

    __device__ __forceinline__ RecLoad(int c, int n) : at(c + V <= n ? c : n - V), cut(V == 2 && c == n - 1) {}
    __device__ __forceinline__ Raw load(const E *row) const
    {
        typedef uint32_t word_at_2 __attribute__((aligned(2)));
        if constexpr (V == 2) return *reinterpret_cast<const word_at_2 *>(row + at);
        else return row[at];
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

// s(z) and s(-z) from one exponential of a number that is not positive: neither overflows or cancels
__device__ __forceinline__ void sigmoids(float z, float &a, float &rest)
{
    const float e = expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
    a = z >= 0.0f ? r : e * r;
    rest = z >= 0.0f ? e * r : r;
}

template <bool SIG, typename A>
__device__ __forceinline__ void gate_of(A z, A &a, A &rest)
{
    if constexpr (SIG) sigmoids(z, a, rest);
    else { a = z; rest = one_of(z); }
}

template <typename A>
__device__ __forceinline__ A step_of(bool cut, A a, A h, A b)
{
    return cut ? b : mac(b, a, h);
}

// Chunks compose by products of many factors, which may overflow where nothing is there to be multiplied.
template <typename A>
__device__ __forceinline__ A chunk_of(bool cut, A a, A h, A b)
{
    return cut || is_zero(h) ? b : mac(b, a, h);
}

// carry behind chunk j (columns past the end repeat the last one)
template <int V, typename A>
__device__ __forceinline__ void compose(const RecurrenceArgs &p, int j, int64_t b, int c, int n, A (&carry)[V])
{
    const int64_t at = (j * p.batch + b) * n;
    const bool cut = p.chunk_cut[j * p.batch + b];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = c + v < n ? c + v : n - 1;
        const A ca = reinterpret_cast<const A *>(p.chunk_a)[at + col], cb = reinterpret_cast<const A *>(p.chunk_b)[at + col];
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
            carry[v] = step_of(cut_w, ca, carry[v], cb);
        }
    }
}

// The resets of a wavefront's S steps as bits, steps past `end` unset.
__device__ __forceinline__ uint64_t reset_bits(const RecurrenceArgs &a, int64_t b, int64_t t, int64_t end, int steps, int lane)
{
    if (!a.reset) return 0;
    const bool in = lane < steps && t + lane < end;
    const uint8_t r = in ? a.reset[b * a.reset_b + (t + lane) * a.reset_t] : 0;
    return __ballot(r != 0);
}

// grid (batch x groups, chunks); 64 x waves threads.  AGGREGATE: forms the chunks' (A, B) and writes nothing else.
template <typename Tr, bool SIG, bool AGGREGATE>
__global__ __launch_bounds__(64 * kRecWaves) void recurrence_fw_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    using E = typename Tr::Elem;
    constexpr int V = Tr::V, S = Tr::S;
    __shared__ Runs<Tr> runs;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t b = blockIdx.x / (unsigned)p.groups;
    const int c = ((int)(blockIdx.x % (unsigned)p.groups) * 64 + lane) * V, n = p.channels;
    const int64_t begin = (int64_t)blockIdx.y * p.chunk;
    const int64_t end = begin + p.chunk < p.steps ? begin + p.chunk : p.steps;
    const E *gate = reinterpret_cast<const E *>(p.gate) + b * p.gate_b;
    const E *x = reinterpret_cast<const E *>(p.x) + b * p.x_b;
    using Raw = typename RecLoad<Tr>::Raw;
    const RecLoad<Tr> in(c, n);

    A carry[V], whole[V];
    bool any_cut = false;
    if constexpr (AGGREGATE) {
#pragma unroll
        for (int v = 0; v < V; ++v) { carry[v] = zero_of(A()); whole[v] = one_of(A()); }
    } else {
        get_state<V>(p.state ? reinterpret_cast<const A *>(p.state) + b * n : nullptr, c, n, carry);
#pragma unroll 4
        for (int j = 0; j < (int)blockIdx.y; ++j) compose(p, j, b, c, n, carry);
    }

    Raw next_z[S], next_x[S];
    uint64_t next_cut = 0;
    auto fetch = [&](int64_t t0) {
        const int64_t t = t0 + wave * S;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int64_t at = t + s < end ? t + s : end - 1;
            next_z[s] = in.load(gate + at * p.gate_t);
            next_x[s] = in.load(x + at * p.x_t);
        }
        next_cut = reset_bits(p, b, t, end, S, lane);
    };
    fetch(begin);
    int turn = 0;
    for (int64_t t0 = begin; t0 < end; t0 += waves * S, turn ^= 1) {
        const int64_t t = t0 + wave * S;
        const int count = (int)(end - t < 0 ? 0 : end - t < S ? end - t : S);
        const uint64_t cuts = next_cut;
        A za[S][V], zb[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            in.widen(next_z[s], za[s]);
            in.widen(next_x[s], zb[s]);
        }
        if (t0 + waves * S < end) fetch(t0 + waves * S);
        A ra[V], rb[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { ra[v] = one_of(A()); rb[v] = zero_of(A()); }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool cut = (cuts >> s) & 1;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A a, rest;
                gate_of<SIG>(za[s][v], a, rest);
                if constexpr (SIG) zb[s][v] = mul(rest, zb[s][v]);
                za[s][v] = a;
                if (s >= count) continue;   // steps past the end change nothing
                rb[v] = step_of(cut, a, rb[v], zb[s][v]);
                ra[v] = cut ? zero_of(A()) : mul(ra[v], a);
            }
        }
        A mine[V];
        if constexpr (AGGREGATE) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                runs.a[turn][wave][v][lane] = ra[v];
                runs.b[turn][wave][v][lane] = rb[v];
            }
            if (lane == 0) runs.cut[turn][wave] = cuts != 0;
            __syncthreads();
            for (int w = 0; w < waves; ++w) {
                const bool cut = runs.cut[turn][w];
                any_cut |= cut;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const A ca = runs.a[turn][w][v][lane];
                    carry[v] = step_of(cut, ca, carry[v], runs.b[turn][w][v][lane]);
                    whole[v] = mul(whole[v], ca);
                }
            }
        } else {
            exchange<Tr, false>(runs, turn, wave, waves, lane, cuts != 0, ra, rb, carry, mine);
            E *out = reinterpret_cast<E *>(p.h) + (b * p.steps + t) * n;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool cut = (cuts >> s) & 1;
#pragma unroll
                for (int v = 0; v < V; ++v) mine[v] = step_of(cut, za[s][v], mine[v], zb[s][v]);
                if (s < count) put(out + (int64_t)s * n, c, n, mine);
            }
        }
    }
    if (wave != 0) return;
    if constexpr (AGGREGATE) {
        const int64_t at = (blockIdx.y * p.batch + b) * n;
        put_state<V>(reinterpret_cast<A *>(p.chunk_a) + at, c, n, whole);
        put_state<V>(reinterpret_cast<A *>(p.chunk_b) + at, c, n, carry);
        if (lane == 0 && c == 0) p.chunk_cut[blockIdx.y * p.batch + b] = any_cut;
    } else if (p.last && blockIdx.y == gridDim.y - 1) {
        put_state<V>(reinterpret_cast<A *>(p.last) + b * n, c, n, carry);
    }
}

// The same from the last step back, on c: c -> conj(a) (grad + c).
template <typename Tr, bool SIG, bool AGGREGATE>
__global__ __launch_bounds__(64 * kRecWaves) void recurrence_bw_kernel(RecurrenceArgs p)
{
    using A = typename Tr::Acc;
    using E = typename Tr::Elem;
    constexpr int V = Tr::V, S = Tr::SB;
    __shared__ Runs<Tr> runs;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t b = blockIdx.x / (unsigned)p.groups;
    const int c = ((int)(blockIdx.x % (unsigned)p.groups) * 64 + lane) * V, n = p.channels;
    const int64_t begin = (int64_t)blockIdx.y * p.chunk;
    const int64_t end = begin + p.chunk < p.steps ? begin + p.chunk : p.steps;
    const E *gate = reinterpret_cast<const E *>(p.gate) + b * p.gate_b;
    const E *x = reinterpret_cast<const E *>(p.x) + b * p.x_b;
    const E *grad = p.grad ? reinterpret_cast<const E *>(p.grad) + b * p.grad_b : nullptr;
    const E *h = reinterpret_cast<const E *>(p.h) + b * p.steps * n;
    using Raw = typename RecLoad<Tr>::Raw;
    const RecLoad<Tr> in(c, n);

    A carry[V], whole[V];
    bool any_cut = false;
    if constexpr (AGGREGATE) {
#pragma unroll
        for (int v = 0; v < V; ++v) { carry[v] = zero_of(A()); whole[v] = one_of(A()); }
    } else {
        get_state<V>(p.grad_last ? reinterpret_cast<const A *>(p.grad_last) + b * n : nullptr, c, n, carry);
#pragma unroll 4
        for (int j = (int)gridDim.y - 1; j > (int)blockIdx.y; --j) compose(p, j, b, c, n, carry);
    }

    Raw next_z[S], next_g[S], next_x[S], next_p[S];
    uint64_t next_cut = 0;
    auto fetch = [&](int64_t t0) {
        const int64_t t = t0 + wave * S;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int64_t at = t + s < end ? t + s : end - 1;
            next_z[s] = in.load(gate + at * p.gate_t);
            next_g[s] = grad ? in.load(grad + at * p.grad_t) : Raw();
            if constexpr (!AGGREGATE) {
                if constexpr (SIG) next_x[s] = in.load(x + at * p.x_t);
                next_p[s] = in.load(h + (at > 0 ? at - 1 : 0) * n);
            }
        }
        next_cut = reset_bits(p, b, t, end, S, lane);
    };
    const int tile = waves * S;
    const int64_t first = begin + (end - 1 - begin) / tile * tile;   // the chunk's last tile
    fetch(first);
    int turn = 0;
    for (int64_t t0 = first; t0 >= begin; t0 -= tile, turn ^= 1) {
        const int64_t t = t0 + wave * S;
        const int count = (int)(end - t < 0 ? 0 : end - t < S ? end - t : S);
        const uint64_t cuts = next_cut;
        A za[S][V], zg[S][V], zr[S][V], zp[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            in.widen(next_z[s], za[s]);
            in.widen(next_g[s], zg[s]);
            if constexpr (!AGGREGATE) {
                in.widen(next_p[s], zp[s]);
                if constexpr (SIG) in.widen(next_x[s], zr[s]);
            }
        }
        if constexpr (!AGGREGATE) {
            if (t == 0) {
                A first_state[V];
                get_state<V>(p.state ? reinterpret_cast<const A *>(p.state) + b * n : nullptr, c, n, first_state);
#pragma unroll
                for (int v = 0; v < V; ++v) zp[0][v] = first_state[v];
            }
        }
        if (t0 - tile >= begin) fetch(t0 - tile);
        A ra[V], rb[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { ra[v] = one_of(A()); rb[v] = zero_of(A()); }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            const bool cut = (cuts >> s) & 1;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A a, rest;
                gate_of<SIG>(za[s][v], a, rest);
                if constexpr (!AGGREGATE) {
                    if (cut) zp[s][v] = zero_of(A());
                    if constexpr (SIG) {
                        zp[s][v] = (zp[s][v] - zr[s][v]) * (a * rest);
                        zr[s][v] = rest;
                    }
                }
                za[s][v] = conj_of(a);
                if (s >= count) continue;
                rb[v] = cut ? zero_of(A()) : mul(za[s][v], add(zg[s][v], rb[v]));
                ra[v] = cut ? zero_of(A()) : mul(ra[v], za[s][v]);
            }
        }
        if constexpr (AGGREGATE) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                runs.a[turn][wave][v][lane] = ra[v];
                runs.b[turn][wave][v][lane] = rb[v];
            }
            if (lane == 0) runs.cut[turn][wave] = cuts != 0;
            __syncthreads();
            for (int w = waves - 1; w >= 0; --w) {
                const bool cut = runs.cut[turn][w];
                any_cut |= cut;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const A ca = runs.a[turn][w][v][lane];
                    carry[v] = step_of(cut, ca, carry[v], runs.b[turn][w][v][lane]);
                    whole[v] = mul(whole[v], ca);
                }
            }
        } else {
            A mine[V];
            exchange<Tr, true>(runs, turn, wave, waves, lane, cuts != 0, ra, rb, carry, mine);
            E *dz = reinterpret_cast<E *>(p.d_gate) + (b * p.steps + t) * n;
            E *dx = reinterpret_cast<E *>(p.d_x) + (b * p.steps + t) * n;
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const bool cut = (cuts >> s) & 1;
                if (s >= count) continue;
                A out_z[V], out_x[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const A e = add(zg[s][v], mine[v]);
                    out_z[v] = mul(e, conj_of(zp[s][v]));
                    if constexpr (SIG) out_x[v] = mul(e, zr[s][v]);
                    else out_x[v] = e;
                    mine[v] = cut ? zero_of(A()) : mul(za[s][v], e);
                }
                put(dz + (int64_t)s * n, c, n, out_z);
                put(dx + (int64_t)s * n, c, n, out_x);
            }
        }
    }
    if (wave != 0) return;
    if constexpr (AGGREGATE) {
        const int64_t at = (blockIdx.y * p.batch + b) * n;
        put_state<V>(reinterpret_cast<A *>(p.chunk_a) + at, c, n, whole);
        put_state<V>(reinterpret_cast<A *>(p.chunk_b) + at, c, n, carry);
        if (lane == 0 && c == 0) p.chunk_cut[blockIdx.y * p.batch + b] = any_cut;
    } else if (p.d_state && blockIdx.y == 0) {
        put_state<V>(reinterpret_cast<A *>(p.d_state) + b * n, c, n, carry);
    }
}

// One step of every sequence, the state updated in place.  grid (channels / 256 rounded up, batch).
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
            gate_of<SIG>(z[v], a, rest);
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
