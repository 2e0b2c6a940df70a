// Gated linear recurrence h_t = a_t h_{t-1} + b_t along the rows of (batch, rows, dim) arrays, its
// backward pass and its single-row step.
//
// Mathematics.  A run of rows maps the state entering it affinely, h -> A h + B, with A = prod a_t and B
// the recurrence started from 0, and two runs compose to (A2 A1, A2 B1 + B2).  The backward pass is the
// same recurrence from the other end in u_t = a_t g_t, the gradient handed to row t - 1: with d_t the
// derivatives of h_t, g_t = d_t + u_{t+1}, dx_t = g_t (or (1 - a_t) g_t) and da_t = g_t (h_{t-1} - [x_t]).
//
// Split.  One element costs three to six values of traffic and a handful of operations, so everything
// here is about keeping enough loads in flight.  A CTA owns a strip of CL * V neighbouring channels and
// TP * S rows at a time: thread (tt, tc) holds S consecutive rows of V channels in registers, reduces them
// to one (A, B), and reads the (A, B) of the threads before it from shared memory to get the state that
// enters its rows; a second walk over its registers then gives the S states.  Every input is read once,
// every output written once, and the state that crosses an iteration stays in registers, in 32 bits (64
// for float64 inputs).  A run is folded into the state one S-row map at a time, so the products of gates
// that are formed are S long (CTA-row long across a cluster) and no longer.
//
// Packed sequences are one scan over all rows in which the first row of a sequence drops what enters it:
// the drop is a flag beside (A, B), not a gate of 0, so that a NaN or an infinity of one sequence
// stays inside it.
#pragma once

#include "sequence.h"
#include "sequence_types.cuh"

namespace sigb200 {

struct RecurrencePlan {
    int log_lanes;     // CL = 1 << log_lanes threads side by side in the channels
    int log_parts;     // TP = 1 << log_parts threads behind each other in the rows
    unsigned strips;   // strips of CL * V channels
    int fold_log;      // backward, shared gates: lanes folded into one partial sum, log2
};

namespace {

__device__ __forceinline__ int64_t offset_at(const void* offsets, bool wide, int64_t i) {
    return wide ? static_cast<const long long*>(offsets)[i] : static_cast<const int*>(offsets)[i];
}

// Walks the packed sequences along increasing rows.  `seq` is the last sequence whose offset is at or before
// the row (-1 before the first, `count` behind the last); it spans rows [begin, next).  Offsets are only
// compared with rows, so values that are out of order or out of range take no access out of bounds.
struct SequenceWalk {
    const void* offsets;
    int64_t count, seq, begin, next;
    bool wide;

    __device__ __forceinline__ void settle() {
        begin = seq >= 0 ? offset_at(offsets, wide, seq) : INT64_MIN;
        next = seq < count ? offset_at(offsets, wide, seq + 1) : INT64_MAX;
    }
    __device__ void seek(const void* o, bool w, int64_t n, int64_t row) {
        offsets = o; wide = w; count = n;
        int64_t lo = 0, hi = n + 1;  // first of the n + 1 offsets that is > row
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (offset_at(o, w, mid) <= row) lo = mid + 1; else hi = mid;
        }
        seq = lo - 1;
        settle();
    }
    __device__ __forceinline__ void advance(int64_t row) {
        while (next <= row) { ++seq; settle(); }
    }
    __device__ __forceinline__ bool inside() const { return seq >= 0 && seq < count; }
    // no sequence starts or ends in [row, row + n), and all of those rows are in one
    __device__ __forceinline__ bool quiet(int64_t row, int n) const { return inside() && begin < row && next > row + n; }
};

// What happens in a thread's S rows, one bit a row: a sequence starts, a sequence ends, the row is in none.
struct RowEvents {
    unsigned starts = 0, ends = 0, dead = 0;
};

template <int S>
__device__ __forceinline__ RowEvents row_events(SequenceWalk walk, int64_t row0, int64_t rows) {
    RowEvents e;
    if (walk.quiet(row0, S)) return e;
    for (int s = 0; s < S && row0 + s < rows; ++s) {
        walk.advance(row0 + s);
        if (!walk.inside()) e.dead |= 1u << s;
        else {
            if (walk.begin == row0 + s) e.starts |= 1u << s;
            if (walk.next == row0 + s + 1) e.ends |= 1u << s;
        }
    }
    return e;
}

// Sequence that row `row` belongs to, walking from a thread's first row.
__device__ __forceinline__ int64_t sequence_of(SequenceWalk walk, int64_t row) {
    walk.advance(row);
    return walk.seq;
}

// a and 1 - a, neither by cancellation: exp and expm1 for logarithms; for logits both come from e^-|v|.
__device__ __forceinline__ void gate_factors(int form, float v, float& a, float& rest) {
    if (form == kGateValue) { a = v; rest = 1.0f - v; }
    else if (form == kGateLog) { a = expf(v); rest = -expm1f(v); }
    else {
        const float e = expf(-fabsf(v)), r = 1.0f / (1.0f + e), s = e * r;
        a = v >= 0.0f ? r : s;
        rest = v >= 0.0f ? s : r;
    }
}
__device__ __forceinline__ void gate_factors(int form, double v, double& a, double& rest) {
    if (form == kGateValue) { a = v; rest = 1.0 - v; }
    else if (form == kGateLog) { a = exp(v); rest = -expm1(v); }
    else {
        const double e = exp(-fabs(v)), r = 1.0 / (1.0 + e), s = e * r;
        a = v >= 0.0 ? r : s;
        rest = v >= 0.0 ? s : r;
    }
}

__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }

// S rows of V values each; rows at or beyond `rows` and channels beyond the last one read as zero.
template <typename T, int V, int S>
__device__ __forceinline__ void load_rows(Pack<T, V> (&r)[S], const T* base, int64_t row0, int64_t rows, int64_t stride,
                                          bool live) {
#pragma unroll
    for (int s = 0; s < S; ++s)
        r[s] = live && row0 + s < rows ? load_pack<T, V>(base + (row0 + s) * stride) : Pack<T, V>{};
}

// Bytes of shared memory: `kinds` value arrays (A and the Bs) and the drop flags, of both buffers.
template <typename A, int V>
constexpr size_t recurrence_smem(int kinds, int lanes, int parts) {
    return 2 * (sizeof(A) * size_t(kinds) * lanes * parts * V + size_t(parts));
}

// Folds the maps of the parts, in the direction of the scan, into the
// state that enters each: `run` goes from the state entering the CTA's rows to the one leaving them, `in`
// is the state entering part tt.
template <typename A, int V, bool REVERSE>
__device__ __forceinline__ void fold_parts(const A* ma, const A* mb, const unsigned char* md, unsigned bit, int parts,
                                           int lanes, int tt, int tc, A (&run)[V], A (&in)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = run[v];
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        const int t = REVERSE ? parts - 1 - i : i;
        const bool drop = md[t] & bit;
        const Pack<A, V> fa = load_pack<A, V>(ma + (t * lanes + tc) * V), fb = load_pack<A, V>(mb + (t * lanes + tc) * V);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (t == tt) in[v] = run[v];
            run[v] = drop ? fb.v[v] : fma_(fa.v[v], run[v], fb.v[v]);
        }
    }
}

template <typename X, typename G, int V, int S, bool SHARED>
__global__ void __launch_bounds__(256) recurrence_forward_kernel(const RecurrenceArgs p, const RecurrencePlan plan) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lanes = 1 << plan.log_lanes, parts = 1 << plan.log_parts, width = lanes * V;
    const int tc = threadIdx.x & (lanes - 1), tt = threadIdx.x >> plan.log_lanes;
    A* maps = reinterpret_cast<A*>(smem);  // [buffer][A, B][parts][width]
    unsigned char* drops = smem + sizeof(A) * 4 * parts * width;  // [buffer][parts]

    const uint64_t b = blockIdx.x / plan.strips;
    const uint64_t c0 = (uint64_t(blockIdx.x % plan.strips) * lanes + tc) * V;
    const bool live = c0 < p.dim, packed = p.sequences > 0;
    const int64_t rows = int64_t(p.rows), dim = int64_t(p.dim);
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + c0;
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const A* initial = p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr;
    X* out = p.out ? static_cast<X*>(p.out) + b * p.rows * p.dim + c0 : nullptr;
    A* state = p.state ? static_cast<A*>(p.state) + c0 : nullptr;
    A* marks = p.checkpoints
        ? static_cast<A*>(p.checkpoints) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + c0 : nullptr;

    A run[V];  // the state that enters the iteration's first row
#pragma unroll
    for (int v = 0; v < V; ++v) run[v] = !packed && initial && live ? initial[b * p.dim + v] : A(0);
    if (packed && state && live)  // sequences without rows hand their initial state on
        for (int64_t j = tt; j < int64_t(p.sequences); j += parts)
            if (offset_at(p.offsets, p.wide_offsets, j + 1) <= offset_at(p.offsets, p.wide_offsets, j))
                for (int v = 0; v < V; ++v) state[j * dim + v] = initial ? initial[j * dim + v] : A(0);

    SequenceWalk walk;
    if (packed) walk.seek(p.offsets, p.wide_offsets, p.sequences, int64_t(tt) * S);
    int buf = 0;
    for (int64_t base = 0; base < rows; base += int64_t(parts) * S, buf ^= 1) {
        const int64_t row0 = base + int64_t(tt) * S;
        Pack<X, V> rx[S];
        Pack<G, GV> rg[S];
        load_rows<X, V, S>(rx, x, row0, rows, p.x_row, live);
        load_rows<G, GV, S>(rg, gate, row0, rows, p.gate_row, live);
        RowEvents e;
        if (packed) {
            walk.advance(row0);
            e = row_events<S>(walk, row0, rows);
        }
        A a[S][V], u[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A rest;
                gate_factors(p.form, widen(rg[s].v[SHARED ? 0 : v]), a[s][v], rest);
                u[s][v] = widen(rx[s].v[v]);
                if (p.complement) u[s][v] *= rest;
                if (row0 + s >= rows || (e.dead >> s & 1u)) { a[s][v] = A(1); u[s][v] = A(0); }
            }
        // the initial state of a sequence that starts here joins b: its first row is then b alone
        if (e.starts && initial && live)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (e.starts >> s & 1u) {
                    const A* in = initial + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) u[s][v] = fma_(a[s][v], in[v], u[s][v]);
                }
        Pack<A, V> fa, fb;
#pragma unroll
        for (int v = 0; v < V; ++v) { fa.v[v] = A(1); fb.v[v] = A(0); }
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                fb.v[v] = (e.starts >> s & 1u) ? u[s][v] : fma_(a[s][v], fb.v[v], u[s][v]);
                fa.v[v] *= a[s][v];
            }
        A* ma = maps + buf * 2 * parts * width;
        A* mb = ma + parts * width;
        unsigned char* md = drops + buf * parts;
        store_pack<A, V>(ma + threadIdx.x * V, fa);
        store_pack<A, V>(mb + threadIdx.x * V, fb);
        if (tc == 0) md[tt] = e.starts != 0;
        __syncthreads();
        A h[V];
        fold_parts<A, V, false>(ma, mb, md, 1u, parts, lanes, tt, tc, run, h);
        if (!live || row0 >= rows) continue;
        if (marks && row0 % int64_t(kCheckpointRows) == 0)
#pragma unroll
            for (int v = 0; v < V; ++v) marks[row0 / int64_t(kCheckpointRows) * dim + v] = h[v];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            Pack<X, V> y;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = (e.starts >> s & 1u) ? u[s][v] : fma_(a[s][v], h[v], u[s][v]);
                y.v[v] = narrow<X>((e.dead >> s & 1u) ? A(0) : h[v]);
            }
            if (out && row0 + s < rows) store_pack<X, V>(out + (row0 + s) * dim, y);
            if (state && (e.ends >> s & 1u)) {
                A* to = state + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                for (int v = 0; v < V; ++v) to[v] = h[v];
            }
        }
    }
    if (!packed && state && live && tt == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) state[b * p.dim + v] = run[v];
}

// One iteration goes forward through its rows from a checkpoint (for h_{t-1}, kept in registers) and
// backward through the same registers, so that x, the gates and the derivatives are read once and h,
// rounded or not, is not read at all.
// Shared gates: each thread sums its V channels, 1 << fold_log neighbouring lanes are folded by shuffles,
// and `partial` takes one value per row and fold (dgate itself where a fold is a whole gate).
template <typename X, typename G, int V, int S, bool SHARED>
__global__ void __launch_bounds__(256) recurrence_backward_kernel(const RecurrenceArgs p, const RecurrencePlan plan,
                                                                  Acc<X>* partial) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lanes = 1 << plan.log_lanes, parts = 1 << plan.log_parts, width = lanes * V;
    const int tc = threadIdx.x & (lanes - 1), tt = threadIdx.x >> plan.log_lanes;
    A* maps = reinterpret_cast<A*>(smem);  // [buffer][A, forward B, backward B][parts][width]
    unsigned char* drops = smem + sizeof(A) * 6 * parts * width;  // [buffer][parts], bit 0 starts, bit 1 ends

    const uint64_t b = blockIdx.x / plan.strips;
    const uint64_t c0 = (uint64_t(blockIdx.x % plan.strips) * lanes + tc) * V;
    const bool live = c0 < p.dim, packed = p.sequences > 0;
    const int64_t rows = int64_t(p.rows), dim = int64_t(p.dim);
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + c0;
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const X* derivs = static_cast<const X*>(p.derivs) + b * p.d_batch + c0;
    const A* initial = p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr;
    const A* state_derivs = p.state_derivs ? static_cast<const A*>(p.state_derivs) + c0 : nullptr;
    const A* marks = static_cast<const A*>(p.marks) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + c0;
    X* dx = static_cast<X*>(p.dx) + b * p.rows * p.dim + c0;
    A* dinitial = p.dinitial ? static_cast<A*>(p.dinitial) + c0 : nullptr;
    const int64_t folds = SHARED ? (dim / V) >> plan.fold_log : 0;
    G* dgate = static_cast<G*>(p.dgate) + b * p.rows * p.gate_dim + (SHARED ? 0 : c0);

    A run[V];  // the gradient that enters the iteration's last row from behind
#pragma unroll
    for (int v = 0; v < V; ++v) run[v] = !packed && state_derivs && live ? state_derivs[b * p.dim + v] : A(0);
    if (packed && dinitial && live)
        for (int64_t j = tt; j < int64_t(p.sequences); j += parts)
            if (offset_at(p.offsets, p.wide_offsets, j + 1) <= offset_at(p.offsets, p.wide_offsets, j))
                for (int v = 0; v < V; ++v) dinitial[j * dim + v] = state_derivs ? state_derivs[j * dim + v] : A(0);

    const int64_t span = int64_t(parts) * S;
    int buf = 0;
    for (int64_t base = (rows - 1) / span * span; base >= 0; base -= span, buf ^= 1) {
        const int64_t row0 = base + int64_t(tt) * S;
        Pack<X, V> rx[S], rd[S];
        Pack<G, GV> rg[S];
        load_rows<X, V, S>(rx, x, row0, rows, p.x_row, live);
        load_rows<G, GV, S>(rg, gate, row0, rows, p.gate_row, live);
        load_rows<X, V, S>(rd, derivs, row0, rows, p.d_row, live);
        A h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = live ? marks[base / int64_t(kCheckpointRows) * dim + v] : A(0);
        RowEvents e;
        SequenceWalk walk;
        if (packed && row0 < rows) {
            walk.seek(p.offsets, p.wide_offsets, p.sequences, row0);
            e = row_events<S>(walk, row0, rows);
        }
        A a[S][V], rest[S][V], u[S][V], d[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gate_factors(p.form, widen(rg[s].v[SHARED ? 0 : v]), a[s][v], rest[s][v]);
                u[s][v] = widen(rx[s].v[v]);
                if (p.complement) u[s][v] *= rest[s][v];
                d[s][v] = widen(rd[s].v[v]);
                if (row0 + s >= rows || (e.dead >> s & 1u)) { a[s][v] = A(1); u[s][v] = d[s][v] = A(0); }
            }
        // the gradient of a state joins the derivatives of the row that it was taken from
        if (e.ends && state_derivs && live)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (e.ends >> s & 1u) {
                    const A* in = state_derivs + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) d[s][v] += in[v];
                }
        Pack<A, V> fa, fb, gb;
#pragma unroll
        for (int v = 0; v < V; ++v) { fa.v[v] = A(1); fb.v[v] = gb.v[v] = A(0); }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (e.starts >> s & 1u) {
                const A* in = initial && live ? initial + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
                for (int v = 0; v < V; ++v) fb.v[v] = in ? in[v] : A(0);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                fb.v[v] = fma_(a[s][v], fb.v[v], u[s][v]);
                fa.v[v] *= a[s][v];
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s)
#pragma unroll
            for (int v = 0; v < V; ++v)
                gb.v[v] = a[s][v] * ((e.ends >> s & 1u) ? d[s][v] : d[s][v] + gb.v[v]);
        A* ma = maps + buf * 3 * parts * width;
        A* mf = ma + parts * width;
        A* mg = mf + parts * width;
        unsigned char* md = drops + buf * parts;
        store_pack<A, V>(ma + threadIdx.x * V, fa);
        store_pack<A, V>(mf + threadIdx.x * V, fb);
        store_pack<A, V>(mg + threadIdx.x * V, gb);
        if (tc == 0) md[tt] = (e.starts ? 1 : 0) | (e.ends ? 2 : 0);
        __syncthreads();
        A w[V], in[V];
        fold_parts<A, V, false>(ma, mf, md, 1u, parts, lanes, tt, tc, h, in);
        fold_parts<A, V, true>(ma, mg, md, 2u, parts, lanes, tt, tc, run, w);
        A before[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (e.starts >> s & 1u) {
                const A* from = initial && live ? initial + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
                for (int v = 0; v < V; ++v) in[v] = from ? from[v] : A(0);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                before[s][v] = in[v];
                in[v] = fma_(a[s][v], in[v], u[s][v]);
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            const bool dead = e.dead >> s & 1u, stored = live && row0 + s < rows;
            Pack<X, V> gx;
            Pack<G, V> gg;
            A sum = A(0);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const A g = (e.ends >> s & 1u) ? d[s][v] : d[s][v] + w[v];
                gx.v[v] = narrow<X>(dead ? A(0) : p.complement ? rest[s][v] * g : g);
                A da = g * (p.complement ? before[s][v] - widen(rx[s].v[v]) : before[s][v]);
                if (p.form != kGateValue) da *= a[s][v];
                if (p.form == kGateLogit) da *= rest[s][v];
                if (dead) da = A(0);
                gg.v[v] = narrow<G>(da);
                sum += da;
                w[v] = a[s][v] * g;
            }
            if (stored) store_pack<X, V>(dx + (row0 + s) * dim, gx);
            if (SHARED) {
                sum = stored ? sum : A(0);
                for (int k = 1; k < 1 << plan.fold_log; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                const int64_t fold = int64_t(c0 / V) >> plan.fold_log;
                if (stored && (tc & ((1 << plan.fold_log) - 1)) == 0) {
                    if (partial) partial[(b * rows + row0 + s) * folds + fold] = sum;
                    else dgate[(row0 + s) * int64_t(p.gate_dim) + fold] = narrow<G>(sum);
                }
            } else if (stored) {
                store_pack<G, V>(dgate + (row0 + s) * dim, gg);
            }
            if (dinitial && live && (e.starts >> s & 1u)) {
                A* to = dinitial + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                for (int v = 0; v < V; ++v) to[v] = w[v];
            }
        }
    }
    if (!packed && dinitial && live && tt == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) dinitial[b * p.dim + v] = run[v];
}

// dgate[row, h] = sum of the `count` partial sums of gate h, in their order.
template <typename A, typename G>
__global__ void fold_partials_kernel(const A* __restrict__ partial, G* __restrict__ dgate, uint64_t n, uint64_t count) {
    const uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n) return;
    A sum = A(0);
    for (uint64_t k = 0; k < count; ++k) sum += partial[i * count + k];
    dgate[i] = narrow<G>(sum);
}

// One row for each state: state = a state + b, out = the new state rounded.  Two reads, one read and write
// of the state and one write; a grid over all values, since nothing is shared between them.
template <typename X, typename G, int V, bool SHARED>
__global__ void __launch_bounds__(256) recurrence_step_kernel(const RecurrenceArgs p) {
    using A = Acc<X>;
    const uint64_t columns = p.dim / V;
    const uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= p.rows * columns) return;
    const uint64_t row = i / columns, c0 = (i - row * columns) * V;
    const Pack<X, V> x = load_pack<X, V>(static_cast<const X*>(p.x) + row * p.x_row + c0);
    const G* gate = static_cast<const G*>(p.gate) + row * p.gate_row;
    const Pack<G, SHARED ? 1 : V> g = load_pack<G, SHARED ? 1 : V>(gate + (SHARED ? c0 / (p.dim / p.gate_dim) : c0));
    A* at = static_cast<A*>(p.state) + row * p.dim + c0;
    Pack<A, V> h = load_pack<A, V>(at);
    Pack<X, V> y;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A a, rest, u = widen(x.v[v]);
        gate_factors(p.form, widen(g.v[SHARED ? 0 : v]), a, rest);
        if (p.complement) u *= rest;
        h.v[v] = fma_(a, h.v[v], u);
        y.v[v] = narrow<X>(h.v[v]);
    }
    store_pack<A, V>(at, h);
    store_pack<X, V>(static_cast<X*>(p.out) + row * p.dim + c0, y);
}

}  // namespace
}  // namespace sigb200
