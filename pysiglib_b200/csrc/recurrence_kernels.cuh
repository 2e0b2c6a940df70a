// Gated linear recurrence h_t = a_t h_{t-1} + b_t along the rows of (batch, rows, dim) arrays, its
// backward pass and its single-row step.
//
// Mathematics.  A run of rows maps the state entering it affinely, h -> A h + B, with A = prod a_t and B
// the recurrence started from 0, and two runs compose to (A2 A1, A2 B1 + B2).  The backward pass is the
// same recurrence from the other end in u_t = a_t g_t, the gradient handed to row t - 1: with d_t the
// derivatives of h_t, g_t = d_t + u_{t+1}, dx_t = g_t (or (1 - a_t) g_t) and da_t = g_t (h_{t-1} - [x_t]).
//
// Split.  A value costs three to five values of traffic and a few dozen operations at most, so the loads have to
// be in flight all the time.  A CTA owns a strip of CL * V neighbouring channels and walks down the rows, W warps
// times 32 / CL parts times S rows at a time: each thread holds S consecutive rows of V channels in
// registers and reduces them to one map.  The maps of a warp are composed by shuffles, those of the warps go
// through shared memory, and a second walk over the registers gives the S states.  The next
// iteration's inputs are copied into shared memory (asynchronously, into slots that only the thread itself reads)
// while this one's are folded and stored.  Every input is read once, every output written once, and the
// state that crosses an iteration stays in registers, in 32 bits (64 for float64 inputs).
//
// Where strips are too few to fill the GPU, a cluster of CTAs shares one: each takes a block of rows of every
// iteration and writes its map into the shared memory of the others; the cluster's barrier is the only wait.
//
// Packed sequences are one scan over all rows in which the first row of a sequence drops what enters it:
// the drop is a flag beside (A, B), not a gate of 0, so that a NaN or an infinity of one sequence
// stays inside it.
#pragma once

#include <cooperative_groups.h>

#include "sequence.h"
#include "sequence_types.cuh"

namespace sigb200 {

struct RecurrencePlan {
    int log_lanes;     // CL = 1 << log_lanes threads side by side in the channels, 32 / CL parts in a warp
    int warps;         // W
    int cluster;       // CTAs that share a strip
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
    __device__ __forceinline__ void retreat(int64_t row) {
        while (begin > row) { --seq; settle(); }
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

// a and 1 - a, neither by cancellation: exp and expm1 for logarithms; for logits both from e^-|v|, with the
// hardware's reciprocal (within 2 ulp on [1, 2]) in place of a division.
template <int FORM>
__device__ __forceinline__ void gate_factors(float v, float& a, float& rest) {
    if (FORM == kGateValue) { a = v; rest = 1.0f - v; }
    else if (FORM == kGateLog) { a = expf(v); rest = -expm1f(v); }
    else {
        const float e = expf(-fabsf(v)), r = __fdividef(1.0f, 1.0f + e), s = e * r;
        a = v >= 0.0f ? r : s;
        rest = v >= 0.0f ? s : r;
    }
}
template <int FORM>
__device__ __forceinline__ void gate_factors(double v, double& a, double& rest) {
    if (FORM == kGateValue) { a = v; rest = 1.0 - v; }
    else if (FORM == kGateLog) { a = exp(v); rest = -expm1(v); }
    else {
        const double e = exp(-fabs(v)), r = 1.0 / (1.0 + e), s = e * r;
        a = v >= 0.0 ? r : s;
        rest = v >= 0.0 ? s : r;
    }
}

__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }

// The next iteration's S rows of V values of one array.  4 bytes and more go asynchronously to
// slot [row][thread] of shared memory; single 16-bit values, which that copy does not know, to registers.
// Rows before 0, at or beyond `rows`, and channels beyond the last one read as zero.
template <typename T, int V, int S>
struct Prefetch {
    static constexpr int kBytes = sizeof(T) * V;
    static constexpr bool kShared = kBytes >= 4;
    static constexpr size_t smem(int threads) { return kShared ? size_t(kBytes) * S * threads : 0; }
    Pack<T, V> held[kShared ? 1 : S];
    Pack<T, V>* slot;

    __device__ __forceinline__ void issue(const T* base, int64_t row0, int64_t rows, int64_t stride, bool live) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool on = live && row0 + s >= 0 && row0 + s < rows;
            const T* from = base + (on ? (row0 + s) * stride : 0);
            if constexpr (kShared) {
                const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(slot + s * blockDim.x));
                const int bytes = on ? kBytes : 0;
                if constexpr (kBytes == 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
                else
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(kBytes), "r"(bytes) : "memory");
            } else {
                held[s] = on ? *reinterpret_cast<const Pack<T, V>*>(from) : Pack<T, V>{};
            }
        }
    }
    __device__ __forceinline__ Pack<T, V> take(int s) const {
        if constexpr (kShared) return slot[s * blockDim.x];
        else return held[s];
    }
};

__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void await_copies() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// The affine map of a run of rows on V channels; `drop`: what enters the run does not leave it.
template <typename A, int V>
struct Map {
    A a[V], b[V];
    bool drop;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int v = 0; v < V; ++v) { a[v] = A(1); b[v] = A(0); }
        drop = false;
    }
    // this map behind `earlier`
    __device__ __forceinline__ void behind(const Map& earlier) {
        if (drop) return;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            b[v] = fma_(a[v], earlier.b[v], b[v]);
            a[v] *= earlier.a[v];
        }
        drop = earlier.drop;
    }
    __device__ __forceinline__ void apply(A (&h)[V]) const {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = drop ? b[v] : fma_(a[v], h[v], b[v]);
    }
};

// Maps in shared memory: [warp or CTA][A, B][lane of the strip], with a flag each.
template <typename A, int V>
struct MapStore {
    Pack<A, V>* values;
    unsigned char* drops;
    int lanes;

    __device__ __forceinline__ void put(int i, int tc, const Map<A, V>& m) const {
        Pack<A, V> a, b;
#pragma unroll
        for (int v = 0; v < V; ++v) { a.v[v] = m.a[v]; b.v[v] = m.b[v]; }
        values[(2 * i) * lanes + tc] = a;
        values[(2 * i + 1) * lanes + tc] = b;
        if (tc == 0) drops[i] = m.drop;
    }
    template <bool PACKED>
    __device__ __forceinline__ Map<A, V> get(int i, int tc) const {
        const Pack<A, V> a = values[(2 * i) * lanes + tc], b = values[(2 * i + 1) * lanes + tc];
        Map<A, V> m;
#pragma unroll
        for (int v = 0; v < V; ++v) { m.a[v] = a.v[v]; m.b[v] = b.v[v]; }
        m.drop = PACKED && drops[i];
        return m;
    }
};

// Bytes of shared memory behind the prefetch slots: both buffers of the warps' maps (`scans` of them) and of
// the cluster's maps, flags included.
template <typename A, int V>
__host__ __device__ constexpr size_t map_bytes(int lanes, int count) { return 2 * sizeof(A) * V * size_t(lanes) * count + 16 * ((count + 15) / 16); }
template <typename A, int V>
__host__ __device__ constexpr size_t scan_bytes(int lanes, int warps, int cluster, int scans) {
    return 2 * (scans * map_bytes<A, V>(lanes, warps) + (cluster > 1 ? map_bytes<A, V>(lanes, cluster) : 0));
}

template <typename A, int V>
__device__ __forceinline__ MapStore<A, V> map_store(unsigned char* at, int lanes, int count) {
    MapStore<A, V> m;
    m.values = reinterpret_cast<Pack<A, V>*>(at);
    m.drops = at + 2 * sizeof(A) * V * size_t(lanes) * count;
    m.lanes = lanes;
    return m;
}

// Scan of the threads' maps over the parts of a warp (REVERSE: from the last part to the first).  On return
// `m` is the map of everything in the warp that comes before this part, and lanes of the last part in scan
// order have put the whole warp's map into `store`.
template <typename A, int V, bool REVERSE, bool PACKED>
__device__ __forceinline__ void scan_warp(Map<A, V>& m, int log_lanes, const MapStore<A, V>& store) {
    const int lane = threadIdx.x & 31, lanes = 1 << log_lanes, parts = 32 >> log_lanes;
    const int part = REVERSE ? parts - 1 - (lane >> log_lanes) : lane >> log_lanes;
    for (int k = 1; k < parts; k <<= 1) {
        Map<A, V> e;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            e.a[v] = REVERSE ? __shfl_down_sync(0xffffffffu, m.a[v], k << log_lanes) : __shfl_up_sync(0xffffffffu, m.a[v], k << log_lanes);
            e.b[v] = REVERSE ? __shfl_down_sync(0xffffffffu, m.b[v], k << log_lanes) : __shfl_up_sync(0xffffffffu, m.b[v], k << log_lanes);
        }
        e.drop = false;
        if (PACKED) e.drop = REVERSE ? __shfl_down_sync(0xffffffffu, int(m.drop), k << log_lanes) : __shfl_up_sync(0xffffffffu, int(m.drop), k << log_lanes);
        if (part >= k) m.behind(e);
    }
    if (part == parts - 1) store.put(threadIdx.x >> 5, lane & (lanes - 1), m);
    if (parts > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            m.a[v] = REVERSE ? __shfl_down_sync(0xffffffffu, m.a[v], lanes) : __shfl_up_sync(0xffffffffu, m.a[v], lanes);
            m.b[v] = REVERSE ? __shfl_down_sync(0xffffffffu, m.b[v], lanes) : __shfl_up_sync(0xffffffffu, m.b[v], lanes);
        }
        if (PACKED) m.drop = REVERSE ? __shfl_down_sync(0xffffffffu, int(m.drop), lanes) : __shfl_up_sync(0xffffffffu, int(m.drop), lanes);
    }
    if (part == 0) m.clear();
}

// The state that enters this thread's rows, from `run`, the state that enters the iteration's first row (in
// scan order), and `m`, the map of the parts before it in its warp; `run` moves on to the next iteration.
// One CTA: the warps' maps are applied in their order.  A cluster: each CTA composes its own, hands the
// composition to all and applies what lies before it.
template <typename A, int V, bool REVERSE, bool PACKED>
__device__ __forceinline__ void enter(A (&run)[V], A (&in)[V], const Map<A, V>& m, const MapStore<A, V>& store,
                                      const MapStore<A, V>& shared, int warps, int cluster, int rank, int tc) {
    const int warp = threadIdx.x >> 5;
    if (cluster == 1) {
#pragma unroll 4
        for (int i = 0; i < warps; ++i) {
            const int w = REVERSE ? warps - 1 - i : i;
            if (w == warp) {
#pragma unroll
                for (int v = 0; v < V; ++v) in[v] = run[v];
            }
            store.template get<PACKED>(w, tc).apply(run);
        }
    } else {
        Map<A, V> all;
        all.clear();
        for (int i = 0; i < warps; ++i) {
            Map<A, V> next = store.template get<PACKED>(REVERSE ? warps - 1 - i : i, tc);
            next.behind(all);
            all = next;
        }
        auto group = cooperative_groups::this_cluster();
        // each warp serves some of the CTAs
        if ((threadIdx.x & 31) < (1 << (31 - __clz(store.lanes))))
            for (int r = warp; r < cluster; r += warps) {
                MapStore<A, V> there = shared;
                there.values = group.map_shared_rank(shared.values, r);
                there.drops = group.map_shared_rank(shared.drops, r);
                there.put(rank, tc, all);
            }
        group.sync();
#pragma unroll
        for (int v = 0; v < V; ++v) in[v] = run[v];
        for (int i = 0; i < cluster; ++i) {
            const int r = REVERSE ? cluster - 1 - i : i;
            if (r == rank) {
#pragma unroll
                for (int v = 0; v < V; ++v) in[v] = run[v];
            }
            shared.template get<PACKED>(r, tc).apply(run);
        }
        for (int i = 0; i < (REVERSE ? warps - 1 - warp : warp); ++i)
            store.template get<PACKED>(REVERSE ? warps - 1 - i : i, tc).apply(in);
    }
    m.apply(in);
}

// a, x and, where REST, 1 - a of S rows from the prefetched inputs; without REST x is b already.
template <int FORM, bool REST, typename X, typename G, int V, int GV, int S, typename A>
__device__ __forceinline__ void factors(const Prefetch<X, V, S>& fx, const Prefetch<G, GV, S>& fg, bool complement,
                                        A (&a)[S][V], A (&u)[S][V], A (&rest)[REST ? S : 1][V]) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const Pack<X, V> x = fx.take(s);
        const Pack<G, GV> g = fg.take(s);
        A ga[GV], gr[GV];
#pragma unroll
        for (int v = 0; v < GV; ++v) gate_factors<FORM>(A(widen(g.v[v])), ga[v], gr[v]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a[s][v] = ga[v % GV];
            u[s][v] = widen(x.v[v]);
            if (REST) rest[s % (REST ? S : 1)][v] = gr[v % GV];
            else if (complement) u[s][v] *= gr[v % GV];
        }
    }
}

template <bool REST, typename X, typename G, int V, int GV, int S, typename A>
__device__ __forceinline__ void factors(int form, const Prefetch<X, V, S>& fx, const Prefetch<G, GV, S>& fg, bool complement,
                                        A (&a)[S][V], A (&u)[S][V], A (&rest)[REST ? S : 1][V]) {
    if (form == kGateValue) factors<kGateValue, REST>(fx, fg, complement, a, u, rest);
    else if (form == kGateLog) factors<kGateLog, REST>(fx, fg, complement, a, u, rest);
    else factors<kGateLogit, REST>(fx, fg, complement, a, u, rest);
}

template <typename X, typename G, int V, int S, bool SHARED, bool PACKED>
__global__ void __launch_bounds__(256, 2) recurrence_forward_kernel(const RecurrenceArgs p, const RecurrencePlan plan) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lanes = 1 << plan.log_lanes, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tc = lane & (lanes - 1), parts = 32 >> plan.log_lanes;
    const int cluster = plan.cluster, rank = cluster > 1 ? int(blockIdx.x % cluster) : 0;
    const uint64_t strip = blockIdx.x / cluster, b = strip / plan.strips;
    const uint64_t c0 = ((strip % plan.strips) * lanes + tc) * V;
    const bool live = c0 < p.dim;
    const int64_t rows = int64_t(p.rows), dim = int64_t(p.dim);
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + (live ? c0 : 0);
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (!live ? 0 : SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const A* initial = p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr;
    X* out = p.out ? static_cast<X*>(p.out) + b * p.rows * p.dim + c0 : nullptr;
    A* state = p.state ? static_cast<A*>(p.state) + c0 : nullptr;
    A* marks = p.checkpoints
        ? static_cast<A*>(p.checkpoints) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + c0 : nullptr;

    Prefetch<X, V, S> fx;
    Prefetch<G, GV, S> fg;
    fx.slot = reinterpret_cast<Pack<X, V>*>(smem) + threadIdx.x;
    unsigned char* at = smem + fx.smem(blockDim.x);
    fg.slot = reinterpret_cast<Pack<G, GV>*>(at) + threadIdx.x;
    at += (fg.smem(blockDim.x) + 15) / 16 * 16;
    MapStore<A, V> stores[2], shared[2];
    for (int k = 0; k < 2; ++k, at += map_bytes<A, V>(lanes, plan.warps)) stores[k] = map_store<A, V>(at, lanes, plan.warps);
    for (int k = 0; k < 2 && cluster > 1; ++k, at += map_bytes<A, V>(lanes, cluster)) shared[k] = map_store<A, V>(at, lanes, cluster);

    A run[V];  // the state that enters the iteration's first row
#pragma unroll
    for (int v = 0; v < V; ++v) run[v] = !PACKED && initial && live ? initial[b * p.dim + v] : A(0);
    const int part = warp * parts + (lane >> plan.log_lanes);
    if (PACKED && state && live && rank == 0)  // sequences without rows hand their initial state on
        for (int64_t j = part; j < int64_t(p.sequences); j += plan.warps * parts)
            if (offset_at(p.offsets, p.wide_offsets, j + 1) <= offset_at(p.offsets, p.wide_offsets, j))
                for (int v = 0; v < V; ++v) state[j * dim + v] = initial ? initial[j * dim + v] : A(0);

    const int64_t span = int64_t(plan.warps) * parts * cluster * S;
    int64_t row0 = (int64_t(rank) * plan.warps * parts + part) * S;
    SequenceWalk walk;
    if (PACKED) walk.seek(p.offsets, p.wide_offsets, p.sequences, row0);
    fx.issue(x, row0, rows, p.x_row, live);
    fg.issue(gate, row0, rows, p.gate_row, live);
    commit_copies();
    int buf = 0;
    for (int64_t base = 0; base < rows; base += span, row0 += span, buf ^= 1) {
        RowEvents e;
        if (PACKED) {
            walk.advance(row0);
            e = row_events<S>(walk, row0, rows);
        }
        A a[S][V], u[S][V], unused[1][V];
        await_copies();
        factors<false>(p.form, fx, fg, p.complement, a, u, unused);
        if (row0 + S > rows || (PACKED && e.dead))
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (row0 + s >= rows || (e.dead >> s & 1u)) { a[s][v] = A(1); u[s][v] = A(0); }
        // the initial state of a sequence that starts here joins b: its first row is then b alone
        if (PACKED && e.starts && initial && live)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (e.starts >> s & 1u) {
                    const A* in = initial + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) u[s][v] = fma_(a[s][v], in[v], u[s][v]);
                }
        Map<A, V> m;
        m.clear();
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m.b[v] = PACKED && (e.starts >> s & 1u) ? u[s][v] : fma_(a[s][v], m.b[v], u[s][v]);
                m.a[v] *= a[s][v];
            }
        m.drop = PACKED && e.starts;
        scan_warp<A, V, false, PACKED>(m, plan.log_lanes, stores[buf]);
        __syncthreads();
        fx.issue(x, row0 + span, rows, p.x_row, live);  // the slots were read before the barrier
        fg.issue(gate, row0 + span, rows, p.gate_row, live);
        commit_copies();
        A h[V];
        enter<A, V, false, PACKED>(run, h, m, stores[buf], shared[buf], plan.warps, cluster, rank, tc);
        if (!live || row0 >= rows) continue;
        if (marks && row0 % int64_t(kCheckpointRows) == 0)
#pragma unroll
            for (int v = 0; v < V; ++v) marks[row0 / int64_t(kCheckpointRows) * dim + v] = h[v];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            Pack<X, V> y;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = PACKED && (e.starts >> s & 1u) ? u[s][v] : fma_(a[s][v], h[v], u[s][v]);
                y.v[v] = narrow<X>(PACKED && (e.dead >> s & 1u) ? A(0) : h[v]);
            }
            if (out && row0 + s < rows) store_pack<X, V>(out + (row0 + s) * dim, y);
            if (PACKED && state && (e.ends >> s & 1u)) {
                A* to = state + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                for (int v = 0; v < V; ++v) to[v] = h[v];
            }
        }
    }
    if (!PACKED && state && live && part == 0 && rank == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) state[b * p.dim + v] = run[v];
}

// One iteration goes forward through its rows from a checkpoint (for h_{t-1}, kept in registers) and
// backward through the same registers, so that x, the gates and the derivatives are read once and h,
// rounded or not, is not read at all.
// Shared gates: each thread sums its V channels, 1 << fold_log neighbouring lanes are folded by shuffles,
// and `partial` takes one value per row and fold (dgate itself where a fold is a whole gate).
template <typename X, typename G, int V, int S, bool SHARED, bool PACKED>
__global__ void __launch_bounds__(256, 2) recurrence_backward_kernel(const RecurrenceArgs p, const RecurrencePlan plan,
                                                                     Acc<X>* partial) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lanes = 1 << plan.log_lanes, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tc = lane & (lanes - 1), parts = 32 >> plan.log_lanes;
    const int cluster = plan.cluster, rank = cluster > 1 ? int(blockIdx.x % cluster) : 0;
    const uint64_t strip = blockIdx.x / cluster, b = strip / plan.strips;
    const uint64_t c0 = ((strip % plan.strips) * lanes + tc) * V;
    const bool live = c0 < p.dim;
    const int64_t rows = int64_t(p.rows), dim = int64_t(p.dim);
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + (live ? c0 : 0);
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (!live ? 0 : SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const X* derivs = static_cast<const X*>(p.derivs) + b * p.d_batch + (live ? c0 : 0);
    const A* initial = p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr;
    const A* state_derivs = p.state_derivs ? static_cast<const A*>(p.state_derivs) + c0 : nullptr;
    const A* marks = static_cast<const A*>(p.marks) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + c0;
    X* dx = static_cast<X*>(p.dx) + b * p.rows * p.dim + c0;
    A* dinitial = p.dinitial ? static_cast<A*>(p.dinitial) + c0 : nullptr;
    const int64_t folds = SHARED ? (dim / V) >> plan.fold_log : 0;
    G* dgate = static_cast<G*>(p.dgate) + b * p.rows * p.gate_dim + (SHARED ? 0 : c0);

    Prefetch<X, V, S> fx, fd;
    Prefetch<G, GV, S> fg;
    fx.slot = reinterpret_cast<Pack<X, V>*>(smem) + threadIdx.x;
    fd.slot = fx.slot + S * blockDim.x;
    unsigned char* at = smem + 2 * fx.smem(blockDim.x);
    fg.slot = reinterpret_cast<Pack<G, GV>*>(at) + threadIdx.x;
    at += (fg.smem(blockDim.x) + 15) / 16 * 16;
    MapStore<A, V> ahead[2], stores[2], shared[2];
    for (int k = 0; k < 2; ++k, at += map_bytes<A, V>(lanes, plan.warps)) ahead[k] = map_store<A, V>(at, lanes, plan.warps);
    for (int k = 0; k < 2; ++k, at += map_bytes<A, V>(lanes, plan.warps)) stores[k] = map_store<A, V>(at, lanes, plan.warps);
    for (int k = 0; k < 2 && cluster > 1; ++k, at += map_bytes<A, V>(lanes, cluster)) shared[k] = map_store<A, V>(at, lanes, cluster);

    A run[V];  // the gradient that enters the iteration's last row from behind
#pragma unroll
    for (int v = 0; v < V; ++v) run[v] = !PACKED && state_derivs && live ? state_derivs[b * p.dim + v] : A(0);
    const int part = warp * parts + (lane >> plan.log_lanes);
    if (PACKED && dinitial && live && rank == 0)
        for (int64_t j = part; j < int64_t(p.sequences); j += plan.warps * parts)
            if (offset_at(p.offsets, p.wide_offsets, j + 1) <= offset_at(p.offsets, p.wide_offsets, j))
                for (int v = 0; v < V; ++v) dinitial[j * dim + v] = state_derivs ? state_derivs[j * dim + v] : A(0);

    const int64_t block = int64_t(plan.warps) * parts * S, span = block * cluster;
    int64_t base = (rows - 1) / span * span, row0 = base + rank * block + int64_t(part) * S;
    SequenceWalk walk;
    if (PACKED) walk.seek(p.offsets, p.wide_offsets, p.sequences, row0);
    fx.issue(x, row0, rows, p.x_row, live);
    fg.issue(gate, row0, rows, p.gate_row, live);
    fd.issue(derivs, row0, rows, p.d_row, live);
    commit_copies();
    int buf = 0;
    for (; base >= 0; base -= span, row0 -= span, buf ^= 1) {
        A h[V];
        const int64_t own = base + rank * block;  // the CTA's first row
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = live && own < rows ? marks[own / int64_t(kCheckpointRows) * dim + v] : A(0);
        RowEvents e;
        if (PACKED) {
            walk.retreat(row0);
            e = row_events<S>(walk, row0, rows);
        }
        A a[S][V], rest[S][V], x_[S][V], d[S][V];
        await_copies();
        factors<true>(p.form, fx, fg, p.complement, a, x_, rest);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const Pack<X, V> rd = fd.take(s);
#pragma unroll
            for (int v = 0; v < V; ++v) d[s][v] = widen(rd.v[v]);
        }
        if (row0 + S > rows || (PACKED && e.dead))
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (row0 + s >= rows || (e.dead >> s & 1u)) { a[s][v] = A(1); rest[s][v] = x_[s][v] = d[s][v] = A(0); }
        // the gradient of a state joins the derivatives of the row that it was taken from
        if (PACKED && e.ends && state_derivs && live)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (e.ends >> s & 1u) {
                    const A* in = state_derivs + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) d[s][v] += in[v];
                }
        Map<A, V> m, g;
        m.clear();
        g.clear();
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (PACKED && (e.starts >> s & 1u)) {
                const A* in = initial && live ? initial + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
                for (int v = 0; v < V; ++v) m.b[v] = in ? in[v] : A(0);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m.b[v] = fma_(a[s][v], m.b[v], p.complement ? rest[s][v] * x_[s][v] : x_[s][v]);
                m.a[v] *= a[s][v];
            }
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s)
#pragma unroll
            for (int v = 0; v < V; ++v)
                g.b[v] = a[s][v] * (PACKED && (e.ends >> s & 1u) ? d[s][v] : d[s][v] + g.b[v]);
#pragma unroll
        for (int v = 0; v < V; ++v) g.a[v] = m.a[v];
        m.drop = PACKED && e.starts;
        g.drop = PACKED && e.ends;
        scan_warp<A, V, false, PACKED>(m, plan.log_lanes, ahead[buf]);
        scan_warp<A, V, true, PACKED>(g, plan.log_lanes, stores[buf]);
        __syncthreads();
        fx.issue(x, row0 - span, rows, p.x_row, live);  // the slots were read before the barrier
        fg.issue(gate, row0 - span, rows, p.gate_row, live);
        fd.issue(derivs, row0 - span, rows, p.d_row, live);
        commit_copies();
        A in[V], w[V];
        enter<A, V, false, PACKED>(h, in, m, ahead[buf], ahead[buf], plan.warps, 1, 0, tc);
        enter<A, V, true, PACKED>(run, w, g, stores[buf], shared[buf], plan.warps, cluster, rank, tc);
        // backward through the rows: d becomes g
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (!(PACKED && (e.ends >> s & 1u))) d[s][v] += w[v];
                w[v] = a[s][v] * d[s][v];
            }
            if (PACKED && dinitial && live && (e.starts >> s & 1u)) {
                A* to = dinitial + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                for (int v = 0; v < V; ++v) to[v] = w[v];
            }
        }
        // forward through them with h_{t-1} in `in`
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (PACKED && (e.starts >> s & 1u)) {
                const A* from = initial && live ? initial + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
                for (int v = 0; v < V; ++v) in[v] = from ? from[v] : A(0);
            }
            const bool dead = PACKED && (e.dead >> s & 1u), stored = live && row0 + s < rows;
            Pack<X, V> gx;
            Pack<G, V> gg;
            A sum = A(0);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const A g_ = d[s][v];
                gx.v[v] = narrow<X>(dead ? A(0) : p.complement ? rest[s][v] * g_ : g_);
                A da = g_ * (p.complement ? in[v] - x_[s][v] : in[v]);
                if (p.form != kGateValue) da *= a[s][v];
                if (p.form == kGateLogit) da *= rest[s][v];
                if (dead) da = A(0);
                gg.v[v] = narrow<G>(da);
                sum += da;
                in[v] = fma_(a[s][v], in[v], p.complement ? rest[s][v] * x_[s][v] : x_[s][v]);
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
        }
    }
    if (!PACKED && dinitial && live && part == 0 && rank == 0)
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
        const A t = widen(g.v[SHARED ? 0 : v]);
        if (p.form == kGateValue) gate_factors<kGateValue>(t, a, rest);
        else if (p.form == kGateLog) gate_factors<kGateLog>(t, a, rest);
        else gate_factors<kGateLogit>(t, a, rest);
        if (p.complement) u *= rest;
        h.v[v] = fma_(a, h.v[v], u);
        y.v[v] = narrow<X>(h.v[v]);
    }
    store_pack<A, V>(at, h);
    store_pack<X, V>(static_cast<X*>(p.out) + row * p.dim + c0, y);
}

}  // namespace
}  // namespace sigb200
