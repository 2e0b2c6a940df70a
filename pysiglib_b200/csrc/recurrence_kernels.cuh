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

#include <climits>

#include "sequence.h"
#include "sequence_types.cuh"

namespace sigb200 {

struct RecurrencePlan {
    int log_lanes;     // CL = 1 << log_lanes threads side by side in the channels, 32 / CL parts in a warp
    int warps;         // W
    int cluster;       // CTAs that share a strip
    unsigned strips;   // strips of CL * V channels
    bool pairs;        // 8-byte neighbours are aligned to 16 bytes in every array
    int fold_log;      // backward, shared gates: lanes folded into one partial sum, log2
};

namespace {

__device__ __forceinline__ int saturated(long long v) {
    return v < INT_MIN ? INT_MIN : v > INT_MAX ? INT_MAX : int(v);
}
__device__ __forceinline__ int offset_at(const void* offsets, bool wide, int i) {
    return wide ? saturated(static_cast<const long long*>(offsets)[i]) : static_cast<const int*>(offsets)[i];
}

// Offsets of packed sequences that a CTA keeps in shared memory, where there are no more of them.
constexpr int kLocalOffsets = 512;

// Walks the packed sequences along the rows.  `seq` is the last sequence whose offset is at or before the row
// (-1 before the first, `count` behind the last); it spans rows [begin, next).  Offsets are only compared
// with rows, so values that are out of order or out of range take no access out of bounds.
struct SequenceWalk {
    const void* offsets;
    int count, seq, begin, next;
    bool wide;

    __device__ __forceinline__ void settle() {
        begin = seq >= 0 ? offset_at(offsets, wide, seq) : INT_MIN;
        next = seq < count ? offset_at(offsets, wide, seq + 1) : INT_MAX;
    }
    __device__ void seek(int row) {
        int lo = 0, hi = count + 1;  // first of the count + 1 offsets that is > row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (offset_at(offsets, wide, mid) <= row) lo = mid + 1; else hi = mid;
        }
        seq = lo - 1;
        settle();
    }
    // all threads: copies the offsets to `local` where they fit (behind a barrier)
    __device__ __forceinline__ void open(const RecurrenceArgs& p, int* local) {
        offsets = p.offsets; wide = p.wide_offsets; count = int(p.sequences);
        if (count + 1 <= kLocalOffsets) {
            for (int i = threadIdx.x; i <= count; i += blockDim.x) local[i] = offset_at(p.offsets, p.wide_offsets, i);
            __syncthreads();
            offsets = local;
            wide = false;
        }
    }
    __device__ __forceinline__ void advance(int row) {
        while (next <= row && seq < count) { ++seq; settle(); }
    }
    __device__ __forceinline__ void retreat(int row) {
        while (begin > row && seq >= 0) { --seq; settle(); }
    }
    __device__ __forceinline__ bool inside() const { return seq >= 0 && seq < count; }
    // no sequence starts or ends in [row, row + n), and all of those rows are in one
    __device__ __forceinline__ bool quiet(int row, int n) const { return inside() && begin < row && next > row + n; }
};

// What happens in a thread's S rows, one bit a row: a sequence starts, a sequence ends, the row is in none.
struct RowEvents {
    unsigned starts = 0, ends = 0, dead = 0;
};

template <int S>
__device__ __forceinline__ RowEvents row_events(SequenceWalk walk, int row0, int rows) {
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
__device__ __forceinline__ int64_t sequence_of(SequenceWalk walk, int row) {
    walk.advance(row);
    return walk.seq;
}

// a and 1 - a, neither by cancellation: exp and expm1 for logarithms; for logits, with e = e^-v kept finite,
// a = 1 / (1 + e) and 1 - a = e a.  The reciprocal is the hardware's (within 1 ulp).
// FAST (gates of 16 bits): exponentials as 2^(v log2 e) in single precision, off by up to 2 + 1.2 |v| ulp.  A gate
// of 8 or 11 bits leaves e^v uncertain by |v| 2^-9 or 2^-12 of itself, thousands of times more.
__device__ __forceinline__ float exponential(float v, bool fast) {
    if (!fast) return expf(v);
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
    return r;
}
__device__ __forceinline__ double exponential(double v, bool) { return exp(v); }
__device__ __forceinline__ float minus_expm1(float v) { return -expm1f(v); }
__device__ __forceinline__ double minus_expm1(double v) { return -expm1(v); }
__device__ __forceinline__ float below(float v) {  // at most 2^100, NaN kept
    float r;
    asm("min.NaN.f32 %0, %1, 0f71800000;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double below(double v) { return v > 0x1p1000 ? 0x1p1000 : v; }
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }
template <int FORM, bool FAST, typename A>
__device__ __forceinline__ void gate_factors(A v, A& a, A& rest) {
    if (FORM == kGateValue) { a = v; rest = A(1) - v; }
    else if (FORM == kGateLog) { a = exponential(v, FAST); rest = minus_expm1(v); }
    else {
        const A e = below(exponential(-v, FAST));
        a = reciprocal(A(1) + e);
        rest = e * a;
    }
}

__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }

#ifndef SIG_ROOM
#define SIG_ROOM 100
#endif
constexpr int kCtaThreads = 256;  // at most; also the stride of the prefetch slots

// One copy of B bytes (4, 8 or 16) to shared memory, asynchronous; `on` false writes zeros.
template <int B>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool on) {
    const unsigned at = static_cast<unsigned>(__cvta_generic_to_shared(to));
    const int bytes = on ? B : 0;
    if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(at), "l"(from), "n"(B), "r"(bytes) : "memory");
}
template <int B>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    const unsigned at = static_cast<unsigned>(__cvta_generic_to_shared(to));
    if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(B) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until all groups of the warp but the last N are there
template <int N>
__device__ __forceinline__ void await_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}

// The coming iterations' S rows of V values of one array.  4 bytes and more go asynchronously to
// slot [stage][row][thread] of shared memory; single 16-bit values, which that copy does not know, to
// registers, one iteration ahead.  Rows from `count` on read as zero (as anything, where there are none).
// Copies of less than 16 bytes pass through L1, whose free part bounds how many are in flight.  Where 8-byte
// neighbours are aligned as a pair, the even thread therefore copies both of an even row and the odd thread
// both of an odd row; a warp reads only what its own threads copied.
template <typename T, int V, int S>
struct Prefetch {
    static constexpr int kBytes = sizeof(T) * V;
    static constexpr bool kShared = kBytes >= 4, kPairs = V > 1 && kBytes == 8;
    static constexpr size_t kStage = kShared ? size_t(kBytes) * S * kCtaThreads : 0;
    Pack<T, V> held[kShared ? 1 : S];
    Pack<T, V>* slot;
    int odd;     // pairs: 1 for the thread that copies the odd rows
    bool pairs;

    __device__ __forceinline__ void place(unsigned char* at, int tc, bool in_pairs) {
        slot = reinterpret_cast<Pack<T, V>*>(at) + threadIdx.x;
        pairs = kPairs && in_pairs;
        odd = pairs ? tc & 1 : 0;
    }
    // where this thread's copies of the rows from `first` on start
    __device__ __forceinline__ const T* start(const T* first, int64_t stride) const { return odd ? first + stride - V : first; }

    __device__ __forceinline__ void issue(int stage, const T* base, const T* from, int64_t stride, int count) {
        if constexpr (kShared) {
            Pack<T, V>* to = slot + stage * S * kCtaThreads;
            if (kPairs && pairs) {
                to += odd * (kCtaThreads - 1);
                const int left = count - odd;
                stride *= 2;
                if (count == S) {
#pragma unroll
                    for (int s = 0; s < S; s += 2, from += stride) copy_async<16>(to + s * kCtaThreads, from);
                } else if (count > 0) {
#pragma unroll
                    for (int s = 0; s < S; s += 2, from += stride) copy_async<16>(to + s * kCtaThreads, s < left ? from : base, s < left);
                }
            } else if (count == S) {
#pragma unroll
                for (int s = 0; s < S; ++s, from += stride) copy_async<kBytes>(to + s * kCtaThreads, from);
            } else if (count > 0) {
#pragma unroll
                for (int s = 0; s < S; ++s, from += stride) copy_async<kBytes>(to + s * kCtaThreads, s < count ? from : base, s < count);
            }
        }
    }
    __device__ __forceinline__ void hold(const T* from, int64_t stride, int count) {
        if constexpr (!kShared) {
#pragma unroll
            for (int s = 0; s < S; ++s, from += stride) held[s] = s < count ? *reinterpret_cast<const Pack<T, V>*>(from) : Pack<T, V>{};
        }
    }
    __device__ __forceinline__ Pack<T, V> take(int stage, int s) const {
        if constexpr (kShared) return slot[(stage * S + s) * kCtaThreads];
        else return held[s];
    }
};

// Iterations whose inputs are in shared memory or on their way: as many as two CTAs an SM have room for.
template <typename X, typename G, int V, int GV, int S, int ARRAYS>
struct Stages {
    static constexpr size_t kBytes = ARRAYS * Prefetch<X, V, S>::kStage + Prefetch<G, GV, S>::kStage;
    static constexpr int kCount = kBytes * 4 <= SIG_ROOM * 1024 ? 4 : kBytes * 3 <= SIG_ROOM * 1024 ? 3 : 2;
};

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
    __device__ __forceinline__ void apply(A (&h)[V]) const {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = drop ? b[v] : fma_(a[v], h[v], b[v]);
    }
};

// Shared memory of one scan: the maps of the warps, the state that enters each of them, the state that enters
// the next iteration, and, twice by turns, the maps that the CTAs of a cluster hand to one another.
template <typename A>
struct ScanMemory {
    A *maps, *carry, *run, *others;  // [warp][A, B][width], [warp][width], [width], [turn][CTA][A, B][width]
    unsigned char *drops, *other_drops;  // [warp], [turn][CTA]
    int width;

    __host__ __device__ static constexpr size_t bytes(int width, int warps, int cluster) {
        return sizeof(A) * width * (3 * size_t(warps) + 1 + (cluster > 1 ? 4 * size_t(cluster) : 0)) + 16 * size_t(1 + (warps + 2 * cluster) / 16);
    }
    __device__ __forceinline__ void place(unsigned char* at, int w, int warps, int cluster) {
        width = w;
        maps = reinterpret_cast<A*>(at);
        carry = maps + 2 * warps * width;
        run = carry + warps * width;
        others = run + width;
        drops = reinterpret_cast<unsigned char*>(others + (cluster > 1 ? 4 * cluster * width : 0));
        other_drops = drops + warps;
    }
};

// Scan of the threads' maps over the parts of a warp (REVERSE: from the last part to the first).  On return
// `m` is the map of this part and everything in the warp before it; the whole warp's is in `memory`.
template <typename A, int V, bool REVERSE, bool PACKED>
__device__ __forceinline__ void scan_warp(Map<A, V>& m, int log_lanes, const ScanMemory<A>& memory) {
    const int lane = threadIdx.x & 31, lanes = 1 << log_lanes, parts = 32 >> log_lanes;
    const int part = REVERSE ? parts - 1 - (lane >> log_lanes) : lane >> log_lanes;
    const auto from = [&](auto value, int by) {
        return REVERSE ? __shfl_down_sync(0xffffffffu, value, by) : __shfl_up_sync(0xffffffffu, value, by);
    };
    for (int k = 1; k < parts; k <<= 1) {
        const bool earlier_drop = PACKED && from(int(m.drop), k << log_lanes);
        const bool take = part >= k && !(PACKED && m.drop);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const A ea = from(m.a[v], k << log_lanes), eb = from(m.b[v], k << log_lanes);
            if (take) {
                m.b[v] = fma_(m.a[v], eb, m.b[v]);
                m.a[v] *= ea;
            }
        }
        if (take) m.drop = earlier_drop;
    }
    if (part == parts - 1) {
        Pack<A, V> a, b;
#pragma unroll
        for (int v = 0; v < V; ++v) { a.v[v] = m.a[v]; b.v[v] = m.b[v]; }
        A* to = memory.maps + 2 * int(threadIdx.x >> 5) * memory.width + (lane & (lanes - 1)) * V;
        store_pack<A, V>(to, a);
        store_pack<A, V>(to + memory.width, b);
        if (PACKED && (lane & (lanes - 1)) == 0) memory.drops[threadIdx.x >> 5] = m.drop;
    }
}

// The state that enters this thread's rows, from the one that enters its warp's and the inclusive maps.
template <typename A, int V, bool REVERSE>
__device__ __forceinline__ void enter_rows(const Map<A, V>& m, int log_lanes, const A* carry, A (&h)[V]) {
    const int lane = threadIdx.x & 31, lanes = 1 << log_lanes;
    const Pack<A, V> in = load_pack<A, V>(carry);
    A behind[V];
#pragma unroll
    for (int v = 0; v < V; ++v) behind[v] = in.v[v];
    m.apply(behind);
    const bool first = REVERSE ? lane >= 32 - lanes : lane < lanes;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const A e = REVERSE ? __shfl_down_sync(0xffffffffu, behind[v], lanes) : __shfl_up_sync(0xffffffffu, behind[v], lanes);
        h[v] = first ? in.v[v] : e;
    }
}

// Column c of the strip, one thread each: the state `r` that enters the CTA's rows goes through the warps'
// maps, and what enters each warp is left in `carry`.
template <typename A, bool REVERSE, bool PACKED>
__device__ __forceinline__ A carry_through(const ScanMemory<A>& m, int warps, int c, A r) {
#pragma unroll 4
    for (int i = 0; i < warps; ++i) {
        const int w = REVERSE ? warps - 1 - i : i;
        m.carry[w * m.width + c] = r;
        const A b = m.maps[(2 * w + 1) * m.width + c];
        r = PACKED && m.drops[w] ? b : fma_(m.maps[2 * w * m.width + c], r, b);
    }
    return r;
}

// The same across a cluster: each CTA composes its warps' maps and writes the composition into every CTA's
// memory; behind the cluster's barrier each applies those before its own.  All threads call it.
template <typename A, bool REVERSE, bool PACKED>
__device__ __forceinline__ void carry_across(const ScanMemory<A>& m, int warps, int cluster, int rank, int turn) {
    auto group = cooperative_groups::this_cluster();
    A* others = m.others + turn * 2 * cluster * m.width;
    unsigned char* drops = m.other_drops + turn * cluster;
    for (int c = threadIdx.x; c < m.width; c += blockDim.x) {
        A a = A(1), b = A(0);
        bool drop = false;
        for (int i = 0; i < warps; ++i) {
            const int w = REVERSE ? warps - 1 - i : i;
            const A wa = m.maps[2 * w * m.width + c], wb = m.maps[(2 * w + 1) * m.width + c];
            const bool wd = PACKED && m.drops[w];
            b = wd ? wb : fma_(wa, b, wb);
            a *= wa;
            drop |= wd;
        }
        for (int r = 0; r < cluster; ++r) {
            A* there = group.map_shared_rank(others, r) + 2 * rank * m.width + c;
            there[0] = a;
            there[m.width] = b;
            if (PACKED && c == 0) group.map_shared_rank(drops, r)[rank] = drop;
        }
    }
    // only the threads that wrote order their writes before the barrier: a release by all would wait for every
    // thread's stores of outputs as well
    if (threadIdx.x < m.width) asm volatile("fence.acq_rel.cluster;" ::: "memory");
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int c = threadIdx.x; c < m.width; c += blockDim.x) {
        A r = m.run[c], mine = r;
        for (int i = 0; i < cluster; ++i) {
            const int k = REVERSE ? cluster - 1 - i : i;
            if (k == rank) mine = r;
            const A b = others[(2 * k + 1) * m.width + c];
            r = PACKED && drops[k] ? b : fma_(others[2 * k * m.width + c], r, b);
        }
        m.run[c] = r;
        carry_through<A, REVERSE, PACKED>(m, warps, c, mine);
    }
}

// a, x and, where REST, 1 - a of S rows from the prefetched inputs; without REST x is b already.
template <int FORM, bool REST, bool COMPLEMENT, typename X, typename G, int V, int GV, int S, typename A>
__device__ __forceinline__ void factors(const Prefetch<X, V, S>& fx, const Prefetch<G, GV, S>& fg, int stage, A (&a)[S][V],
                                        A (&u)[S][V], A (&rest)[REST ? S : 1][V]) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const Pack<X, V> x = fx.take(stage, s);
        const Pack<G, GV> g = fg.take(stage, s);
        A ga[GV], gr[GV];
#pragma unroll
        for (int v = 0; v < GV; ++v) gate_factors<FORM, sizeof(G) == 2>(A(widen(g.v[v])), ga[v], gr[v]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a[s][v] = ga[v % GV];
            u[s][v] = widen(x.v[v]);
            if (COMPLEMENT) u[s][v] *= gr[v % GV];
            if (REST) rest[s % (REST ? S : 1)][v] = gr[v % GV];
        }
    }
}

template <bool REST, bool COMPLEMENT, typename X, typename G, int V, int GV, int S, typename A>
__device__ __forceinline__ void factors(int form, const Prefetch<X, V, S>& fx, const Prefetch<G, GV, S>& fg, int stage, A (&a)[S][V],
                                        A (&u)[S][V], A (&rest)[REST ? S : 1][V]) {
    if (form == kGateValue) factors<kGateValue, REST, COMPLEMENT>(fx, fg, stage, a, u, rest);
    else if (form == kGateLog) factors<kGateLog, REST, COMPLEMENT>(fx, fg, stage, a, u, rest);
    else factors<kGateLogit, REST, COMPLEMENT>(fx, fg, stage, a, u, rest);
}

// Where a thread stands: its strip, channels and rows.
struct Place {
    int lanes, lane, warp, tc, parts, part, cluster, rank;
    uint64_t batch, first, c0;  // batch entry, first channel of the strip and of the thread
    bool live;

    __device__ __forceinline__ Place(const RecurrencePlan& plan, uint64_t dim, int V) {
        lanes = 1 << plan.log_lanes;
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        tc = lane & (lanes - 1);
        parts = 32 >> plan.log_lanes;
        part = warp * parts + (lane >> plan.log_lanes);
        cluster = plan.cluster;
        rank = cluster > 1 ? int(blockIdx.x % cluster) : 0;
        const uint64_t strip = cluster > 1 ? blockIdx.x / cluster : blockIdx.x;
        batch = strip / plan.strips;
        first = (strip % plan.strips) * lanes * V;
        c0 = first + uint64_t(tc) * V;
        live = c0 < dim;
    }
};

// How many of the S rows from row0 on there are (row0 may lie before 0 as a whole).
template <int S>
__device__ __forceinline__ int rows_left(int rows, int row0, bool live) {
    return live && row0 >= 0 ? max(0, min(S, rows - row0)) : 0;
}

template <typename X, typename G, int V, int S, bool SHARED, bool PACKED>
__global__ void __launch_bounds__(kCtaThreads, 2) recurrence_forward_kernel(const RecurrenceArgs p, const RecurrencePlan plan) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V, kStages = Stages<X, G, V, GV, S, 1>::kCount;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place at(plan, p.dim, V);
    const uint64_t b = at.batch, c0 = at.c0;
    const bool live = at.live;
    const int rows = int(p.rows);
    const int64_t dim = int64_t(p.dim);
    const A* initial = p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr;
    A* state = p.state ? static_cast<A*>(p.state) + c0 : nullptr;
    A* marks = p.checkpoints
        ? static_cast<A*>(p.checkpoints) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + c0 : nullptr;

    Prefetch<X, V, S> fx;
    Prefetch<G, GV, S> fg;
    unsigned char* next = smem;
    fx.place(next, at.tc, plan.pairs);
    next += kStages * fx.kStage;
    fg.place(next, at.tc, plan.pairs);
    next += kStages * fg.kStage;
    ScanMemory<A> memory;
    memory.place(next, at.lanes * V, plan.warps, at.cluster);
    for (int c = threadIdx.x; c < memory.width; c += blockDim.x)
        memory.run[c] = !PACKED && p.initial && at.first + c < p.dim ? static_cast<const A*>(p.initial)[b * p.dim + at.first + c] : A(0);
    const int span = plan.warps * at.parts * at.cluster * S;
    int row0 = (at.rank * plan.warps * at.parts + at.part) * S;
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + (live ? c0 : 0);
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (!live ? 0 : SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const int64_t x_row = int64_t(p.x_row), gate_row = int64_t(p.gate_row);
    const int64_t x_span = span * x_row, gate_span = span * gate_row, out_span = span * dim;
    const X* px = fx.start(x + int64_t(row0) * x_row, x_row);
    const G* pg = fg.start(gate + int64_t(row0) * gate_row, gate_row);
    X* out = p.out ? static_cast<X*>(p.out) + (int64_t(b * p.rows) + row0) * dim + c0 : nullptr;
    int coming = row0;  // the row that the next copies are for
    const auto fetch = [&](int stage) {
        const int n = rows_left<S>(rows, coming, live);
        fx.issue(stage, x, px, x_row, n);
        fg.issue(stage, gate, pg, gate_row, n);
        commit_copies();
        px += x_span;
        pg += gate_span;
        coming += span;
    };
    const auto hold = [&](int row) {
        const int n = rows_left<S>(rows, row, live);
        fx.hold(x + int64_t(row) * x_row, x_row, n);
        fg.hold(gate + int64_t(row) * gate_row, gate_row, n);
    };
    for (int k = 0; k < kStages - 1; ++k) fetch(k);
    hold(row0);
    if (at.cluster > 1) cooperative_groups::this_cluster().sync();  // all of it runs before any writes to another
    SequenceWalk walk;
    if (PACKED) {
        walk.open(p, reinterpret_cast<int*>(next + ScanMemory<A>::bytes(memory.width, plan.warps, at.cluster)));
        walk.seek(row0);
        if (state && live && at.rank == 0)  // sequences without rows hand their initial state on
            for (int j = at.part; j < walk.count; j += plan.warps * at.parts)
                if (offset_at(walk.offsets, walk.wide, j + 1) <= offset_at(walk.offsets, walk.wide, j))
                    for (int v = 0; v < V; ++v) state[j * dim + v] = initial ? initial[j * dim + v] : A(0);
    }
    int turn = 0, stage = 0;
    for (int base = 0; base < rows; base += span, row0 += span, turn ^= 1, stage = stage + 1 == kStages ? 0 : stage + 1) {
        const int count = rows_left<S>(rows, row0, live);
        fetch(stage == 0 ? kStages - 1 : stage - 1);  // its slots were read in the last iteration, before a barrier
        RowEvents e;
        if (PACKED) {
            walk.advance(row0);
            e = row_events<S>(walk, row0, rows);
        }
        A a[S][V], u[S][V], unused[1][V];
        await_copies<kStages - 1>();
        if (p.complement) factors<false, true>(p.form, fx, fg, stage, a, u, unused);
        else factors<false, false>(p.form, fx, fg, stage, a, u, unused);
        hold(row0 + span);
        if (count < S || (PACKED && e.dead)) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (s >= count || (e.dead >> s & 1u)) {
#pragma unroll
                    for (int v = 0; v < V; ++v) { a[s][v] = A(1); u[s][v] = A(0); }
                }
        }
        const bool events = PACKED && e.starts | e.ends | e.dead;
        // the initial state of a sequence that starts here joins b: its first row is then b alone
        if (events && e.starts && initial && live) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (e.starts >> s & 1u) {
                    const A* in = initial + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) u[s][v] = fma_(a[s][v], in[v], u[s][v]);
                }
        }
        Map<A, V> m;
        m.clear();
        if (!events) {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    m.b[v] = s ? fma_(a[s][v], m.b[v], u[s][v]) : u[s][v];
                    m.a[v] = s ? m.a[v] * a[s][v] : a[s][v];
                }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    m.b[v] = e.starts >> s & 1u ? u[s][v] : fma_(a[s][v], m.b[v], u[s][v]);
                    m.a[v] *= a[s][v];
                }
            m.drop = e.starts;
        }
        __syncwarp();
        scan_warp<A, V, false, PACKED>(m, plan.log_lanes, memory);
        __syncthreads();
        if (at.cluster == 1) {
            for (int c = threadIdx.x; c < memory.width; c += blockDim.x)
                memory.run[c] = carry_through<A, false, PACKED>(memory, plan.warps, c, memory.run[c]);
        } else {
            carry_across<A, false, PACKED>(memory, plan.warps, at.cluster, at.rank, turn);
        }
        __syncthreads();
        A h[V];
        enter_rows<A, V, false>(m, plan.log_lanes, memory.carry + at.warp * memory.width + at.tc * V, h);
        if (count) {
            if (marks && row0 % int(kCheckpointRows) == 0)
#pragma unroll
                for (int v = 0; v < V; ++v) marks[int64_t(row0 / int(kCheckpointRows)) * dim + v] = h[v];
            if (!events) {
                X* to = out;
                const int stored = out ? count : 0;
                if (stored == S) {
#pragma unroll
                    for (int s = 0; s < S; ++s, to += dim) {
#pragma unroll
                        for (int v = 0; v < V; ++v) h[v] = fma_(a[s][v], h[v], u[s][v]);
                        store_pack<X, V>(to, narrow_pack<X, V>(h));
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < S; ++s, to += dim) {
#pragma unroll
                        for (int v = 0; v < V; ++v) h[v] = fma_(a[s][v], h[v], u[s][v]);
                        if (s < stored) store_pack<X, V>(to, narrow_pack<X, V>(h));
                    }
                }
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    A y[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        h[v] = e.starts >> s & 1u ? u[s][v] : fma_(a[s][v], h[v], u[s][v]);
                        y[v] = e.dead >> s & 1u ? A(0) : h[v];
                    }
                    if (out && s < count) store_pack<X, V>(out + s * dim, narrow_pack<X, V>(y));
                    if (state && (e.ends >> s & 1u)) {
                        A* to = state + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                        for (int v = 0; v < V; ++v) to[v] = h[v];
                    }
                }
            }
        }
        if (out) out += out_span;
    }
    if (!PACKED && p.state && at.rank == 0)
        for (int c = threadIdx.x; c < memory.width && at.first + c < p.dim; c += blockDim.x)
            static_cast<A*>(p.state)[b * p.dim + at.first + c] = memory.run[c];
}

// One iteration takes its rows backward and then, from a checkpoint, forward again (for h_{t-1}), both in
// registers, so that x, the gates and the derivatives are read once and h, rounded or not, is not read at all.
// Shared gates: each thread sums its V channels, 1 << fold_log neighbouring lanes are folded by shuffles,
// and `partial` takes one value per row and fold (dgate itself where a fold is a whole gate).
template <typename X, typename G, int V, int S, bool SHARED, bool PACKED, bool COMPLEMENT>
__global__ void __launch_bounds__(kCtaThreads, 2) recurrence_backward_kernel(const RecurrenceArgs p, const RecurrencePlan plan,
                                                                     Acc<X>* partial) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V, kStages = Stages<X, G, V, GV, S, 2>::kCount;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place at(plan, p.dim, V);
    const uint64_t b = at.batch, c0 = at.c0;
    const bool live = at.live;
    const int rows = int(p.rows);
    const int64_t dim = int64_t(p.dim);
    const A* initial = p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr;
    const A* state_derivs = p.state_derivs ? static_cast<const A*>(p.state_derivs) + c0 : nullptr;
    A* dinitial = p.dinitial ? static_cast<A*>(p.dinitial) + c0 : nullptr;
    const A* marks = static_cast<const A*>(p.marks) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + at.first;

    Prefetch<X, V, S> fx, fd;
    Prefetch<G, GV, S> fg;
    unsigned char* next = smem;
    fx.place(next, at.tc, plan.pairs);
    next += kStages * fx.kStage;
    fd.place(next, at.tc, plan.pairs);
    next += kStages * fd.kStage;
    fg.place(next, at.tc, plan.pairs);
    next += kStages * fg.kStage;
    ScanMemory<A> ahead, back;
    ahead.place(next, at.lanes * V, plan.warps, 1);
    next += ScanMemory<A>::bytes(ahead.width, plan.warps, 1);
    back.place(next, ahead.width, plan.warps, at.cluster);
    A* entering = reinterpret_cast<A*>(next + ScanMemory<A>::bytes(ahead.width, plan.warps, at.cluster));  // [stage][width]
    for (int c = threadIdx.x; c < back.width; c += blockDim.x)
        back.run[c] = !PACKED && p.state_derivs && at.first + c < p.dim ? static_cast<const A*>(p.state_derivs)[b * p.dim + at.first + c] : A(0);
    const int block = plan.warps * at.parts * S, span = block * at.cluster;
    int base = (rows - 1) / span * span, row0 = base + at.rank * block + at.part * S;
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + (live ? c0 : 0);
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (!live ? 0 : SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const X* derivs = static_cast<const X*>(p.derivs) + b * p.d_batch + (live ? c0 : 0);
    const int64_t x_row = int64_t(p.x_row), gate_row = int64_t(p.gate_row), d_row = int64_t(p.d_row);
    const int64_t x_span = span * x_row, gate_span = span * gate_row, d_span = span * d_row;
    const X* px = fx.start(x + int64_t(row0) * x_row, x_row);
    const G* pg = fg.start(gate + int64_t(row0) * gate_row, gate_row);
    const X* pd = fd.start(derivs + int64_t(row0) * d_row, d_row);
    const int64_t out_span = span * dim;
    X* dx = static_cast<X*>(p.dx) + (int64_t(b) * rows + row0) * dim + c0;
    G* dgate = static_cast<G*>(p.dgate) + (SHARED ? 0 : (int64_t(b) * rows + row0) * dim + c0);
    int coming = row0, coming_base = base;
    const auto fetch = [&](int stage) {
        const int n = rows_left<S>(rows, coming, live);
        fx.issue(stage, x, px, x_row, n);
        fg.issue(stage, gate, pg, gate_row, n);
        fd.issue(stage, derivs, pd, d_row, n);
        // the checkpoint that enters the CTA's rows: each column's thread copies its own
        const int own = coming_base + at.rank * block;
        const A* mark = marks + int64_t(own / int(kCheckpointRows)) * dim;
        for (int c = threadIdx.x; c < ahead.width; c += blockDim.x) {
            const bool on = own >= 0 && own < rows && at.first + c < p.dim;
            copy_async<sizeof(A)>(entering + stage * ahead.width + c, on ? mark + c : static_cast<const A*>(p.marks), on);
        }
        commit_copies();
        px -= x_span;
        pg -= gate_span;
        pd -= d_span;
        coming -= span;
        coming_base -= span;
    };
    const auto hold = [&](int row) {
        const int n = rows_left<S>(rows, row, live);
        fx.hold(x + int64_t(row) * x_row, x_row, n);
        fg.hold(gate + int64_t(row) * gate_row, gate_row, n);
        fd.hold(derivs + int64_t(row) * d_row, d_row, n);
    };
    for (int k = 0; k < kStages - 1; ++k) fetch(k);
    hold(row0);
    if (at.cluster > 1) cooperative_groups::this_cluster().sync();  // all of it runs before any writes to another
    SequenceWalk walk;
    if (PACKED) {
        walk.open(p, reinterpret_cast<int*>(entering + kStages * ahead.width));
        walk.seek(row0);
        if (dinitial && live && at.rank == 0)
            for (int j = at.part; j < walk.count; j += plan.warps * at.parts)
                if (offset_at(walk.offsets, walk.wide, j + 1) <= offset_at(walk.offsets, walk.wide, j))
                    for (int v = 0; v < V; ++v) dinitial[j * dim + v] = state_derivs ? state_derivs[j * dim + v] : A(0);
    }
    int turn = 0, stage = 0;
    for (; base >= 0; base -= span, row0 -= span, turn ^= 1, stage = stage + 1 == kStages ? 0 : stage + 1) {
        const int count = rows_left<S>(rows, row0, live);
        fetch(stage == 0 ? kStages - 1 : stage - 1);  // its slots were read in the last iteration, before a barrier
        RowEvents e;
        if (PACKED) {
            walk.retreat(row0);
            e = row_events<S>(walk, row0, rows);
        }
        A a[S][V], rest[S][V], x_[S][V], d[S][V];
        await_copies<kStages - 1>();
        factors<true, false>(p.form, fx, fg, stage, a, x_, rest);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const Pack<X, V> rd = fd.take(stage, s);
#pragma unroll
            for (int v = 0; v < V; ++v) d[s][v] = widen(rd.v[v]);
        }
        hold(row0 - span);
        if (count < S || (PACKED && e.dead)) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (s >= count || (e.dead >> s & 1u)) {
#pragma unroll
                    for (int v = 0; v < V; ++v) { a[s][v] = A(1); rest[s][v] = x_[s][v] = d[s][v] = A(0); }
                }
        }
        const bool events = PACKED && e.starts | e.ends | e.dead;
        // the gradient of a state joins the derivatives of the row that it was taken from
        if (events && e.ends && state_derivs && live) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (e.ends >> s & 1u) {
                    const A* in = state_derivs + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) d[s][v] += in[v];
                }
        }
        Map<A, V> m, g;
        m.clear();
        g.clear();
        const auto input = [&](int s, int v) { return COMPLEMENT ? rest[s][v] * x_[s][v] : x_[s][v]; };
        if (!events) {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int q = S - 1 - s;
                    m.b[v] = s ? fma_(a[s][v], m.b[v], input(s, v)) : input(s, v);
                    m.a[v] = s ? m.a[v] * a[s][v] : a[s][v];
                    g.b[v] = a[q][v] * (s ? d[q][v] + g.b[v] : d[q][v]);
                }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (e.starts >> s & 1u) {
                    const A* in = initial && live ? initial + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
                    for (int v = 0; v < V; ++v) m.b[v] = in ? in[v] : A(0);
                }
                const int q = S - 1 - s;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    m.b[v] = fma_(a[s][v], m.b[v], input(s, v));
                    m.a[v] *= a[s][v];
                    g.b[v] = a[q][v] * (e.ends >> q & 1u ? d[q][v] : d[q][v] + g.b[v]);
                }
            }
            m.drop = e.starts;
            g.drop = e.ends;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) g.a[v] = m.a[v];
        __syncwarp();
        scan_warp<A, V, false, PACKED>(m, plan.log_lanes, ahead);
        scan_warp<A, V, true, PACKED>(g, plan.log_lanes, back);
        __syncthreads();
        for (int c = threadIdx.x; c < ahead.width; c += blockDim.x) carry_through<A, false, PACKED>(ahead, plan.warps, c, entering[stage * ahead.width + c]);
        if (at.cluster == 1) {
            for (int c = threadIdx.x; c < back.width; c += blockDim.x)
                back.run[c] = carry_through<A, true, PACKED>(back, plan.warps, c, back.run[c]);
        } else {
            carry_across<A, true, PACKED>(back, plan.warps, at.cluster, at.rank, turn);
        }
        __syncthreads();
        A in[V], w[V];
        enter_rows<A, V, false>(m, plan.log_lanes, ahead.carry + at.warp * ahead.width + at.tc * V, in);
        enter_rows<A, V, true>(g, plan.log_lanes, back.carry + at.warp * back.width + at.tc * V, w);
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
        X* to_x = dx;
        G* to_gate = dgate;
        dx -= out_span;
        dgate -= SHARED ? 0 : out_span;
#pragma unroll
        for (int s = 0; s < S; ++s, to_x += dim, to_gate += SHARED ? 0 : dim) {
            if (PACKED && (e.starts >> s & 1u)) {
                const A* from = initial && live ? initial + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
                for (int v = 0; v < V; ++v) in[v] = from ? from[v] : A(0);
            }
            A gx[V], gg[V], sum = A(0);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gx[v] = COMPLEMENT ? rest[s][v] * d[s][v] : d[s][v];
                gg[v] = d[s][v] * (COMPLEMENT ? in[v] - x_[s][v] : in[v]);
                if (p.form != kGateValue) gg[v] *= a[s][v];
                if (p.form == kGateLogit) gg[v] *= rest[s][v];
                if (PACKED && (e.dead >> s & 1u)) gx[v] = gg[v] = A(0);
                sum += gg[v];
                in[v] = fma_(a[s][v], in[v], input(s, v));
            }
            if (s < count) store_pack<X, V>(to_x, narrow_pack<X, V>(gx));
            if (SHARED) {
                sum = s < count ? sum : A(0);
                for (int k = 1; k < 1 << plan.fold_log; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                if (s < count && (at.tc & ((1 << plan.fold_log) - 1)) == 0) {
                    const int64_t fold = int64_t(c0 / V) >> plan.fold_log, row = int64_t(b) * rows + row0 + s;
                    if (partial) partial[row * ((dim / V) >> plan.fold_log) + fold] = sum;
                    else to_gate[row * int64_t(p.gate_dim) + fold] = narrow<G>(sum);
                }
            } else if (s < count) {
                if constexpr (std::is_same_v<Acc<G>, A>) store_pack<G, V>(to_gate, narrow_pack<G, V>(gg));
            }
        }
    }
    if (!PACKED && p.dinitial && at.rank == 0)
        for (int c = threadIdx.x; c < back.width && at.first + c < p.dim; c += blockDim.x)
            static_cast<A*>(p.dinitial)[b * p.dim + at.first + c] = back.run[c];
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
        if (p.form == kGateValue) gate_factors<kGateValue, sizeof(G) == 2>(t, a, rest);
        else if (p.form == kGateLog) gate_factors<kGateLog, sizeof(G) == 2>(t, a, rest);
        else gate_factors<kGateLogit, sizeof(G) == 2>(t, a, rest);
        if (p.complement) u *= rest;
        h.v[v] = fma_(a, h.v[v], u);
        y.v[v] = narrow<X>(h.v[v]);
    }
    store_pack<A, V>(at, h);
    store_pack<X, V>(static_cast<X*>(p.out) + row * p.dim + c0, y);
}

}  // namespace
}  // namespace sigb200
