// Gated linear recurrence h_t = a_t h_{t-1} + b_t along the rows of (batch, rows, dim) arrays, its
// backward pass and its single-row step.
//
// Mathematics.  A run of rows maps the state entering it affinely, h -> A h + B, with A = prod a_t and B
// the recurrence started from 0, and two runs compose to (A2 A1, A2 B1 + B2).  The backward pass is the
// same recurrence from the other end in u_t = a_t g_t, the gradient handed to row t - 1: with d_t the
// derivatives of h_t, g_t = d_t + u_{t+1}, dx_t = g_t (or (1 - a_t) g_t) and da_t = g_t (h_{t-1} - [x_t]).
//
// Split.  A value costs three to five values of traffic and a few dozen operations at most, so the loads have to
// be in flight all the time and nothing may stand still.  A CTA owns a strip of CL * V neighbouring channels and
// walks down the rows, W warps times 32 / CL parts times S rows at a time: each thread holds S consecutive
// rows of V channels in registers and reduces them to one map, the maps of a warp are composed by shuffles, the
// state goes round the ring of warps, each handing it to the next as soon as its map has been applied,
// and a second walk over the registers gives the S states.  No barrier holds all warps: while some wait
// for the state the others load and reduce.  The coming iterations' inputs are copied into shared memory
// asynchronously, into slots that only the warp itself reads.  Every input is read once, every output
// written once, and the state is held in 32 bits (64 for float64 inputs).
//
// Where the strips are too few to fill the GPU, the rows are cut into segments as well.  A first kernel reduces
// every segment to its map, each thread a contiguous run of rows and without any exchange on the way; the
// main kernel starts each segment from the maps before it.  That reads the inputs twice, the second
// time from L2 where they fit.
//
// Packed sequences are one scan over all rows in which the first row of a sequence drops what enters it:
// the drop is a flag beside (A, B), not a gate of 0, so that a NaN or an infinity of one sequence
// stays inside it.
#pragma once

#include <climits>

#include "sequence.h"
#include "sequence_types.cuh"

namespace sigb200 {

struct RecurrencePlan {
    int log_lanes;     // CL = 1 << log_lanes threads side by side in the channels, 32 / CL parts in a warp
    int warps;         // W
    int stages;        // iterations whose inputs are in shared memory or on their way, 2 to 4
    unsigned strips;   // strips of CL * V channels
    int segments;      // of the rows
    int segment_rows;  // a multiple of the rows of an iteration and, where there are several, of a checkpoint's
    bool pairs;        // 8-byte neighbours are aligned to 16 bytes in every array
    int fold_log;      // backward, shared gates: lanes folded into one partial sum, log2
    void* maps;        // [batch][segment][A, B][dim] of the segments, and
    int* drops;        // [batch][segment]
    bool follows;      // the launch right behind the one of those maps: it may begin before they are there
};

namespace {

__device__ __forceinline__ int saturated(long long v) {
    return v < INT_MIN ? INT_MIN : v > INT_MAX ? INT_MAX : int(v);
}
__device__ __forceinline__ int offset_at(const void* offsets, bool wide, int i) {
    return wide ? saturated(static_cast<const long long*>(offsets)[i]) : static_cast<const int*>(offsets)[i];
}

// Offsets of packed sequences that a CTA keeps in shared memory, where there are no more of them: what is left
// beside the backward pass's stages of 16-bit inputs with two CTAs an SM.
constexpr int kLocalOffsets = 240;

// Bytes of shared memory that they take.
__host__ __device__ inline size_t offset_room(const RecurrenceArgs& p) {
    return p.sequences && p.sequences < uint64_t(kLocalOffsets) ? (p.sequences + 4) / 4 * 16 : 0;
}

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

__device__ __forceinline__ float exponential(float v) { return expf(v); }
__device__ __forceinline__ double exponential(double v) { return exp(v); }
// a = e^v and 1 - a together: v = n ln 2 + f with |f| <= ln 2 / 2 (ln 2 in two parts), p = e^f - 1 by its Taylor
// series (the first term left out, f^8 / 8!, is below 2^-25 of p), a = 2^n + 2^n p and 1 - a = (1 - 2^n) - 2^n p,
// both halved on the way so that 2^n stays finite.  Below e^-87 a is 0.
__device__ __forceinline__ void exponential_pair(float v, float& a, float& rest) {
    float c;  // v within [-87, 89], NaN kept
    asm("{\n .reg .f32 t;\n max.NaN.f32 t, %1, 0fC2AE0000;\n min.NaN.f32 %0, t, 0f42B20000;\n}" : "=f"(c) : "f"(v));
    const float n = rintf(c * 1.4426950408889634f);
    const float f = fmaf(n, 1.9046543e-9f, fmaf(n, -0.69314718246459961f, c));
    float p = fmaf(f, 1.0f / 5040, 1.0f / 720);
    p = fmaf(p, f, 1.0f / 120);
    p = fmaf(p, f, 1.0f / 24);
    p = fmaf(p, f, 1.0f / 6);
    p = fmaf(p, f, 0.5f);
    p = fmaf(p * f, f, f);
    const float s = __int_as_float((__float2int_rn(n) + 126) << 23);  // 2^(n - 1), 0 for n = -126
    a = 2.0f * fmaf(s, p, s);
    rest = 2.0f * fmaf(-s, p, 0.5f - s);
}
__device__ __forceinline__ void exponential_pair(double v, double& a, double& rest) { a = exp(v); rest = -expm1(v); }
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }

// r = a b + c, a b, a + b and a - b on V values: two at a time where they are float32, which halves the issue slots
// (what bounds these kernels for 16-bit inputs).
template <typename A, int V> constexpr bool kTwo = std::is_same_v<A, float> && V % 2 == 0;
template <typename A, int V>
__device__ __forceinline__ void v_fma(A (&r)[V], const A (&a)[V], const A (&b)[V], const A (&c)[V]) {
    if constexpr (kTwo<A, V>) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
            const float2 t = __ffma2_rn(make_float2(a[v], a[v + 1]), make_float2(b[v], b[v + 1]), make_float2(c[v], c[v + 1]));
            r[v] = t.x;
            r[v + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = fma_(a[v], b[v], c[v]);
    }
}
template <typename A, int V>
__device__ __forceinline__ void v_mul(A (&r)[V], const A (&a)[V], const A (&b)[V]) {
    if constexpr (kTwo<A, V>) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
            const float2 t = __fmul2_rn(make_float2(a[v], a[v + 1]), make_float2(b[v], b[v + 1]));
            r[v] = t.x;
            r[v + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = a[v] * b[v];
    }
}
template <typename A, int V>
__device__ __forceinline__ void v_add(A (&r)[V], const A (&a)[V], const A (&b)[V]) {
    if constexpr (kTwo<A, V>) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
            const float2 t = __fadd2_rn(make_float2(a[v], a[v + 1]), make_float2(b[v], b[v + 1]));
            r[v] = t.x;
            r[v + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = a[v] + b[v];
    }
}
template <typename A, int V>
__device__ __forceinline__ void v_sub(A (&r)[V], const A (&a)[V], const A (&b)[V]) {
    if constexpr (kTwo<A, V>) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {  // -1 b + a is exact up to its one rounding
            const float2 t = __ffma2_rn(make_float2(b[v], b[v + 1]), make_float2(-1.0f, -1.0f), make_float2(a[v], a[v + 1]));
            r[v] = t.x;
            r[v + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = a[v] - b[v];
    }
}
template <typename A, int V>
__device__ __forceinline__ void v_fill(A (&r)[V], A value) {
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = value;
}

// 1 - a for a = 1 / (1 + e): e a, and 1 from 2^60 on, where it is 1 to the last bit long before a becomes 0 and e a
// meaningless (a gate of -infinity closes exactly).  NaN is kept.
template <typename A>
__device__ __forceinline__ A complement_of(A e, A a) { return e >= A(0x1p60) ? A(1) : e * a; }

// a, and where PAIR 1 - a, of V gate values, neither by cancellation; for logits, with e = e^-v, a = 1 / (1 + e) and
// 1 - a = e a.  The reciprocal is the hardware's (within 1 ulp).
// FAST (gates of 16 bits): exponentials as 2^(v log2 e) in single precision, off by up to 2 + 1.2 |v| ulp.  A gate
// of 8 or 11 bits leaves e^v uncertain by |v| 2^-9 or 2^-12 of itself, thousands of times more.
template <int FORM, bool FAST, bool PAIR, typename A, int V>
__device__ __forceinline__ void gate_factors(const A (&g)[V], A (&a)[V], A (&rest)[V]) {
    if constexpr (FORM == kGateValue) {
        A one[V];
        v_fill(one, A(1));
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = g[v];
        if (PAIR) v_sub(rest, one, g);
    } else if constexpr (FORM == kGateLog && PAIR) {
#pragma unroll
        for (int v = 0; v < V; ++v) exponential_pair(g[v], a[v], rest[v]);
    } else if constexpr (std::is_same_v<A, float> && FAST) {
        A t[V], unit[V];
        v_fill(t, FORM == kGateLogit ? -1.4426950408889634f : 1.4426950408889634f);
        v_mul(t, t, g);
#pragma unroll
        for (int v = 0; v < V; ++v) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t[v]) : "f"(t[v]));
        if constexpr (FORM == kGateLog) {
#pragma unroll
            for (int v = 0; v < V; ++v) a[v] = t[v];
        } else {
            v_fill(unit, 1.0f);
            v_add(unit, unit, t);
#pragma unroll
            for (int v = 0; v < V; ++v) a[v] = reciprocal(unit[v]);
            if (PAIR) {
#pragma unroll
                for (int v = 0; v < V; ++v) rest[v] = complement_of(t[v], a[v]);
            }
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (FORM == kGateLog) a[v] = exponential(g[v]);
            else {
                const A e = exponential(-g[v]);
                a[v] = reciprocal(A(1) + e);
                rest[v] = complement_of(e, a[v]);
            }
        }
    }
}

constexpr int kCtaThreads = 256;  // at most

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
// until all groups of the warp but the last `stages - 1` are there
__device__ __forceinline__ void await_copies(int stages) {
    if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (stages == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
}

// The coming iterations' S rows of V values of one array.  4 bytes and more go asynchronously to
// slot [stage][warp][row][lane] of shared memory.  Single 16-bit values, which that copy does not know, and the
// gates that channels share (REGISTERS), one for several lanes, go to registers, one iteration ahead.  Rows
// from `count` on read as zero.
// Copies of less than 16 bytes pass through L1, whose free part bounds how many are in flight.  Where 8-byte
// neighbours are aligned as a pair, the even thread therefore copies both of an even row and the odd thread
// both of an odd row; a warp reads only what its own threads copied.
template <typename T, int V, int S, bool REGISTERS>
struct Prefetch {
    static constexpr int kBytes = sizeof(T) * V;
    static constexpr bool kShared = !REGISTERS && kBytes >= 4, kPairs = V > 1 && kBytes == 8;
    static constexpr size_t kWarp = kShared ? size_t(kBytes) * S * 32 : 0;  // of a stage
    Pack<T, V> held[kShared ? 1 : S];
    Pack<T, V>* slot;
    int per_stage;  // packs
    int odd;        // pairs: 1 for the thread that copies the odd rows
    bool pairs;

    // takes `stages` stages of shared memory at `at` and returns its end
    __device__ __forceinline__ unsigned char* place(unsigned char* at, int stages, int warps, int tc, bool in_pairs) {
        slot = reinterpret_cast<Pack<T, V>*>(at) + (threadIdx.x >> 5) * S * 32 + (threadIdx.x & 31);
        per_stage = warps * S * 32;
        pairs = kPairs && in_pairs;
        odd = pairs ? tc & 1 : 0;
        return at + stages * warps * kWarp;
    }
    // where this thread's copies of the rows from `first` on start
    __device__ __forceinline__ const T* start(const T* first, int64_t stride) const { return odd ? first + stride - V : first; }

    // `base`: the array's start, the source of the copies that bring zeros.  They too have to be aligned to their
    // size, which a thread's own channels need not be where pairs are copied.
    __device__ __forceinline__ void issue(int stage, const T* base, const T* from, int64_t stride, int count) {
        if constexpr (kShared) {
            Pack<T, V>* to = slot + stage * per_stage;
            if (kPairs && pairs) {
                to += odd * 31;
                const int left = count - odd;
                stride *= 2;
                if (count == S) {
#pragma unroll
                    for (int s = 0; s < S; s += 2, from += stride) copy_async<16>(to + s * 32, from);
                } else {
#pragma unroll
                    for (int s = 0; s < S; s += 2, from += stride) copy_async<16>(to + s * 32, s < left ? from : base, s < left);
                }
            } else if (count == S) {
#pragma unroll
                for (int s = 0; s < S; ++s, from += stride) copy_async<kBytes>(to + s * 32, from);
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s, from += stride) copy_async<kBytes>(to + s * 32, s < count ? from : base, s < count);
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
        if constexpr (kShared) return slot[stage * per_stage + s * 32];
        else return held[s];
    }
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
};

// Scan of the threads' maps over the parts of a warp (REVERSE: from the last part to the first): `m` becomes the map of
// this part and everything in the warp before it.
template <typename A, int V, bool REVERSE, bool PACKED>
__device__ __forceinline__ void scan_warp(Map<A, V>& m, int log_lanes) {
    const int lane = threadIdx.x & 31, parts = 32 >> log_lanes;
    const int part = REVERSE ? parts - 1 - (lane >> log_lanes) : lane >> log_lanes;
    const auto from = [&](auto value, int by) {
        return REVERSE ? __shfl_down_sync(0xffffffffu, value, by) : __shfl_up_sync(0xffffffffu, value, by);
    };
    for (int k = 1; k < parts; k <<= 1) {
        const bool earlier_drop = PACKED && from(int(m.drop), k << log_lanes);
        const bool take = part >= k && !(PACKED && m.drop);
        A ea[V], eb[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            ea[v] = from(m.a[v], k << log_lanes);
            eb[v] = from(m.b[v], k << log_lanes);
        }
        if (take) {
            v_fma(m.b, m.a, eb, m.b);
            v_mul(m.a, m.a, ea);
            m.drop = earlier_drop;
        }
    }
}

// The state that enters this thread's rows, from `in`, which enters its warp's, and the maps of scan_warp; lanes of the
// part that comes last put what leaves the warp at `leaving`, before `pass_on`.
template <typename A, int V, bool REVERSE, typename PassOn>
__device__ __forceinline__ void enter_rows(const Map<A, V>& m, int log_lanes, const A (&in)[V], A (&h)[V], A* leaving, const PassOn& pass_on) {
    const int lane = threadIdx.x & 31, lanes = 1 << log_lanes;
    Pack<A, V> behind;
    v_fma(behind.v, m.a, in, m.b);
    if (m.drop) {
#pragma unroll
        for (int v = 0; v < V; ++v) behind.v[v] = m.b[v];
    }
    if (REVERSE ? lane < lanes : lane >= 32 - lanes) store_pack<A, V>(leaving, behind);
    pass_on();  // the next warp waits for it
    const bool first = REVERSE ? lane >= 32 - lanes : lane < lanes;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const A e = REVERSE ? __shfl_down_sync(0xffffffffu, behind.v[v], lanes) : __shfl_up_sync(0xffffffffu, behind.v[v], lanes);
        h[v] = first ? in[v] : e;
    }
}

// Hand-over between two warps of a CTA: the one that gives arrives, the one that takes waits for it.
// Both in whole warps.
__device__ __forceinline__ void give(int link) {
    __syncwarp();
    asm volatile("bar.arrive %0, 64;" ::"r"(link) : "memory");
}
__device__ __forceinline__ void take_over(int link) {
    __syncwarp();
    asm volatile("bar.sync %0, 64;" ::"r"(link) : "memory");
}

// Backward: whether the memory of through_segments is that of the rings (2 W rows of `width`), which are not yet in
// use: a strip of 64 channels and more leaves it room there.
__host__ __device__ constexpr bool fold_in_ring(int width) { return width >= 64; }

// What enters the strip's columns of a segment: `first`, which enters the first segment in scan order (null: 0), through
// the maps of the segments before this one.  All threads call it: groups of them compose runs of
// segments, which then go one after another.  `memory`: [group][A, B][width] and [group] drops; the result is left
// in its first `width` values.  A state of 0 meets no factor, so that a product of large gates that
// overflowed does it no harm.
template <typename A, bool REVERSE, bool PACKED>
__device__ __forceinline__ void through_segments(const RecurrencePlan& plan, uint64_t batch, int segment, uint64_t dim, uint64_t strip,
                                                 int width, const A* first, A* memory) {
    const int groups = max(1, int(blockDim.x) / width), before = REVERSE ? plan.segments - 1 - segment : segment;
    int* drops = reinterpret_cast<int*>(memory + 2 * groups * width);
    const int run = (before + groups - 1) / groups;
    for (int i = threadIdx.x; i < groups * width; i += blockDim.x) {
        const int group = i / width, c = i - group * width;
        A a = A(1), b = A(0);
        int drop = 0;
        if (strip + c < dim) {
#pragma unroll 8
            for (int k = group * run; k < min(before, (group + 1) * run); ++k) {
                const uint64_t at = batch * plan.segments + (REVERSE ? plan.segments - 1 - k : k);
                const A* map = static_cast<const A*>(plan.maps) + 2 * at * dim + strip + c;
                const A ma = map[0], mb = map[dim];
                const bool drops_here = PACKED && plan.drops[at];
                b = drops_here || b == A(0) ? mb : fma_(ma, b, mb);
                a *= ma;
                drop |= drops_here;
            }
        }
        memory[2 * group * width + c] = a;
        memory[(2 * group + 1) * width + c] = b;
        if (c == 0) drops[group] = drop;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
        A r = first && strip + c < dim ? first[strip + c] : A(0);
        for (int g = 0; g < groups; ++g) {
            const A b = memory[(2 * g + 1) * width + c];
            r = drops[g] || r == A(0) ? b : fma_(memory[2 * g * width + c], r, b);
        }
        memory[c] = r;  // this column's own
    }
    __syncthreads();
}

// a and b of S rows from the prefetched inputs.
template <int FORM, bool COMPLEMENT, typename X, typename G, int V, int GV, int S, bool R, typename A>
__device__ __forceinline__ void factors(const Prefetch<X, V, S, false>& fx, const Prefetch<G, GV, S, R>& fg, int stage, A (&a)[S][V],
                                        A (&u)[S][V]) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const Pack<X, V> x = fx.take(stage, s);
        const Pack<G, GV> g = fg.take(stage, s);
        A wide[GV], ga[GV], gr[GV], rest[V];
#pragma unroll
        for (int v = 0; v < GV; ++v) wide[v] = widen(g.v[v]);
        gate_factors<FORM, sizeof(G) == 2, COMPLEMENT>(wide, ga, gr);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a[s][v] = ga[v % GV];
            rest[v] = gr[v % GV];
            u[s][v] = widen(x.v[v]);
        }
        if (COMPLEMENT) v_mul(u[s], u[s], rest);
    }
}

template <bool COMPLEMENT, typename X, typename G, int V, int GV, int S, bool R, typename A>
__device__ __forceinline__ void factors(int form, const Prefetch<X, V, S, false>& fx, const Prefetch<G, GV, S, R>& fg, int stage, A (&a)[S][V],
                                        A (&u)[S][V]) {
    if (form == kGateValue) factors<kGateValue, COMPLEMENT>(fx, fg, stage, a, u);
    else if (form == kGateLog) factors<kGateLog, COMPLEMENT>(fx, fg, stage, a, u);
    else factors<kGateLogit, COMPLEMENT>(fx, fg, stage, a, u);
}

// Where a thread stands: its strip, channels and segment of the rows.
struct Place {
    int lanes, lane, warp, tc, parts, part, segment;
    uint64_t batch, c0;  // batch entry, the thread's first channel
    bool live;

    __device__ __forceinline__ Place(const RecurrencePlan& plan, uint64_t dim, int V) {
        lanes = 1 << plan.log_lanes;
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        tc = lane & (lanes - 1);
        parts = 32 >> plan.log_lanes;
        part = warp * parts + (lane >> plan.log_lanes);
        unsigned block = blockIdx.x;
        const unsigned strip = block % plan.strips;
        block /= plan.strips;
        segment = int(block % unsigned(plan.segments));
        batch = block / unsigned(plan.segments);
        c0 = (uint64_t(strip) * lanes + tc) * V;
        live = c0 < dim;
    }
};

// How many of the S rows from row0 on there are (row0 may lie before 0 as a whole).
template <int S>
__device__ __forceinline__ int rows_left(int rows, int row0, bool live) {
    return live && row0 >= 0 ? max(0, min(S, rows - row0)) : 0;
}

// Rows of a thread with what a packed sequence does in them.
template <typename A, int V, int S>
struct Rows {
    A a[S][V], u[S][V];  // u: b in the forward direction, d in the backward one
    RowEvents e;
    int count;
};

// Rows that are not there, or in no sequence, become the identity; the initial state of a sequence that starts here
// (0 without one, which a gate that is not finite does not leave 0) joins b, and its first row is then b alone (in
// the backward direction: the gradient of a state joins the derivatives of the row it was taken from).
template <bool REVERSE, typename A, int V, int S>
__device__ __forceinline__ void settle_rows(Rows<A, V, S>& r, const SequenceWalk& walk, int row0, const A* joins, int64_t dim, bool live) {
    if (r.count < S || r.e.dead) {
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s >= r.count || (r.e.dead >> s & 1u)) {
#pragma unroll
                for (int v = 0; v < V; ++v) { r.a[s][v] = A(1); r.u[s][v] = A(0); }
            }
    }
    const unsigned at = REVERSE ? r.e.ends : r.e.starts;
    if (at && live) {
        if (joins) {
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (at >> s & 1u) {
                    const A* in = joins + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) r.u[s][v] = REVERSE ? r.u[s][v] + in[v] : fma_(r.a[s][v], in[v], r.u[s][v]);
                }
        } else if (!REVERSE) {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) r.u[s][v] = at >> s & 1u ? fma_(r.a[s][v], A(0), r.u[s][v]) : r.u[s][v];
        }
    }
}

// Appends the rows to a map, in scan order.
template <bool REVERSE, bool PACKED, typename A, int V, int S>
__device__ __forceinline__ void append_rows(Map<A, V>& m, const Rows<A, V, S>& r) {
    const unsigned drops = REVERSE ? r.e.ends : r.e.starts;
    if (PACKED && drops) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int s = REVERSE ? S - 1 - i : i;
            const bool drop = drops >> s & 1u;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (REVERSE) m.b[v] = r.a[s][v] * (drop ? r.u[s][v] : r.u[s][v] + m.b[v]);
                else m.b[v] = drop ? r.u[s][v] : fma_(r.a[s][v], m.b[v], r.u[s][v]);
                m.a[v] *= r.a[s][v];
            }
        }
        m.drop = true;
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int s = REVERSE ? S - 1 - i : i;
            if (REVERSE) {
                v_add(m.b, r.u[s], m.b);
                v_mul(m.b, r.a[s], m.b);
            } else {
                v_fma(m.b, r.a[s], m.b, r.u[s]);
            }
            v_mul(m.a, m.a, r.a[s]);
        }
    }
}

// Measured (B200, eight launches between two events; the bytes alone would take what stands behind the bar): bfloat16
// 8x4096x2048 81 us | 61, 8x8192x4096 268 to 287 | 245 (the power cap moves the clock), float32 64x512x272 21 | 16: about
// 23 instructions a value at 61 % of the issue slots, 13.5 of the 16 warps an SM that 128 registers a thread admit.
// In segments, with the kernel of their maps: float32 1x65536x192 45 us | 23, bfloat16 16000x1536 in 23 sequences
// 48 | 15; there the warps wait for one another.
template <typename X, typename G, int V, int S, bool SHARED, bool PACKED>
__global__ void __launch_bounds__(kCtaThreads, 2) recurrence_forward_kernel(const RecurrenceArgs p, const RecurrencePlan plan) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place at(plan, p.dim, V);
    const uint64_t b = at.batch, c0 = at.c0;
    const bool live = at.live;
    const int stages = plan.stages, warps = plan.warps;
    const int64_t dim = int64_t(p.dim);
    const int first = at.segment * plan.segment_rows, rows = min(int(p.rows), first + plan.segment_rows);
    // made where they are needed, rather than held in registers all along
    const auto initial = [&] { return p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr; };
    const auto state = [&] { return static_cast<A*>(p.state) + c0; };

    Prefetch<X, V, S, false> fx;
    Prefetch<G, GV, S, SHARED> fg;
    unsigned char* next = smem;
    next = fx.place(next, stages, warps, at.tc, plan.pairs);
    next = fg.place(next, stages, warps, at.tc, plan.pairs);
    const int width = at.lanes * V;
    A* carry = reinterpret_cast<A*>(next) + at.tc * V;  // [warp][width]: the state on its way into each warp
    next += sizeof(A) * width * warps;

    const int span = warps * at.parts * S;
    int row0 = first + at.part * S;
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
        fx.issue(stage, static_cast<const X*>(p.x), px, x_row, n);
        fg.issue(stage, static_cast<const G*>(p.gate), pg, gate_row, n);
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
    for (int k = 0; k < stages - 1; ++k) fetch(k);
    hold(row0);
    A in[V];  // the state that enters the warp's rows
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = !PACKED && p.initial && live ? initial()[b * p.dim + v] : A(0);
    if (plan.segments > 1) {
        cudaGridDependencySynchronize();  // the maps; what is above runs beside the kernel that makes them
        A* fold = reinterpret_cast<A*>(next + offset_room(p));
        through_segments<A, false, PACKED>(plan, b, at.segment, p.dim, c0 - uint64_t(at.tc) * V, width,
                                           PACKED || !p.initial ? nullptr : static_cast<const A*>(p.initial) + b * p.dim, fold);
#pragma unroll
        for (int v = 0; v < V; ++v) in[v] = fold[at.tc * V + v];
    }
    SequenceWalk walk;
    if (PACKED) {
        walk.open(p, reinterpret_cast<int*>(next));
        walk.seek(row0);
        if (p.state && live && at.segment == 0)  // sequences without rows hand their initial state on
            for (int j = at.part; j < walk.count; j += warps * at.parts)
                if (offset_at(walk.offsets, walk.wide, j + 1) <= offset_at(walk.offsets, walk.wide, j))
                    for (int v = 0; v < V; ++v) state()[j * dim + v] = p.initial ? initial()[j * dim + v] : A(0);
    }
    const int link = 1 + at.warp, link_before = at.warp ? at.warp : warps;
    A* leaving = carry + (at.warp + 1 == warps ? 0 : at.warp + 1) * width;
    int stage = 0;
    for (int base = first; base < rows; base += span, row0 += span, stage = stage + 1 == stages ? 0 : stage + 1) {
        __syncwarp();
        fetch(stage == 0 ? stages - 1 : stage - 1);  // its slots were read in the last iteration
        Rows<A, V, S> r;
        r.count = rows_left<S>(rows, row0, live);
        if (PACKED) {
            walk.advance(row0);
            r.e = row_events<S>(walk, row0, rows);
        }
        await_copies(stages);
        if (p.complement) factors<true>(p.form, fx, fg, stage, r.a, r.u);
        else factors<false>(p.form, fx, fg, stage, r.a, r.u);
        hold(row0 + span);
        settle_rows<false>(r, walk, row0, initial(), dim, live);
        Map<A, V> m;
        m.clear();
        append_rows<false, PACKED>(m, r);
        __syncwarp();
        scan_warp<A, V, false, PACKED>(m, plan.log_lanes);
        if (base != first || at.warp) {  // one warp alone has one iteration (make_plan)
            take_over(link_before);
            const Pack<A, V> c = load_pack<A, V>(carry + at.warp * width);
#pragma unroll
            for (int v = 0; v < V; ++v) in[v] = c.v[v];
        }
        A h[V];
        enter_rows<A, V, false>(m, plan.log_lanes, in, h, leaving,
                                [&] { if (at.warp + 1 < warps || base + span < rows) give(link); });
        if (r.count) {
            if (p.checkpoints && row0 % int(kCheckpointRows) == 0) {
                Pack<A, V> mark;
#pragma unroll
                for (int v = 0; v < V; ++v) mark.v[v] = h[v];
                const int64_t n = b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) + row0 / int(kCheckpointRows);
                store_pack<A, V>(static_cast<A*>(p.checkpoints) + n * dim + c0, mark);
            }
            const int stored = out ? r.count : 0;
            X* to = out;
            if (!(PACKED && (r.e.starts | r.e.ends | r.e.dead))) {
                if (stored == S) {
#pragma unroll
                    for (int s = 0; s < S; ++s, to += dim) {
                        v_fma(h, r.a[s], h, r.u[s]);
                        store_pack<X, V>(to, narrow_pack<X, V>(h));
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < S; ++s, to += dim) {
                        v_fma(h, r.a[s], h, r.u[s]);
                        if (s < stored) store_pack<X, V>(to, narrow_pack<X, V>(h));
                    }
                }
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s, to += dim) {
                    A y[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        h[v] = r.e.starts >> s & 1u ? r.u[s][v] : fma_(r.a[s][v], h[v], r.u[s][v]);
                        y[v] = r.e.dead >> s & 1u ? A(0) : h[v];
                    }
                    if (s < stored) store_pack<X, V>(to, narrow_pack<X, V>(y));
                    if (p.state && (r.e.ends >> s & 1u)) {
                        A* last = state() + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                        for (int v = 0; v < V; ++v) last[v] = h[v];
                    }
                }
            }
        }
        if (out) out += out_span;
    }
    // what left the last warp's last part
    if (!PACKED && p.state && live && at.segment + 1 == plan.segments && at.warp + 1 == warps && at.lane >= 32 - at.lanes)
#pragma unroll
        for (int v = 0; v < V; ++v) state()[b * p.dim + v] = leaving[v];
}

// Sums S values each over 1 << log >= S neighbouring lanes.  Each of the first rounds halves the values a lane still
// holds, so that S - 1 + log - log2 S exchanges do instead of S log.  Returns the value whose sum this lane's
// sums[0] is, -1 where another lane has it too.
template <typename A, int S>
__device__ __forceinline__ int fold_rows(A (&sums)[S], int log, int tc) {
    int row = 0;
#pragma unroll
    for (int half = S / 2, bit = 0; half >= 1; half /= 2, ++bit) {
        const bool upper = tc >> bit & 1;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const A mine = upper ? sums[half + i] : sums[i], other = upper ? sums[i] : sums[half + i];
            sums[i] = mine + __shfl_xor_sync(0xffffffffu, other, 1 << bit);
        }
        row += upper ? half : 0;
    }
    constexpr int kRounds = S == 8 ? 3 : S == 4 ? 2 : 1;
    for (int k = kRounds; k < log; ++k) sums[0] += __shfl_xor_sync(0xffffffffu, sums[0], 1 << k);
    return (tc & ((1 << log) - 1)) >> kRounds ? -1 : row;
}

// What the backward pass takes twice from its slots, or keeps where they do not hold it: x and, for shared gates, 1 - a.
template <typename A, int V, int GV, int S>
struct Kept {
    A x[V > 1 ? 1 : S][V], rest[GV > 1 ? 1 : S][GV];
};

// First walk of the backward pass through its rows, upward: a and the derivatives into `r`, the rows appended to the map
// `m` of the state.  QUIET: all S rows are there and no sequence starts, ends or is missing in them.
template <int FORM, bool COMPLEMENT, bool QUIET, typename X, typename G, int V, int GV, int S, bool R, typename A, typename Start>
__device__ __forceinline__ void walk_up(const Prefetch<X, V, S, false>& fx, const Prefetch<X, V, S, false>& fd, const Prefetch<G, GV, S, R>& fg,
                                        int stage, Rows<A, V, S>& r, Map<A, V>& m, Kept<A, V, GV, S>& kept, const Start& first_state) {
    constexpr bool kPair = COMPLEMENT || (GV == 1 && FORM == kGateLogit);
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const Pack<X, V> x = fx.take(stage, s), d = fd.take(stage, s);
        const Pack<G, GV> g = fg.take(stage, s);
        A wide[GV], ga[GV], gr[GV], rest[V], b[V];
#pragma unroll
        for (int v = 0; v < GV; ++v) wide[v] = widen(g.v[v]);
        gate_factors<FORM, sizeof(G) == 2, kPair>(wide, ga, gr);
        if (GV == 1 && kPair) kept.rest[GV > 1 ? 0 : s][0] = gr[0];
        const bool gone = !QUIET && (s >= r.count || (r.e.dead >> s & 1u));
        if (!QUIET && (r.e.starts >> s & 1u)) first_state(s, m.b);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            b[v] = widen(x.v[v]);
            rest[v] = gr[v % GV];
            if (V == 1) kept.x[V > 1 ? 0 : s][v] = b[v];
            r.a[s][v] = gone ? A(1) : ga[v % GV];
            r.u[s][v] = gone ? A(0) : A(widen(d.v[v]));
        }
        if (COMPLEMENT) v_mul(b, b, rest);
        if (gone) v_fill(b, A(0));
        v_fma(m.b, r.a[s], m.b, b);
    }
}

template <bool COMPLEMENT, bool QUIET, typename X, typename G, int V, int GV, int S, bool R, typename A, typename Start>
__device__ __forceinline__ void walk_up(int form, const Prefetch<X, V, S, false>& fx, const Prefetch<X, V, S, false>& fd,
                                        const Prefetch<G, GV, S, R>& fg, int stage, Rows<A, V, S>& r, Map<A, V>& m, Kept<A, V, GV, S>& kept,
                                        const Start& first_state) {
    if (form == kGateValue) walk_up<kGateValue, COMPLEMENT, QUIET>(fx, fd, fg, stage, r, m, kept, first_state);
    else if (form == kGateLog) walk_up<kGateLog, COMPLEMENT, QUIET>(fx, fd, fg, stage, r, m, kept, first_state);
    else walk_up<kGateLogit, COMPLEMENT, QUIET>(fx, fd, fg, stage, r, m, kept, first_state);
}

// Last walk, upward again with h_{t-1} in `h` and the gradients g in r.u: dx and dgate of each row go to `store`.
template <int FORM, bool COMPLEMENT, bool QUIET, typename X, typename G, int V, int GV, int S, bool R, typename A, typename Start, typename Store>
__device__ __forceinline__ void walk_out(const Prefetch<X, V, S, false>& fx, const Prefetch<G, GV, S, R>& fg, int stage, const Rows<A, V, S>& r,
                                         const Kept<A, V, GV, S>& kept, A (&h)[V], const Start& first_state, const Store& store) {
    constexpr bool kPair = COMPLEMENT || FORM == kGateLogit;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (!QUIET && (r.e.starts >> s & 1u)) first_state(s, h);
        A x[V], rest[V], dx[V], dgate[V];
        if (V > 1) {
            const Pack<X, V> again = fx.take(stage, s);
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = widen(again.v[v]);
        } else {
            x[0] = kept.x[V > 1 ? 0 : s][0];
        }
        if constexpr (kPair && GV > 1) {
            const Pack<G, GV> g = fg.take(stage, s);
            A wide[GV], unused[GV];
#pragma unroll
            for (int v = 0; v < GV; ++v) wide[v] = widen(g.v[v]);
            gate_factors<FORM, sizeof(G) == 2, true>(wide, unused, rest);
        } else if (kPair) {
            v_fill(rest, kept.rest[GV > 1 ? 0 : s][0]);
        }
        const bool dead = !QUIET && (r.e.dead >> s & 1u);
        if (COMPLEMENT) {
            v_mul(dx, rest, r.u[s]);
            v_sub(dgate, h, x);
            v_mul(dgate, dgate, r.u[s]);
            v_mul(x, x, rest);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) dx[v] = r.u[s][v];
            v_mul(dgate, h, r.u[s]);
        }
        if (FORM != kGateValue) v_mul(dgate, dgate, r.a[s]);
        if (FORM == kGateLogit) v_mul(dgate, dgate, rest);
        if (dead) {
            v_fill(dx, A(0));
            v_fill(dgate, A(0));
        }
        v_fma(h, r.a[s], h, x);
        store(std::bool_constant<QUIET>{}, s, dx, dgate);
    }
}

template <bool COMPLEMENT, bool QUIET, typename X, typename G, int V, int GV, int S, bool R, typename A, typename Start, typename Store>
__device__ __forceinline__ void walk_out(int form, const Prefetch<X, V, S, false>& fx, const Prefetch<G, GV, S, R>& fg, int stage,
                                         const Rows<A, V, S>& r, const Kept<A, V, GV, S>& kept, A (&h)[V], const Start& first_state, const Store& store) {
    if (form == kGateValue) walk_out<kGateValue, COMPLEMENT, QUIET>(fx, fg, stage, r, kept, h, first_state, store);
    else if (form == kGateLog) walk_out<kGateLog, COMPLEMENT, QUIET>(fx, fg, stage, r, kept, h, first_state, store);
    else walk_out<kGateLogit, COMPLEMENT, QUIET>(fx, fg, stage, r, kept, h, first_state, store);
}

// One iteration walks up its rows (factors and maps), down (gradients) and up again from a checkpoint (h_{t-1} and
// the outputs), with a and the gradients in registers and x and the gates read again from shared memory, so that
// x, the gates and the derivatives are read once and h, rounded or not, is not read at all.
// Checkpoints are near enough for a warp to start from one, or from the warp before; the gradient goes round
// the ring of warps, from the last to the first.
// Shared gates: each thread sums its V channels, 1 << fold_log neighbouring lanes are folded by shuffles,
// and `partial` takes one value per row and fold (dgate itself where a fold is a whole gate).
// Measured (as above): bfloat16 8x4096x2048 153 us | 102, float32 64x512x272 38 | 27: about 45 instructions a value
// at 60 % of the issue slots, 256 CTAs for 296 places; in segments float32 1x65536x192 62 us | 38, bfloat16 16000x1536
// 79 | 23.
template <typename X, typename G, int V, int S, bool SHARED, bool PACKED, bool COMPLEMENT>
__global__ void __launch_bounds__(kCtaThreads, 2) recurrence_backward_kernel(const RecurrenceArgs p, const RecurrencePlan plan,
                                                                     Acc<X>* partial) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place at(plan, p.dim, V);
    const uint64_t b = at.batch, c0 = at.c0;
    const bool live = at.live;
    const int stages = plan.stages, warps = plan.warps;
    const int64_t dim = int64_t(p.dim);
    const int first = at.segment * plan.segment_rows, rows = min(int(p.rows), first + plan.segment_rows);
    // made where they are needed, rather than held in registers all along
    const auto initial = [&] { return p.initial ? static_cast<const A*>(p.initial) + c0 : nullptr; };
    const auto state_derivs = [&] { return p.state_derivs ? static_cast<const A*>(p.state_derivs) + c0 : nullptr; };
    const auto dinitial = [&] { return static_cast<A*>(p.dinitial) + c0; };

    Prefetch<X, V, S, false> fx, fd;
    Prefetch<G, GV, S, SHARED> fg;
    unsigned char* next = smem;
    next = fx.place(next, stages, warps, at.tc, plan.pairs);
    next = fd.place(next, stages, warps, at.tc, plan.pairs);
    next = fg.place(next, stages, warps, at.tc, plan.pairs);
    const int width = at.lanes * V;
    A* ahead = reinterpret_cast<A*>(next) + at.tc * V;  // [warp][width]: the state on its way into each warp
    A* back = ahead + warps * width;                    // [warp][width]: the gradient
    A* entering = back + (warps + at.warp) * width;     // [stage][warp][width]: checkpoints
    next += sizeof(A) * width * warps * (2 + stages);

    const int span = warps * at.parts * S;
    int base = first + (rows - 1 - first) / span * span, row0 = base + at.part * S;
    const int last_base = base;
    const X* x = static_cast<const X*>(p.x) + b * p.x_batch + (live ? c0 : 0);
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (!live ? 0 : SHARED ? c0 / (p.dim / p.gate_dim) : c0);
    const X* derivs = static_cast<const X*>(p.derivs) + b * p.d_batch + (live ? c0 : 0);
    const int64_t x_row = int64_t(p.x_row), gate_row = int64_t(p.gate_row), d_row = int64_t(p.d_row);
    const int64_t x_span = span * x_row, gate_span = span * gate_row, d_span = span * d_row;
    const X* px = fx.start(x + int64_t(row0) * x_row, x_row);
    const G* pg = fg.start(gate + int64_t(row0) * gate_row, gate_row);
    const X* pd = fd.start(derivs + int64_t(row0) * d_row, d_row);
    // warps whose first row is a checkpoint's start from it, the others from the warp before
    const int warp_rows = at.parts * S;
    const bool marked = at.warp * warp_rows % int(kCheckpointRows) == 0;
    const bool passes = at.warp + 1 < warps && (at.warp + 1) * warp_rows % int(kCheckpointRows) != 0;
    const A* marks = static_cast<const A*>(p.marks) + b * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim + c0;
    const int64_t out_span = span * dim;
    X* dx = static_cast<X*>(p.dx) + (int64_t(b * p.rows) + row0) * dim + c0;
    G* dgate = static_cast<G*>(p.dgate) + (SHARED ? 0 : (int64_t(b * p.rows) + row0) * dim + c0);
    int coming = row0, coming_base = base;
    const auto fetch = [&](int stage) {
        const int n = coming_base >= first ? rows_left<S>(rows, coming, live) : 0;
        fx.issue(stage, static_cast<const X*>(p.x), px, x_row, n);
        fg.issue(stage, static_cast<const G*>(p.gate), pg, gate_row, n);
        fd.issue(stage, static_cast<const X*>(p.derivs), pd, d_row, n);
        const int own = coming_base + at.warp * warp_rows;  // the warp's first row
        if (marked && live && at.lane < at.lanes && coming_base >= first && own < rows)
            copy_async<sizeof(A) * V>(entering + stage * warps * width, marks + int64_t(own / int(kCheckpointRows)) * dim);
        commit_copies();
        px -= x_span;
        pg -= gate_span;
        pd -= d_span;
        coming -= span;
        coming_base -= span;
    };
    const auto hold = [&](int row, bool on) {
        const int n = on ? rows_left<S>(rows, row, live) : 0;
        fx.hold(x + int64_t(row) * x_row, x_row, n);
        fg.hold(gate + int64_t(row) * gate_row, gate_row, n);
        fd.hold(derivs + int64_t(row) * d_row, d_row, n);
    };
    for (int k = 0; k < stages - 1; ++k) fetch(k);
    hold(row0, true);
    A w[V];  // the gradient that enters the warp's rows from behind
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = !PACKED && p.state_derivs && live ? state_derivs()[b * p.dim + v] : A(0);
    if (plan.segments > 1) {
        cudaGridDependencySynchronize();  // the maps; what is above runs beside the kernel that makes them
        A* fold = fold_in_ring(width) ? ahead - at.tc * V : reinterpret_cast<A*>(next + offset_room(p));
        through_segments<A, true, PACKED>(plan, b, at.segment, p.dim, c0 - uint64_t(at.tc) * V, width,
                                          PACKED || !p.state_derivs ? nullptr : static_cast<const A*>(p.state_derivs) + b * p.dim, fold);
#pragma unroll
        for (int v = 0; v < V; ++v) w[v] = fold[at.tc * V + v];
        if (fold_in_ring(width)) __syncthreads();
    }
    SequenceWalk walk;
    if (PACKED) {
        walk.open(p, reinterpret_cast<int*>(next));
        walk.seek(row0);
        if (p.dinitial && live && at.segment == 0)
            for (int j = at.part; j < walk.count; j += warps * at.parts)
                if (offset_at(walk.offsets, walk.wide, j + 1) <= offset_at(walk.offsets, walk.wide, j))
                    for (int v = 0; v < V; ++v) dinitial()[j * dim + v] = p.state_derivs ? state_derivs()[j * dim + v] : A(0);
    }
    // hand-overs: 1 .. W of the gradient to the warp before (or from the first to the last), W + 1 .. of the state
    const int link = 1 + at.warp, link_behind = at.warp + 1 == warps ? 1 : 2 + at.warp;
    A* leaving = back + (at.warp ? at.warp - 1 : warps - 1) * width;
    int stage = 0;
    for (; base >= first; base -= span, row0 -= span, stage = stage + 1 == stages ? 0 : stage + 1) {
        __syncwarp();
        fetch(stage == 0 ? stages - 1 : stage - 1);  // its slots were read in the last iteration
        Rows<A, V, S> r;  // u: derivatives, later their sums
        r.count = rows_left<S>(rows, row0, live);
        if (PACKED) {
            walk.retreat(row0);
            r.e = row_events<S>(walk, row0, rows);
        }
        const auto first_state = [&](int s, A (&h)[V]) {
            const A* from = p.initial && live ? initial() + sequence_of(walk, row0 + s) * dim : nullptr;
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = from ? from[v] : A(0);
        };
        const bool quiet = r.count == S && !(PACKED && (r.e.starts | r.e.ends | r.e.dead));
        Map<A, V> m, g;
        m.clear();
        Kept<A, V, GV, S> kept;
        await_copies(stages);
        if (quiet) walk_up<COMPLEMENT, true>(p.form, fx, fd, fg, stage, r, m, kept, first_state);
        else walk_up<COMPLEMENT, false>(p.form, fx, fd, fg, stage, r, m, kept, first_state);
        hold(row0 - span, base > first);
        if (PACKED && r.e.ends && p.state_derivs && live) settle_rows<true>(r, walk, row0, state_derivs(), dim, live);
        g.clear();
        append_rows<true, PACKED>(g, r);
#pragma unroll
        for (int v = 0; v < V; ++v) m.a[v] = g.a[v];
        m.drop = PACKED && r.e.starts;
        __syncwarp();
        scan_warp<A, V, false, PACKED>(m, plan.log_lanes);
        scan_warp<A, V, true, PACKED>(g, plan.log_lanes);
        // forward: the checkpoint, or what the warp before left
        A in[V], h[V];
        if (!marked) take_over(warps + at.warp);
        {
            const Pack<A, V> c = load_pack<A, V>(marked ? entering + stage * warps * width : ahead + at.warp * width);
#pragma unroll
            for (int v = 0; v < V; ++v) in[v] = c.v[v];
        }
        enter_rows<A, V, false>(m, plan.log_lanes, in, h, ahead + (at.warp + 1 == warps ? 0 : at.warp + 1) * width,
                                [&] { if (passes) give(warps + 1 + at.warp); });
        // backward: the gradient
        if (base != last_base || at.warp + 1 < warps) {
            take_over(link_behind);
            const Pack<A, V> c = load_pack<A, V>(back + at.warp * width);
#pragma unroll
            for (int v = 0; v < V; ++v) w[v] = c.v[v];
        }
        A behind[V];
        enter_rows<A, V, true>(g, plan.log_lanes, w, behind, leaving, [&] { if (at.warp || base > first) give(link); });
        // backward through the rows: the derivatives become g
        if (PACKED && !quiet) {
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                if (!(r.e.ends >> s & 1u)) v_add(r.u[s], r.u[s], behind);
                v_mul(behind, r.a[s], r.u[s]);
                if (p.dinitial && live && (r.e.starts >> s & 1u)) {
                    A* to = dinitial() + sequence_of(walk, row0 + s) * dim;
#pragma unroll
                    for (int v = 0; v < V; ++v) to[v] = behind[v];
                }
            }
        } else {
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                v_add(r.u[s], r.u[s], behind);
                v_mul(behind, r.a[s], r.u[s]);
            }
        }
        A sums[SHARED ? S : 1];
        X* to_x = dx;
        G* to_gate = dgate;
        dx -= out_span;
        dgate -= SHARED ? 0 : out_span;
        const auto store = [&](auto all, int s, const A (&gx)[V], const A (&gg)[V]) {
            if (all || s < r.count) store_pack<X, V>(to_x, narrow_pack<X, V>(gx));
            to_x += dim;
            if constexpr (SHARED) {
                A sum = gg[0];
#pragma unroll
                for (int v = 1; v < V; ++v) sum += gg[v];
                sums[s] = sum;
            } else {
                if constexpr (std::is_same_v<Acc<G>, A>)
                    if (all || s < r.count) store_pack<G, V>(to_gate, narrow_pack<G, V>(gg));
                to_gate += dim;
            }
        };
        if (quiet) walk_out<COMPLEMENT, true>(p.form, fx, fg, stage, r, kept, h, first_state, store);
        else walk_out<COMPLEMENT, false>(p.form, fx, fg, stage, r, kept, h, first_state, store);
        if constexpr (SHARED) {
            const int64_t fold = int64_t(c0 / V) >> plan.fold_log, folds = (dim / V) >> plan.fold_log;
            const auto store_sum = [&](int row, A sum) {
                const int64_t place = (int64_t(b * p.rows) + row0 + row) * folds + fold;
                if (partial) partial[place] = sum;
                else dgate[place] = narrow<G>(sum);
            };
            if (1 << plan.fold_log >= S) {
                const int row = fold_rows<A, S>(sums, plan.fold_log, at.tc);
                if (row >= 0 && row < r.count) store_sum(row, sums[0]);
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    for (int k = 1; k < 1 << plan.fold_log; k <<= 1) sums[s] += __shfl_xor_sync(0xffffffffu, sums[s], k);
                    if (s < r.count && (at.tc & ((1 << plan.fold_log) - 1)) == 0) store_sum(s, sums[s]);
                }
            }
        }
    }
    // what left the first warp's first part
    if (!PACKED && p.dinitial && live && at.segment == 0 && at.warp == 0 && at.lane < at.lanes)
#pragma unroll
        for (int v = 0; v < V; ++v) dinitial()[b * p.dim + v] = leaving[v];
}

// Map of every segment of the rows: of the recurrence (x, initial states), or REVERSE of the gradient (derivatives in
// the place of x, gradients of states).  Each thread takes a contiguous run of rows, S at a time, and
// appends them to its map; parts and warps are composed once, at the end.
// Of packed sequences only the last (REVERSE: the first) one in a segment decides what leaves it: the rows before
// (behind) it are not read.  Measured: float32 1x65536x192, 101 MB in 21 us, 60 % of the HBM's rate; bfloat16
// 16000x1536 in 23 sequences 17 to 19 us instead of 24.
template <typename X, typename G, int V, int S, bool SHARED, bool PACKED, bool REVERSE>
__global__ void __launch_bounds__(kCtaThreads, 2) recurrence_maps_kernel(const RecurrenceArgs p, const RecurrencePlan plan) {
    using A = Acc<X>;
    constexpr int GV = SHARED ? 1 : V;
    cudaTriggerProgrammaticLaunchCompletion();  // the main kernel's CTAs may come as these leave
    extern __shared__ __align__(16) unsigned char smem[];
    const Place at(plan, p.dim, V);
    const uint64_t b = at.batch, c0 = at.c0;
    const bool live = at.live;
    const int stages = plan.stages, warps = plan.warps;
    const int64_t dim = int64_t(p.dim);
    const A* joins = static_cast<const A*>(REVERSE ? p.state_derivs : p.initial);
    if (joins) joins += c0;
    const int64_t x_row = int64_t(REVERSE ? p.d_row : p.x_row), gate_row = int64_t(p.gate_row);
    const X* x = static_cast<const X*>(REVERSE ? p.derivs : p.x) + b * (REVERSE ? p.d_batch : p.x_batch) + (live ? c0 : 0);
    const G* gate = static_cast<const G*>(p.gate) + b * p.gate_batch + (!live ? 0 : SHARED ? c0 / (p.dim / p.gate_dim) : c0);

    Prefetch<X, V, S, false> fx;
    Prefetch<G, GV, S, SHARED> fg;
    unsigned char* next = smem;
    next = fx.place(next, stages, warps, at.tc, plan.pairs);
    next = fg.place(next, stages, warps, at.tc, plan.pairs);
    const int width = at.lanes * V;
    A* maps = reinterpret_cast<A*>(next);  // [warp][A, B][width]
    next += sizeof(A) * 2 * width * warps;
    int* drops = reinterpret_cast<int*>(next);  // [warp]
    next += sizeof(int) * warps;
    int first = at.segment * plan.segment_rows, rows = min(int(p.rows), first + plan.segment_rows);
    SequenceWalk walk;
    if (PACKED) {  // nothing leaves the segment from before its last sequence (from behind its first)
        walk.open(p, reinterpret_cast<int*>(next));
        walk.seek(REVERSE ? first : rows - 1);
        if (walk.inside()) {
            if (REVERSE) rows = min(rows, walk.next);
            else first = max(first, walk.begin);
        }
    }
    const int round = warps * at.parts * S, run = (rows - first + round - 1) / round * S;  // rows of a thread
    const int begin = first + at.part * run, end = min(rows, begin + run);
    if (PACKED) walk.seek(REVERSE ? begin + run : begin);
    int coming = REVERSE ? begin + run - S : begin;
    const auto fetch = [&](int stage) {
        const int n = coming >= begin ? rows_left<S>(end, coming, live) : 0;
        fx.issue(stage, static_cast<const X*>(REVERSE ? p.derivs : p.x), fx.start(x + int64_t(coming) * x_row, x_row), x_row, n);
        fg.issue(stage, static_cast<const G*>(p.gate), fg.start(gate + int64_t(coming) * gate_row, gate_row), gate_row, n);
        commit_copies();
        coming += REVERSE ? -S : S;
    };
    const auto hold = [&](int row) {
        const int n = row >= begin ? rows_left<S>(end, row, live) : 0;
        fx.hold(x + int64_t(row) * x_row, x_row, n);
        fg.hold(gate + int64_t(row) * gate_row, gate_row, n);
    };
    hold(coming);
    for (int k = 0; k < stages - 1; ++k) fetch(k);
    Map<A, V> m;
    m.clear();
    int stage = 0;
    for (int done = 0; done < run; done += S, stage = stage + 1 == stages ? 0 : stage + 1) {
        const int row0 = REVERSE ? begin + run - S - done : begin + done;
        __syncwarp();
        fetch(stage == 0 ? stages - 1 : stage - 1);
        Rows<A, V, S> r;
        r.count = rows_left<S>(end, row0, live);
        if (PACKED) {
            if (REVERSE) walk.retreat(row0); else walk.advance(row0);
            r.e = row_events<S>(walk, row0, end);
        }
        await_copies(stages);
        if (!REVERSE && p.complement) factors<true>(p.form, fx, fg, stage, r.a, r.u);
        else factors<false>(p.form, fx, fg, stage, r.a, r.u);
        hold(REVERSE ? row0 - S : row0 + S);
        settle_rows<REVERSE>(r, walk, row0, joins, dim, live);
        append_rows<REVERSE, PACKED>(m, r);
    }
    __syncwarp();
    scan_warp<A, V, REVERSE, PACKED>(m, plan.log_lanes);
    if (REVERSE ? at.lane < at.lanes : at.lane >= 32 - at.lanes) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            maps[2 * at.warp * width + at.tc * V + v] = m.a[v];
            maps[(2 * at.warp + 1) * width + at.tc * V + v] = m.b[v];
        }
        if (at.tc == 0) drops[at.warp] = m.drop;
    }
    __syncthreads();
    const uint64_t to = b * plan.segments + at.segment, strip = c0 - uint64_t(at.tc) * V;
    for (int c = threadIdx.x; c < width && strip + c < p.dim; c += blockDim.x) {
        A a = A(1), f = A(0);
        int drop = 0;
        for (int i = 0; i < warps; ++i) {
            const int w = REVERSE ? warps - 1 - i : i;
            const A wb = maps[(2 * w + 1) * width + c], wa = maps[2 * w * width + c];
            f = drops[w] ? wb : fma_(wa, f, wb);
            a *= wa;
            drop |= drops[w];
        }
        A* map = static_cast<A*>(plan.maps) + 2 * to * p.dim + strip + c;
        map[0] = a;
        map[p.dim] = f;
        if (c == 0 && strip == 0) plan.drops[to] = drop;
    }
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
// The launch is most of it: bfloat16 16x512 with float32 gates takes 3.2 us, one launch behind the other, its 131 KB
// would take 0.02 us.
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
    constexpr int GV = SHARED ? 1 : V;
    A wide[GV], a[GV], rest[GV];
#pragma unroll
    for (int v = 0; v < GV; ++v) wide[v] = widen(g.v[v]);
    if (p.form == kGateValue) gate_factors<kGateValue, sizeof(G) == 2, true>(wide, a, rest);
    else if (p.form == kGateLog) gate_factors<kGateLog, sizeof(G) == 2, true>(wide, a, rest);
    else gate_factors<kGateLogit, sizeof(G) == 2, true>(wide, a, rest);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A u = widen(x.v[v]);
        if (p.complement) u *= rest[v % GV];
        h.v[v] = fma_(a[v % GV], h.v[v], u);
        y.v[v] = narrow<X>(h.v[v]);
    }
    store_pack<A, V>(at, h);
    store_pack<X, V>(static_cast<X*>(p.out) + row * p.dim + c0, y);
}

}  // namespace
}  // namespace sigb200
