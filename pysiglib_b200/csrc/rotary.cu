// Rotary positions: every pair of channels of a row is turned by the angle position * frequency.
//
// Mathematics.  (y_p, y_q) = scale * (x_p cos w - x_q sin w, x_p sin w + x_q cos w) with w = p_t f_i, for the
// pairs (i, i + r/2) or (2i, 2i + 1) of the first r channels; the others are copied.  The adjoint is the
// turn by -w.  Angles are formed in 64 bits, as quarter turns p_t * (f_i 2 / pi) less the nearest integer, so that a
// position of millions keeps all the bits that the sine needs.  The sine and cosine of the remainder are
// taken in the type of the arithmetic (64 bits for float64 rows, of radians; else 32) by their Taylor series within an
// eighth of a turn, and each output is rounded once.
//
// Split.  One read and one write per value bound it, as long as the sines are shared: a thread takes V pairs of
// one position and walks over the rows (heads, batch entries) that have that position; where
// every row has its own it takes four positions, loads them all, and turns one after the other.
// Measured (B200, eight launches between two events; the copy alone would take what stands behind the bar): bfloat16 2x32768x16x128 193 us | 164,
// 4x2048x32x128 33 | 20; float32 64x1023x272 with a time stamp a row 56 | 43.  What is left is the sines where they
// are not shared and the loads' latency at the start and the end of short threads.
#include <algorithm>
#include <type_traits>

#include "algebra_host.h"
#include "sequence.h"
#include "sequence_types.cuh"

namespace sigb200 {
namespace {

struct RotaryGrid {
    uint64_t threads, turning;        // in all; the first ones, which turn pairs
    uint32_t turned, copied;          // chunks of a row that hold pairs, and that do not
    uint64_t units;                   // row blocks, of one row where positions are shared, else of four
    uint64_t outer1;                  // inner axis of the rows that differ in position beside the row axis
    uint64_t shared, shared1;         // rows that share a position, and their inner axis
    uint64_t per_thread, groups;      // shared rows of a thread, threads that share them out
    int64_t xo0, xo1, yo0, yo1, po0, po1, xs0, xs1, ys0, ys1;  // strides of those axes
};

constexpr int kInFlight = 4;  // rows of an unshared position, or of a copy

// Sine and cosine of a number of quarter turns.  The nearest integer comes off in 64 bits; what is left, t of at most a
// half, is rounded to 32 bits once, and the series in t have the powers of pi / 2 in their coefficients (the first
// one in two parts).  Where 64 bits hold no fraction of a turn any more, t is 0.
__device__ __forceinline__ void sine_cosine(double quarters, float& s, float& c) {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer, its last bits
    constexpr double h = 1.57079632679489661923, h2 = h * h, h4 = h2 * h2, h8 = h4 * h4;
    constexpr float kHigh = float(h), kLow = float(h - kHigh);
    const double whole = quarters + kMagic;
    float t = static_cast<float>(quarters - (whole - kMagic));
    if (fabsf(t) > 0.5f) t = 0.0f;
    const float z = t * t;
    float p = fmaf(z, float(h8 * h / 362880), float(-h4 * h2 * h / 5040)), q = fmaf(z, float(-h8 * h2 / 3628800), float(h8 / 40320));
    p = fmaf(p, z, float(h4 * h / 120));
    q = fmaf(q, z, float(-h4 * h2 / 720));
    p = fmaf(p, z, float(-h2 * h / 6));
    q = fmaf(q, z, float(h4 / 24));
    p = fmaf(p, z, kLow);
    q = fmaf(q, z, float(-h2 / 2));
    const float sine = fmaf(t, kHigh, t * p), cosine = fmaf(q, z, 1.0f);
    const int k = __double2loint(whole);
    const float a = k & 1 ? cosine : sine, b = k & 1 ? sine : cosine;
    s = k & 2 ? -a : a;
    c = (k + 1) & 2 ? -b : b;
}
// In 64 bits of an angle: less the nearest number of quarter turns, pi / 2 in two parts, then the Taylor series (the
// terms left out are below 2^-60 of what they belong to).  What the remainder t loses when it is rounded is the angle's
// error; kept as `low`, it turns sine and cosine by its first-order term.  Where an angle's neighbours are more than a
// turn away, t is 0.
__device__ __forceinline__ void sine_cosine(double angle, double& s, double& c) {
    constexpr double kMagic = 6755399441055744.0, kHigh = 1.57079632679489661923, kLow = 6.123233995736766e-17;
    const double whole = fma(angle, 0.63661977236758134308, kMagic), n = whole - kMagic;
    const double product = __dmul_rn(n, kHigh), rest = __dsub_rn(angle, product);  // rest is exact
    const double off = fma(n, kLow, fma(n, kHigh, -product));
    double t = __dsub_rn(rest, off), low = __dsub_rn(__dsub_rn(rest, t), off);
    if (fabs(t) > 1.0) t = low = 0.0;
    const double z = t * t;
    double p = fma(z, 1.0 / 355687428096000, -1.0 / 1307674368000), q = fma(z, 1.0 / 20922789888000, -1.0 / 87178291200);
    p = fma(p, z, 1.0 / 6227020800);
    q = fma(q, z, 1.0 / 479001600);
    p = fma(p, z, -1.0 / 39916800);
    q = fma(q, z, -1.0 / 3628800);
    p = fma(p, z, 1.0 / 362880);
    q = fma(q, z, 1.0 / 40320);
    p = fma(p, z, -1.0 / 5040);
    q = fma(q, z, -1.0 / 720);
    p = fma(p, z, 1.0 / 120);
    q = fma(q, z, 1.0 / 24);
    p = fma(p, z, -1.0 / 6);
    q = fma(q, z, -0.5);
    const double first = fma(p * z, t, t), second = fma(q, z, 1.0);
    const double sine = fma(second, low, first), cosine = fma(-first, low, second);
    const int k = __double2loint(whole);
    const double a = k & 1 ? cosine : sine, b = k & 1 ? sine : cosine;
    s = k & 2 ? -a : a;
    c = (k + 1) & 2 ? -b : b;
}

template <typename P>
__device__ __forceinline__ double position_at(const void* positions, int64_t at, uint64_t row) {
    if constexpr (std::is_void_v<P>) return static_cast<double>(row);
    else return static_cast<double>(static_cast<const P*>(positions)[at]);
}

// The 2 V channels of V pairs, in the order they are loaded: V and V.  Interleaved pairs lie side by side within each
// of the two (a thread takes V / 2 pairs from either half of the channels, so that its neighbours' loads join
// up); for V = 1 the two are the pair.
template <typename X, int V>
struct Pairs {
    Pack<X, V> p, q;
};

template <typename X, int V, bool INTERLEAVED, typename A>
__device__ __forceinline__ Pairs<X, V> turned(const Pairs<X, V>& x, const A (&s)[V], const A (&c)[V]) {
    A yp[V], yq[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const A a = widen(INTERLEAVED ? (2 * v < V ? x.p.v[(2 * v) % V] : x.q.v[(2 * v) % V]) : x.p.v[v]);
        const A b = widen(INTERLEAVED ? (2 * v + 1 < V ? x.p.v[(2 * v + 1) % V] : x.q.v[(2 * v + 1) % V]) : x.q.v[v]);
        const A ya = a * c[v] - b * s[v], yb = a * s[v] + b * c[v];
        if (INTERLEAVED) {
            (2 * v < V ? yp : yq)[(2 * v) % V] = ya;
            (2 * v + 1 < V ? yp : yq)[(2 * v + 1) % V] = yb;
        } else {
            yp[v] = ya;
            yq[v] = yb;
        }
    }
    return {narrow_pack<X, V>(yp), narrow_pack<X, V>(yq)};
}

// SHARED: several rows have a thread's position.  Else each row has its own.
template <typename X, typename P, int V, bool INTERLEAVED, bool SHARED>
__global__ void __launch_bounds__(256, SHARED || sizeof(X) == 2 ? 2 : 3) rotary_kernel(const RotaryArgs p, const RotaryGrid g) {
    using A = Acc<X>;
    uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= g.threads) return;
    const bool turning = i < g.turning;
    if (!turning) i -= g.turning;
    const uint32_t chunks = turning ? g.turned : g.copied;
    const uint32_t chunk = static_cast<uint32_t>(i % chunks);
    i /= chunks;
    const uint64_t unit = i % g.units;
    i /= g.units;
    const uint64_t group = SHARED ? i % g.groups : 0, outer = SHARED ? i / g.groups : i;
    const uint64_t o0 = outer / g.outer1, o1 = outer - o0 * g.outer1;
    const uint64_t row = SHARED ? unit : unit * kInFlight;
    const int64_t cp = turning ? (INTERLEAVED && V == 1 ? 2 * int64_t(chunk) : int64_t(chunk) * V) : int64_t(p.rotary_dim) + int64_t(chunk) * V;
    const int64_t cq = INTERLEAVED && V == 1 ? 1 : int64_t(p.rotary_dim / 2);  // from cp on
    const X* x = static_cast<const X*>(p.x) + int64_t(o0) * g.xo0 + int64_t(o1) * g.xo1 + int64_t(row) * int64_t(p.x_row) + cp;
    X* y = static_cast<X*>(p.out) + int64_t(o0) * g.yo0 + int64_t(o1) * g.yo1 + int64_t(row) * int64_t(p.out_row) + cp;

    // the rows of this thread: `count` of them, `x_step` and `y_step` apart, with a jump after every `inner`
    int64_t x_step = int64_t(p.x_row), y_step = int64_t(p.out_row), x_jump = 0, y_jump = 0;
    uint64_t count = min(uint64_t(kInFlight), p.rows - row), inner = ~0ull, at = 0;
    if (SHARED) {
        const uint64_t first = group * g.per_thread, k0 = first / g.shared1;
        count = min(g.per_thread, g.shared - first);
        inner = g.shared1;
        at = first - k0 * g.shared1;
        x += int64_t(k0) * g.xs0 + int64_t(at) * g.xs1;
        y += int64_t(k0) * g.ys0 + int64_t(at) * g.ys1;
        x_step = g.xs1;
        y_step = g.ys1;
        x_jump = g.xs0 - int64_t(g.shared1) * g.xs1;
        y_jump = g.ys0 - int64_t(g.shared1) * g.ys1;
    }
    uint64_t y_at = at;
    const auto next_x = [&] {
        x += x_step;
        if (SHARED && ++at == inner) { at = 0; x += x_jump; }
    };
    const auto next_y = [&] {
        y += y_step;
        if (SHARED && ++y_at == inner) { y_at = 0; y += y_jump; }
    };

    if (!turning) {
        Pack<X, V> r[kInFlight], ahead[kInFlight];
        const auto read = [&](Pack<X, V> (&to)[kInFlight], uint64_t k) {
#pragma unroll
            for (int n = 0; n < kInFlight; ++n)
                if (k + n < count) {
                    to[n] = load_pack<X, V>(x);
                    next_x();
                }
        };
        read(r, 0);
        for (uint64_t k = 0; k < count; k += kInFlight) {
            read(ahead, k + kInFlight);
#pragma unroll
            for (int n = 0; n < kInFlight; ++n)
                if (k + n < count) {
                    store_pack<X, V>(y, r[n]);
                    next_y();
                    r[n] = ahead[n];
                }
        }
        return;
    }
    A s[V], c[V];
    double rate[V];  // quarter turns (float64: radians) for each unit of position
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const uint64_t pair = !INTERLEAVED || V == 1 ? uint64_t(chunk) * V + v : (v < V / 2 ? cp : cp + cq - V) / 2 + v;
        rate[v] = p.frequencies[pair] * (std::is_same_v<A, double> ? 1.0 : 0.63661977236758134308);
    }
    const A scale = static_cast<A>(p.scale), signed_scale = static_cast<A>(p.inverse ? -p.scale : p.scale);
    const auto turn_at = [&](double position) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            sine_cosine(position * rate[v], s[v], c[v]);
            s[v] *= signed_scale;
            c[v] *= scale;
        }
    };
    const int64_t place = int64_t(o0) * g.po0 + int64_t(o1) * g.po1 + int64_t(row) * int64_t(p.p_row);
    const auto load = [&] {
        Pairs<X, V> r;
        r.p = load_pack<X, V>(x);
        r.q = load_pack<X, V>(x + cq);
        next_x();
        return r;
    };
    const auto store = [&](const Pairs<X, V>& r) {
        const Pairs<X, V> t = turned<X, V, INTERLEAVED>(r, s, c);
        store_pack<X, V>(y, t.p);
        store_pack<X, V>(y + cq, t.q);
        next_y();
    };
    if constexpr (SHARED) {
        // two rows in flight while two are turned
        Pairs<X, V> r[2], ahead[2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
            if (uint64_t(n) < count) r[n] = load();
        turn_at(position_at<P>(p.positions, place, row));
        uint64_t k = 0;
        for (; k + 4 <= count; k += 2) {
            ahead[0] = load();
            ahead[1] = load();
            store(r[0]);
            store(r[1]);
            r[0] = ahead[0];
            r[1] = ahead[1];
        }
        if (k + 3 == count) ahead[0] = load();
#pragma unroll
        for (int n = 0; n < 2; ++n)
            if (k + n < count) store(r[n]);
        if (k + 3 == count) store(ahead[0]);
    } else {
        Pairs<X, V> r[kInFlight];
        double position[kInFlight];
#pragma unroll
        for (int n = 0; n < kInFlight; ++n)
            if (uint64_t(n) < count) {
                r[n] = load();
                position[n] = position_at<P>(p.positions, place + n * int64_t(p.p_row), row + n);
            }
#pragma unroll
        for (int n = 0; n < kInFlight; ++n)
            if (uint64_t(n) < count) {
                turn_at(position[n]);
                store(r[n]);
            }
    }
}

template <typename X, typename P, int V>
void launch(const RotaryArgs& p, cudaStream_t stream) {
    RotaryGrid g{};
    g.turned = static_cast<uint32_t>(p.rotary_dim / 2 / V);
    g.copied = static_cast<uint32_t>((p.dim - p.rotary_dim) / V);
    // axes along which the positions do not change are walked by one thread
    const bool same0 = p.n0 == 1 || p.p0 == 0 || std::is_void_v<P>, same1 = p.n1 == 1 || p.p1 == 0 || std::is_void_v<P>;
    uint64_t outer = 1;
    g.outer1 = g.shared = g.shared1 = 1;
    const auto x0 = int64_t(p.x0), x1 = int64_t(p.x1), y0 = int64_t(p.out0), y1 = int64_t(p.out1), p0 = int64_t(p.p0), p1 = int64_t(p.p1);
    if (same0 && same1) {
        g.shared = p.n0 * p.n1; g.shared1 = p.n1;
        g.xs0 = x0; g.xs1 = x1; g.ys0 = y0; g.ys1 = y1;
    } else if (same1) {
        outer = p.n0; g.xo0 = x0; g.yo0 = y0; g.po0 = p0;
        g.shared = g.shared1 = p.n1; g.xs1 = x1; g.ys1 = y1;
    } else if (same0) {
        outer = p.n1; g.xo0 = x1; g.yo0 = y1; g.po0 = p1;
        g.shared = g.shared1 = p.n0; g.xs1 = x0; g.ys1 = y0;
    } else {
        outer = p.n0 * p.n1; g.outer1 = p.n1;
        g.xo0 = x0; g.xo1 = x1; g.yo0 = y0; g.yo1 = y1; g.po0 = p0; g.po1 = p1;
    }
    const bool shared = g.shared > 1;
    g.units = shared ? p.rows : (p.rows + kInFlight - 1) / kInFlight;
    // enough threads for every SM before one takes more of the rows that share a position
    const uint64_t lines = uint64_t(g.turned + g.copied) * g.units * outer;
    const uint64_t wanted = uint64_t(device_context(current_device()).sm_count) * 1024;
    g.groups = std::max<uint64_t>(1, std::min<uint64_t>(g.shared, (wanted + lines - 1) / lines));
    g.per_thread = (g.shared + g.groups - 1) / g.groups;
    g.groups = (g.shared + g.per_thread - 1) / g.per_thread;
    g.turning = g.turned * g.units * outer * g.groups;
    g.threads = lines * g.groups;
    const unsigned grid = grid_1d(g.threads, 256);
    if (p.interleaved) {
        if (shared) rotary_kernel<X, P, V, true, true><<<grid, 256, 0, stream>>>(p, g);
        else rotary_kernel<X, P, V, true, false><<<grid, 256, 0, stream>>>(p, g);
    } else {
        if (shared) rotary_kernel<X, P, V, false, true><<<grid, 256, 0, stream>>>(p, g);
        else rotary_kernel<X, P, V, false, false><<<grid, 256, 0, stream>>>(p, g);
    }
    check_launch("rotary kernel");
}

template <typename X, int V>
void launch_positions(const RotaryArgs& p, cudaStream_t stream) {
    switch (p.position_type) {
        case kPositionNone: return launch<X, void, V>(p, stream);
        case kPositionInt32: return launch<X, int, V>(p, stream);
        case kPositionInt64: return launch<X, long long, V>(p, stream);
        case kPositionFloat32: return launch<X, float, V>(p, stream);
        default: return launch<X, double, V>(p, stream);
    }
}

// Whether V channels at a time are aligned everywhere: the pairs, the copied channels and every stride.
bool fits(const RotaryArgs& p, uint64_t V, size_t size) {
    for (uint64_t n : {p.rotary_dim / 2, p.dim - p.rotary_dim, p.x0, p.x1, p.x_row, p.out0, p.out1, p.out_row})
        if (n % V) return false;
    return reinterpret_cast<uintptr_t>(p.x) % (V * size) == 0 && reinterpret_cast<uintptr_t>(p.out) % (V * size) == 0;
}

// 16 bytes a load where all is aligned to it; else two values where that fits (bfloat16 8x4096x8x132, 68 turned: 44
// against 70 us one by one), else one.
template <typename X>
void launch_type(const RotaryArgs& p, cudaStream_t stream) {
    constexpr int W = 16 / sizeof(X);
    if (fits(p, W, sizeof(X))) launch_positions<X, W>(p, stream);
    else if (W > 2 && fits(p, 2, sizeof(X))) launch_positions<X, 2>(p, stream);
    else launch_positions<X, 1>(p, stream);
}

void run(const RotaryArgs& p, cudaStream_t stream) {
    switch (p.type) {
        case kFloat32: return launch_type<float>(p, stream);
        case kFloat64: return launch_type<double>(p, stream);
        case kBFloat16: return launch_type<__nv_bfloat16>(p, stream);
        default: return launch_type<__half>(p, stream);
    }
}

size_t position_size(int type) { return type == kPositionInt64 || type == kPositionFloat64 ? 8 : 4; }

}  // namespace

void rotary_entry(const RotaryArgs& args, const CallOptions& opt) {
    const char* who = "rotary";
    const RotaryArgs& p = args;
    if (p.type < kFloat32 || p.type > kFloat16) throw std::invalid_argument("rotary: unknown element type");
    if (p.position_type < kPositionNone || p.position_type > kPositionFloat64)
        throw std::invalid_argument("rotary: unknown type of positions");
    if (p.rotary_dim % 2 || p.rotary_dim > p.dim) throw std::invalid_argument("rotary: the turned channels must be an even number, at most all");
    const uint64_t rows = checked_mul(checked_mul(p.n0, p.n1, who), p.rows, who);
    const uint64_t n = checked_mul(rows, p.dim, who);
    if (n == 0) return;
    if (n >= 1ull << 59 || p.dim >= 1ull << 31) throw std::out_of_range("rotary: size overflow");
    if (!p.x || !p.out || (p.rotary_dim && !p.frequencies) || (p.position_type != kPositionNone && !p.positions))
        throw std::invalid_argument("rotary received a null pointer");
    const void* positions = p.position_type == kPositionNone ? nullptr : p.positions;
    const void* frequencies = p.rotary_dim ? p.frequencies : nullptr;
    int device = opt.known_device;
    if (device >= 0 || all_on_device({p.x, p.out, positions, frequencies}, who, &device)) {
        DeviceGuard guard(device);
        run(p, opt.stream);
        if (opt.synchronize) SIG_CUDA_CHECK(cudaStreamSynchronize(opt.stream));
        return;
    }
    const auto dense = [&](uint64_t s0, uint64_t s1, uint64_t s_row, uint64_t width) {
        return (s_row == width || p.rows == 1) && (s1 == p.rows * width || p.n1 == 1) && (s0 == p.n1 * p.rows * width || p.n0 == 1);
    };
    if (!dense(p.x0, p.x1, p.x_row, p.dim) || !dense(p.out0, p.out1, p.out_row, p.dim) || (positions && !dense(p.p0, p.p1, p.p_row, 1)))
        throw std::invalid_argument("rotary: host buffers must be contiguous");
    const size_t bytes = n * element_size(p.type);
    run_staged({{p.x, nullptr, bytes}, {nullptr, p.out, bytes}, {positions, nullptr, positions ? rows * position_size(p.position_type) : 0},
                {frequencies, nullptr, frequencies ? p.rotary_dim / 2 * sizeof(double) : 0}},
               opt.device, [&](const std::vector<void*>& d, cudaStream_t stream) {
                   RotaryArgs q = p;
                   q.x = d[0]; q.out = d[1];
                   q.positions = positions ? d[2] : nullptr;
                   q.frequencies = static_cast<const double*>(d[3]);
                   run(q, stream);
               });
}

}  // namespace sigb200
