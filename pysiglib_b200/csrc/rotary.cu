// Rotary positions: every pair of channels of a row is turned by the angle position * frequency.
//
// Mathematics.  (y_p, y_q) = scale * (x_p cos w - x_q sin w, x_p sin w + x_q cos w) with w = p_t f_i, for the
// pairs (i, i + r/2) or (2i, 2i + 1) of the first r channels; the others are copied.  The adjoint is the
// turn by -w.  Angles are formed in 64 bits as turns, p_t * (f_i / 2 pi) less the nearest integer, so that a
// position of millions keeps all the bits that the sine needs; the sine and cosine of the remainder are
// taken in the type of the arithmetic (32 bits, 64 for float64 rows) and each output is rounded once.
//
// Split.  One read and one write per value bound it, as long as the sines are shared: a thread takes V
// pairs of one position and walks over the rows (heads, batch entries) that have that position.
#include <algorithm>
#include <type_traits>

#include "algebra_host.h"
#include "sequence.h"
#include "sequence_types.cuh"

namespace sigb200 {
namespace {

struct RotaryGrid {
    uint64_t threads;                 // in all
    uint32_t chunks, turned;          // chunks a row is cut into, the first `turned` of them hold pairs
    uint64_t outer, outer1;           // rows that differ in position beside the row axis, and their inner axis
    uint64_t shared, shared1;         // rows that share a position, and their inner axis
    uint64_t per_thread, groups;      // shared rows of a thread, threads that share them out
    uint64_t xo0, xo1, yo0, yo1, po0, po1, xs0, xs1, ys0, ys1;  // strides of those axes
};

__device__ __forceinline__ void sine_cosine(double turns, float& s, float& c) { sincospif(2.0f * static_cast<float>(turns), &s, &c); }
__device__ __forceinline__ void sine_cosine(double turns, double& s, double& c) { sincospi(2.0 * turns, &s, &c); }

template <typename P>
__device__ __forceinline__ double position_at(const void* positions, uint64_t at, uint64_t row) {
    if constexpr (std::is_void_v<P>) return static_cast<double>(row);
    else return static_cast<double>(static_cast<const P*>(positions)[at]);
}

template <typename X, typename P, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs p, const RotaryGrid g) {
    using A = Acc<X>;
    constexpr int U = 4;  // rows in flight
    uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= g.threads) return;
    const uint32_t chunk = static_cast<uint32_t>(i % g.chunks);
    i /= g.chunks;
    const uint64_t row = i % p.rows;
    i /= p.rows;
    const uint64_t group = i % g.groups, outer = i / g.groups;
    const uint64_t o0 = outer / g.outer1, o1 = outer % g.outer1;
    const X* x = static_cast<const X*>(p.x) + o0 * g.xo0 + o1 * g.xo1 + row * p.x_row;
    X* y = static_cast<X*>(p.out) + o0 * g.yo0 + o1 * g.yo1 + row * p.out_row;
    const uint64_t first = group * g.per_thread, last = min(first + g.per_thread, g.shared);
    uint64_t k0 = first / g.shared1, k1 = first % g.shared1;

    if (chunk >= g.turned) {  // channels that are not turned
        const uint64_t c = p.rotary_dim + uint64_t(chunk - g.turned) * V;
        for (uint64_t k = first; k < last; ++k) {
            store_pack<X, V>(y + k0 * g.ys0 + k1 * g.ys1 + c, load_pack<X, V>(x + k0 * g.xs0 + k1 * g.xs1 + c));
            if (++k1 == g.shared1) { k1 = 0; ++k0; }
        }
        return;
    }
    const uint64_t pair = uint64_t(chunk) * V;
    const uint64_t cp = INTERLEAVED ? 2 * pair : pair, cq = INTERLEAVED ? 2 * pair + V : pair + p.rotary_dim / 2;
    const double at = position_at<P>(p.positions, o0 * g.po0 + o1 * g.po1 + row * p.p_row, row);
    A s[V], c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const double turns = at * (p.frequencies[pair + v] * 0.15915494309189533577);
        sine_cosine(turns - rint(turns), s[v], c[v]);
        s[v] *= static_cast<A>(p.inverse ? -p.scale : p.scale);
        c[v] *= static_cast<A>(p.scale);
    }
    for (uint64_t k = first; k < last; k += U) {
        Pack<X, V> rp[U], rq[U];
        uint64_t j0 = k0, j1 = k1;
#pragma unroll
        for (int n = 0; n < U; ++n)
            if (k + n < last) {
                const X* from = x + j0 * g.xs0 + j1 * g.xs1;
                rp[n] = load_pack<X, V>(from + cp);
                rq[n] = load_pack<X, V>(from + cq);
                if (++j1 == g.shared1) { j1 = 0; ++j0; }
            }
#pragma unroll
        for (int n = 0; n < U; ++n)
            if (k + n < last) {
                Pack<X, V> up, uq;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    // interleaved pairs lie side by side in the 2 V values of rp and rq together
                    const A a = widen(INTERLEAVED ? (2 * v < V ? rp[n].v[(2 * v) % V] : rq[n].v[(2 * v) % V]) : rp[n].v[v]);
                    const A b = widen(INTERLEAVED ? (2 * v + 1 < V ? rp[n].v[(2 * v + 1) % V] : rq[n].v[(2 * v + 1) % V]) : rq[n].v[v]);
                    const X ya = narrow<X>(a * c[v] - b * s[v]), yb = narrow<X>(a * s[v] + b * c[v]);
                    if (INTERLEAVED) {
                        (2 * v < V ? up : uq).v[(2 * v) % V] = ya;
                        (2 * v + 1 < V ? up : uq).v[(2 * v + 1) % V] = yb;
                    } else {
                        up.v[v] = ya;
                        uq.v[v] = yb;
                    }
                }
                X* to = y + k0 * g.ys0 + k1 * g.ys1;
                store_pack<X, V>(to + cp, up);
                store_pack<X, V>(to + cq, uq);
                if (++k1 == g.shared1) { k1 = 0; ++k0; }
            }
    }
}

template <typename X, typename P, int V>
void launch(const RotaryArgs& p, cudaStream_t stream) {
    RotaryGrid g{};
    g.turned = static_cast<uint32_t>(p.rotary_dim / 2 / V);
    g.chunks = g.turned + static_cast<uint32_t>((p.dim - p.rotary_dim) / V);
    // axes along which the positions do not change are walked by one thread
    const bool same0 = p.n0 == 1 || p.p0 == 0 || std::is_void_v<P>, same1 = p.n1 == 1 || p.p1 == 0 || std::is_void_v<P>;
    g.outer = g.outer1 = g.shared = g.shared1 = 1;
    if (same0 && same1) {
        g.shared = p.n0 * p.n1; g.shared1 = p.n1;
        g.xs0 = p.x0; g.xs1 = p.x1; g.ys0 = p.out0; g.ys1 = p.out1;
    } else if (same1) {
        g.outer = p.n0; g.xo0 = p.x0; g.yo0 = p.out0; g.po0 = p.p0;
        g.shared = g.shared1 = p.n1; g.xs1 = p.x1; g.ys1 = p.out1;
    } else if (same0) {
        g.outer = p.n1; g.xo0 = p.x1; g.yo0 = p.out1; g.po0 = p.p1;
        g.shared = g.shared1 = p.n0; g.xs1 = p.x0; g.ys1 = p.out0;
    } else {
        g.outer = p.n0 * p.n1; g.outer1 = p.n1;
        g.xo0 = p.x0; g.xo1 = p.x1; g.yo0 = p.out0; g.yo1 = p.out1; g.po0 = p.p0; g.po1 = p.p1;
    }
    // enough threads for every SM twice over before one takes several of the rows that share a position
    const uint64_t lines = g.chunks * p.rows * g.outer;
    const uint64_t wanted = uint64_t(device_context(current_device()).sm_count) * 4096;
    g.groups = std::max<uint64_t>(1, std::min<uint64_t>(g.shared, (wanted + lines - 1) / lines));
    g.per_thread = (g.shared + g.groups - 1) / g.groups;
    g.groups = (g.shared + g.per_thread - 1) / g.per_thread;
    g.threads = lines * g.groups;
    const unsigned grid = grid_1d(g.threads, 256);
    if (p.interleaved) rotary_kernel<X, P, V, true><<<grid, 256, 0, stream>>>(p, g);
    else rotary_kernel<X, P, V, false><<<grid, 256, 0, stream>>>(p, g);
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

// 16 bytes a load where all is aligned to it; else single values.
template <typename X>
void launch_type(const RotaryArgs& p, cudaStream_t stream) {
    constexpr int W = 16 / sizeof(X);
    if (fits(p, W, sizeof(X))) launch_positions<X, W>(p, stream);
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
    int device = -1;
    if (all_on_device({p.x, p.out, positions, frequencies}, who, &device)) {
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
