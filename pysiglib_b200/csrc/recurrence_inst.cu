// Launchers of the recurrence kernels for one pair of element types (SIG_RECURRENCE_PART picks it; one
// object each, so that the pairs compile side by side).
#include <algorithm>
#include <atomic>

#include "recurrence.h"
#include "recurrence_kernels.cuh"

namespace sigb200 {
namespace {

// Channels a thread holds: 16 bytes of float32 or float64, 8 of the 16-bit types (whose gates and states
// widen to the same registers).
template <typename X> constexpr int kWide = sizeof(X) == 8 ? 2 : 4;
// Rows a thread holds: as many as leave the arrays of S * V values in registers and two CTAs an SM their stages
// (float16 with float32 gates, packed 8000x1536 backward: 4 rows 74 us, 8 rows 107 us).
template <typename X, typename G, int V, bool SHARED>
constexpr int kBackwardRows = V > 1 && (sizeof(X) > 2 || (!SHARED && sizeof(G) > 2)) ? 4 : 8;
template <typename X, int V> constexpr int kForwardRows = V > 1 && sizeof(X) > 2 ? 4 : 8;

constexpr int kMostShared = 227 * 1024;  // of a CTA

int log2_ceil(uint64_t n) {
    int k = 0;
    while ((1ull << k) < n) ++k;
    return k;
}

// Whether the inputs' rows and the cuts between groups of `bytes` of their channels are aligned to `bytes`
// (a shared gate's are not cut).
bool aligned_to(const RecurrenceArgs& p, size_t bytes) {
    const auto fits = [&](const void* ptr, size_t size, uint64_t width, uint64_t batch, uint64_t row) {
        return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && width * size % bytes == 0 && batch * size % bytes == 0 && row * size % bytes == 0;
    };
    const size_t e = element_size(p.type);
    return fits(p.x, e, p.dim, p.x_batch, p.x_row) && fits(p.derivs, e, p.dim, p.d_batch, p.d_row) &&
           (p.gate_dim != p.dim || fits(p.gate, element_size(p.gate_type), p.dim, p.gate_batch, p.gate_row));
}

// Up to 8 warps whose lanes lie side by side in the channels as far as 128 bytes of a row go (full lines), and
// behind one another in the rows beyond that; an SM holds two such CTAs.  Where full lines make fewer strips
// than there are SMs, half lines do if that is enough; else the rows are cut into segments, as many as fill the
// SMs (float32 1x65536x192, forward: 94 segments 46 us; 8 CTAs of a cluster to each strip took 71 us, one CTA 246 us).
template <typename X>
RecurrencePlan make_plan(const RecurrenceArgs& p, int V, int S) {
    constexpr uint64_t kResident = 16;  // warps an SM holds at 128 registers a thread
    const uint64_t per_row = (p.dim + V - 1) / V, sms = device_context(current_device()).sm_count;
    const int columns = log2_ceil(per_row), needed = log2_ceil((p.rows + S - 1) / S);
    RecurrencePlan plan{};
    plan.log_lanes = std::min({columns, log2_ceil(128 / (V * sizeof(X))), 5});
    const auto ctas = [&](int log_lanes) { return p.batch * (((per_row - 1) >> log_lanes) + 1); };
    if (plan.log_lanes > 0 && ctas(plan.log_lanes) < sms && ctas(plan.log_lanes - 1) >= sms) --plan.log_lanes;
    // two lines wide where that pads no more channels and leaves strips for one and a half rounds of the SMs:
    // half the parts to compose (training, two lines against one: float32 48x400x320 40 against 48 us, 100x300x256 47
    // against 57, 20x800x1024 97 against 105, 40x600x512 76 against 78, 64x2000x512 365 against 356; bfloat16 64x500x768
    // 89 against 92, 16x2000x2048 203 against 202, 12x3000x2304 245 against 246)
    if (plan.log_lanes < std::min(columns, 5) && 2 * ctas(plan.log_lanes + 1) >= 3 * sms && ctas(plan.log_lanes + 1) * 2 == ctas(plan.log_lanes))
        ++plan.log_lanes;
    // and where there will be segments: the rows make up for the strips, as long as a thread of a CTA composes no more
    // than 32 of the segments' maps (through_segments), which are twice as many then.  Training, two lines wide against
    // one: 25 maps float32 1x65536x192 108 against 111 us, 1x90000x192 146 against 149; 30 bfloat16 5x30000x128 89
    // against 94; 25 1x50000x768 166 against 174; 12 16000x1536 packed 132 against 140; 37 float32 1x50000x128 66
    // against 64; 49 bfloat16 3x30000x128 73 against 71; 148 1x30000x128 49 against 41
    else if (plan.log_lanes < std::min(columns, 5) && ctas(plan.log_lanes) < sms && ctas(plan.log_lanes + 1) * 2 == ctas(plan.log_lanes) &&
             kResident * sms * (V << (plan.log_lanes + 1)) <= 32 * 8 * kCtaThreads * ctas(plan.log_lanes + 1))
        ++plan.log_lanes;
    // short inputs: no more parts than there are rows for, the lanes go to the channels instead
    plan.log_lanes = std::max(plan.log_lanes, std::min(columns, 5 - std::min(needed, 5)));
    // fewer than eight warps hold all rows in one iteration
    plan.warps = 1 << std::min(3, std::max(0, needed - (5 - plan.log_lanes)));
    plan.pairs = plan.log_lanes > 0 && aligned_to(p, 16);
    if (ctas(plan.log_lanes) > 0x7fffffffull)
        throw std::invalid_argument("linear_recurrence: problem too large for one kernel launch");
    plan.strips = static_cast<unsigned>(((per_row - 1) >> plan.log_lanes) + 1);
    const uint64_t strips = ctas(plan.log_lanes), warp_rows = uint64_t(32 >> plan.log_lanes) * S, round = 2 * sms;
    // Rings of four warps, twice as many on an SM, where CTAs of eight would leave most of a second round empty or have
    // few iterations, whose start and end then count: three at most, or four where all CTAs of four warps fit one
    // round.  Four against eight warps, forward and backward, in float32, float64 and bfloat16 of three widths: 330
    // strips of 140 to 1200 rows 0.81 to 1.02 of the time, mostly 0.9; 480 to 2000 strips of 140 rows 0.69 to 0.86, of
    // 257 rows 0.78 to 0.97; 480 and 560 strips of 400 rows 0.82 to 0.95, of 512 rows 0.89 to 1.04, of 640 rows 0.93 to
    // 1.12; 640 to 2000 strips of 400 rows 0.83 to 1.07, of 512 rows 0.92 to 1.20.
    const uint64_t iterations = (p.rows + 8 * warp_rows - 1) / (8 * warp_rows);
    if (plan.warps == 8 && strips > round && (2 * strips <= 3 * round || iterations <= (strips <= 2 * round ? 4 : 3)) && 4 * warp_rows % kCheckpointRows == 0)
        plan.warps = 4;
    const uint64_t span = plan.warps * warp_rows, blocks = (p.rows + span - 1) / span;
    uint64_t segments = 1;
    if (strips < sms) segments = std::min(blocks, kResident * sms / (strips * plan.warps));
    const uint64_t length = (blocks + segments - 1) / segments;
    plan.segments = static_cast<int>((blocks + length - 1) / length);
    plan.segment_rows = static_cast<int>(length * span);
    return plan;
}

void check(const char* what) {
    count_launch();
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) throw CudaFailure(err, std::string(what) + ": " + cudaGetErrorString(err));
}

// Shared memory behind the rings: the offsets of packed sequences and what composes the segments.
template <typename A>
size_t front_bytes(const RecurrenceArgs& p, const RecurrencePlan& plan, int width, bool in_ring = false) {
    const int values = std::max(32 * plan.warps, width);
    return offset_room(p) + (plan.segments > 1 && !in_ring ? 2 * values * sizeof(A) + (values / width + 1) * sizeof(int) : 0);
}

// As many stages as the resident CTAs of an SM (16 warps) have room for; returns the bytes of shared memory of a CTA.
size_t shared_memory(RecurrencePlan& plan, size_t stage_of_warp, size_t fixed) {
    const size_t room = size_t(228) * 1024 / (16 / plan.warps) - 1024;
    plan.stages = 4;
    while (plan.stages > 2 && fixed + plan.stages * plan.warps * stage_of_warp > room) --plan.stages;
    return fixed + plan.stages * plan.warps * stage_of_warp;
}

// The kernels' limit of shared memory is raised once on each device.
template <auto Kernel, typename... Args>
void launch(const RecurrenceArgs& p, const RecurrencePlan& plan, size_t smem, cudaStream_t stream, Args... args) {
    static std::atomic<uint64_t> raised{0};
    if (smem > 48 * 1024) {
        const uint64_t bit = 1ull << (current_device() & 63);
        if (!(raised.load(std::memory_order_acquire) & bit)) {
            SIG_CUDA_CHECK(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
            if (current_device() < 64) raised.fetch_or(bit, std::memory_order_release);
        }
    }
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(p.batch) * plan.strips * unsigned(plan.segments));
    config.blockDim = dim3(32 * plan.warps);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = &overlap;
    config.numAttrs = plan.follows ? 1 : 0;
    count_launch();
    const cudaError_t err = cudaLaunchKernelEx(&config, Kernel, p, plan, args...);
    if (err != cudaSuccess) throw CudaFailure(err, std::string("linear recurrence kernel: ") + cudaGetErrorString(err));
}

// Scratch for the segments' maps and, behind them, their drops.
template <typename A>
size_t maps_bytes(const RecurrenceArgs& p, const RecurrencePlan& plan) {
    return plan.segments > 1 ? p.batch * plan.segments * (2 * p.dim * sizeof(A) + sizeof(int)) : 0;
}

template <typename X, typename G, int V, bool SHARED, bool REVERSE>
void reduce_segments(const RecurrenceArgs& p, RecurrencePlan plan, cudaStream_t stream) {
    constexpr int S = V == 1 || sizeof(X) == 2 ? 8 : 4;  // float32 as in the main kernels; 4 for 16 bits: packed 16000x1536 56 -> 62 us
    const size_t smem = shared_memory(plan, Prefetch<X, V, S, false>::kWarp + Prefetch<G, SHARED ? 1 : V, S, SHARED>::kWarp,
                                      plan.warps * (2 * sizeof(Acc<X>) * (V << plan.log_lanes) + sizeof(int)) + 16 + offset_room(p));
    if (p.sequences) launch<recurrence_maps_kernel<X, G, V, S, SHARED, true, REVERSE>>(p, plan, smem, stream);
    else launch<recurrence_maps_kernel<X, G, V, S, SHARED, false, REVERSE>>(p, plan, smem, stream);
}

template <typename A>
void place_maps(const RecurrenceArgs& p, RecurrencePlan& plan, void* memory) {
    plan.maps = memory;
    plan.drops = reinterpret_cast<int*>(static_cast<A*>(memory) + p.batch * plan.segments * 2 * p.dim);
}

template <typename X, typename G, int V, bool SHARED>
void forward(const RecurrenceArgs& p, cudaStream_t stream) {
    constexpr int S = kForwardRows<X, V>;
    RecurrencePlan plan = make_plan<X>(p, V, S);
    Scratch maps(maps_bytes<Acc<X>>(p, plan), stream);
    if (plan.segments > 1) {
        place_maps<Acc<X>>(p, plan, maps.get());
        reduce_segments<X, G, V, SHARED, false>(p, plan, stream);
        plan.follows = true;
    }
    const int width = V << plan.log_lanes;
    const size_t smem = shared_memory(plan, Prefetch<X, V, S, false>::kWarp + Prefetch<G, SHARED ? 1 : V, S, SHARED>::kWarp,
                                      sizeof(Acc<X>) * width * plan.warps + front_bytes<Acc<X>>(p, plan, width));
    if (p.sequences) launch<recurrence_forward_kernel<X, G, V, S, SHARED, true>>(p, plan, smem, stream);
    else launch<recurrence_forward_kernel<X, G, V, S, SHARED, false>>(p, plan, smem, stream);
}

template <typename X, typename G, int V, bool SHARED>
void backward(const RecurrenceArgs& p, cudaStream_t stream) {
    constexpr int S = kBackwardRows<X, G, V, SHARED>;
    RecurrencePlan plan = make_plan<X>(p, V, S);
    Scratch maps(maps_bytes<Acc<X>>(p, plan), stream);
    if (plan.segments > 1) {
        place_maps<Acc<X>>(p, plan, maps.get());
        reduce_segments<X, G, V, SHARED, true>(p, plan, stream);
        plan.follows = true;
    }
    Acc<X>* partial = nullptr;
    uint64_t per_gate = 0;
    if (SHARED) {  // lanes whose channels share a gate, as far as a power of two goes
        per_gate = p.dim / p.gate_dim / V;
        while (plan.fold_log < plan.log_lanes && per_gate % 2 == 0) { per_gate /= 2; ++plan.fold_log; }
    }
    const uint64_t n = p.batch * p.rows * p.gate_dim;
    Scratch scratch(per_gate > 1 ? checked_mul(n, per_gate * sizeof(Acc<X>), "linear_recurrence_backprop") : 0, stream);
    if (per_gate > 1) partial = scratch.as<Acc<X>>();
    const int width = V << plan.log_lanes;
    const size_t column = width * sizeof(Acc<X>);
    const size_t smem = shared_memory(plan, 2 * Prefetch<X, V, S, false>::kWarp + Prefetch<G, SHARED ? 1 : V, S, SHARED>::kWarp + column,
                                      2 * plan.warps * column + front_bytes<Acc<X>>(p, plan, width, fold_in_ring(width)));
    if (p.complement) {
        if (p.sequences) launch<recurrence_backward_kernel<X, G, V, S, SHARED, true, true>>(p, plan, smem, stream, partial);
        else launch<recurrence_backward_kernel<X, G, V, S, SHARED, false, true>>(p, plan, smem, stream, partial);
    } else {
        if (p.sequences) launch<recurrence_backward_kernel<X, G, V, S, SHARED, true, false>>(p, plan, smem, stream, partial);
        else launch<recurrence_backward_kernel<X, G, V, S, SHARED, false, false>>(p, plan, smem, stream, partial);
    }
    if (partial) {
        if (n / 256 >= 0x7fffffffull) throw std::invalid_argument("linear_recurrence_backprop: problem too large for one kernel launch");
        fold_partials_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(partial, static_cast<G*>(p.dgate), n, per_gate);
        check("linear recurrence gate gradient kernel");
    }
}

template <typename X, typename G, int V, bool SHARED>
void step(const RecurrenceArgs& p, cudaStream_t stream) {
    const uint64_t n = p.rows * (p.dim / V);
    if (n / 256 >= 0x7fffffffull) throw std::invalid_argument("linear_recurrence_step: problem too large for one kernel launch");
    recurrence_step_kernel<X, G, V, SHARED><<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(p);
    check("linear recurrence step kernel");
}

// Whether every access of a thread's V channels is one aligned load or store.
template <typename X, typename G, int V>
bool aligned(const RecurrenceArgs& p, bool shared) {
    const auto fits = [](const void* ptr, size_t bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; };
    const uint64_t group = p.dim / p.gate_dim;
    if (p.dim % V || p.x_batch % V || p.x_row % V || p.d_batch % V || p.d_row % V) return false;
    for (const void* ptr : {p.x, p.derivs, static_cast<const void*>(p.out), static_cast<const void*>(p.dx)})
        if (!fits(ptr, V * sizeof(X))) return false;
    for (const void* ptr : {static_cast<const void*>(p.state), static_cast<const void*>(p.checkpoints), p.marks})
        if (!fits(ptr, V * sizeof(Acc<X>))) return false;
    if (shared) return group % V == 0;
    return p.gate_batch % V == 0 && p.gate_row % V == 0 && fits(p.gate, V * sizeof(G)) && fits(p.dgate, V * sizeof(G));
}

}  // namespace

template <typename X, typename G>
void launch_recurrence(RecurrencePass pass, const RecurrenceArgs& p, cudaStream_t stream) {
    constexpr int W = kWide<X>;
    const bool shared = p.gate_dim != p.dim;
    const bool wide = aligned<X, G, W>(p, shared);
#define SIG_RECURRENCE(fn)                                                                   \
    wide ? (shared ? fn<X, G, W, true>(p, stream) : fn<X, G, W, false>(p, stream))           \
         : (shared ? fn<X, G, 1, true>(p, stream) : fn<X, G, 1, false>(p, stream))
    switch (pass) {
        case RecurrencePass::forward: SIG_RECURRENCE(forward); break;
        case RecurrencePass::backward: SIG_RECURRENCE(backward); break;
        case RecurrencePass::step: SIG_RECURRENCE(step); break;
    }
#undef SIG_RECURRENCE
}

#define SIG_INSTANTIATE(X, G) template void launch_recurrence<X, G>(RecurrencePass, const RecurrenceArgs&, cudaStream_t);
#if SIG_RECURRENCE_PART == 0
SIG_INSTANTIATE(float, float)
#elif SIG_RECURRENCE_PART == 1
SIG_INSTANTIATE(double, double)
#elif SIG_RECURRENCE_PART == 2
SIG_INSTANTIATE(__nv_bfloat16, __nv_bfloat16)
#elif SIG_RECURRENCE_PART == 3
SIG_INSTANTIATE(__nv_bfloat16, float)
#elif SIG_RECURRENCE_PART == 4
SIG_INSTANTIATE(__half, __half)
#else
SIG_INSTANTIATE(__half, float)
#endif

}  // namespace sigb200
