// Host side of the gated linear recurrence: checks, staging of host arrays, dispatch on element types.
#include "recurrence.h"

#include "algebra_host.h"

namespace sigb200 {
namespace {

void dispatch(RecurrencePass pass, const RecurrenceArgs& p, cudaStream_t stream) {
    if (p.type == kFloat32) launch_recurrence<float, float>(pass, p, stream);
    else if (p.type == kFloat64) launch_recurrence<double, double>(pass, p, stream);
    else if (p.type == kBFloat16 && p.gate_type == kBFloat16) launch_recurrence<__nv_bfloat16, __nv_bfloat16>(pass, p, stream);
    else if (p.type == kBFloat16) launch_recurrence<__nv_bfloat16, float>(pass, p, stream);
    else if (p.gate_type == kFloat16) launch_recurrence<__half, __half>(pass, p, stream);
    else launch_recurrence<__half, float>(pass, p, stream);
}

struct Sizes {
    uint64_t values, gates, states, marks;  // elements of x, the gates, the states, the checkpoints
};

Sizes checked(const RecurrenceArgs& p, const char* who) {
    const std::string name(who);
    if (p.type < kFloat32 || p.type > kFloat16) throw std::invalid_argument(name + ": unknown element type");
    if (p.gate_type != p.type && !(p.gate_type == kFloat32 && (p.type == kBFloat16 || p.type == kFloat16)))
        throw std::invalid_argument(name + ": gates must have the type of x, or float32 for 16-bit x");
    if (p.form < kGateValue || p.form > kGateLogit) throw std::invalid_argument(name + ": unknown gate form");
    if (p.dim == 0 || p.gate_dim == 0 || p.dim % p.gate_dim)
        throw std::invalid_argument(name + ": the number of gates must divide the number of channels");
    if (!p.x || !p.gate) throw std::invalid_argument(name + " received a null pointer");
    if (p.sequences && (p.batch != 1 || !p.offsets))
        throw std::invalid_argument(name + ": packed sequences need offsets and a batch of 1");
    if (p.rows >= kMaxRows || p.sequences >= kMaxRows) throw std::out_of_range(name + ": 2^30 rows or sequences and more are not supported");
    const uint64_t rows = checked_mul(p.batch, p.rows, who);
    Sizes s{};
    s.values = checked_mul(rows, p.dim, who);
    if (s.values >= 1ull << 59) throw std::out_of_range(name + ": size overflow");
    s.gates = rows * p.gate_dim;
    s.states = checked_mul(p.sequences ? p.sequences : p.batch, p.dim, who);
    s.marks = p.batch * ((p.rows + kCheckpointRows - 1) / kCheckpointRows) * p.dim;
    return s;
}

// Host arrays are staged whole and without gaps.
void require_dense(uint64_t batch, uint64_t rows, uint64_t width, uint64_t batch_stride, uint64_t row_stride, const char* who) {
    if (row_stride != width || (batch > 1 && batch_stride != rows * width))
        throw std::invalid_argument(std::string(who) + ": host buffers must be contiguous");
}

void require_dense_inputs(const RecurrenceArgs& p, const char* who) {
    require_dense(p.batch, p.rows, p.dim, p.x_batch, p.x_row, who);
    require_dense(p.batch, p.rows, p.gate_dim, p.gate_batch, p.gate_row, who);
    if (p.derivs) require_dense(p.batch, p.rows, p.dim, p.d_batch, p.d_row, who);
}

StagedOperand input(const void* p, size_t bytes) { return {p, nullptr, p ? bytes : 0}; }
StagedOperand output(void* p, size_t bytes) { return {nullptr, p, p ? bytes : 0}; }
template <typename T> T staged(T host, void* device) { return host ? static_cast<T>(device) : nullptr; }

void backward_on_device(RecurrenceArgs p, const Sizes& s, cudaStream_t stream) {
    Scratch marks(p.marks ? 0 : s.marks * state_size(p.type), stream);
    if (!p.marks) {  // the states entering every 16th row, by a forward pass that stores nothing else
        RecurrenceArgs f = p;
        f.out = f.state = nullptr;
        f.derivs = nullptr;
        f.dx = f.dgate = nullptr;
        f.checkpoints = marks.get();
        dispatch(RecurrencePass::forward, f, stream);
        p.marks = marks.get();
    }
    p.state = nullptr;
    dispatch(RecurrencePass::backward, p, stream);
}

}  // namespace

void recurrence_entry(const RecurrenceArgs& args, const CallOptions& opt) {
    const char* who = "linear_recurrence";
    RecurrenceArgs p = args;
    if (p.batch == 0 || p.rows == 0) return;
    const Sizes s = checked(p, who);
    if (!p.out) throw std::invalid_argument("linear_recurrence received a null pointer");
    int device = opt.known_device;
    if (device >= 0 || all_on_device({p.x, p.gate, p.initial, p.offsets, p.out, p.state, p.checkpoints}, who, &device)) {
        DeviceGuard guard(device);
        dispatch(RecurrencePass::forward, p, opt.stream);
        if (opt.synchronize) SIG_CUDA_CHECK(cudaStreamSynchronize(opt.stream));
        return;
    }
    require_dense_inputs(p, who);
    const size_t e = element_size(p.type), st = state_size(p.type);
    run_staged({input(p.x, s.values * e), input(p.gate, s.gates * element_size(p.gate_type)), input(p.initial, s.states * st),
                input(p.offsets, (p.sequences + 1) * (p.wide_offsets ? 8 : 4)), output(p.out, s.values * e),
                output(p.state, s.states * st), output(p.checkpoints, s.marks * st)},
               opt.device, [&](const std::vector<void*>& d, cudaStream_t stream) {
                   RecurrenceArgs q = p;
                   q.x = d[0]; q.gate = d[1];
                   q.initial = staged(p.initial, d[2]); q.offsets = staged(p.offsets, d[3]);
                   q.out = d[4]; q.state = staged(p.state, d[5]); q.checkpoints = staged(p.checkpoints, d[6]);
                   dispatch(RecurrencePass::forward, q, stream);
               });
}

void recurrence_backprop_entry(const RecurrenceArgs& args, const CallOptions& opt) {
    const char* who = "linear_recurrence_backprop";
    RecurrenceArgs p = args;
    if (p.batch == 0 || p.rows == 0) return;
    const Sizes s = checked(p, who);
    if (!p.derivs || !p.dx || !p.dgate) throw std::invalid_argument("linear_recurrence_backprop received a null pointer");
    int device = opt.known_device;
    if (device >= 0 || all_on_device({p.derivs, p.x, p.gate, p.initial, p.offsets, p.state_derivs, p.marks, p.dx, p.dgate, p.dinitial}, who, &device)) {
        DeviceGuard guard(device);
        backward_on_device(p, s, opt.stream);
        if (opt.synchronize) SIG_CUDA_CHECK(cudaStreamSynchronize(opt.stream));
        return;
    }
    require_dense_inputs(p, who);
    const size_t e = element_size(p.type), st = state_size(p.type), ge = element_size(p.gate_type);
    run_staged({input(p.x, s.values * e), input(p.gate, s.gates * ge), input(p.initial, s.states * st),
                input(p.offsets, (p.sequences + 1) * (p.wide_offsets ? 8 : 4)), input(p.derivs, s.values * e),
                input(p.state_derivs, s.states * st), input(p.marks, s.marks * st), output(p.dx, s.values * e),
                output(p.dgate, s.gates * ge), output(p.dinitial, s.states * st)},
               opt.device, [&](const std::vector<void*>& d, cudaStream_t stream) {
                   RecurrenceArgs q = p;
                   q.x = d[0]; q.gate = d[1];
                   q.initial = staged(p.initial, d[2]); q.offsets = staged(p.offsets, d[3]);
                   q.derivs = d[4]; q.state_derivs = staged(p.state_derivs, d[5]); q.marks = staged(p.marks, d[6]);
                   q.dx = d[7]; q.dgate = d[8]; q.dinitial = staged(p.dinitial, d[9]);
                   backward_on_device(q, s, stream);
               });
}

void recurrence_step_entry(const RecurrenceArgs& args, const CallOptions& opt) {
    const char* who = "linear_recurrence_step";
    RecurrenceArgs p = args;
    if (p.rows == 0) return;
    const Sizes s = checked(p, who);
    if (!p.out || !p.state) throw std::invalid_argument("linear_recurrence_step received a null pointer");
    int device = opt.known_device;
    if (device >= 0 || all_on_device({p.x, p.gate, p.out, p.state}, who, &device)) {
        DeviceGuard guard(device);
        dispatch(RecurrencePass::step, p, opt.stream);
        if (opt.synchronize) SIG_CUDA_CHECK(cudaStreamSynchronize(opt.stream));
        return;
    }
    require_dense_inputs(p, who);
    const size_t e = element_size(p.type), st = state_size(p.type);
    run_staged({input(p.x, s.values * e), input(p.gate, s.gates * element_size(p.gate_type)),
                {p.state, p.state, s.values * st}, output(p.out, s.values * e)},
               opt.device, [&](const std::vector<void*>& d, cudaStream_t stream) {
                   RecurrenceArgs q = p;
                   q.x = d[0]; q.gate = d[1]; q.state = d[2]; q.out = d[3];
                   dispatch(RecurrencePass::step, q, stream);
               });
}

}  // namespace sigb200
