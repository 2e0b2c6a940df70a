// Entry points of the sequence operators (gated linear recurrences, rotary positions): argument
// blocks shared by the C ABI, the host dispatch and the kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "dispatch.h"

namespace sigb200 {

// Element types of the sequence operators, as the C ABI numbers them.
enum ElementType : int { kFloat32 = 0, kFloat64 = 1, kBFloat16 = 2, kFloat16 = 3 };
// Types of rotary positions.
enum PositionType : int { kPositionNone = 0, kPositionInt32 = 1, kPositionInt64 = 2, kPositionFloat32 = 3, kPositionFloat64 = 4 };
// How a gate value v gives the factor a of the recurrence: a = v, exp(v), 1 / (1 + exp(-v)).
enum GateForm : int { kGateValue = 0, kGateLog = 1, kGateLogit = 2 };

inline size_t element_size(int type) { return type == kFloat64 ? 8 : type == kFloat32 ? 4 : 2; }
// States, checkpoints and their gradients: float64 for float64 inputs, else float32.
inline size_t state_size(int type) { return type == kFloat64 ? 8 : 4; }

// Rows between two checkpoints of a recurrence (the state entering rows 0, 16, 32, ..): near enough for the
// backward pass to start each warp's rows without waiting for the others', for 1/16 of a state's bytes a row.
constexpr uint64_t kCheckpointRows = 16;

// Rows are counted in 32 bits, with room for the blocks that an iteration looks ahead.
constexpr uint64_t kMaxRows = 1ull << 30;

struct RecurrenceArgs {
    int type, gate_type;
    uint64_t batch, rows, dim, gate_dim, sequences;  // sequences > 0: packed, batch == 1
    const void *x, *gate, *initial, *offsets;        // initial, offsets may be null
    void *out, *state, *checkpoints;                 // any of them may be null
    const void *derivs, *state_derivs, *marks;       // backward: marks = checkpoints of the forward pass
    void *dx, *dgate, *dinitial;                     // backward
    uint64_t x_batch, x_row, gate_batch, gate_row, d_batch, d_row;  // strides in elements
    int form;
    bool complement, wide_offsets;
};

void recurrence_entry(const RecurrenceArgs& args, const CallOptions& opt);
void recurrence_backprop_entry(const RecurrenceArgs& args, const CallOptions& opt);
// x, gate (rows, dim | gate_dim) contiguous; state (rows, dim) is read and overwritten.
void recurrence_step_entry(const RecurrenceArgs& args, const CallOptions& opt);

struct RotaryArgs {
    int type, position_type;
    uint64_t n0, n1, rows, dim, rotary_dim;
    const void* x;
    const double* frequencies;
    const void* positions;
    void* out;
    uint64_t x0, x1, x_row, out0, out1, out_row, p0, p1, p_row;  // strides in elements
    bool interleaved, inverse;
    double scale;
};

void rotary_entry(const RotaryArgs& args, const CallOptions& opt);

}  // namespace sigb200
