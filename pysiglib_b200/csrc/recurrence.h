// Launch interface of the recurrence kernels: enqueues one pass on `stream` for the current device.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "runtime.h"
#include "sequence.h"

namespace sigb200 {

enum class RecurrencePass { forward, backward, step };

template <typename X, typename G>
void launch_recurrence(RecurrencePass pass, const RecurrenceArgs& p, cudaStream_t stream);

}  // namespace sigb200
