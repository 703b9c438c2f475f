// context.hpp -- what the entry points outside bridge.cpp use of a context
// (bridge.cpp defines these).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "smoe_hip.h"

namespace smoe {

struct ContextView {
    int device;
    hipStream_t stream;
    uint32_t* err;        // device error word
};
ContextView context_view(const SmoeMetalCtx* ctx);

// The attention scratch of the context, at least `bytes` long: SMOE_OK,
// SMOE_ERR_CAPTURE (would grow under stream capture) or SMOE_ERR_HIP.  What it
// outgrows lives until the context is destroyed if a captured graph may hold it.
int context_attention_scratch(SmoeMetalCtx* ctx, size_t bytes, float** p);

// runs launch(arg), timed as `kind` when profiling; SMOE_OK or SMOE_ERR_HIP
int context_launch(SmoeMetalCtx* ctx, uint32_t kind, const char* what, hipError_t (*launch)(void*), void* arg);

// `rc`, with `why` for smoe_hip_last_error
int context_refuse(SmoeMetalCtx* ctx, int rc, const char* why);

}  // namespace smoe
