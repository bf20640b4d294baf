// linear.hip -- linear attention with a decay for each head: a call's launches (by linear_plan.h).
#include "iq4xs_internal.h"
#include "linear_device.h"
#include "linear_internal.h"
#include "linear_launch.h"

namespace iq4xs {

static LinearArgs args_of(const iq4xs_linear_attention_args& g) {
    return {g.q, g.k, g.v, g.decay, g.starts, g.states, g.from_slots, g.to_slots, g.out, g.q_stride, g.k_stride, g.v_stride,
            g.decay_stride, g.states ? g.slots : 0, (int)g.total, (int)g.most_q, (int)g.seqs, g.heads, g.heads / g.qk_heads,
            g.out_type, g.scale};
}

hipError_t linear_attention_workspace(const iq4xs_linear_attention_args& g, size_t* bytes) {
    LinearPlan p;
    if (!linear_plan(g, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    *bytes = p.state_bytes + p.decay_bytes;
    return hipSuccess;
}

hipError_t launch_linear_attention(const iq4xs_linear_attention_args& g, void* ws, size_t ws_bytes, hipStream_t stream) {
    LinearPlan p;
    if (!linear_plan(g, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    const size_t need = p.state_bytes + p.decay_bytes;
    if (ws_bytes < need || (need && (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0))) return hipErrorInvalidValue;
    clear_launch_error();
    const LinearArgs a = args_of(g);
    if (p.steps) {
        launch_linear_steps(a, g.dk, g.dv, g.in_type, p.units, stream);
    } else {
        float* states = static_cast<float*>(ws);
        static_assert(sizeof(SegmentDecay) == SEGMENT_DECAY_BYTES, "as the workspace counts them");
        const LinearSegments segments{states, reinterpret_cast<SegmentDecay*>(states + p.state_bytes / sizeof(float)),
                                      p.segments, p.length, p.runs, p.kept, p.join_rows, p.grid};
        launch_linear_chunks(a, segments, g.dk, g.dv, g.in_type, stream);
    }
    return hipGetLastError();
}

}  // namespace iq4xs
