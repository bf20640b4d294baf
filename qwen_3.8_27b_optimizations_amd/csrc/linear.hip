// linear.hip -- linear attention with a decay for each head: which kernel takes a call.
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
    if (g.seqs > 0x7FFFFFFF / g.heads / 8) return hipErrorInvalidConfiguration;
    *bytes = 0;
    return hipSuccess;
}

hipError_t launch_linear_attention(const iq4xs_linear_attention_args& g, void* ws, size_t ws_bytes, hipStream_t stream) {
    size_t need;
    const hipError_t err = linear_attention_workspace(g, &need);
    if (err != hipSuccess) return err;
    if (ws_bytes < need || (need && (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0))) return hipErrorInvalidValue;
    clear_launch_error();
    launch_linear_step(args_of(g), g.dk, g.dv, g.in_type, linear_step_grid(g), stream);
    return hipGetLastError();
}

}  // namespace iq4xs
