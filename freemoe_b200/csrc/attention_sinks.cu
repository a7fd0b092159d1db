// attention_sinks.cu -- the kernels of attention over a paged cache for windows behind which
// the first keys stay visible: a unit of their own, so that the two sets build side by side.
#include "attention_launch.cuh"

namespace fmb {

int launch_attention_sinks(const fmcuda_paged_attention_args &a, const AttnPlan &n, const AttnParams &p, uint8_t *ws,
                           cudaStream_t s) {
    return launch_attention_of<true>(a, n, p, ws, s);
}

} // namespace fmb
