// Attention over the 8-bit KV cache, e4m3 codes: the kernel instantiations.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wunused-function"  // (the headers' other kernels)
#include "attention_q8.hpp"
#pragma clang diagnostic pop

namespace hm {

void launch_attn_q8_e4m3(const AttnQ8Params& P, int head_dim, const Q8Plan& plan, bool two, hipStream_t s) {
    launch_attn_q8<RK_NPU_HIP_KV_E4M3>(P, head_dim, plan, two, s);
}

}  // namespace hm
