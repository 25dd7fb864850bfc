// Attention over the 8-bit KV cache, i8 codes: the kernel instantiations.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wunused-function"  // (the headers' other kernels)
#include "attention_q8.hpp"
#pragma clang diagnostic pop

namespace hm {

void launch_attn_q8_i8(const AttnQ8Params& P, int head_dim, const Q8Plan& plan, bool two, hipStream_t s) {
    launch_attn_q8<RK_NPU_HIP_KV_I8>(P, head_dim, plan, two, s);
}

}  // namespace hm
