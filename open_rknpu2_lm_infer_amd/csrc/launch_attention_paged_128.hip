// The attention over the paged cache, head_dim 128.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wunused-function"  // (the headers' other kernels)
#include "attention_paged.hpp"
#pragma clang diagnostic pop

namespace hm {

void launch_attn_paged_128(const AttnPagedParams& P, const PagedPlan& plan, hipStream_t s) {
    launch_attn_paged<128>(P, plan, s);
}

}  // namespace hm
