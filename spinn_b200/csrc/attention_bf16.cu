// attention_bf16.cu -- paged attention over bf16 caches.
#include "attention.cuh"

namespace spinn {

AttnPlan attention_plan_bf16(const AttnParams& p, int sms, bool weights) {
  return attention_plan_t<__nv_bfloat16>(p, sms, weights);
}
int attention_launch_bf16(AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  return attention_launch_t<__nv_bfloat16>(p, pl, st);
}

}  // namespace spinn
