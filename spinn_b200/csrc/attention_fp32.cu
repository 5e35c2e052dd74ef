// attention_fp32.cu -- paged attention over fp32 caches.
#include "attention.cuh"

namespace spinn {

AttnPlan attention_plan_fp32(const AttnParams& p, int sms, bool weights) {
  return attention_plan_t<float>(p, sms, weights);
}
int attention_launch_fp32(AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  return attention_launch_t<float>(p, pl, st);
}

}  // namespace spinn
