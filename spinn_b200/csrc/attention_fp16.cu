// attention_fp16.cu -- paged attention over fp16 caches.
#include "attention.cuh"

namespace spinn {

AttnPlan attention_plan_fp16(const AttnParams& p, int sms, bool weights) {
  return attention_plan_t<__half>(p, sms, weights);
}
int attention_launch_fp16(AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  return attention_launch_t<__half>(p, pl, st);
}

}  // namespace spinn
