// The bf16 kernels of the biased attention's gradients (attn_bias_back.h).
#include "attn_bias_back.h"

namespace jh {

void grad_launch_bf16(const BiasBack& b, const GradPlan& plan, int bias, bool cap, hipStream_t st) {
    grad_launch<true>(b, plan, bias, cap, st);
}

}  // namespace jh
