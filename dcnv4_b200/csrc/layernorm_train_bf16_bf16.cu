// LayerNorm training kernels for one pair of tensor types (see layernorm_train.cuh).
#include "layernorm_train.cuh"

namespace dcnb200 {

cudaError_t ln_train_run_bf16_bf16(bool backward, int mode, int act, const ln::Plan& p, const LnTrainArgs& a, cudaStream_t s) {
  return ln::run<__nv_bfloat16, __nv_bfloat16>(backward, mode, act, p, a, s);
}

}  // namespace dcnb200
