// LayerNorm training kernels for one pair of tensor types (see layernorm_train.cuh).
#include "layernorm_train.cuh"

namespace dcnb200 {

cudaError_t ln_train_run_f16_f32(bool backward, int mode, int act, const ln::Plan& p, const LnTrainArgs& a, cudaStream_t s) {
  return ln::run<__half, float>(backward, mode, act, p, a, s);
}

}  // namespace dcnb200
