// LayerNorm training passes: choice of the instantiation, and the reduction of the parameter gradients.
#include "layernorm_train.cuh"

namespace dcnb200 {

cudaError_t ln_train_run_f32_f32(bool, int, int, const ln::Plan&, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_f16_f16(bool, int, int, const ln::Plan&, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_f16_f32(bool, int, int, const ln::Plan&, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_bf16_bf16(bool, int, int, const ln::Plan&, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_bf16_f32(bool, int, int, const ln::Plan&, const LnTrainArgs&, cudaStream_t);

namespace {

constexpr int kCols = 32, kSlices = 32;

// Column sums of the CTAs' partial (A, B): a CTA takes 32 columns, each of its 32 warps a slice of the partials.
// The order of the additions depends on the sizes alone.
template <typename P>
__global__ void __launch_bounds__(kCols * kSlices)
ln_train_params_kernel(const LnTrainArgs a, int mode) {
  __shared__ float2 part[kSlices][kCols + 1];
  const int col = blockIdx.x * kCols + (threadIdx.x % kCols), slice = threadIdx.x / kCols;
  pdl_trigger();
  pdl_wait();
  float2 t = make_float2(0.f, 0.f);
  if (col < a.C) {
    for (int i = slice; i < a.n_partial; i += kSlices) {
      const float* p = a.partial + (size_t)i * 2 * a.C + col;
      t.x += p[0];
      t.y += p[a.C];
    }
  }
  part[slice][threadIdx.x % kCols] = t;
  __syncthreads();
  if (slice != 0 || col >= a.C) return;
  float sa = 0.f, sb = 0.f;
#pragma unroll
  for (int i = 0; i < kSlices; ++i) { const float2 u = part[i][threadIdx.x]; sa += u.x; sb += u.y; }
  ln::finish_column<P>(a, mode == ln::kPost, col, sa, sb);
}

}  // namespace

int ln_train_max_channels() { return ln::kMaxChannels; }

// Element sizes of types 0 fp32, 1 fp16, 2 bf16.
static int size_of(int d) { return d == 0 ? 4 : 2; }

// Alignment decides the kernel: bulk copies want every loaded tensor on 16 bytes, the vector stores every stored one.
static ln::Plan plan_of(bool backward, int mode, int xd, int yd, const LnTrainArgs& a) {
  auto on = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  const bool base = on(a.x, 16) && on(a.res, 16) && on(a.h, 16) && on(a.gy, 16) && on(a.gh, 16);
  const bool vec = on(a.y, 16) && on(a.h, 16) && on(a.dx, 16) && on(a.dx2, 16);
  return ln::plan_for(backward, mode, size_of(xd), size_of(yd), a.gh != nullptr, a.res != nullptr, base, vec, a.rows, a.C);
}

// Partial sums of the backward pass: one (2, C) fp32 block per CTA, for whichever kernel the alignment will choose.
size_t ln_train_workspace_bytes(int xd, int rows, int C) {
  const int direct = ln::direct_grid(rows, ln::geometry(C, 1, 0).lpr);
  const int n = direct > ln::kSms ? direct : (rows < ln::kSms ? rows : ln::kSms);
  return (size_t)n * 2 * C * sizeof(float);
}

// xd / yd: tensor types of the branch input and of residual / result / gradients; yd is xd or fp32.  Parameters are
// fp32 or of type xd.
static cudaError_t run(bool backward, int mode, int act, int xd, int yd, const ln::Plan& p, const LnTrainArgs& a, cudaStream_t s) {
  if (xd == 0) return ln_train_run_f32_f32(backward, mode, act, p, a, s);
  if (xd == 1) return yd == 0 ? ln_train_run_f16_f32(backward, mode, act, p, a, s) : ln_train_run_f16_f16(backward, mode, act, p, a, s);
  return yd == 0 ? ln_train_run_bf16_f32(backward, mode, act, p, a, s) : ln_train_run_bf16_bf16(backward, mode, act, p, a, s);
}

cudaError_t launch_ln_train_fwd(int mode, int act, int xd, int yd, const LnTrainArgs& a, cudaStream_t s) {
  return run(false, mode, act, xd, yd, plan_of(false, mode, xd, yd, a), a, s);
}

cudaError_t launch_ln_train_bwd(int mode, int act, int xd, int yd, const LnTrainArgs& a, cudaStream_t s) {
  const ln::Plan p = plan_of(true, mode, xd, yd, a);
  if (cudaError_t e = run(true, mode, act, xd, yd, p, a, s)) return e;
  if (!p.direct && p.grid == 1) return cudaSuccess;
  LnTrainArgs f = a;
  f.n_partial = p.grid;
  const dim3 grid((unsigned)((a.C + kCols - 1) / kCols)), threads(kCols * kSlices);
  if (xd == 1) return launch_overlapped(ln_train_params_kernel<__half>, grid, threads, 0, s, f, mode);
  if (xd == 2) return launch_overlapped(ln_train_params_kernel<__nv_bfloat16>, grid, threads, 0, s, f, mode);
  return launch_overlapped(ln_train_params_kernel<float>, grid, threads, 0, s, f, mode);
}

}  // namespace dcnb200
