// LayerNorm training passes: choice of the instantiation, and the reduction of the parameter gradients.
#include "layernorm_train.cuh"

namespace dcnb200 {

cudaError_t ln_train_run_f32_f32(bool, int, int, bool, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_f16_f16(bool, int, int, bool, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_f16_f32(bool, int, int, bool, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_bf16_bf16(bool, int, int, bool, const LnTrainArgs&, cudaStream_t);
cudaError_t ln_train_run_bf16_f32(bool, int, int, bool, const LnTrainArgs&, cudaStream_t);

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
  auto put = [&](void* dst, float v) {
    if (a.param_f32) static_cast<float*>(dst)[col] = v;
    else static_cast<P*>(dst)[col] = from_f32<P>(v);
  };
  if (mode == ln::kPost && a.gamma != nullptr) {
    const float g = ln::param<P>(a.gamma, col, a.param_f32);
    put(a.dgamma, fmaf(ln::param<P>(a.w, col, a.param_f32), sa, ln::param<P>(a.b, col, a.param_f32) * sb));
    put(a.dw, g * sa);
    put(a.db, g * sb);
  } else {
    put(a.dw, sa);
    put(a.db, sb);
  }
}

}  // namespace

// Whether the 16-byte vectors of the wide instantiation may be used: every row of every tensor starts on 16 bytes.
static bool vectors_ok(int xd, int yd, const LnTrainArgs& a) {
  const int ex = xd == 0 ? 4 : 2, ey = yd == 0 ? 4 : 2;
  const int v = xd == 0 ? 4 : 8;
  if (a.C % v != 0 || (long long)a.C * ex % 16 != 0 || (long long)a.C * ey % 16 != 0) return false;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  return al(a.x) && al(a.res) && al(a.y) && al(a.h) && al(a.gy) && al(a.gh) && al(a.dx) && al(a.dx2);
}

static ln::Geometry geometry_of(int xd, int C, bool vec) {
  const int v = xd == 0 ? 4 : 8;
  return ln::geometry(vec ? C / v : C, !vec, v == 8 ? 3 : 4);
}

int ln_train_max_channels() { return ln::kMaxChannels; }

// Partial sums of the backward pass: one (2, C) fp32 block per CTA.  The scalar instantiation's grid is the larger
// one wherever both exist; the workspace covers either.
size_t ln_train_workspace_bytes(int xd, int rows, int C) {
  const int v = xd == 0 ? 4 : 8;
  int n = ln::grid_for(rows, geometry_of(xd, C, false), ln::kBwdPerSm);
  if (C % v == 0) {
    const int m = ln::grid_for(rows, geometry_of(xd, C, true), ln::kBwdPerSm);
    n = n > m ? n : m;
  }
  return (size_t)n * 2 * C * sizeof(float);
}

// xd / yd: tensor types (0 fp32, 1 fp16, 2 bf16) of the branch input and of residual / result / gradients; yd is
// xd or fp32.  Parameters are fp32 or of type xd.
static cudaError_t run(bool backward, int mode, int act, int xd, int yd, const LnTrainArgs& a, cudaStream_t s) {
  const bool vec = vectors_ok(xd, yd, a);
  if (xd == 0) return ln_train_run_f32_f32(backward, mode, act, vec, a, s);
  if (xd == 1) return yd == 0 ? ln_train_run_f16_f32(backward, mode, act, vec, a, s) : ln_train_run_f16_f16(backward, mode, act, vec, a, s);
  return yd == 0 ? ln_train_run_bf16_f32(backward, mode, act, vec, a, s) : ln_train_run_bf16_bf16(backward, mode, act, vec, a, s);
}

cudaError_t launch_ln_train_fwd(int mode, int act, int xd, int yd, const LnTrainArgs& a, cudaStream_t s) {
  return run(false, mode, act, xd, yd, a, s);
}

cudaError_t launch_ln_train_bwd(int mode, int act, int xd, int yd, const LnTrainArgs& a, cudaStream_t s) {
  if (cudaError_t e = run(true, mode, act, xd, yd, a, s)) return e;
  LnTrainArgs f = a;
  f.n_partial = ln::grid_for(a.rows, geometry_of(xd, a.C, vectors_ok(xd, yd, a)), ln::kBwdPerSm);
  const dim3 grid((unsigned)((a.C + kCols - 1) / kCols)), threads(kCols * kSlices);
  if (xd == 1) return launch_overlapped(ln_train_params_kernel<__half>, grid, threads, 0, s, f, mode);
  if (xd == 2) return launch_overlapped(ln_train_params_kernel<__nv_bfloat16>, grid, threads, 0, s, f, mode);
  return launch_overlapped(ln_train_params_kernel<float>, grid, threads, 0, s, f, mode);
}

}  // namespace dcnb200
