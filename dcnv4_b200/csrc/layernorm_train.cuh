// LayerNorm for training: forward passes that keep each row's statistics, and the backward passes with the
// reductions of the parameter gradients, for the three places a FlashInternImage layer normalises:
//
//   plain   y   = act(z),                       z = xh * w + b,  xh = (x - mean) * rstd
//   post    out = residual + s * gamma * z      (post-norm block: layer scale gamma, stochastic depth s per sample)
//   pre     h   = residual + s * x,  y = LN(h)  (seam of two pre-norm branches)
//
// Backward, with g the gradient that reaches z (times the activation's derivative, times s) and w' = w or w * gamma:
//   dx = rstd * (g w' - mean_c(g w') - xh * mean_c(g w' xh))      [+ grad_h for `pre`]
//   A  = sum_rows g * xh,   B = sum_rows g
//   plain, pre: dw = A, db = B;   post: dw = gamma A, db = gamma B, dgamma = w A + b B
// so one row kernel and one small reduction over the CTAs' partial (A, B) serve all three.
//
// A row belongs to a team of `lpr` lanes: 2..32 lanes of a warp, or a whole CTA of 2..16 warps.  A lane keeps its
// NV vectors of the row in registers (each element is read once and written once), its slice of the parameters and
// of A and B for the whole launch; statistics and sums are fp32, two passes over registers (mean, then squared
// deviations).  Nothing is accumulated with atomics: the order of every sum is fixed by the sizes alone, so
// results repeat bit for bit.
//
// The reference builds these norms from torch.nn.LayerNorm, layer-scale products, timm's DropPath and residual
// additions (classification/models/flash_intern_image.py:34-56, 414-432); it has no kernel for them.
#pragma once

#include "common.cuh"

namespace dcnb200 {

struct LnTrainArgs {
  const void* x;         // branch input (plain, post: the normalised tensor)
  const void* res;       // residual (post, pre)
  const void* w;         // LayerNorm weight, bias, layer scale (may be null): all in the parameter type
  const void* b;
  const void* gamma;
  const float* s;        // per-sample factor or null
  void* y;               // forward result
  void* h;               // pre: the sum
  float* mean;
  float* rstd;
  // backward
  const void* gy;        // gradient of y / out
  const void* gh;        // pre: gradient of h or null
  void* dx;              // gradient of the normalised tensor (pre: of the residual)
  void* dx2;             // pre: gradient of the branch input, or null when it equals dx
  float* partial;        // (CTAs, 2, C)
  void* dw;
  void* db;
  void* dgamma;
  int rows, C;
  int lpr;               // lanes of a team (32 * warps when a row takes the whole CTA)
  int param_f32;         // parameters are fp32 (else: the type TP of the instantiation)
  unsigned rows_per_sample;
  int n_partial;
  float eps;
};

namespace ln {

constexpr int kMaxChannels = 8192;
constexpr int kSms = 148;              // B200: fixes the grid, hence the order of sums and the workspace size

// One lane's vector of N elements as raw words; N * sizeof(T) is 16 or 32 bytes, or N is 1.
template <typename T, int N> struct Words { uint32_t r[(N * sizeof(T) + 3) / 4]; };

template <typename T, int N>
__device__ __forceinline__ void load(Words<T, N>& v, const T* p, bool ok) {
  if constexpr (N == 1) {
    if constexpr (sizeof(T) == 4) v.r[0] = ok ? __float_as_uint(__ldg((const float*)p)) : 0u;
    else v.r[0] = ok ? (uint32_t)__ldg((const unsigned short*)p) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T)) / 16; ++i) {
      uint4 t = make_uint4(0u, 0u, 0u, 0u);
      if (ok) t = __ldg(reinterpret_cast<const uint4*>(p) + i);
      v.r[4 * i] = t.x; v.r[4 * i + 1] = t.y; v.r[4 * i + 2] = t.z; v.r[4 * i + 3] = t.w;
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void to_floats(const Words<T, N>& v, float (&f)[N]) {
  if constexpr (N == 1) {
    if constexpr (sizeof(T) == 4) f[0] = __uint_as_float(v.r[0]);
    else { const unsigned short u = (unsigned short)v.r[0]; f[0] = to_f32(*reinterpret_cast<const T*>(&u)); }
  } else {
    widen(v.r, f, (const T*)nullptr);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&f)[N]) {
  if constexpr (N == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    uint32_t r[N * sizeof(T) / 4];
    narrow(f, r, (const T*)nullptr);
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T)) / 16; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
  }
}

// Parameters are fp32 or the 16-bit type P; read once per launch.
template <typename P>
__device__ __forceinline__ float param(const void* p, int i, int f32) {
  return f32 ? __ldg(static_cast<const float*>(p) + i) : to_f32(static_cast<const P*>(p)[i]);
}

__device__ __forceinline__ float warp_sum(float v, int lanes) {
  if (lanes > 16) v += __shfl_xor_sync(0xffffffffu, v, 16);
  if (lanes > 8) v += __shfl_xor_sync(0xffffffffu, v, 8);
  if (lanes > 4) v += __shfl_xor_sync(0xffffffffu, v, 4);
  if (lanes > 2) v += __shfl_xor_sync(0xffffffffu, v, 2);
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v;
}
// Sum of two values over the team.  `red` is [2][16] float2; teams wider than a warp are the whole CTA and meet at
// one barrier per call: the slots alternate, so the next call cannot overwrite what a slow warp still reads.
__device__ __forceinline__ float2 team_sum(float a, float b, int lpr, float2 (*red)[16], int& flip) {
  a = warp_sum(a, lpr);
  b = warp_sum(b, lpr);
  if (lpr > 32) {
    float2* slot = red[flip];
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = 0.f; b = 0.f;
    for (int i = 0; i < (lpr >> 5); ++i) { const float2 t = slot[i]; a += t.x; b += t.y; }
  }
  return make_float2(a, b);
}

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;

enum : int { kPlain = 0, kPost = 1, kPre = 2 };

// ------------------------------------------------------------------------------------ forward

template <typename TX, typename TY, int VEC, int NV, int MODE, bool GELU>
__global__ void __launch_bounds__(512)
ln_train_fwd_kernel(const LnTrainArgs a) {
  using P = TX;
  __shared__ float2 red[2][16];
  const int lpr = a.lpr, C = a.C;
  const bool wide = lpr > 32;
  const int sub = wide ? threadIdx.x : (threadIdx.x & 31) % lpr;
  const int team0 = wide ? blockIdx.x : (blockIdx.x * blockDim.x + threadIdx.x) / lpr;
  const int n_teams = wide ? gridDim.x : gridDim.x * blockDim.x / lpr;
  const float inv_c = 1.f / (float)C;
  int flip = 0;
  pdl_trigger();
  pdl_wait();

  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = (sub + v * lpr) * VEC + e;
      const bool ok = c < C;
      w[v][e] = ok ? param<P>(a.w, c, a.param_f32) : 0.f;
      b[v][e] = ok ? param<P>(a.b, c, a.param_f32) : 0.f;
      if (MODE == kPost && a.gamma != nullptr) {
        const float g = ok ? param<P>(a.gamma, c, a.param_f32) : 0.f;
        w[v][e] *= g;
        b[v][e] *= g;
      }
    }
  // the lanes of a warp stay in the loop together: the team sums shuffle across it
  const int row_step = n_teams;
  for (int r0 = wide ? team0 : team0 - (int)(threadIdx.x & 31) / lpr; r0 < a.rows; r0 += row_step) {
    const int row = wide ? r0 : r0 + (int)(threadIdx.x & 31) / lpr;
    const bool live = row < a.rows;
    const long long base = (long long)row * C;
    Words<TX, VEC> rx[NV];
    Words<TY, VEC> rr[MODE == kPlain ? 1 : NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (sub + v * lpr) * VEC;
      load<TX, VEC>(rx[v], static_cast<const TX*>(a.x) + base + c, live && c < C);
      if (MODE != kPlain) load<TY, VEC>(rr[v], static_cast<const TY*>(a.res) + base + c, live && c < C);
    }
    float s = 1.f;
    if (MODE != kPlain && a.s != nullptr) s = live ? __ldg(a.s + (unsigned)row / a.rows_per_sample) : 0.f;
    float xv[NV][VEC];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      to_floats<TX, VEC>(rx[v], xv[v]);
      if (MODE == kPre) {
        float rv[VEC];
        to_floats<TY, VEC>(rr[v], rv);
#pragma unroll
        for (int e = 0; e < VEC; ++e) xv[v][e] = fmaf(s, xv[v][e], rv[e]);
        const int c = (sub + v * lpr) * VEC;
        if (live && c < C) store<TY, VEC>(static_cast<TY*>(a.h) + base + c, xv[v]);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += xv[v][e];
    }
    const float mean = team_sum(sum, 0.f, lpr, red, flip).x * inv_c;
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if ((sub + v * lpr) * VEC < C) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const float d = xv[v][e] - mean; sq = fmaf(d, d, sq); }
      }
    const float rstd = rsqrtf(team_sum(sq, 0.f, lpr, red, flip).x * inv_c + a.eps);
    if (!live) continue;
    if (sub == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (sub + v * lpr) * VEC;
      if (c >= C) continue;
      float o[VEC], rv[VEC];
      if (MODE == kPost) to_floats<TY, VEC>(rr[v], rv);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        o[e] = fmaf((xv[v][e] - mean) * rstd, w[v][e], b[v][e]);
        if (GELU) o[e] = 0.5f * o[e] * (1.f + erff(o[e] * kSqrtHalf));
        if (MODE == kPost) o[e] = fmaf(s, o[e], rv[e]);
      }
      store<TY, VEC>(static_cast<TY*>(a.y) + base + c, o);
    }
  }
}

// ----------------------------------------------------------------------------------- backward

// TL: type of the normalised tensor and of its gradient; TG: type of the incoming gradients; T2: type of the branch
// gradient of `pre`; P: parameter type when not fp32.
template <typename TL, typename TG, typename T2, typename P, int VEC, int NV, int MODE, bool GELU>
__global__ void __launch_bounds__(512)
ln_train_bwd_kernel(const LnTrainArgs a) {
  __shared__ float2 red[2][16];
  extern __shared__ float acc_smem[];    // [2][C]
  const int lpr = a.lpr, C = a.C;
  const bool wide = lpr > 32;
  const int lane = threadIdx.x & 31;
  const int sub = wide ? threadIdx.x : lane % lpr;
  const int team0 = wide ? blockIdx.x : (blockIdx.x * blockDim.x + threadIdx.x) / lpr;
  const int n_teams = wide ? gridDim.x : gridDim.x * blockDim.x / lpr;
  const float inv_c = 1.f / (float)C;
  int flip = 0;
  pdl_trigger();
  pdl_wait();

  float w[NV][VEC], b[GELU ? NV : 1][VEC], sa[NV][VEC], sb[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = (sub + v * lpr) * VEC + e;
      const bool ok = c < C;
      w[v][e] = ok ? param<P>(a.w, c, a.param_f32) : 0.f;
      if (GELU) b[v][e] = ok ? param<P>(a.b, c, a.param_f32) : 0.f;
      if (MODE == kPost && a.gamma != nullptr && ok) w[v][e] *= param<P>(a.gamma, c, a.param_f32);
      sa[v][e] = 0.f;
      sb[v][e] = 0.f;
    }
  for (int r0 = wide ? team0 : team0 - lane / lpr; r0 < a.rows; r0 += n_teams) {
    const int row = wide ? r0 : r0 + lane / lpr;
    const bool live = row < a.rows;
    const long long base = (long long)row * C;
    Words<TL, VEC> rx[NV];
    Words<TG, VEC> rg[NV], rh[MODE == kPre ? NV : 1];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (sub + v * lpr) * VEC;
      const bool ok = live && c < C;
      load<TL, VEC>(rx[v], static_cast<const TL*>(MODE == kPre ? a.h : a.x) + base + c, ok);
      load<TG, VEC>(rg[v], static_cast<const TG*>(a.gy) + base + c, ok);
      if (MODE == kPre) load<TG, VEC>(rh[v], static_cast<const TG*>(a.gh) + base + c, ok && a.gh != nullptr);
    }
    const float mean = live ? __ldg(a.mean + row) : 0.f, rstd = live ? __ldg(a.rstd + row) : 0.f;
    float s = 1.f;
    if (MODE != kPlain && a.s != nullptr) s = live ? __ldg(a.s + (unsigned)row / a.rows_per_sample) : 0.f;
    float xh[NV][VEC], gw[NV][VEC];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float g[VEC];
      to_floats<TL, VEC>(rx[v], xh[v]);
      to_floats<TG, VEC>(rg[v], g);
      const bool ok = live && (sub + v * lpr) * VEC < C;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        xh[v][e] = ok ? (xh[v][e] - mean) * rstd : 0.f;
        if (MODE == kPost) g[e] *= s;
        if (GELU) {
          const float z = fmaf(xh[v][e], w[v][e], b[v][e]);
          const float cdf = 0.5f * (1.f + erff(z * kSqrtHalf));
          g[e] *= fmaf(z * kInvSqrt2Pi, __expf(-0.5f * z * z), cdf);
        }
        sa[v][e] = fmaf(g[e], xh[v][e], sa[v][e]);
        sb[v][e] += g[e];
        gw[v][e] = g[e] * w[v][e];
        s1 += gw[v][e];
        s2 = fmaf(gw[v][e], xh[v][e], s2);
      }
    }
    const float2 t = team_sum(s1, s2, lpr, red, flip);
    const float m1 = t.x * inv_c, m2 = t.y * inv_c;
    if (!live) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (sub + v * lpr) * VEC;
      if (c >= C) continue;
      float o[VEC], hv[VEC];
      if (MODE == kPre) to_floats<TG, VEC>(rh[v], hv);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        o[e] = rstd * (gw[v][e] - fmaf(xh[v][e], m2, m1));
        if (MODE == kPre) o[e] += hv[e];
      }
      store<TL, VEC>(static_cast<TL*>(a.dx) + base + c, o);
      if (MODE == kPre && a.dx2 != nullptr) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] *= s;
        store<T2, VEC>(static_cast<T2*>(a.dx2) + base + c, o);
      }
    }
  }

  // this CTA's sums: over the teams of each warp by shuffles, then warp after warp into shared memory
  if (!wide) {
    for (int o = lpr; o < 32; o <<= 1) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sa[v][e] += __shfl_xor_sync(0xffffffffu, sa[v][e], o);
          sb[v][e] += __shfl_xor_sync(0xffffffffu, sb[v][e], o);
        }
    }
    const int n_warps = blockDim.x >> 5;
    for (int q = 0; q < n_warps; ++q) {
      if ((int)(threadIdx.x >> 5) == q && lane < lpr) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int c = (sub + v * lpr) * VEC + e;
            if (c < C) {
              acc_smem[c] = (q ? acc_smem[c] : 0.f) + sa[v][e];
              acc_smem[C + c] = (q ? acc_smem[C + c] : 0.f) + sb[v][e];
            }
          }
      }
      __syncthreads();
    }
    float* dst = a.partial + (size_t)blockIdx.x * 2 * C;
    for (int i = threadIdx.x; i < 2 * C; i += blockDim.x) dst[i] = acc_smem[i];
  } else {
    float* dst = a.partial + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = (sub + v * lpr) * VEC + e;
        if (c < C) { dst[c] = sa[v][e]; dst[C + c] = sb[v][e]; }
      }
  }
}

// --------------------------------------------------------------------------------- dispatch

// Team width and vectors per lane for `n_vec` vectors a row.
struct Geometry {
  int lpr, nv, threads;
  bool ok;
};
// NV candidates: 1..4 vectors, or 4 / 16 scalars.  The fewest idle vector slots win; ties go to the wider team
// (fewer registers).  Teams stop at 512 lanes.
inline Geometry geometry(int n_vec, bool scalar, int max_nv) {
  Geometry best{0, 0, 0, false};
  double best_cost = 1e30;
  for (int lpr = 2; lpr <= 512; lpr *= 2) {
    int nv = (n_vec + lpr - 1) / lpr;
    if (scalar) nv = nv <= 4 ? 4 : (nv <= 16 ? 16 : 1000);
    if (nv > (scalar ? 16 : max_nv)) continue;
    const double cost = (double)lpr * nv / n_vec;
    if (cost <= best_cost * 1.0001) { best_cost = cost; best = Geometry{lpr, nv, lpr > 32 ? lpr : 256, true}; }
  }
  return best;
}

// CTAs of a launch over `rows` rows: what the rows fill, at most `per_sm` per SM.
inline int grid_for(int rows, const Geometry& g, int per_sm) {
  const int rows_per_cta = g.lpr > 32 ? 1 : g.threads / g.lpr;
  const long long need = ((long long)rows + rows_per_cta - 1) / rows_per_cta;
  const long long cap = (long long)kSms * per_sm;
  return (int)(need < cap ? (need < 1 ? 1 : need) : cap);
}

template <typename T> struct FullVec { static constexpr int n = 16 / (int)sizeof(T); };

template <typename TX, typename TY, int VEC, int NV>
cudaError_t fwd_nv(int mode, int act, const LnTrainArgs& a, int grid, int threads, cudaStream_t s) {
  const dim3 g((unsigned)grid), t((unsigned)threads);
  if (mode == kPost) return launch_overlapped(ln_train_fwd_kernel<TX, TY, VEC, NV, kPost, false>, g, t, 0, s, a);
  if (mode == kPre) return launch_overlapped(ln_train_fwd_kernel<TX, TY, VEC, NV, kPre, false>, g, t, 0, s, a);
  if (act) return launch_overlapped(ln_train_fwd_kernel<TX, TY, VEC, NV, kPlain, true>, g, t, 0, s, a);
  return launch_overlapped(ln_train_fwd_kernel<TX, TY, VEC, NV, kPlain, false>, g, t, 0, s, a);
}
template <typename TX, typename TY, int VEC, int NV>
cudaError_t bwd_nv(int mode, int act, const LnTrainArgs& a, int grid, int threads, cudaStream_t s) {
  const dim3 g((unsigned)grid), t((unsigned)threads);
  const size_t smem = a.lpr > 32 ? 0 : (size_t)2 * a.C * sizeof(float);
  if (mode == kPre) return launch_overlapped(ln_train_bwd_kernel<TY, TY, TX, TX, VEC, NV, kPre, false>, g, t, smem, s, a);
  if (mode == kPost) return launch_overlapped(ln_train_bwd_kernel<TX, TY, TX, TX, VEC, NV, kPost, false>, g, t, smem, s, a);
  if (act) return launch_overlapped(ln_train_bwd_kernel<TX, TY, TX, TX, VEC, NV, kPlain, true>, g, t, smem, s, a);
  return launch_overlapped(ln_train_bwd_kernel<TX, TY, TX, TX, VEC, NV, kPlain, false>, g, t, smem, s, a);
}

// CTAs per SM of the backward grid: enough rows in flight, few enough partial sums.
constexpr int kFwdPerSm = 8, kBwdPerSm = 2;

template <typename TX, typename TY>
cudaError_t run(bool backward, int mode, int act, bool vec_ok, const LnTrainArgs& a0, cudaStream_t s) {
  constexpr int V = FullVec<TX>::n;
  LnTrainArgs a = a0;
  const bool scalar = !vec_ok;
  const Geometry g = geometry(scalar ? a.C : a.C / V, scalar, V == 8 ? 3 : 4);
  if (!g.ok) return cudaErrorInvalidValue;
  a.lpr = g.lpr;
  const int grid = grid_for(a.rows, g, backward ? kBwdPerSm : kFwdPerSm);
  a.n_partial = grid;
#define LN_RUN(VV, NN) \
  return backward ? bwd_nv<TX, TY, VV, NN>(mode, act, a, grid, g.threads, s) : fwd_nv<TX, TY, VV, NN>(mode, act, a, grid, g.threads, s)
  if (scalar) {
    if (g.nv == 4) { LN_RUN(1, 4); }
    LN_RUN(1, 16);
  }
  switch (g.nv) {
    case 1: LN_RUN(V, 1);
    case 2: LN_RUN(V, 2);
    case 3: LN_RUN(V, 3);
    default:
      if constexpr (V == 4) { LN_RUN(V, 4); }
      return cudaErrorInvalidValue;
  }
#undef LN_RUN
}

}  // namespace ln
}  // namespace dcnb200
