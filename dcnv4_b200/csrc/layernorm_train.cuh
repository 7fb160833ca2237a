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
// The statistics of `pre` are those of the fp32 sum, of which a 16-bit h has lost bits: xh of the stored h with them would
// carry h's rounding into every gradient, and a row whose spread is small beside that rounding would get an xh of
// anything up to |h| 2^-9 / sqrt(eps).  So where h has 16 bits the backward pass reads residual and branch and forms the
// sum again, by the forward's own fma, hence bit for bit (one more 16-bit tensor read; an fp32 h is the sum itself).  A
// caller who has kept the 16-bit h alone gets the gradient at h as stored: the mean is h's own, and 1/sigma is the given
// one or what h's own spread allows, whichever is less.
//
// Their floor is memory: a few operations per element, each tensor read and written once.  Reached (forward + backward, us, inputs
// beyond L2; floor in brackets): 2048 x 4096 fp32, pre: 25.4 + 34.7 (20.4 + 25.5); 131072 x 160 bf16 -> fp32, plain: 24.7 + 34.7
// (19.2 + 25.5); 802816 x 32 fp16 with GELU: 33.1 + 46.4 (15.6 + 23.5); 200704 x 80 bf16, post: 23.4 + 28.4 (14.7 + 14.7).  In 16 bits
// no unit is full (issue slots 31-53 %, DRAM 9-34 %): three to six warps a scheduler wait for results of their own.  Rows are contiguous,
// so a tile of rows is one span per tensor, and a ring of such tiles is kept in flight with bulk copies (cp.async.bulk,
// mbarriers, bounded waits) while the CTA's 12 or 16 warps compute: the bytes in flight do not depend on how many
// registers a row takes.  A span only has to start on 16 bytes, so rows of any width use the ring; with a width that no
// vector divides, teams keep to rows that start at the same distance from a vector boundary.
//
// A row belongs to a team of `lpr` lanes: 2..32 lanes of a warp, or 2..16 whole warps.  A lane keeps its
// NV vectors of the row, its slice of the parameters and of A and B in registers; statistics and sums are fp32, two
// passes over registers (mean, then squared deviations), two elements per instruction (fma.rn.f32x2).  Nothing is
// accumulated with atomics: the order of every sum is fixed by the sizes alone, so results repeat bit for bit.
//
// Tensors that do not start on 16 bytes (a view into the middle of another), and odd rows too wide for the ring, take
// the element-wise kernels at the end, which load straight from global memory.
//
// The reference builds these norms from torch.nn.LayerNorm, layer-scale products, timm's DropPath and residual
// additions (classification/models/flash_intern_image.py:34-56, 414-432); it has no kernel for them.
#pragma once

#include "common.cuh"

namespace dcnb200 {

struct LnTrainArgs {
  const void* x;         // branch input (plain, post: the normalised tensor); backward of pre: with res, to form the sum again
  const void* res;       // residual (post, pre; backward: pre with a 16-bit sum, or null)
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
  int lpr;               // lanes of a team
  int param_f32;         // parameters are fp32 (else: the type TP of the instantiation)
  unsigned rows_per_sample;
  unsigned long long per_mul;  // row / rows_per_sample == (row * per_mul) >> per_shift for row < 2^31
  int per_shift;
  int n_partial;
  float eps;
  int* status;           // device status word
  int tile_rows, stages; // ring: rows of a tile, tiles in flight
};

__device__ __forceinline__ unsigned sample_of(const LnTrainArgs& a, unsigned row) {
  return (unsigned)((row * a.per_mul) >> a.per_shift);
}

namespace ln {

constexpr int kMaxChannels = 8192;
constexpr int kSms = 148;              // B200: fixes the grid, hence the order of sums and the workspace size

// One element, or 0 where there is none; the word is widened when it is used, so that a row's loads go out together.
template <typename T>
__device__ __forceinline__ uint32_t load(const T* p, bool ok) {
  if constexpr (sizeof(T) == 4) return ok ? __float_as_uint(__ldg((const float*)p)) : 0u;
  else return ok ? (uint32_t)__ldg((const unsigned short*)p) : 0u;
}
template <typename T>
__device__ __forceinline__ float as_float(uint32_t r) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r);
  else { const unsigned short u = (unsigned short)r; return to_f32(*reinterpret_cast<const T*>(&u)); }
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

// ------------------------------------------------------------------------------ arithmetic

// Pairs of fp32: one instruction for two elements (sm_100).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Normal distribution function and density of two values, each from one exponential: Phi by formula 7.1.26 of Abramowitz
// and Stegun (erf to 1.5e-7), the density is that formula's own exp(-z^2 / 2) / sqrt(2 pi).  With the approximate
// exponential and reciprocal z Phi(z) is off by at most 2.5e-7 |z| (measured over [-8, 8]; erff gives 1.0e-7 |z|): fewer bits
// than fp32 has, of which a 16-bit result shows nothing.
__device__ __forceinline__ void normal(float2 z, float2& cdf, float2& density) {
  const float2 x = mul2(make_float2(fabsf(z.x), fabsf(z.y)), both(kSqrtHalf));
  const float2 y = mul2(mul2(x, x), both(-1.4426950408889634f));
  float2 e, t = fma2(x, both(0.3275911f), both(1.f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(y.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(y.y));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(t.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(t.y));
  float2 q = fma2(both(1.061405429f), t, both(-1.453152027f));
  q = fma2(q, t, both(1.421413741f));
  q = fma2(q, t, both(-0.284496736f));
  q = fma2(q, t, both(0.254829592f));
  // erf|x| = 1 - q t e, hence Phi = 1/2 + sign(z) (1/2 - q t e / 2)
  const float2 half = fma2(mul2(mul2(q, t), e), both(-0.5f), both(0.5f));
  cdf = add2(make_float2(copysignf(half.x, z.x), copysignf(half.y, z.y)), both(0.5f));
  density = mul2(e, both(kInvSqrt2Pi));
}

// ------------------------------------------------------------------------------ the ring of row tiles

constexpr int kMaxStages = 8;
constexpr int kRingHeader = 512;    // barriers, abort flag, team sums
struct RingHeader {
  uint64_t full[kMaxStages], empty[kMaxStages];
  int abort;
  int pad;
  float2 red[2][16];
};
static_assert(sizeof(RingHeader) <= kRingHeader, "ring header");

// Warps of a CTA: as many as the registers of NE elements a lane leave room for.  Parameters live in registers up to
// 16 elements, beyond that in shared memory.
constexpr int warps_for(int ne) { return ne <= 16 ? 16 : 12; }
// CTAs per SM of the forward kernels: where parameters are in shared memory two fit (200704 x 80 bf16, post-norm: 21.4
// against 23.5 us with one; 131072 x 160 bf16 to fp32: 26.5 against 28.6), elsewhere the registers would spill (2048 x 4096
// fp32: 33 against 23 us).
constexpr int fwd_ctas(int ne) { return ne > 16 ? 2 : 1; }
template <int NE> constexpr int ring_warps() { return warps_for(NE); }
template <int VEC, int NV> constexpr bool params_in_smem() { return VEC * NV > 16 || (VEC == 1 && NV > 8); }

__device__ __forceinline__ void ring_wait(uint64_t* bar, uint32_t parity, RingHeader* h, int* status) {
  if (*(volatile int*)&h->abort) return;
  if (!mbar_wait_bounded(bar, parity)) { atomicExch(status, kStatusStageTimeout); *(volatile int*)&h->abort = 1; }
}
// One thread; the other threads see the barriers after the CTA's first __syncthreads.
__device__ __forceinline__ void ring_init(RingHeader* h, int stages, int warps) {
  for (int s = 0; s < stages; ++s) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&h->full[s])) : "memory");
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&h->empty[s])), "r"(warps) : "memory");
  }
  h->abort = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void ring_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One tensor's span of a tile: whole 16-byte units by bulk copy, the last tile's remainder by plain stores, which the
// arrival that follows makes visible.  Returns the bytes the barrier has to expect.
__device__ __forceinline__ uint32_t span_bytes(int n, int C, int es) { return (uint32_t)n * (uint32_t)C * (uint32_t)es; }
template <typename T>
__device__ __forceinline__ void span_tail(unsigned char* dst, const T* src, uint32_t bytes) {
  for (uint32_t i = (bytes & ~15u) / sizeof(T); i < bytes / sizeof(T); ++i) reinterpret_cast<T*>(dst)[i] = src[i];
}

// Fills the ring.  One lane of the first warp asks for a tile of up to four tensors; it refills a slot when it starts the
// tile after the one the slot held, so it waits for the slowest warp of that tile and no warp does nothing else.
template <typename T0, typename T1, typename T2, typename T3 = T2>
struct RingFill {
  const T0* p0; const T1* p1; const T2* p2; const T3* p3;
  unsigned char* ring;
  RingHeader* h;
  int tiles;

  __device__ __forceinline__ uint32_t slot0(const LnTrainArgs& a) const { return span_bytes(a.tile_rows, a.C, sizeof(T0)); }
  __device__ __forceinline__ uint32_t slot1(const LnTrainArgs& a) const { return p1 ? span_bytes(a.tile_rows, a.C, sizeof(T1)) : 0; }
  __device__ __forceinline__ uint32_t slot2(const LnTrainArgs& a) const { return p2 ? span_bytes(a.tile_rows, a.C, sizeof(T2)) : 0; }
  __device__ __forceinline__ uint32_t slot3(const LnTrainArgs& a) const { return p3 ? span_bytes(a.tile_rows, a.C, sizeof(T3)) : 0; }

  // tile `t` into slot `stage`, which is free
  __device__ void issue(const LnTrainArgs& a, int t, int stage) const {
    const uint32_t z0 = slot0(a), z1 = slot1(a), z2 = slot2(a);
    const long long row0 = (long long)t * a.tile_rows;
    const int n = (int)(a.rows - row0 < a.tile_rows ? a.rows - row0 : a.tile_rows);
    const uint32_t b0 = span_bytes(n, a.C, sizeof(T0)), b1 = p1 ? span_bytes(n, a.C, sizeof(T1)) : 0;
    const uint32_t b2 = p2 ? span_bytes(n, a.C, sizeof(T2)) : 0, b3 = p3 ? span_bytes(n, a.C, sizeof(T3)) : 0;
    unsigned char* d = ring + (size_t)stage * (z0 + z1 + z2 + slot3(a));
    const T0* s0 = p0 + row0 * a.C;
    const T1* s1 = p1 ? p1 + row0 * a.C : nullptr;
    const T2* s2 = p2 ? p2 + row0 * a.C : nullptr;
    const T3* s3 = p3 ? p3 + row0 * a.C : nullptr;
    span_tail(d, s0, b0);
    if (p1) span_tail(d + z0, s1, b1);
    if (p2) span_tail(d + z0 + z1, s2, b2);
    if (p3) span_tail(d + z0 + z1 + z2, s3, b3);
    mbar_expect_tx(&h->full[stage], (b0 & ~15u) + (b1 & ~15u) + (b2 & ~15u) + (b3 & ~15u));
    if (b0 & ~15u) bulk_g2s(d, s0, b0 & ~15u, &h->full[stage]);
    if (b1 & ~15u) bulk_g2s(d + z0, s1, b1 & ~15u, &h->full[stage]);
    if (b2 & ~15u) bulk_g2s(d + z0 + z1, s2, b2 & ~15u, &h->full[stage]);
    if (b3 & ~15u) bulk_g2s(d + z0 + z1 + z2, s3, b3 & ~15u, &h->full[stage]);
  }
  __device__ void start(const LnTrainArgs& a) const {
    for (int s = 0; s < a.stages; ++s) {
      const long long t = blockIdx.x + (long long)s * gridDim.x;
      if (t < tiles) issue(a, (int)t, s);
    }
  }
  // before this CTA's tile `t` (its k-th, k > 0): the slot of the tile before gets the tile `stages` further on
  __device__ void refill(const LnTrainArgs& a, int t, int stage, uint32_t phase) const {
    const long long next = (long long)t + (long long)(a.stages - 1) * gridDim.x;
    if (next >= tiles) return;
    const int prev = stage == 0 ? a.stages - 1 : stage - 1;
    ring_wait(&h->empty[prev], stage == 0 ? phase ^ 1 : phase, h, a.status);
    if (!*(volatile int*)&h->abort) issue(a, (int)next, prev);
  }
};

// Widths that no vector divides.  Row r then starts r * C mod VEC elements behind a vector boundary, a pattern that repeats
// after VEC / gcd(C, VEC) rows.  A team that takes rows of one residue only meets one shift: it reads and writes whole
// vectors on the boundaries, its lanes own columns k * VEC + e - shift, and only the first and the last vector of a row
// hold elements of the neighbouring rows, which are masked.
// Word i of a vector whose elements [lo, hi) belong to the row.
template <typename T>
__device__ __forceinline__ uint32_t word_mask(int i, int lo, int hi) {
  if constexpr (sizeof(T) == 4) return i >= lo && i < hi ? 0xffffffffu : 0u;
  else return (2 * i >= lo && 2 * i < hi ? 0x0000ffffu : 0u) | (2 * i + 1 >= lo && 2 * i + 1 < hi ? 0xffff0000u : 0u);
}

// A lane's elements of a row in shared memory, as pairs.  VEC > 1: vectors sub, sub + lpr, ... of VEC elements, of which
// only the last can lie beyond C (NV is the least that covers a row; with a shift, the last two, and the first is
// partial); VEC == 1: elements sub, sub + lpr, ...
template <typename T, int VEC, int NV, bool SHIFT = false>
__device__ __forceinline__ void row_load(float2 (&f)[NV * VEC / 2], const T* row, int sub, int lpr, int C, bool live,
                                         int shift = 0) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int v = 0; v < NV; v += 2) {
      const int c0 = sub + v * lpr, c1 = c0 + lpr;
      f[v / 2].x = live && c0 < C ? to_f32(row[c0]) : 0.f;
      f[v / 2].y = live && c1 < C ? to_f32(row[c1]) : 0.f;
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (sub + v * lpr) * VEC - (SHIFT ? shift : 0);
      const bool edge = SHIFT && (v == 0 || v + 2 >= NV);
      constexpr int W = VEC * (int)sizeof(T) / 4;
      const bool in = live && ((v + 1 < NV && !edge) || c < C);
      uint32_t r[W];
      if constexpr (W == 2) {
        uint2 t = make_uint2(0u, 0u);
        if (in) t = *reinterpret_cast<const uint2*>(row + c);
        r[0] = t.x; r[1] = t.y;
      }
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        uint4 t = make_uint4(0u, 0u, 0u, 0u);
        if (in) t = reinterpret_cast<const uint4*>(row + c)[i];
        r[4 * i] = t.x; r[4 * i + 1] = t.y; r[4 * i + 2] = t.z; r[4 * i + 3] = t.w;
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < W; ++i) r[i] &= word_mask<T>(i, -c, C - c);
      }
      float w[VEC];
      widen(r, w, (const T*)nullptr);
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) f[v * VEC / 2 + e] = make_float2(w[2 * e], w[2 * e + 1]);
    }
  }
}
// The same from global memory (parameters).
template <typename T, int VEC, int NV>
__device__ __forceinline__ void row_fetch(float2 (&f)[NV * VEC / 2], const T* row, int sub, int lpr, int C) {
  row_load<T, VEC, NV>(f, row, sub, lpr, C, true);
}
template <typename T, int VEC, int NV, bool SHIFT = false>
__device__ __forceinline__ void row_store(T* row, const float2 (&f)[NV * VEC / 2], int sub, int lpr, int C, int shift = 0) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int v = 0; v < NV; v += 2) {
      const int c0 = sub + v * lpr, c1 = c0 + lpr;
      if (c0 < C) row[c0] = from_f32<T>(f[v / 2].x);
      if (c1 < C) row[c1] = from_f32<T>(f[v / 2].y);
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (sub + v * lpr) * VEC - (SHIFT ? shift : 0);
      const bool edge = SHIFT && (v == 0 || v + 2 >= NV);
      float w[VEC];
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) { w[2 * e] = f[v * VEC / 2 + e].x; w[2 * e + 1] = f[v * VEC / 2 + e].y; }
      if (edge ? c >= 0 && c + VEC <= C : v + 1 < NV || c < C) {
        uint32_t r[VEC * sizeof(T) / 4];
        narrow(w, r, (const T*)nullptr);
        stg_raw(row + c, r);   // 8 or 16 bytes in one instruction
      } else if (edge) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (c + e >= 0 && c + e < C) row[c + e] = from_f32<T>(w[e]);
      }
    }
  }
}
// Parameter slice in the same order; zero outside the row.
template <typename P, int VEC, int NV>
__device__ __forceinline__ void param_load(float2 (&f)[NV * VEC / 2], const void* p, int sub, int lpr, int C, int f32,
                                           int shift = 0) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = (sub + v * lpr) * VEC + e - shift, i = v * VEC + e;
      const float t = c >= 0 && c < C ? param<P>(p, c, f32) : 0.f;
      if (i & 1) f[i / 2].y = t;
      else f[i / 2].x = t;
    }
}
// 16-byte loads where the parameters allow it: a launch's first rows wait for these.
template <typename P, int VEC, int NV, bool SHIFT>
__device__ __forceinline__ void param_fetch(float2 (&f)[NV * VEC / 2], const void* p, int sub, int lpr, int C, int f32,
                                            int shift) {
  if constexpr (VEC > 1 && !SHIFT) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      if (f32) { row_fetch<float, VEC, NV>(f, static_cast<const float*>(p), sub, lpr, C); return; }
      if constexpr (sizeof(P) == 2) { row_fetch<P, VEC, NV>(f, static_cast<const P*>(p), sub, lpr, C); return; }
    }
  }
  param_load<P, VEC, NV>(f, p, sub, lpr, C, f32, shift);
}
// One fp32 parameter vector in shared memory, filled by the whole CTA.  For vectors of 8 their halves lie in two arrays, so
// that the 16-byte loads of neighbouring lanes are neighbours (interleaved, they would meet in the same banks).
template <int VEC>
__device__ __forceinline__ int staged_at(int c, int C) {
  return VEC == 8 ? (c & 4) / 4 * (C / 2) + c / 8 * 4 + (c & 3) : c;
}
template <typename P, int VEC>
__device__ __forceinline__ void param_stage(float* dst, const void* p, const void* factor, int C, int f32) {
  for (int c = threadIdx.x; c < C; c += blockDim.x)
    dst[staged_at<VEC>(c, C)] = param<P>(p, c, f32) * (factor != nullptr ? param<P>(factor, c, f32) : 1.f);
}
template <int VEC, int NV>
__device__ __forceinline__ void param_row(float2 (&f)[NV * VEC / 2], const float* p, int sub, int lpr, int C) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int k = sub + v * lpr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
        if (v + 1 < NV || k * 8 < C) t = reinterpret_cast<const float4*>(p + h * (C / 2))[k];
        f[v * 4 + 2 * h] = make_float2(t.x, t.y);
        f[v * 4 + 2 * h + 1] = make_float2(t.z, t.w);
      }
    }
  } else {
    row_load<float, VEC, NV>(f, p, sub, lpr, C, true);
  }
}
// Parameter gradients of one column from its sums.
template <typename P>
__device__ __forceinline__ void finish_column(const LnTrainArgs& a, bool post, int c, float sa, float sb) {
  auto put = [&](void* dst, float v) {
    if (a.param_f32) static_cast<float*>(dst)[c] = v;
    else static_cast<P*>(dst)[c] = from_f32<P>(v);
  };
  if (post && a.gamma != nullptr) {
    const float g = param<P>(a.gamma, c, a.param_f32);
    put(a.dgamma, fmaf(param<P>(a.w, c, a.param_f32), sa, param<P>(a.b, c, a.param_f32) * sb));
    put(a.dw, g * sa);
    put(a.db, g * sb);
  } else {
    put(a.dw, sa);
    put(a.db, sb);
  }
}
// Column of a lane's element i.
template <int VEC> __device__ __forceinline__ int column(int i, int sub, int lpr) { return (sub + i / VEC * lpr) * VEC + i % VEC; }

// Sum of two values over the team.  The warps of a wider team meet at a named barrier of their own, one per call (the
// slots alternate, so the next call cannot overwrite what a slow warp still reads).
__device__ __forceinline__ float2 ring_sum(float2 t, int lpr, RingHeader* h, int& flip) {
#pragma unroll 1
  for (int o = lpr > 32 ? 16 : lpr >> 1; o > 0; o >>= 1) {
    const float2 u = make_float2(__shfl_xor_sync(0xffffffffu, t.x, o), __shfl_xor_sync(0xffffffffu, t.y, o));
    t = add2(t, u);
  }
  if (lpr > 32) {
    float2* slot = h->red[flip];
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = t;
    const int team = threadIdx.x / lpr;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(lpr) : "memory");
    t = make_float2(0.f, 0.f);
    for (int i = 0; i < (lpr >> 5); ++i) t = add2(t, slot[team * (lpr >> 5) + i]);
  }
  return t;
}

__device__ __forceinline__ float ring_sum(float t, int lpr, RingHeader* h, int& flip) {
#pragma unroll 1
  for (int o = lpr > 32 ? 16 : lpr >> 1; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lpr > 32) {
    float2* slot = h->red[flip];
    flip ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5].x = t;
    const int team = threadIdx.x / lpr;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(lpr) : "memory");
    t = 0.f;
    for (int i = 0; i < (lpr >> 5); ++i) t += slot[team * (lpr >> 5) + i].x;
  }
  return t;
}

// Sum of a lane's elements.  Two chains of additions, here and below: a warp's own latency is what short rows wait for.
template <int N>
__device__ __forceinline__ float lane_sum(const float2 (&x)[N]) {
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i & 1] = add2(sum[i & 1], x[i]);
  sum[0] = add2(sum[0], sum[1]);
  return sum[0].x + sum[0].y;
}
// Takes the mean off a lane's elements; returns the sum of the squares of those that belong to the row.
template <int VEC, int NV, bool SHIFT>
__device__ __forceinline__ float lane_centre(float2 (&x)[NV * VEC / 2], float mean, int sub, int lpr, int C, int shift) {
  float2 sq[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) {
    x[i] = add2(x[i], both(-mean));
    if (VEC > 1 && (SHIFT ? 2 * i / VEC != 0 && 2 * i / VEC + 2 < NV : 2 * i / VEC + 1 < NV)) {
      sq[i & 1] = fma2(x[i], x[i], sq[i & 1]);
    } else if (VEC > 1 && !SHIFT) {
      if (column<VEC>(2 * i, sub, lpr) < C) sq[i & 1] = fma2(x[i], x[i], sq[i & 1]);
    } else {      // the elements of a pair may differ in whether they belong to the row
      const int c0 = column<VEC>(2 * i, sub, lpr) - shift, c1 = column<VEC>(2 * i + 1, sub, lpr) - shift;
      if (c0 >= 0 && c0 < C) sq[i & 1].x = fmaf(x[i].x, x[i].x, sq[i & 1].x);
      if (c1 >= 0 && c1 < C) sq[i & 1].y = fmaf(x[i].y, x[i].y, sq[i & 1].y);
    }
  }
  sq[0] = add2(sq[0], sq[1]);
  return sq[0].x + sq[0].y;
}

template <typename TX, typename TY, int VEC, int NV, bool SHIFT, int MODE, bool GELU>
__global__ void __launch_bounds__(32 * ring_warps<VEC * NV>(), fwd_ctas(VEC * NV))
ln_ring_fwd_kernel(const LnTrainArgs a) {
  using P = TX;
  constexpr int NE = VEC * NV, W = ring_warps<NE>();
  extern __shared__ __align__(128) unsigned char smem[];
  RingHeader* h = reinterpret_cast<RingHeader*>(smem);
  unsigned char* ring = smem + kRingHeader;
  const int lpr = a.lpr, C = a.C, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (a.rows + a.tile_rows - 1) / a.tile_rows;
  const RingFill<TX, TY, TY> fill{static_cast<const TX*>(a.x), MODE == kPlain ? nullptr : static_cast<const TY*>(a.res), nullptr,
                                  nullptr, ring, h, tiles};
  // the first thread sets up and fills the ring while the others fetch the parameters
  if (threadIdx.x == 0) ring_init(h, a.stages, W);
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) fill.start(a);
  {
    const int sub = (int)threadIdx.x % lpr, team = (int)threadIdx.x / lpr;
    const int per_pass = W * 32 / lpr;                     // rows of one pass of the CTA
    const int first = lpr > 32 ? team : warp * (32 / lpr);  // first row of this warp in a pass
    const int shift = SHIFT ? (int)((unsigned)team * (unsigned)C % VEC) : 0;
    const int passes = (a.tile_rows + per_pass - 1) / per_pass;
    const float inv_c = 1.f / (float)C;
    const uint32_t slot0 = fill.slot0(a), slot = slot0 + fill.slot1(a);
    int flip = 0;
    constexpr bool kStaged = params_in_smem<VEC, NV>();
    float2 w[NE / 2], b[NE / 2];
    float* ws = reinterpret_cast<float*>(ring + (size_t)a.stages * slot);
    float* bs = ws + (C + 3) / 4 * 4;
    if constexpr (kStaged) {
      const void* g = MODE == kPost ? a.gamma : nullptr;
      param_stage<P, VEC>(ws, a.w, g, C, a.param_f32);
      param_stage<P, VEC>(bs, a.b, g, C, a.param_f32);
    } else {
      param_fetch<P, VEC, NV, SHIFT>(w, a.w, sub, lpr, C, a.param_f32, shift);
      param_fetch<P, VEC, NV, SHIFT>(b, a.b, sub, lpr, C, a.param_f32, shift);
      if (MODE == kPost && a.gamma != nullptr) {
        float2 g[NE / 2];
        param_fetch<P, VEC, NV, SHIFT>(g, a.gamma, sub, lpr, C, a.param_f32, shift);
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) { w[i] = mul2(w[i], g[i]); b[i] = mul2(b[i], g[i]); }
      }
    }
    __syncthreads();
    const bool scaled = MODE != kPlain && a.s != nullptr;
    auto factor = [&](int t, int pass) {        // s of this team's row, asked for one pass ahead
      const int lr = pass * per_pass + team;
      const long long row = (long long)t * a.tile_rows + lr;
      return t < tiles && lr < a.tile_rows && row < a.rows ? __ldg(a.s + sample_of(a, (unsigned)row)) : 0.f;
    };
    float s = 1.f, s_next = scaled ? factor(blockIdx.x, 0) : 1.f;
    int stage = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      if (threadIdx.x == 0 && t != (int)blockIdx.x) fill.refill(a, t, stage, phase);
      __syncwarp();
      ring_wait(&h->full[stage], phase, h, a.status);
      const unsigned char* base = ring + (size_t)stage * slot;
      const int row0 = t * a.tile_rows;
      const int n = a.rows - row0 < a.tile_rows ? a.rows - row0 : a.tile_rows;
      for (int pass = 0; pass < passes; ++pass) {
        if (scaled) {
          s = s_next;
          s_next = pass + 1 < passes ? factor(t, pass + 1) : factor(t + gridDim.x, 0);
        }
        const int lr = pass * per_pass + team;
        if (pass * per_pass + first >= n) continue;        // no row of this warp's
        const bool live = lr < n;
        const int row = row0 + lr;
        float2 x[NE / 2], r[MODE == kPlain ? 1 : NE / 2];
        row_load<TX, VEC, NV, SHIFT>(x, reinterpret_cast<const TX*>(base) + (size_t)lr * C, sub, lpr, C, live, shift);
        if constexpr (MODE != kPlain) row_load<TY, VEC, NV, SHIFT>(r, reinterpret_cast<const TY*>(base + slot0) + (size_t)lr * C, sub, lpr, C, live, shift);
        if constexpr (MODE == kPre) {
#pragma unroll
          for (int i = 0; i < NE / 2; ++i) x[i] = fma2(both(s), x[i], r[i]);
          if (live) row_store<TY, VEC, NV, SHIFT>(static_cast<TY*>(a.h) + (long long)row * C, x, sub, lpr, C, shift);
        }
        const float mean = ring_sum(lane_sum(x), lpr, h, flip) * inv_c;
        const float rstd = rsqrtf(ring_sum(lane_centre<VEC, NV, SHIFT>(x, mean, sub, lpr, C, shift), lpr, h, flip) * inv_c + a.eps);
        if (!live) continue;
        if constexpr (kStaged) {
          param_row<VEC, NV>(w, ws, sub, lpr, C);
          param_row<VEC, NV>(b, bs, sub, lpr, C);
        }
        if (sub == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) {
          float2 o = fma2(mul2(x[i], both(rstd)), w[i], b[i]);
          if (GELU) {
            float2 cdf, density;
            normal(o, cdf, density);
            o = mul2(o, cdf);
          }
          if constexpr (MODE == kPost) o = fma2(both(s), o, r[i]);
          x[i] = o;
        }
        row_store<TY, VEC, NV, SHIFT>(static_cast<TY*>(a.y) + (long long)row * C, x, sub, lpr, C, shift);
      }
      __syncwarp();
      if (lane == 0) ring_arrive(&h->empty[stage]);
      if (++stage == a.stages) { stage = 0; phase ^= 1; }
    }
  }
  if (*(volatile int*)&h->abort)       // copies into this CTA's memory may be in flight: give them 20 ms to land
    for (int i = 0; i < 20000; ++i) __nanosleep(1000);
}

template <typename TL, typename TG, typename T2, typename P, int VEC, int NV, bool SHIFT, int MODE, bool GELU>
__global__ void __launch_bounds__(32 * ring_warps<VEC * NV>(), 1)
ln_ring_bwd_kernel(const LnTrainArgs a) {
  constexpr int NE = VEC * NV, W = ring_warps<NE>();
  extern __shared__ __align__(128) unsigned char smem[];
  RingHeader* h = reinterpret_cast<RingHeader*>(smem);
  unsigned char* ring = smem + kRingHeader;
  const int lpr = a.lpr, C = a.C, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (a.rows + a.tile_rows - 1) / a.tile_rows;
  const bool with_gh = MODE == kPre && a.gh != nullptr;
  constexpr bool kNarrow = MODE == kPre && sizeof(TL) == 2;   // h has lost bits of the sum that was normalised
  const bool summed = kNarrow && a.res != nullptr;            // x is the branch, and the sum is formed again
  const int sub = (int)threadIdx.x % lpr, team = (int)threadIdx.x / lpr;
  const int shift = SHIFT ? (int)((unsigned)team * (unsigned)C % VEC) : 0;
  float2 sa[NE / 2], sb[NE / 2];
#pragma unroll
  for (int i = 0; i < NE / 2; ++i) sa[i] = sb[i] = make_float2(0.f, 0.f);
  const RingFill<TL, TG, TG, TL> fill{static_cast<const TL*>(MODE == kPre && !summed ? a.h : a.x), static_cast<const TG*>(a.gy),
                                      with_gh ? static_cast<const TG*>(a.gh) : nullptr,
                                      kNarrow ? static_cast<const TL*>(a.res) : nullptr, ring, h, tiles};
  if (threadIdx.x == 0) ring_init(h, a.stages, W);
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) fill.start(a);
  {
    const int per_pass = W * 32 / lpr;
    const int first = lpr > 32 ? team : warp * (32 / lpr);
    const int passes = (a.tile_rows + per_pass - 1) / per_pass;
    const float inv_c = 1.f / (float)C;
    const uint32_t slot0 = fill.slot0(a), slot1 = fill.slot1(a), slot2 = fill.slot2(a), slot = slot0 + slot1 + slot2 + fill.slot3(a);
    int flip = 0;
    constexpr bool kStaged = params_in_smem<VEC, NV>();
    float2 w[NE / 2], b[GELU ? NE / 2 : 1];
    float* ws = reinterpret_cast<float*>(ring + (size_t)a.stages * slot);
    float* bs = ws + (C + 3) / 4 * 4;
    if constexpr (kStaged) {
      param_stage<P, VEC>(ws, a.w, MODE == kPost ? a.gamma : nullptr, C, a.param_f32);
      if constexpr (GELU) param_stage<P, VEC>(bs, a.b, nullptr, C, a.param_f32);
    } else {
      param_fetch<P, VEC, NV, SHIFT>(w, a.w, sub, lpr, C, a.param_f32, shift);
      if constexpr (GELU) param_fetch<P, VEC, NV, SHIFT>(b, a.b, sub, lpr, C, a.param_f32, shift);
      if (MODE == kPost && a.gamma != nullptr) {
        float2 g[NE / 2];
        param_fetch<P, VEC, NV, SHIFT>(g, a.gamma, sub, lpr, C, a.param_f32, shift);
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) w[i] = mul2(w[i], g[i]);
      }
    }
    __syncthreads();
    const bool scaled = MODE != kPlain && a.s != nullptr;
    // statistics and factor of this team's row, asked for one pass ahead
    auto stats = [&](int t, int pass, float& mean, float& rstd, float& s) {
      const int lr = pass * per_pass + team;
      const long long row = (long long)t * a.tile_rows + lr;
      const bool ok = t < tiles && lr < a.tile_rows && row < a.rows;
      mean = ok ? __ldg(a.mean + row) : 0.f;
      rstd = ok ? __ldg(a.rstd + row) : 0.f;
      if (scaled) s = ok ? __ldg(a.s + sample_of(a, (unsigned)row)) : 0.f;
    };
    float mean_n, rstd_n, s_n = 1.f;
    stats(blockIdx.x, 0, mean_n, rstd_n, s_n);
    int stage = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      if (threadIdx.x == 0 && t != (int)blockIdx.x) fill.refill(a, t, stage, phase);
      __syncwarp();
      ring_wait(&h->full[stage], phase, h, a.status);
      const unsigned char* base = ring + (size_t)stage * slot;
      const int row0 = t * a.tile_rows;
      const int n = a.rows - row0 < a.tile_rows ? a.rows - row0 : a.tile_rows;
      for (int pass = 0; pass < passes; ++pass) {
        float mean = mean_n, rstd = rstd_n;
        const float s = s_n;
        if (pass + 1 < passes) stats(t, pass + 1, mean_n, rstd_n, s_n);
        else stats(t + gridDim.x, 0, mean_n, rstd_n, s_n);
        const int lr = pass * per_pass + team;
        if (pass * per_pass + first >= n) continue;
        const bool live = lr < n;
        const int row = row0 + lr;
        float2 x[NE / 2], g[NE / 2];
        row_load<TL, VEC, NV, SHIFT>(x, reinterpret_cast<const TL*>(base) + (size_t)lr * C, sub, lpr, C, live, shift);
        if constexpr (kNarrow) {
          if (summed) {
            row_load<TL, VEC, NV, SHIFT>(g, reinterpret_cast<const TL*>(base + slot0 + slot1 + slot2) + (size_t)lr * C, sub, lpr, C, live, shift);
#pragma unroll
            for (int i = 0; i < NE / 2; ++i) x[i] = fma2(both(s), x[i], g[i]);
          } else {
            mean = ring_sum(lane_sum(x), lpr, h, flip) * inv_c;
            rstd = fminf(rstd, rsqrtf(ring_sum(lane_centre<VEC, NV, SHIFT>(x, mean, sub, lpr, C, shift), lpr, h, flip) * inv_c));
            mean = 0.f;
          }
        }
        row_load<TG, VEC, NV, SHIFT>(g, reinterpret_cast<const TG*>(base + slot0) + (size_t)lr * C, sub, lpr, C, live, shift);
        // elements beyond C have g = w = 0 and add nothing to any sum
        float2 t1[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, t2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if constexpr (kStaged) {
          param_row<VEC, NV>(w, ws, sub, lpr, C);
          if constexpr (GELU) param_row<VEC, NV>(b, bs, sub, lpr, C);
        }
        const float2 r2 = both(rstd), minus_mean = both(-mean);
#pragma unroll
        for (int i = 0; i < NE / 2; ++i) {
          x[i] = mul2(add2(x[i], minus_mean), r2);
          if (MODE == kPost) g[i] = mul2(g[i], both(s));
          if constexpr (GELU) {
            const float2 z = fma2(x[i], w[i], b[i]);
            float2 cdf, density;
            normal(z, cdf, density);
            g[i] = mul2(g[i], fma2(z, density, cdf));
          }
          sa[i] = fma2(g[i], x[i], sa[i]);
          sb[i] = add2(sb[i], g[i]);
          g[i] = mul2(g[i], w[i]);
          t1[i & 1] = add2(t1[i & 1], g[i]);
          t2[i & 1] = fma2(g[i], x[i], t2[i & 1]);
        }
        t1[0] = add2(t1[0], t1[1]);
        t2[0] = add2(t2[0], t2[1]);
        const float2 m = ring_sum(make_float2(t1[0].x + t1[0].y, t2[0].x + t2[0].y), lpr, h, flip);
        if (!live) continue;
        const float2 m1 = both(-m.x * inv_c * rstd), m2 = both(-m.y * inv_c * rstd);
        if constexpr (MODE == kPre) {
#pragma unroll
          for (int i = 0; i < NE / 2; ++i) x[i] = fma2(x[i], m2, fma2(g[i], r2, m1));
          if (with_gh) {
            row_load<TG, VEC, NV, SHIFT>(g, reinterpret_cast<const TG*>(base + slot0 + slot1) + (size_t)lr * C, sub, lpr, C, true, shift);
#pragma unroll
            for (int i = 0; i < NE / 2; ++i) x[i] = add2(x[i], g[i]);
          }
          row_store<TL, VEC, NV, SHIFT>(static_cast<TL*>(a.dx) + (long long)row * C, x, sub, lpr, C, shift);
          if (a.dx2 != nullptr) {
#pragma unroll
            for (int i = 0; i < NE / 2; ++i) x[i] = mul2(x[i], both(s));
            row_store<T2, VEC, NV, SHIFT>(static_cast<T2*>(a.dx2) + (long long)row * C, x, sub, lpr, C, shift);
          }
        } else {
#pragma unroll
          for (int i = 0; i < NE / 2; ++i) x[i] = fma2(x[i], m2, fma2(g[i], r2, m1));
          row_store<TL, VEC, NV, SHIFT>(static_cast<TL*>(a.dx) + (long long)row * C, x, sub, lpr, C, shift);
        }
      }
      __syncwarp();
      if (lane == 0) ring_arrive(&h->empty[stage]);
      if (++stage == a.stages) { stage = 0; phase ^= 1; }
    }
    // over the teams of each warp (which own the same columns, unless they are shifted)
    for (int o = SHIFT ? 32 : lpr; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < NE / 2; ++i) {
        sa[i].x += __shfl_xor_sync(0xffffffffu, sa[i].x, o);
        sa[i].y += __shfl_xor_sync(0xffffffffu, sa[i].y, o);
        sb[i].x += __shfl_xor_sync(0xffffffffu, sb[i].x, o);
        sb[i].y += __shfl_xor_sync(0xffffffffu, sb[i].y, o);
      }
    }
  }
  if (*(volatile int*)&h->abort)
    for (int i = 0; i < 20000; ++i) __nanosleep(1000);
  // over the warps, or the teams of several warps, through the ring's memory: every tile has been consumed
  __syncthreads();
  float* acc = reinterpret_cast<float*>(ring);     // [slots][2][C]
  const bool by_team = SHIFT || lpr > 32;
  const int slots = by_team ? W * 32 / lpr : W, slot = by_team ? team : warp;
  if (by_team || lane < lpr) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int c = column<VEC>(i, sub, lpr) - shift;
      if (c >= 0 && c < C) {
        acc[(slot * 2) * C + c] = i & 1 ? sa[i / 2].y : sa[i / 2].x;
        acc[(slot * 2 + 1) * C + c] = i & 1 ? sb[i / 2].y : sb[i / 2].x;
      }
    }
  }
  __syncthreads();
  if (gridDim.x == 1) {      // the only CTA: these are the sums over all rows
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      float ta = 0.f, tb = 0.f;
      for (int q = 0; q < slots; ++q) { ta += acc[q * 2 * C + c]; tb += acc[q * 2 * C + C + c]; }
      finish_column<P>(a, MODE == kPost, c, ta, tb);
    }
    return;
  }
  float* dst = a.partial + (size_t)blockIdx.x * 2 * C;
  for (int i = threadIdx.x; i < 2 * C; i += blockDim.x) {
    float t = 0.f;
    for (int q = 0; q < slots; ++q) t += acc[q * 2 * C + i];
    dst[i] = t;
  }
}

// ------------------------------------------------------------------------- element-wise kernels

template <typename TX, typename TY, int NV, int MODE, bool GELU>
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

  float w[NV], b[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = sub + v * lpr;
    const bool ok = c < C;
    w[v] = ok ? param<P>(a.w, c, a.param_f32) : 0.f;
    b[v] = ok ? param<P>(a.b, c, a.param_f32) : 0.f;
    if (MODE == kPost && a.gamma != nullptr) {
      const float g = ok ? param<P>(a.gamma, c, a.param_f32) : 0.f;
      w[v] *= g;
      b[v] *= g;
    }
  }
  // the lanes of a warp stay in the loop together: the team sums shuffle across it
  for (int r0 = wide ? team0 : team0 - (int)(threadIdx.x & 31) / lpr; r0 < a.rows; r0 += n_teams) {
    const int row = wide ? r0 : r0 + (int)(threadIdx.x & 31) / lpr;
    const bool live = row < a.rows;
    const long long base = (long long)row * C;
    uint32_t rx[NV], rr[MODE == kPlain ? 1 : NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = sub + v * lpr;
      rx[v] = load(static_cast<const TX*>(a.x) + base + c, live && c < C);
      if (MODE != kPlain) rr[v] = load(static_cast<const TY*>(a.res) + base + c, live && c < C);
    }
    float s = 1.f;
    if (MODE != kPlain && a.s != nullptr) s = live ? __ldg(a.s + sample_of(a, (unsigned)row)) : 0.f;
    float xv[NV];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = sub + v * lpr;
      xv[v] = as_float<TX>(rx[v]);
      if (MODE == kPre) {
        xv[v] = fmaf(s, xv[v], as_float<TY>(rr[v]));
        if (live && c < C) static_cast<TY*>(a.h)[base + c] = from_f32<TY>(xv[v]);
      }
      sum += xv[v];
    }
    const float mean = team_sum(sum, 0.f, lpr, red, flip).x * inv_c;
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (sub + v * lpr < C) { const float d = xv[v] - mean; sq = fmaf(d, d, sq); }
    const float rstd = rsqrtf(team_sum(sq, 0.f, lpr, red, flip).x * inv_c + a.eps);
    if (!live) continue;
    if (sub == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = sub + v * lpr;
      if (c >= C) continue;
      float o = fmaf((xv[v] - mean) * rstd, w[v], b[v]);
      if (GELU) { float2 cdf, density; normal(both(o), cdf, density); o *= cdf.x; }
      if (MODE == kPost) o = fmaf(s, o, as_float<TY>(rr[v]));
      static_cast<TY*>(a.y)[base + c] = from_f32<TY>(o);
    }
  }
}

// ----------------------------------------------------------------------------------- backward

// TL: type of the normalised tensor and of its gradient; TG: type of the incoming gradients; T2: type of the branch
// gradient of `pre`; P: parameter type when not fp32.
template <typename TL, typename TG, typename T2, typename P, int NV, int MODE, bool GELU>
__global__ void __launch_bounds__(512)
ln_train_bwd_kernel(const LnTrainArgs a) {
  __shared__ float2 red[2][16];
  extern __shared__ float acc_smem[];    // [2][C]
  const int lpr = a.lpr, C = a.C;
  const bool wide = lpr > 32;
  const int lane = threadIdx.x & 31;
  constexpr bool kNarrow = MODE == kPre && sizeof(TL) == 2;   // as in the ring kernel
  const bool summed = kNarrow && a.res != nullptr;
  const int sub = wide ? threadIdx.x : lane % lpr;
  const int team0 = wide ? blockIdx.x : (blockIdx.x * blockDim.x + threadIdx.x) / lpr;
  const int n_teams = wide ? gridDim.x : gridDim.x * blockDim.x / lpr;
  const float inv_c = 1.f / (float)C;
  int flip = 0;
  pdl_trigger();
  pdl_wait();

  float w[NV], b[GELU ? NV : 1], sa[NV], sb[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = sub + v * lpr;
    const bool ok = c < C;
    w[v] = ok ? param<P>(a.w, c, a.param_f32) : 0.f;
    if (GELU) b[v] = ok ? param<P>(a.b, c, a.param_f32) : 0.f;
    if (MODE == kPost && a.gamma != nullptr && ok) w[v] *= param<P>(a.gamma, c, a.param_f32);
    sa[v] = 0.f;
    sb[v] = 0.f;
  }
  for (int r0 = wide ? team0 : team0 - lane / lpr; r0 < a.rows; r0 += n_teams) {
    const int row = wide ? r0 : r0 + lane / lpr;
    const bool live = row < a.rows;
    const long long base = (long long)row * C;
    uint32_t rx[NV], rr[kNarrow ? NV : 1], rg[NV], rh[MODE == kPre ? NV : 1];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = sub + v * lpr;
      const bool ok = live && c < C;
      rx[v] = load(static_cast<const TL*>(MODE == kPre && !summed ? a.h : a.x) + base + c, ok);
      if (kNarrow) rr[v] = load(static_cast<const TL*>(a.res) + base + c, ok && summed);
      rg[v] = load(static_cast<const TG*>(a.gy) + base + c, ok);
      if (MODE == kPre) rh[v] = load(static_cast<const TG*>(a.gh) + base + c, ok && a.gh != nullptr);
    }
    float mean = live ? __ldg(a.mean + row) : 0.f, rstd = live ? __ldg(a.rstd + row) : 0.f;
    float s = 1.f;
    if (MODE != kPlain && a.s != nullptr) s = live ? __ldg(a.s + sample_of(a, (unsigned)row)) : 0.f;
    float xh[NV], gw[NV];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xh[v] = as_float<TL>(rx[v]);
      if (kNarrow && summed) xh[v] = fmaf(s, xh[v], as_float<TL>(rr[v]));
    }
    if (kNarrow && !summed) {
      float sum = 0.f, sq = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) sum += xh[v];
      mean = team_sum(sum, 0.f, lpr, red, flip).x * inv_c;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (sub + v * lpr < C) { const float d = xh[v] - mean; sq = fmaf(d, d, sq); }
      rstd = fminf(rstd, rsqrtf(team_sum(sq, 0.f, lpr, red, flip).x * inv_c));
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float g = as_float<TG>(rg[v]);
      xh[v] = live && sub + v * lpr < C ? (xh[v] - mean) * rstd : 0.f;
      if (MODE == kPost) g *= s;
      if (GELU) {
        const float z = fmaf(xh[v], w[v], b[v]);
        float2 cdf, density;
        normal(both(z), cdf, density);
        g *= fmaf(z, density.x, cdf.x);
      }
      sa[v] = fmaf(g, xh[v], sa[v]);
      sb[v] += g;
      gw[v] = g * w[v];
      s1 += gw[v];
      s2 = fmaf(gw[v], xh[v], s2);
    }
    const float2 t = team_sum(s1, s2, lpr, red, flip);
    const float m1 = t.x * inv_c, m2 = t.y * inv_c;
    if (!live) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = sub + v * lpr;
      if (c >= C) continue;
      float o = rstd * (gw[v] - fmaf(xh[v], m2, m1));
      if (MODE == kPre) o += as_float<TG>(rh[v]);
      static_cast<TL*>(a.dx)[base + c] = from_f32<TL>(o);
      if (MODE == kPre && a.dx2 != nullptr) static_cast<T2*>(a.dx2)[base + c] = from_f32<T2>(o * s);
    }
  }

  // this CTA's sums: over the teams of each warp by shuffles, then warp after warp into shared memory
  float* dst = a.partial + (size_t)blockIdx.x * 2 * C;
  if (wide) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = sub + v * lpr;
      if (c < C) { dst[c] = sa[v]; dst[C + c] = sb[v]; }
    }
    return;
  }
  for (int o = lpr; o < 32; o <<= 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      sa[v] += __shfl_xor_sync(0xffffffffu, sa[v], o);
      sb[v] += __shfl_xor_sync(0xffffffffu, sb[v], o);
    }
  }
  const int n_warps = blockDim.x >> 5;
  for (int q = 0; q < n_warps; ++q) {
    if ((int)(threadIdx.x >> 5) == q && lane < lpr) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = sub + v * lpr;
        if (c < C) {
          acc_smem[c] = (q ? acc_smem[c] : 0.f) + sa[v];
          acc_smem[C + c] = (q ? acc_smem[C + c] : 0.f) + sb[v];
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * C; i += blockDim.x) dst[i] = acc_smem[i];
}

// --------------------------------------------------------------------------------- dispatch

// Team width, elements per lane and computing warps for a row of `n` vectors (or elements).
struct Geometry {
  int lpr, nv, warps;
  bool ok;
};
// A lane holds 1..max_nv vectors (of 8 elements up to 3, of 4 up to 6), or 4, 8, 12 or 16 single elements.  A row costs its team's lanes about as much for its
// bookkeeping as ten more elements a lane would: fewest lanes * (elements + 10) wins.  A team divides the warps of
// the CTA (16, or 12 where a lane holds more than 16 elements).
inline Geometry geometry(int n, int vec, int max_nv, int period = 1) {
  Geometry best{0, 0, 0, false};
  long long best_cost = 0;
  for (int lpr = 2; lpr <= 512; lpr *= 2) {
    int nv = (n + lpr - 1) / lpr;
    if (vec == 1) nv = (nv + 3) / 4 * 4;
    if (nv > (vec == 1 ? 16 : max_nv)) continue;
    const int warps = warps_for(nv * vec);
    if (warps * 32 % lpr != 0 || warps * 32 / lpr % period != 0) continue;   // shifted rows: a team keeps its residue
    const long long cost = (long long)lpr * (nv * vec + 10);
    if (!best.ok || cost < best_cost) { best_cost = cost; best = Geometry{lpr, nv, warps, true}; }
  }
  return best;
}

constexpr size_t kRingBytes = 200 * 1024;   // of 227 KB per SM
// Most of one tile, so that three of them are in flight.
constexpr size_t kTileBytes = 64 * 1024;
// A backward pass this small stays in one CTA and needs no second kernel for the parameter gradients: measured 4.0 against
// 5.8 us at 32 KB, 4.5 against 5.7 at 64 KB, 8.0 against 5.7 at 196 KB.
constexpr size_t kAloneBytes = 64 * 1024;

// Ring of a launch: `row_bytes` of all loaded tensors together, `align` rows make every span a multiple of 16 bytes.
// False where two tiles do not fit.
struct Ring { int tile_rows, stages, grid; size_t smem; };
inline bool ring_for(int rows, const Geometry& g, size_t row_bytes, int align, size_t acc_bytes, size_t param_bytes, int per_sm, Ring* out) {
  const int per_pass = g.warps * 32 / g.lpr;
  // what two CTAs share, unless it is too small for two tiles
  size_t room = kRingBytes / per_sm - param_bytes;
  if (per_sm > 1 && (param_bytes > kRingBytes / per_sm || 2 * (size_t)align * row_bytes > room)) { per_sm = 1; room = kRingBytes - param_bytes; }
  const size_t tile_bytes = kTileBytes / per_sm;
  const int ctas = kSms * per_sm;
  if (2 * (size_t)align * row_bytes > room) return false;
  // A backward pass of a few rows stays in one CTA, which then needs no second kernel for the parameter gradients.
  const bool alone = acc_bytes > 0 && (size_t)rows * row_bytes <= kAloneBytes;
  const long long share = alone ? rows : ((long long)rows + ctas - 1) / ctas;
  // Tiles are whole passes of the CTA: `j` of them cost j + 0.5 a tile (its bookkeeping), times the rounds of tiles that the
  // busiest CTA walks, plus j for the first load and the last computation, which nothing overlaps.
  long long r = share < per_pass ? share : per_pass;
  double best = 1e30;
  for (long long j = 1; share >= per_pass && (j == 1 || (size_t)(j * per_pass) * row_bytes <= tile_bytes); ++j) {
    const long long tiles = ((long long)rows + j * per_pass - 1) / (j * per_pass);
    const double cost = (double)((tiles + ctas - 1) / ctas) * (j + 0.5) + j;
    if (cost < best * 0.99) { best = cost; r = j * per_pass; }
  }
  while (r > 1 && 2 * (size_t)r * row_bytes > room) r = (r + 1) / 2;
  r = (r + align - 1) / align * align;
  if (2 * (size_t)r * row_bytes > room) r = align;
  const long long tiles = ((long long)rows + r - 1) / r;
  out->tile_rows = (int)r;
  out->grid = alone ? 1 : (int)(tiles < ctas ? tiles : ctas);
  long long st = (long long)(room / ((size_t)r * row_bytes));
  const long long walk = (tiles + out->grid - 1) / out->grid;   // tiles of one CTA
  if (st > walk) st = walk;
  if (st > kMaxStages) st = kMaxStages;
  out->stages = (int)st;
  size_t bytes = (size_t)st * r * row_bytes + param_bytes;
  if (bytes < acc_bytes) bytes = acc_bytes;
  out->smem = kRingHeader + bytes;
  return true;
}

// Rows that make rows * C * es a multiple of 16 for the element size (16-bit tensors need the most).
inline int align_rows(int C, int es_min) {
  int r = 1;
  while ((long long)r * C * es_min % 16 != 0) r *= 2;
  return r;
}

// CTAs of the element-wise kernels.
constexpr int kDirectThreads = 256;
inline int direct_grid(int rows, int lpr) {
  const int per_cta = lpr > 32 ? 1 : kDirectThreads / lpr;
  const long long need = ((long long)rows + per_cta - 1) / per_cta, cap = 2LL * kSms;
  return (int)(need < cap ? need : cap);
}

// What a launch will do: shared by the launcher and the workspace size.
struct Plan {
  Geometry g;
  Ring ring;
  int vec;       // elements per vector; 1 element-wise
  bool shift;    // vectors of rows that start between boundaries
  bool direct;
  int grid;
};
inline Plan plan_for(bool backward, int mode, int x_es, int y_es, bool gh, bool summed, bool base16, bool vec_ok, int rows, int C) {
  Plan p;
  const int V = x_es == 4 || y_es == 4 ? 4 : 8;
  p.vec = vec_ok && base16 ? V : 1;
  p.shift = p.vec > 1 && C % V != 0;
  if (p.shift) {   // up to V - 1 elements in front of a row's first; 16 elements a lane, whose parameters are in registers
    int period = V;
    for (int c = C; c % 2 == 0; c /= 2) period /= 2;
    p.g = geometry((C + 2 * V - 2) / V, V, 16 / V, period);
    if (!p.g.ok) { p.shift = false; p.vec = 1; }
  }
  if (!p.shift) p.g = geometry(p.vec > 1 ? C / V : C, p.vec, V == 8 ? 3 : 6);
  const int lx = backward && mode == kPre ? y_es : x_es;      // element size of the normalised tensor
  const size_t row_bytes = (size_t)C * (backward ? lx * (1 + (mode == kPre && summed)) + y_es * (1 + (mode == kPre && gh)) : x_es + (mode == kPlain ? 0 : y_es));
  const int es_min = backward ? (lx < y_es ? lx : y_es) : (mode == kPlain || x_es < y_es ? x_es : y_es);
  const int slots = p.shift || p.g.lpr > 32 ? p.g.warps * 32 / p.g.lpr : p.g.warps;
  const size_t acc = backward ? (size_t)slots * 2 * C * sizeof(float) : 0;
  const size_t params = p.g.nv * p.vec > 16 || (p.vec == 1 && p.g.nv > 8) ? (size_t)2 * ((C + 3) / 4 * 4) * sizeof(float) : 0;
  p.direct = !base16 || acc > kRingBytes || !ring_for(rows, p.g, row_bytes, align_rows(C, es_min), acc, params, backward ? 1 : fwd_ctas(p.g.nv * p.vec), &p.ring);
  if (p.direct) {
    p.vec = 1;
    p.shift = false;
    p.g = geometry(C, 1, 0);
    if (p.g.nv != 4) p.g.nv = 16;   // the element-wise kernels come with 4 and 16
  }
  p.grid = p.direct ? direct_grid(rows, p.g.lpr) : p.ring.grid;
  return p;
}

// Elements of a vector: 16 bytes of the wider tensor type (a 16-bit branch beside fp32 tensors takes 8 bytes: with 8
// elements a lane's fp32 pieces would be 32 bytes apart and meet in the same banks).
template <typename TX, typename TY> struct FullVec { static constexpr int n = sizeof(TX) == 4 || sizeof(TY) == 4 ? 4 : 8; };

template <auto Kern>
cudaError_t launch_ring(const LnTrainArgs& a, const Plan& p, cudaStream_t s) {
  static int limit[64] = {0};   // dynamic shared memory granted so far, per kernel and device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  dev &= 63;
  if (limit[dev] == 0) {
    e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kRingHeader + kRingBytes));
    if (e != cudaSuccess) return e;
    limit[dev] = 1;
  }
  return launch_overlapped(Kern, dim3((unsigned)p.grid), dim3((unsigned)(32 * p.g.warps)), p.ring.smem, s, a);
}

template <typename TX, typename TY, int VEC, int NV, bool SHIFT = false>
cudaError_t ring_run(bool backward, int mode, int act, const LnTrainArgs& a, const Plan& p, cudaStream_t s) {
  if (!backward) {
    if (mode == kPost) return launch_ring<ln_ring_fwd_kernel<TX, TY, VEC, NV, SHIFT, kPost, false>>(a, p, s);
    if (mode == kPre) return launch_ring<ln_ring_fwd_kernel<TX, TY, VEC, NV, SHIFT, kPre, false>>(a, p, s);
    if (act) return launch_ring<ln_ring_fwd_kernel<TX, TY, VEC, NV, SHIFT, kPlain, true>>(a, p, s);
    return launch_ring<ln_ring_fwd_kernel<TX, TY, VEC, NV, SHIFT, kPlain, false>>(a, p, s);
  }
  if (mode == kPre) return launch_ring<ln_ring_bwd_kernel<TY, TY, TX, TX, VEC, NV, SHIFT, kPre, false>>(a, p, s);
  if (mode == kPost) return launch_ring<ln_ring_bwd_kernel<TX, TY, TX, TX, VEC, NV, SHIFT, kPost, false>>(a, p, s);
  if (act) return launch_ring<ln_ring_bwd_kernel<TX, TY, TX, TX, VEC, NV, SHIFT, kPlain, true>>(a, p, s);
  return launch_ring<ln_ring_bwd_kernel<TX, TY, TX, TX, VEC, NV, SHIFT, kPlain, false>>(a, p, s);
}
template <typename TX, typename TY, int NV>
cudaError_t direct_run(bool backward, int mode, int act, const LnTrainArgs& a, const Plan& p, cudaStream_t s) {
  const dim3 g((unsigned)p.grid), t((unsigned)(p.g.lpr > 32 ? p.g.lpr : kDirectThreads));
  if (!backward) {
    if (mode == kPost) return launch_overlapped(ln_train_fwd_kernel<TX, TY, NV, kPost, false>, g, t, 0, s, a);
    if (mode == kPre) return launch_overlapped(ln_train_fwd_kernel<TX, TY, NV, kPre, false>, g, t, 0, s, a);
    if (act) return launch_overlapped(ln_train_fwd_kernel<TX, TY, NV, kPlain, true>, g, t, 0, s, a);
    return launch_overlapped(ln_train_fwd_kernel<TX, TY, NV, kPlain, false>, g, t, 0, s, a);
  }
  const size_t smem = a.lpr > 32 ? 0 : (size_t)2 * a.C * sizeof(float);
  if (mode == kPre) return launch_overlapped(ln_train_bwd_kernel<TY, TY, TX, TX, NV, kPre, false>, g, t, smem, s, a);
  if (mode == kPost) return launch_overlapped(ln_train_bwd_kernel<TX, TY, TX, TX, NV, kPost, false>, g, t, smem, s, a);
  if (act) return launch_overlapped(ln_train_bwd_kernel<TX, TY, TX, TX, NV, kPlain, true>, g, t, smem, s, a);
  return launch_overlapped(ln_train_bwd_kernel<TX, TY, TX, TX, NV, kPlain, false>, g, t, smem, s, a);
}

template <typename TX, typename TY>
cudaError_t run(bool backward, int mode, int act, const Plan& p, const LnTrainArgs& a0, cudaStream_t s) {
  constexpr int V = FullVec<TX, TY>::n;
  if (!p.g.ok) return cudaErrorInvalidValue;
  LnTrainArgs a = a0;
  a.lpr = p.g.lpr;
  if (p.direct) return p.g.nv == 4 ? direct_run<TX, TY, 4>(backward, mode, act, a, p, s) : direct_run<TX, TY, 16>(backward, mode, act, a, p, s);
  a.tile_rows = p.ring.tile_rows;
  a.stages = p.ring.stages;
  if (p.vec == 1) {
    if (p.g.nv == 4) return ring_run<TX, TY, 1, 4>(backward, mode, act, a, p, s);
    if (p.g.nv == 8) return ring_run<TX, TY, 1, 8>(backward, mode, act, a, p, s);
    if (p.g.nv == 12) return ring_run<TX, TY, 1, 12>(backward, mode, act, a, p, s);
    return ring_run<TX, TY, 1, 16>(backward, mode, act, a, p, s);
  }
  if (p.shift) {
    if (p.g.nv == 1) return ring_run<TX, TY, V, 1, true>(backward, mode, act, a, p, s);
    if (p.g.nv == 2) return ring_run<TX, TY, V, 2, true>(backward, mode, act, a, p, s);
    if constexpr (V == 4) {
      if (p.g.nv == 3) return ring_run<TX, TY, V, 3, true>(backward, mode, act, a, p, s);
      if (p.g.nv == 4) return ring_run<TX, TY, V, 4, true>(backward, mode, act, a, p, s);
    }
    return cudaErrorInvalidValue;
  }
  switch (p.g.nv) {
    case 1: return ring_run<TX, TY, V, 1>(backward, mode, act, a, p, s);
    case 2: return ring_run<TX, TY, V, 2>(backward, mode, act, a, p, s);
    case 3: return ring_run<TX, TY, V, 3>(backward, mode, act, a, p, s);
    default:
      if constexpr (V == 4) {
        if (p.g.nv == 4) return ring_run<TX, TY, V, 4>(backward, mode, act, a, p, s);
        if (p.g.nv == 5) return ring_run<TX, TY, V, 5>(backward, mode, act, a, p, s);
        if (p.g.nv == 6) return ring_run<TX, TY, V, 6>(backward, mode, act, a, p, s);
      }
      return cudaErrorInvalidValue;
  }
}

}  // namespace ln
}  // namespace dcnb200
