// Newton-Schulz orthogonalisation of a stack of matrices (the step of the Muon optimiser), sm_100a.
//
//   X_0 = G / (|G|_F + eps);   A = X X^T,   B = b A + c A A,   X <- a X + B X       `steps` times
//
// drives the singular values of G towards 1 while keeping its singular vectors.  With p = min(m, n), q = max(m, n) an
// iteration is p^2 q + p^3 + 2 p^2 q multiply-adds (A and A A symmetric: only the tiles on and below the diagonal are
// computed, the others are mirrored): matrix products of a few hundred rows, so tensor-core work.  For m > n the
// products are taken on the other side (A = X^T X, X <- a X + X B): nothing is ever transposed in memory, the operand
// that needs it is read as an MN-major tile.
//
// Number formats.  Operands of the products are fp16, accumulators fp32.  Every value is bounded by the iteration
// itself (|X| <= 1.3, |A| <= 1.5, |B| <= 5), so fp16's range suffices and its 11 bits are worth having: rounding X
// perturbs every singular direction by about 2^-12 |X|_F / sqrt(p), and each step multiplies the small directions,
// noise included, by up to a = 3.44.  Therefore X is kept as a pair hi + lo / 2048 (22 bits) through all but the last
// two steps and the dominant term a X is formed in fp32 from that pair; only the correction B X sees 11 bits.  Over
// spectra from flat to rank-deficient the result is within 2.5e-3 of the exact iteration (hi alone: 2e-2, and the usual
// bf16 iteration: 2e-1).  In the last two steps nothing is left to amplify: a is folded into B's diagonal and X is hi.
// The result is returned in bf16, whose own rounding is of the size of that error.
//
// One kernel serves the three products; a persistent CTA per SM, ten warps:
//   warp 0     TMA loads of the two operand tiles (128 x 64 and BN x 64, 128-byte swizzle) into a ring
//   warp 1     tcgen05.mma (M 128, N BN, K 16) into one of two accumulators in tensor memory
//   warps 2-9  epilogue: 32 x 32 units from tensor memory; the previous X (hi, lo) or A arrives by TMA in the staging
//              buffer that the result leaves from, one unit ahead
// Every mbarrier wait is bounded; one that runs out sets the device status word and the CTA winds down.
//
// The reference has no optimiser kernels; its trainers use stock AdamW (classification/optimizer.py).
#include <mutex>

#include "tc.cuh"

namespace dcnb200 {

namespace {

using namespace tc;

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreadsNs = 32 * (2 + kEpiWarps);
constexpr int kUnit = 32 * 64;                 // staging unit: 32 rows x 32 fp16 (64-byte swizzle)
constexpr int kStagingWarp = 2 * 2 * kUnit;    // two sets of (hi or result, lo or mirror)
constexpr int kBarBytes = 512;
constexpr float kLoScale = 2048.f;

enum : int { kGram = 0, kPoly = 1, kUpdate = 2 };

template <int BN> constexpr int slot_bytes() { return kBM * kBK * 2 + BN * kBK * 2; }
template <int BN> constexpr int ns_stages() {
  constexpr int room = 227 * 1024 - 1024 - kBarBytes - kEpiWarps * kStagingWarp;
  return room / slot_bytes<BN>() > 6 ? 6 : room / slot_bytes<BN>();
}
template <int BN> constexpr size_t ns_smem() {
  return (size_t)ns_stages<BN>() * slot_bytes<BN>() + kEpiWarps * kStagingWarp + kBarBytes + 1024;
}

struct NsParams {
  int M, N, k_blocks;
  int m_tiles, n_tiles, tiles;   // tiles per matrix (symmetric: the lower triangle)
  int sym;
  long long total;               // tiles of the whole stack
  float a, b, c;
  int residual;                  // kUpdate: out = a * (hi + lo / 2048) + product; else: product
  int write_lo;
  int to_bf16;                   // kUpdate: the result leaves in bf16
  int fold;                      // kPoly: a on the diagonal
  int* status;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// Descriptor of an MN-major tile as the 128-byte swizzled boxes (64 elements of MN x 64 of K) lie in shared memory:
// 8 K-rows every 1024 bytes (stride offset), the next 64 MN-elements every 8192 bytes (leading offset).
__device__ __forceinline__ uint64_t smem_desc_mn(const void* tile) {
  uint64_t d = (uint64_t)((smem_u32(tile) & 0x3FFFF) >> 4);
  d |= (uint64_t)(8192 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

struct Tile { int bi, mt, nt; };
__device__ __forceinline__ Tile tile_of(long long t, const NsParams& p) {
  Tile r;
  r.bi = (int)(t / p.tiles);
  const int i = (int)(t - (long long)r.bi * p.tiles);
  if (p.sym) {  // row mt of the lower triangle starts at mt (mt + 1) / 2
    int mt = (int)((sqrtf(8.f * (float)i + 1.f) - 1.f) * 0.5f);
    while ((mt + 1) * (mt + 2) / 2 <= i) ++mt;
    while (mt * (mt + 1) / 2 > i) --mt;
    r.mt = mt;
    r.nt = i - mt * (mt + 1) / 2;
  } else {
    r.mt = i / p.n_tiles;
    r.nt = i - r.mt * p.n_tiles;
  }
  return r;
}

__device__ __forceinline__ uint32_t pack_h(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_b(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// TA / TB: the operand is MN-major (its rows are the reduction's).
template <int BN, bool TA, bool TB, int EPI>
__global__ void __launch_bounds__(kThreadsNs, 1)
ns_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_r0, const __grid_constant__ CUtensorMap map_r1,
               const __grid_constant__ CUtensorMap map_o0, const __grid_constant__ CUtensorMap map_o1,
               const NsParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kStages = ns_stages<BN>();
  constexpr uint32_t kBytesA = kBM * kBK * 2, kBytesB = BN * kBK * 2;
  unsigned char* ring_a = smem;
  unsigned char* ring_b = smem + kStages * kBytesA;
  unsigned char* staging = smem + kStages * (kBytesA + kBytesB);
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kEpiWarps * kStagingWarp);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* acc_full = bars + 2 * kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* res_bars = acc_empty + 2;            // [kEpiWarps][2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_bars + 2 * kEpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kTmemCols = 2 * BN;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&acc_full[a], 1); mbar_init(&acc_empty[a], kEpiWarps); }
    for (int w = 0; w < 2 * kEpiWarps; ++w) mbar_init(&res_bars[w], 1);
    *abort_flag = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();

  auto give_up = [&] { atomicExch(p.status, kStatusStageTimeout); *abort_flag = 1; };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      pdl_wait();
      for (long long t = blockIdx.x; t < p.total && !*abort_flag; t += gridDim.x) {
        const Tile q = tile_of(t, p);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1)) { give_up(); break; }
          mbar_expect_tx(&full[stage], kBytesA + kBytesB);
          unsigned char* da = ring_a + stage * kBytesA;
          unsigned char* db = ring_b + stage * kBytesB;
          if (TA) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i) tma_load_3d(da + i * 8192, &map_a, q.mt * kBM + i * 64, kb * kBK, q.bi, &full[stage]);
          } else {
            tma_load_3d(da, &map_a, kb * kBK, q.mt * kBM, q.bi, &full[stage]);
          }
          if (TB) {
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) tma_load_3d(db + i * 8192, &map_b, q.nt * BN + i * 64, kb * kBK, q.bi, &full[stage]);
          } else {
            tma_load_3d(db, &map_b, kb * kBK, q.nt * BN, q.bi, &full[stage]);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc<__half>(BN) | ((uint32_t)TA << 15) | ((uint32_t)TB << 16);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (long long t = blockIdx.x; t < p.total && !*abort_flag; t += gridDim.x) {
        if (!mbar_wait_bounded(&acc_empty[acc], acc_phase ^ 1)) { give_up(); break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait_bounded(&full[stage], phase)) { give_up(); break; }
          tc_fence_after();
          const uint64_t da = TA ? smem_desc_mn(ring_a + stage * kBytesA) : smem_desc_sw128(ring_a + stage * kBytesA);
          const uint64_t db = TB ? smem_desc_mn(ring_b + stage * kBytesB) : smem_desc_sw128(ring_b + stage * kBytesB);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)  // 16 of K: 32 bytes along a K-major row, 16 rows of an MN-major tile
            tc_mma_f16(d_tmem, da + (uint64_t)(k * (TA ? 128 : 2)), db + (uint64_t)(k * (TB ? 128 : 2)), idesc, (kb | k) != 0);
          tc_commit(&empty[stage]);
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        tc_commit(&acc_full[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  } else {
    const int quad = warp & 3, group = (warp - 2) >> 2;
    constexpr int kCols = BN / 2, kUnits = kCols / 32;  // columns and units of this warp's share of a tile
    unsigned char* buf = staging + (warp - 2) * kStagingWarp;
    uint64_t* res_bar = &res_bars[2 * (warp - 2)];
    const bool has_res = EPI == kPoly || (EPI == kUpdate && p.residual);
    uint32_t unit = 0;
    pdl_wait();
    // ask for the tile of the previous X or A that unit `u` of tile `t` needs
    auto fetch = [&](long long t, int u, uint32_t k) {
      const Tile q = tile_of(t, p);
      const int col = q.nt * BN + group * kCols + u * 32, row = q.mt * kBM + quad * 32;
      unsigned char* set = buf + (k & 1) * 2 * kUnit;
      mbar_expect_tx(&res_bar[k & 1], EPI == kUpdate ? 2 * kUnit : kUnit);
      tma_load_3d(set, &map_r0, col, row, q.bi, &res_bar[k & 1]);
      if (EPI == kUpdate) tma_load_3d(set + kUnit, &map_r1, col, row, q.bi, &res_bar[k & 1]);
    };
    if (has_res && lane == 0 && blockIdx.x < p.total) fetch(blockIdx.x, 0, 0);
    long long t = blockIdx.x;
    for (uint32_t it = 0; t < p.total && !*abort_flag; t += gridDim.x, ++it) {
      const int acc = (int)(it & 1);
      const Tile q = tile_of(t, p);
      if (!mbar_wait_bounded(&acc_full[acc], (it >> 1) & 1)) { if (lane == 0) give_up(); break; }
      tc_fence_after();
      const int row0 = q.mt * kBM + quad * 32;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN + group * kCols);
#pragma unroll 1
      for (int u = 0; u < kUnits; ++u, ++unit) {
        const int col0 = q.nt * BN + group * kCols + u * 32;
        unsigned char* set = buf + (unit & 1) * 2 * kUnit;
        uint32_t v[32];
        tmem_ld_32x32(taddr + (uint32_t)(u * 32), v);
        if (lane == 0) {
          if (has_res) {
            // the other set is free once the store of the previous unit has read it
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            if (u + 1 < kUnits) fetch(t, u + 1, unit + 1);
            else if (t + gridDim.x < p.total) fetch(t + gridDim.x, 0, unit + 1);
          } else {
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          }
        }
        __syncwarp();
        if (has_res && !mbar_wait_bounded(&res_bar[unit & 1], (unit >> 1) & 1)) { if (lane == 0) give_up(); }
        tmem_ld_wait();
        const bool mirror = EPI != kUpdate && p.sym && q.mt != q.nt;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          // 64-byte swizzle: 16-byte piece index xor bits 1-2 of the row
          const uint32_t off = (uint32_t)lane * 64 + ((((uint32_t)j >> 3) ^ (((uint32_t)lane >> 1) & 3)) << 4);
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(v[j + e]);
          if (EPI == kPoly) {
            const uint4 r = *reinterpret_cast<const uint4*>(set + off);
            const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack_h(rr[e]);
              x[2 * e] = fmaf(p.c, x[2 * e], p.b * f.x);
              x[2 * e + 1] = fmaf(p.c, x[2 * e + 1], p.b * f.y);
            }
            if (p.fold && row0 + lane >= col0 + j && row0 + lane < col0 + j + 8) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (row0 + lane == col0 + j + e) x[e] += p.a;
            }
          }
          if (EPI == kUpdate && p.residual) {
            const uint4 h = *reinterpret_cast<const uint4*>(set + off);
            const uint4 l = *reinterpret_cast<const uint4*>(set + kUnit + off);
            const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack_h(hh[e]), g = unpack_h(ll[e]);
              x[2 * e] = fmaf(p.a, fmaf(g.x, 1.f / kLoScale, f.x), x[2 * e]);
              x[2 * e + 1] = fmaf(p.a, fmaf(g.y, 1.f / kLoScale, f.y), x[2 * e + 1]);
            }
          }
          uint32_t o[4];
          if (EPI == kUpdate && p.to_bf16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack_b(x[2 * e], x[2 * e + 1]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack_h(x[2 * e], x[2 * e + 1]);
          }
          *reinterpret_cast<uint4*>(set + off) = make_uint4(o[0], o[1], o[2], o[3]);
          if (EPI == kUpdate && p.write_lo) {
            uint32_t l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack_h(o[e]);
              l[e] = pack_h((x[2 * e] - f.x) * kLoScale, (x[2 * e + 1] - f.y) * kLoScale);
            }
            *reinterpret_cast<uint4*>(set + kUnit + off) = make_uint4(l[0], l[1], l[2], l[3]);
          }
          if (mirror) {  // the transposed unit: row j + e, column `lane`
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t c = (uint32_t)(j + e);
              const uint32_t at = c * 64 + ((((uint32_t)lane >> 3) ^ ((c >> 1) & 3)) << 4) + ((uint32_t)lane & 7) * 2;
              *reinterpret_cast<uint16_t*>(set + kUnit + at) = (uint16_t)(o[e >> 1] >> ((e & 1) * 16));
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (row0 < p.M && col0 < p.N) {
            tma_store_3d(&map_o0, set, col0, row0, q.bi);
            if (EPI == kUpdate && p.write_lo) tma_store_3d(&map_o1, set + kUnit, col0, row0, q.bi);
            if (mirror) tma_store_3d(&map_o0, set + kUnit, row0, col0, q.bi);
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  // After a wait that ran out, copies into this CTA's shared memory and products may still be in flight: give them
  // 20 ms to land before the memory is handed back.
  if (*abort_flag)
    for (int i = 0; i < 20000; ++i) __nanosleep(1000);
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------- norm and scaling

constexpr int kNormThreads = 256;
constexpr int kMaxChunks = 64;   // partial sums of squares of one matrix

template <typename T> __device__ __forceinline__ float load1(const T* p) { return to_f32(*p); }

// Sum of squares of one slice of one matrix, in 64 bits (fp32 squares of large gradients would overflow).
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
ns_square_kernel(const T* __restrict__ x, double* __restrict__ partial, long long per, long long chunk, int vec) {
  __shared__ double part[kNormThreads / 32];
  pdl_trigger();
  pdl_wait();
  const T* src = x + (long long)blockIdx.y * per;
  const long long lo = (long long)blockIdx.x * chunk;
  const long long hi = lo + chunk < per ? lo + chunk : per;
  double s = 0.0;
  if (vec) {
    constexpr int E = 16 / (int)sizeof(T);
    for (long long i = lo + threadIdx.x * E; i < hi; i += kNormThreads * E) {
      const RawVec<16> r = ldg_raw<16>(src + i, true);
      float v[E];
      widen(r.r, v, (const T*)nullptr);
#pragma unroll
      for (int e = 0; e < E; ++e) s = fma((double)v[e], (double)v[e], s);
    }
  } else {
    for (long long i = lo + threadIdx.x; i < hi; i += kNormThreads) { const double v = load1(src + i); s = fma(v, v, s); }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < kNormThreads / 32; ++i) t += part[i];
    partial[(long long)blockIdx.y * kMaxChunks + blockIdx.x] = t;
  }
}

// X_0 = x / (norm + eps) as the fp16 pair, rows padded to `ld` elements (the padding is never read).
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
ns_scale_kernel(const T* __restrict__ x, const double* __restrict__ partial, __half* __restrict__ hi,
                __half* __restrict__ lo, int rows, int cols, int ld, int n_chunks, float eps, int vec) {
  __shared__ float inv_s;
  pdl_trigger();
  pdl_wait();
  const int bi = blockIdx.y;
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < n_chunks; ++i) t += partial[(long long)bi * kMaxChunks + i];
    inv_s = (float)(1.0 / (sqrt(t) + (double)eps));
  }
  __syncthreads();
  const float inv = inv_s;
  const T* src = x + (long long)bi * rows * cols;
  __half* dh = hi + (long long)bi * rows * ld;
  __half* dl = lo + (long long)bi * rows * ld;
  const long long stride = (long long)gridDim.x * kNormThreads;
  if (vec) {   // whole matrix in vectors of 8: rows are contiguous (cols == ld)
    const long long n8 = (long long)rows * cols / 8;
    for (long long i = (long long)blockIdx.x * kNormThreads + threadIdx.x; i < n8; i += stride) {
      float v[8];
      if constexpr (sizeof(T) == 4) {
        const RawVec<16> r0 = ldg_raw<16>(src + i * 8, true), r1 = ldg_raw<16>(src + i * 8 + 4, true);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = __uint_as_float(r0.r[e]); v[4 + e] = __uint_as_float(r1.r[e]); }
      } else {
        const RawVec<16> r = ldg_raw<16>(src + i * 8, true);
        widen(r.r, v, (const T*)nullptr);
      }
      uint32_t h[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = v[2 * e] * inv, x1 = v[2 * e + 1] * inv;
        h[e] = pack_h(x0, x1);
        const float2 f = unpack_h(h[e]);
        l[e] = pack_h((x0 - f.x) * kLoScale, (x1 - f.y) * kLoScale);
      }
      *reinterpret_cast<uint4*>(dh + i * 8) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(dl + i * 8) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  } else {
    const long long total = (long long)rows * cols;
    for (long long i = (long long)blockIdx.x * kNormThreads + threadIdx.x; i < total; i += stride) {
      const long long r = i / cols;
      const int c = (int)(i - r * cols);
      const float v = load1(src + i) * inv;
      const __half h = __float2half_rn(v);
      dh[r * ld + c] = h;
      dl[r * ld + c] = __float2half_rn((v - __half2float(h)) * kLoScale);
    }
  }
}

// Compact copy of a bf16 result whose rows were padded to `ld` (column counts that 16-byte stores cannot address).
__global__ void __launch_bounds__(kNormThreads)
ns_compact_kernel(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst, long long rows, int cols, int ld) {
  pdl_trigger();
  pdl_wait();
  const long long total = rows * cols, stride = (long long)gridDim.x * kNormThreads;
  for (long long i = (long long)blockIdx.x * kNormThreads + threadIdx.x; i < total; i += stride) {
    const long long r = i / cols;
    dst[i] = src[r * ld + (i - r * cols)];
  }
}

// ------------------------------------------------------------------------------- host side

bool map3(CUtensorMap* m, bool bf16, const void* base, long long batch, long long rows, int cols, int ld, int box_rows,
          int box_cols) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * (cuuint64_t)rows};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
             dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_cols * 2 == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Mat { const void* p; long long rows; int cols, ld; };

template <int BN, bool TA, bool TB, int EPI>
cudaError_t launch_gemm(const Mat& A, const Mat& B, const Mat& r0, const Mat& r1, const Mat& o0, const Mat& o1,
                        long long batch, NsParams p, int M, int N, int K, bool sym, int sms, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaGetDevice(&dev);
  dev = dev < 0 || dev >= 64 ? 0 : dev;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(ns_gemm_kernel<BN, TA, TB, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)ns_smem<BN>());
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  CUtensorMap ma, mb, m0, m1, n0, n1;
  if (!map3(&ma, false, A.p, batch, A.rows, A.cols, A.ld, TA ? 64 : kBM, 64) ||
      !map3(&mb, false, B.p, batch, B.rows, B.cols, B.ld, TB ? 64 : BN, 64) ||
      !map3(&m0, false, r0.p, batch, r0.rows, r0.cols, r0.ld, 32, 32) ||
      !map3(&m1, false, r1.p, batch, r1.rows, r1.cols, r1.ld, 32, 32) ||
      !map3(&n0, p.to_bf16 != 0, o0.p, batch, o0.rows, o0.cols, o0.ld, 32, 32) ||
      !map3(&n1, false, o1.p, batch, o1.rows, o1.cols, o1.ld, 32, 32))
    return cudaErrorNotSupported;
  p.M = M; p.N = N;
  p.k_blocks = (K + kBK - 1) / kBK;
  p.m_tiles = (M + kBM - 1) / kBM;
  p.n_tiles = (N + BN - 1) / BN;
  p.sym = sym;
  p.tiles = sym ? p.m_tiles * (p.m_tiles + 1) / 2 : p.m_tiles * p.n_tiles;
  p.total = batch * p.tiles;
  const unsigned grid = (unsigned)(p.total < sms ? p.total : sms);
  return launch_overlapped(ns_gemm_kernel<BN, TA, TB, EPI>, dim3(grid), dim3(kThreadsNs), ns_smem<BN>(), s, ma, mb, m0,
                           m1, n0, n1, p);
}

inline long long pad8(long long v) { return (v + 7) / 8 * 8; }
inline size_t pad1k(size_t v) { return (v + 1023) / 1024 * 1024; }

struct Layout {
  size_t x[2], l[2], a, b, norm, total;
  int ldn, ldp;
};
Layout layout_of(long long batch, int m, int n) {
  Layout w;
  const int p = m < n ? m : n;
  w.ldn = (int)pad8(n);
  w.ldp = (int)pad8(p);
  const size_t xb = pad1k((size_t)batch * m * w.ldn * 2), ab = pad1k((size_t)batch * p * w.ldp * 2);
  size_t at = 0;
  for (int i = 0; i < 2; ++i) { w.x[i] = at; at += xb; }
  for (int i = 0; i < 2; ++i) { w.l[i] = at; at += xb; }
  w.a = at; at += ab;
  w.b = at; at += ab;
  w.norm = at; at += pad1k((size_t)batch * kMaxChunks * sizeof(double));
  w.total = at;
  return w;
}

template <typename T>
cudaError_t prepare(const void* x, const Layout& w, unsigned char* ws, long long batch, int m, int n, float eps,
                    int sms, cudaStream_t s) {
  const long long per = (long long)m * n;
  const bool vec = n % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  // slices of a matrix: enough to fill the GPU, each a whole number of vector rounds
  long long chunks = (4LL * sms + batch - 1) / batch;
  const long long round = kNormThreads * 8;
  const long long most = (per + round - 1) / round;
  if (chunks > most) chunks = most;
  if (chunks > kMaxChunks) chunks = kMaxChunks;
  long long chunk = ((per + chunks - 1) / chunks + round - 1) / round * round;
  chunks = (per + chunk - 1) / chunk;
  double* partial = reinterpret_cast<double*>(ws + w.norm);
  const T* src = static_cast<const T*>(x);
  cudaError_t e = launch_overlapped(ns_square_kernel<T>, dim3((unsigned)chunks, (unsigned)batch), dim3(kNormThreads), 0, s,
                                    src, partial, per, chunk, (int)vec);
  if (e != cudaSuccess) return e;
  long long blocks = (8LL * sms + batch - 1) / batch;
  if (blocks > most) blocks = most;
  return launch_overlapped(ns_scale_kernel<T>, dim3((unsigned)blocks, (unsigned)batch), dim3(kNormThreads), 0, s, src,
                           (const double*)partial, reinterpret_cast<__half*>(ws + w.x[0]),
                           reinterpret_cast<__half*>(ws + w.l[0]), m, n, w.ldn, (int)chunks, eps, (int)vec);
}

}  // namespace

size_t ns_workspace_bytes(long long batch, int m, int n) { return layout_of(batch, m, n).total; }

// dtype: 0 fp32, 1 fp16, 2 bf16 of x; out is bf16.
cudaError_t launch_newton_schulz(int dtype, const void* x, void* out, void* workspace, long long batch, int m, int n,
                                 int steps, float a, float b, float c, float eps, int sms, int* status, cudaStream_t s) {
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Layout w = layout_of(batch, m, n);
  cudaError_t e = dtype == 0   ? prepare<float>(x, w, ws, batch, m, n, eps, sms, s)
                  : dtype == 1 ? prepare<__half>(x, w, ws, batch, m, n, eps, sms, s)
                               : prepare<__nv_bfloat16>(x, w, ws, batch, m, n, eps, sms, s);
  const bool tall = m > n;
  const int pd = tall ? n : m, qd = tall ? m : n;
  const Mat A{ws + w.a, pd, pd, w.ldp}, B{ws + w.b, pd, pd, w.ldp};
  const bool direct = n % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const int keep = steps - 2;      // steps that carry the pair
  for (int k = 0; k < steps && e == cudaSuccess; ++k) {
    const int cur = k & 1, nxt = cur ^ 1;
    const Mat X{ws + w.x[cur], m, n, w.ldn}, L{ws + w.l[cur], m, n, w.ldn};
    const bool last = k == steps - 1;
    Mat O{ws + w.x[nxt], m, n, w.ldn};
    const Mat OL{ws + w.l[nxt], m, n, w.ldn};
    if (last && direct) O = Mat{out, m, n, n};
    NsParams p = {};
    p.a = a; p.b = b; p.c = c; p.status = status;
    p.residual = k < keep;
    p.fold = !p.residual;
    p.write_lo = k + 1 < keep;
    if (tall) e = launch_gemm<128, true, true, kGram>(X, X, A, A, A, A, batch, p, pd, pd, qd, true, sms, s);
    else e = launch_gemm<128, false, false, kGram>(X, X, A, A, A, A, batch, p, pd, pd, qd, true, sms, s);
    if (e != cudaSuccess) break;
    e = launch_gemm<128, false, false, kPoly>(A, A, A, A, B, B, batch, p, pd, pd, pd, true, sms, s);
    if (e != cudaSuccess) break;
    p.to_bf16 = last;
    if (tall) e = n > 128 ? launch_gemm<256, false, false, kUpdate>(X, B, X, L, O, OL, batch, p, m, n, pd, false, sms, s)
                          : launch_gemm<128, false, false, kUpdate>(X, B, X, L, O, OL, batch, p, m, n, pd, false, sms, s);
    else e = n > 128 ? launch_gemm<256, false, true, kUpdate>(B, X, X, L, O, OL, batch, p, m, n, pd, false, sms, s)
                     : launch_gemm<128, false, true, kUpdate>(B, X, X, L, O, OL, batch, p, m, n, pd, false, sms, s);
  }
  if (e == cudaSuccess && !direct) {
    const long long total = batch * (long long)m * n;
    long long blocks = (total + kNormThreads - 1) / kNormThreads;
    if (blocks > 8LL * sms) blocks = 8LL * sms;
    e = launch_overlapped(ns_compact_kernel, dim3((unsigned)blocks), dim3(kNormThreads), 0, s,
                          (const uint16_t*)(ws + w.x[steps & 1]), static_cast<uint16_t*>(out), batch * (long long)m, n,
                          w.ldn);
  }
  return e;
}

}  // namespace dcnb200
