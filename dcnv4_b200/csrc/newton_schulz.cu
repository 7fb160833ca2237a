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
// two steps and the dominant term a X is formed in fp32 from that pair; only the correction B X sees 11 bits.  Measured on
// 160 x 640, spectra from flat to rank-deficient, before the result's rounding: within 1.5e-3 of the exact iteration in the
// 2-norm (hi alone: 2.3e-2, and the usual bf16 iteration: 1.9e-1).  What can be shown: fifteen roundings of 2^-11, 4.2e-3, where
// many independent ones average out; up to 2.0e-2 for a matrix of a few rows, of which each rounding moves a whole singular
// direction.  In the last two steps nothing is left to amplify: a is folded into B's diagonal and X is hi.  The result is
// returned in bf16, whose rounding adds up to 2^-8 of each element.
//
// fp16 also has a lower end: where eps outweighs |G|, X_0 is as small as their quotient and grows by a factor of a a step.
// Such a matrix is held as 2^k X, with k from an upper bound of |X| that every step carries on, s <- s (|a| + |b| s^2 +
// |c| s^4): then 2^k X is below 1 and not below 1/2 times what the bound overestimates.  The products are those of 2^k X;
// a step's coefficients are b 2^-2k and c 2^-4k, its result is scaled by 2^(k' - k), the last one's by 2^-k.  Powers of two
// are exact, and with |G| >= eps k is 0 throughout.
//
// One persistent kernel runs all products of all steps.  A task is one 128 x BN tile of one product of one matrix; tasks
// are numbered so that a task only needs earlier ones (step by step, product by product), CTAs take them in that order from
// a counter, and each matrix counts its finished tiles: a task starts when its matrix has all tiles of the products
// before.  Nothing waits for a whole product of the whole stack, so one product's last tiles run beside the next one's
// first, and a single small matrix pays a flag in memory between products instead of a kernel launch.  Every task that is
// waited for has been taken by a running CTA, so the order of progress needs no co-residency.  Warps:
//   warp 0     takes tasks, waits for what they need, TMA loads of the two operand tiles (64 x 64 boxes, 128-byte swizzle)
//   warp 1     tcgen05.mma (M 128 or 256, N BN, K 16) into one of two accumulators in tensor memory
//   last warp  counts the finished tiles
//   others     epilogue: 32 x 32 units from tensor memory; the previous X (hi, lo) or A arrives by TMA
//              in the staging buffer that the result leaves from
// Large stacks give the tiles to pairs of CTAs (cta_group::2): a CTA loads its 128 rows of A and half of B's columns, so
// that the operands cost 2/3 of the L2 traffic and of the shared memory's bandwidth, which is what a 128 x 256 tile is
// short of (its 48 KB per 64 of K are written once and read once in the 512 cycles of the products).  The leader takes
// the tasks, hands them to both queues and issues the products; each CTA has its own epilogue and counts its half.  A last
// row block of at most 128 rows is a 128 x BN product (M 128, 64 rows in each CTA), so that no rows are padded to 256.
// What bounds both forms is operand bytes in flight: with three slots of the ring instead of five, pairs took 1.15 times
// as long; the rest of shared memory is the epilogue's staging, which must cover the same latency.
// Every mbarrier wait is bounded; one that runs out sets the device status word and the CTA winds down.
//
// Matrices with p <= 128 and q <= 256 take another kernel: one CTA holds a whole matrix (X and A, B as fp16 operands in shared
// memory, X in fp32 in tensor memory) and runs all steps without leaving the SM, in one launch that includes the norm.
// What bounds it is the chain of 3 * steps products, each a commit, a barrier and a pass of eight warps over the
// accumulator: 64 x 64 takes 22 us, where the tiled kernel's flags and round trips to L2 made it 54.
//
// The reference has no optimiser kernels; its trainers use stock AdamW (classification/optimizer.py).
#include <mutex>

#include "tc.cuh"

namespace dcnb200 {

namespace {

using namespace tc;

constexpr int kBM = 128, kBK = 64;
constexpr int kBox = 64 * 64 * 2;              // operand box: 64 x 64 fp16
// Epilogue warps: four quarters of the accumulator's rows, each in up to four column groups of at least 32.
template <int BN> constexpr int epi_groups() { return BN / 32 < 4 ? BN / 32 : 4; }
template <int BN> constexpr int epi_warps() { return 4 * epi_groups<BN>(); }
template <int BN> constexpr int ns_threads() { return 32 * (3 + epi_warps<BN>()); }
constexpr int kUnit = 32 * 64;                 // staging unit: 32 rows x 32 fp16 (64-byte swizzle)
constexpr int kStagingWarp = 2 * kUnit;        // hi or result, and lo or mirror
constexpr int kBarBytes = 1024;
constexpr int kQueue = 4;                      // tasks between the warp that takes them and the others, tiles to be counted
constexpr float kLoScale = 2048.f;

enum : int { kGram = 0, kPoly = 1, kUpdate = 2 };

// PAIR: two CTAs of a cluster share a 256 x BN tile, each with its 128 rows and half of the columns' operand.
template <bool PAIR> constexpr int tile_m() { return PAIR ? 256 : 128; }
template <int BN, bool PAIR> constexpr int slot_bytes() { return (2 + BN / (PAIR ? 128 : 64)) * kBox; }
template <int BN, bool PAIR> constexpr int ns_stages() {
  constexpr int room = 227 * 1024 - 1024 - kBarBytes - epi_warps<BN>() * kStagingWarp;
  return room / slot_bytes<BN, PAIR>() > 6 ? 6 : room / slot_bytes<BN, PAIR>();
}
template <int BN, bool PAIR> constexpr size_t ns_smem() {
  return (size_t)ns_stages<BN, PAIR>() * slot_bytes<BN, PAIR>() + epi_warps<BN>() * kStagingWarp + kBarBytes + 1024;
}

// Tensor maps of a call: 64 x 64 boxes of the operands, 32 x 32 boxes of what an epilogue reads and writes.
struct NsMaps {
  CUtensorMap x[2], a, b;              // operand boxes
  CUtensorMap xs[2], ls[2], as, bs;    // epilogue boxes
  CUtensorMap out;                     // bf16 result
};

struct NsParams {
  int m, n, p, q;                // p = min, q = max
  int tall;
  int steps, keep;               // steps that carry the pair
  int batch;
  int group1, group2;            // matrices of the task order's first two groups
  int sym_tiles, upd_tiles;      // tiles of a symmetric product, of an update
  int upd_n;                     // tile columns of an update
  unsigned total;                // tasks
  float a;
  const float4* coef;            // [batch][steps] StepCoef
  unsigned* done;                // [batch] finished tiles
  unsigned* ticket;              // next task
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
__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// One lane of a converged warp.  The tensor-core and TMA instructions take their operands from uniform registers: behind
// a plain `lane == 0` the compiler cannot tell that one lane is left and serialises each of them (measured: 0.38 us for
// every 64 of K, whatever the tile's width).
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {   // without suspending, unlike try_wait
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// Global memory written through the async proxy elsewhere and known through a flag is about to be read through it here.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.global;" ::: "memory"); }

// Tile columns of row block i of a symmetric product: those that reach the diagonal or lie left of it.
template <int BN, int TM>
__host__ __device__ inline int sym_cols(int i, int p) {
  const int c = (i * TM + TM - 1) / BN + 1, most = (p + BN - 1) / BN;
  return c < most ? c : most;
}

// ---- range of a matrix ----
constexpr int kMaxScale = 120;       // 2^-120 is a normal number
// k of 2^k X for |X| <= s; 0 for a zero matrix and for NaN.
__device__ __forceinline__ int scale_of(float s) {
  if (!(s > 0.f && s < 0.5f)) return 0;
  const int k = -(ilogbf(s) + 1);
  return k < kMaxScale ? k : kMaxScale;
}
// What a step works with: B = b A + c A A of the scaled matrix, its result times `post`.
struct StepCoef { float b, c, post; };
// Coefficients of a step; s bounds |X| before and after it, k is the scale before and after it.
__device__ __forceinline__ StepCoef step_coef(float a, float b, float c, float& s, int& k, bool last) {
  const float s2 = s * s;
  s *= fabsf(a) + s2 * (fabsf(b) + s2 * fabsf(c));
  const int next = last ? 0 : scale_of(s);
  StepCoef r{b, c, 1.f};
  if (k != 0 || next != 0) { r.b = ldexpf(b, -2 * k); r.c = ldexpf(c, -4 * k); r.post = ldexpf(1.f, next - k); }
  k = next;
  return r;
}
// 2^k X_0 from x and the sum of its squares.  The factor need not be a normal fp32 number (|x| beyond 1e38, or below 1e-38
// with a small eps): such a matrix is scaled in 64 bits.
struct Scaling {
  float s, factor;
  int k;
  double exact;
  bool wide;
  __device__ Scaling(double sum, float eps) {
    const double norm = sqrt(sum), by = norm + (double)eps;
    exact = 1.0 / by;
    s = (float)(norm * exact);
    k = scale_of(s);
    if (k != 0) exact = ldexp(exact, k);
    factor = (float)exact;
    wide = !(factor >= 1.1754944e-38f && factor <= 1.7e38f);
  }
  template <bool WIDE> __device__ __forceinline__ float operator()(float x) const {
    return WIDE ? (float)((double)x * exact) : x * factor;
  }
};

struct Task { int step, kind, bi, mt, nt; };
// Task order.  CTAs take tasks in order, so a task whose matrix is not ready holds up its CTA: the distance between a
// matrix' product and its next one should be a wave of tasks or more.  A = X X^T has the fewest and longest tiles; the
// matrices beyond its first wave of CTAs (group 3) finish it a whole tile later than the others.  So a step goes
//   A of all | A A of groups 1, 2 | B X of 1 | A A of 3 | B X of 2 | B X of 3
// with groups 1 and 2 the halves of the first wave.  (One product after the other for all matrices: CTAs waited 26 % of
// the time at 22 x 640x2560.  Taking ready tiles of any matrix instead, from counters, cost more than it saved.)
template <int BN, int TM>
__device__ __forceinline__ Task task_of(unsigned t, const NsParams& p) {
  Task r;
  const unsigned sym = p.sym_tiles, upd = p.upd_tiles;
  const unsigned per_step = p.batch * (2 * sym + upd);
  r.step = (int)(t / per_step);
  unsigned i = t - r.step * per_step;
  const unsigned g1 = p.group1, g12 = p.group1 + p.group2, g3 = p.batch - g12;
  unsigned first = 0;
  if (i < p.batch * sym) {
    r.kind = kGram;
  } else if ((i -= p.batch * sym) < g12 * sym) {
    r.kind = kPoly;
  } else if ((i -= g12 * sym) < g1 * upd) {
    r.kind = kUpdate;
  } else if ((i -= g1 * upd) < g3 * sym) {
    r.kind = kPoly;
    first = g12;
  } else {           // groups 2 and 3 follow one another
    i -= g3 * sym;
    r.kind = kUpdate;
    first = g1;
  }
  const unsigned per = r.kind == kUpdate ? upd : sym, of = i / per;
  int tile = (int)(i - of * per);
  r.bi = (int)(first + of);
  if (r.kind == kUpdate) {
    r.mt = tile / p.upd_n;
    r.nt = tile - r.mt * p.upd_n;
  } else {
    int mt = 0;
    for (int c = sym_cols<BN, TM>(0, p.p); tile >= c; c = sym_cols<BN, TM>(mt, p.p)) { tile -= c; ++mt; }
    r.mt = mt;
    r.nt = tile;
  }
  return r;
}
// Tiles of the task's matrix that must be finished before it may start.
__device__ __forceinline__ unsigned needs(const Task& t, const NsParams& p) {
  const int per = 2 * p.sym_tiles + p.upd_tiles;
  return (unsigned)(t.step * per + (t.kind == kGram ? 0 : t.kind == kPoly ? p.sym_tiles : 2 * p.sym_tiles));
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

// ---- two CTAs of a cluster ----
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
// Address, in the cluster's window, of a CTA's copy of something in shared memory; rank 0 is the leader.
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity) {   // bounded, as mbar_wait_bounded
  for (int i = 0; i < (1 << 22); ++i) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return true;
  }
  return false;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Into this CTA's shared memory, the bytes counted by a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void mma_f16_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) {     // arrives at this barrier in both CTAs
  const uint16_t both_ctas = 3;
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"(both_ctas) : "memory");
}

template <int BN, bool PAIR>
__global__ void __launch_bounds__(ns_threads<BN>(), 1)
ns_kernel(const __grid_constant__ NsMaps maps, const __grid_constant__ NsParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kStages = ns_stages<BN, PAIR>();
  constexpr uint32_t kSlot = slot_bytes<BN, PAIR>();
  constexpr int kEpiWarps = epi_warps<BN>();
  constexpr int TM = tile_m<PAIR>();
  constexpr int kBoxesB = BN / (PAIR ? 128 : 64);
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  unsigned char* ring = smem;                      // per slot: A (2 boxes), B (kBoxesB boxes)
  unsigned char* staging = smem + kStages * kSlot;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kEpiWarps * kStagingWarp);
  uint64_t* full = bars;
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* task_full = acc_empty + 2;             // [kQueue]
  uint64_t* task_empty = task_full + kQueue;
  uint64_t* tile_done = task_empty + kQueue;       // [kQueue] all stores of a tile complete
  uint64_t* tile_free = tile_done + kQueue;
  uint64_t* res_bars = tile_free + kQueue;         // [kEpiWarps]
  int4* queue = reinterpret_cast<int4*>(res_bars + kEpiWarps);  // [kQueue]: step * 4 + kind (-1: no more), matrix, tile
  volatile int* tile_matrix = reinterpret_cast<volatile int*>(queue + kQueue);   // [kQueue], -1: no more
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(tile_matrix) + kQueue);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kTmemCols = 2 * BN;

  if (threadIdx.x == 0) {
    auto init = [](uint64_t* bar, uint32_t count) {   // one fence for all of them below
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
    };
    for (int s = 0; s < kStages; ++s) { init(&full[s], 1); init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { init(&acc_full[a], 1); init(&acc_empty[a], (PAIR ? 2 : 1) * kEpiWarps); }
    for (int q = 0; q < kQueue; ++q) { init(&task_full[q], 1); init(&task_empty[q], (PAIR ? 2 : 1) * (1 + kEpiWarps)); init(&tile_done[q], kEpiWarps); init(&tile_free[q], 1); }
    for (int w = 0; w < kEpiWarps; ++w) init(&res_bars[w], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();          // the other CTA's barriers are ready
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();

  // Waits and their outcome are a warp's, not a lane's: all lanes leave a loop together.
  auto give_up = [&] { if (lane == 0) { atomicExch(p.status, kStatusStageTimeout); *abort_flag = 1; } };
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, PAIR ? wait_cluster(bar, parity) : mbar_wait_bounded(bar, parity)) != 0;
  };
  // Arrival of one lane at the leader's copy of a barrier.
  auto arrive_leader = [&](uint64_t* bar) {
    if (PAIR && rank != 0) arrive_cluster(at_rank(bar, 0));
    else mbar_arrive(bar);
  };
  auto aborted = [&] { return __any_sync(0xffffffffu, *abort_flag) != 0; };
  // operand orientation of a task: the tile's rows are the reduction's (MN-major)?
  auto a_mn = [&](int kind) { return kind == kGram && p.tall; };
  auto b_mn = [&](int kind) { return kind == kGram ? p.tall != 0 : kind == kUpdate && !p.tall; };
  // a pair's last row block with no more than 128 rows: 64 of them in each CTA
  auto is_half = [&](int kind, int mt) { return PAIR && (kind == kUpdate ? p.m : p.p) - mt * TM <= TM / 2; };
  auto k_blocks = [&](int kind) { return ((kind == kGram ? p.q : p.p) + kBK - 1) / kBK; };

  if (warp == 0) {
    int stage = 0, slot = 0;
    uint32_t phase = 0, qphase = 0;
    pdl_wait();
    unsigned next = 0;                 // lane 0: the next ticket, asked for when the current task's last loads go out
    if (rank == 0 && lane == 0) next = atomicAdd(p.ticket, 1u);
    while (!aborted()) {
      Task q{-1, 3, 0, 0, 0};          // step * 4 + kind == -1: the end
      if (rank == 0) {
        const unsigned t = __shfl_sync(0xffffffffu, next, 0);
        if (t < p.total) {
          q = task_of<BN, TM>(t, p);
          const unsigned want = needs(q, p) * (PAIR ? 2 : 1);     // each CTA of a pair counts a tile
          bool ready = want == 0;
          for (int spins = 0; !ready && spins < (1 << 25); ++spins) ready = load_acquire(p.done + q.bi) >= want;
          if (!__all_sync(0xffffffffu, ready)) { give_up(); break; }
          fence_async();               // for this warp's loads and, by way of the queue, the epilogue's
        }
        if (!wait(&task_empty[slot], qphase ^ 1)) { give_up(); break; }
        if (lane == 0) {
          const int4 code = make_int4(q.step * 4 + q.kind, q.bi, q.mt, q.nt);
          queue[slot] = code;
          if (PAIR) {
            asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};"
                         ::"r"(at_rank(&queue[slot], 1)), "r"(code.x), "r"(code.y), "r"(code.z), "r"(code.w) : "memory");
            arrive_cluster(at_rank(&task_full[slot], 1));
          }
          mbar_arrive(&task_full[slot]);
        }
      } else {
        if (!wait(&task_full[slot], qphase)) { give_up(); break; }
        const int4 code = queue[slot];
        __syncwarp();
        if (lane == 0) arrive_leader(&task_empty[slot]);
        if (code.x >= 0) q = Task{code.x >> 2, code.x & 3, code.y, code.z, code.w};
        fence_async();
      }
      if (++slot == kQueue) { slot = 0; qphase ^= 1; }
      if (q.step < 0) break;
      const bool ta = a_mn(q.kind), tb = b_mn(q.kind);
      const CUtensorMap* mx = &maps.x[q.step & 1];
      const CUtensorMap* ma = q.kind == kGram ? mx : q.kind == kPoly ? &maps.a : (p.tall ? mx : &maps.b);
      const CUtensorMap* mb = q.kind == kGram ? mx : q.kind == kPoly ? &maps.a : (p.tall ? &maps.b : mx);
      const int kb_n = k_blocks(q.kind);
      const bool half = is_half(q.kind, q.mt);
      const int row = q.mt * TM + (int)rank * (half ? kBM / 2 : kBM), col = q.nt * BN + (int)rank * (BN / 2);
      __syncwarp();
      for (int kb = 0; kb < kb_n; ++kb) {
        if (rank == 0 && kb == kb_n - 1 && lane == 0) next = atomicAdd(p.ticket, 1u);
        if (!wait(&empty[stage], phase ^ 1)) { give_up(); break; }
        if (elect_one()) {
          unsigned char* da = ring + stage * kSlot;
          unsigned char* db = da + 2 * kBox;
          if (rank == 0) mbar_expect_tx(&full[stage], (PAIR ? 2 : 1) * (half ? kSlot - kBox : kSlot));
          const uint32_t pair_bar = PAIR ? at_rank(&full[stage], 0) : 0;
          auto load = [&](void* dst, const CUtensorMap* map, bool mn_major, int mn) {
            const int c0 = mn_major ? mn : kb * kBK, c1 = mn_major ? kb * kBK : mn;
            if (PAIR) tma_load_3d_pair(dst, map, c0, c1, q.bi, pair_bar);
            else tma_load_3d(dst, map, c0, c1, q.bi, &full[stage]);
          };
          load(da, ma, ta, row);
          if (!half) load(da + kBox, ma, ta, row + 64);
#pragma unroll
          for (int i = 0; i < kBoxesB; ++i) load(db + i * kBox, mb, tb, col + i * 64);
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    if (PAIR && !aborted())            // the leader's last arrivals at this CTA's barriers have come in
      for (int s = 0; s < kStages; ++s) {
        if (!wait(&empty[stage], phase ^ 1)) { give_up(); break; }
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
  } else if (warp == 1) {
    int stage = 0, acc = 0, slot = 0;
    uint32_t phase = 0, acc_phase = 0, qphase = 0;
    while (rank == 0 && !aborted()) {
      if (!wait(&task_full[slot], qphase)) { give_up(); break; }
      const int4 task = queue[slot];
      const int code = task.x, kind = code & 3;
      __syncwarp();
      if (lane == 0) mbar_arrive(&task_empty[slot]);
      if (++slot == kQueue) { slot = 0; qphase ^= 1; }
      if (code < 0) break;
      const bool ta = a_mn(kind), tb = b_mn(kind);
      const uint32_t idesc = instr_desc<__half>(BN, is_half(kind, task.z) ? TM / 2 : TM) | ((uint32_t)ta << 15) | ((uint32_t)tb << 16);
      const uint64_t step_a = ta ? 128 : 2, step_b = tb ? 128 : 2;  // 16 of K: 16 rows of an MN-major box, 32 bytes of a K-major row
      const int kb_n = k_blocks(kind);
      if (!wait(&acc_empty[acc], acc_phase ^ 1)) { give_up(); break; }
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
      for (int kb = 0; kb < kb_n; ++kb) {
        if (!wait(&full[stage], phase)) { give_up(); break; }
        tc_fence_after();
        if (elect_one()) {
          unsigned char* da = ring + stage * kSlot;
          const uint64_t a0 = ta ? smem_desc_mn(da) : smem_desc_sw128(da);
          const uint64_t b0 = tb ? smem_desc_mn(da + 2 * kBox) : smem_desc_sw128(da + 2 * kBox);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            if (PAIR) mma_f16_pair(d_tmem, a0 + k * step_a, b0 + k * step_b, idesc, (kb | k) != 0);
            else tc_mma_f16(d_tmem, a0 + k * step_a, b0 + k * step_b, idesc, (kb | k) != 0);
          }
          if (PAIR) {
            commit_pair(&empty[stage]);
            if (kb == kb_n - 1) commit_pair(&acc_full[acc]);
          } else {
            tc_commit(&empty[stage]);
            if (kb == kb_n - 1) tc_commit(&acc_full[acc]);
          }
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  } else if (warp == 2 + kEpiWarps) {
    // Counts finished tiles: the release makes a whole CTA's stores visible and takes a microsecond or two, which the
    // epilogue warps do not wait for.
    int slot = 0;
    uint32_t phase = 0;
    for (;;) {
      if (!wait(&tile_done[slot], phase)) {
        if (aborted()) break;
        continue;                        // long dependencies elsewhere; the waits that matter give up by themselves
      }
      const int bi = tile_matrix[slot];
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&tile_free[slot]);
        if (bi >= 0) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.done + bi) : "memory");
      }
      if (bi < 0) break;
      if (++slot == kQueue) { slot = 0; phase ^= 1; }
    }
  } else {
    const int quad = warp & 3, group = (warp - 2) >> 2;
    constexpr int kCols = BN / epi_groups<BN>(), kUnits = kCols / 32;  // columns and units of this warp's share of a tile
    unsigned char* set = staging + (warp - 2) * kStagingWarp;
    uint64_t* res_bar = &res_bars[warp - 2];
    uint32_t fetch_phase = 0;
    int slot = 0, acc = 0;
    uint32_t qphase = 0, acc_phase = 0;
    // A tile counts for its matrix once its stores are complete, some microseconds after they were issued.  With another
    // task at hand the warp goes on and reports the tile a task later; without one it waits, since that task may wait
    // for this tile.
    int pending = -1;                                    // matrix of the tile not yet reported
    int tslot = 0;
    uint32_t tphase = 0;
    auto report = [&](int bi) {                          // the whole warp; this warp's stores of the tile are complete
      if (warp == 2) {                                   // one warp names the matrix
        if (!wait(&tile_free[tslot], tphase ^ 1)) give_up();
        if (lane == 0) tile_matrix[tslot] = bi;
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&tile_done[tslot]);
      if (++tslot == kQueue) { tslot = 0; tphase ^= 1; }
    };
    pdl_wait();
    while (!aborted()) {
      if (pending >= 0 && !__all_sync(0xffffffffu, mbar_test(&task_full[slot], qphase))) {
        if (elect_one()) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
        report(pending);
        pending = -1;
      }
      if (!wait(&task_full[slot], qphase)) { give_up(); break; }
      const int4 code = queue[slot];
      __syncwarp();
      if (lane == 0) arrive_leader(&task_empty[slot]);
      if (++slot == kQueue) { slot = 0; qphase ^= 1; }
      if (code.x < 0) break;
      const Task q{code.x >> 2, code.x & 3, code.y, code.z, code.w};
      const int kind = q.kind;
      const bool pair = q.step < p.keep, last = q.step == p.steps - 1;
      const bool res = kind == kUpdate && pair;          // a * (hi + lo / 2048) is added
      const bool has_res = kind == kPoly || res;
      const bool write_lo = kind == kUpdate && q.step + 1 < p.keep;
      const bool bf16 = kind == kUpdate && last;
      const float diag = kind == kPoly && !pair ? p.a : 0.f;  // a folded into B
      const CUtensorMap* r0 = kind == kPoly ? &maps.as : &maps.xs[q.step & 1];
      const CUtensorMap* r1 = &maps.ls[q.step & 1];
      const CUtensorMap* o0 = kind == kGram ? &maps.as : kind == kPoly ? &maps.bs : (last ? &maps.out : &maps.xs[(q.step & 1) ^ 1]);
      const CUtensorMap* o1 = &maps.ls[(q.step & 1) ^ 1];
      const int rows = kind == kUpdate ? p.m : p.p, cols = kind == kUpdate ? p.n : p.p;
      // A half block's 64 rows of a CTA lie in the upper lanes for the tile's left columns, in the lower for its right.
      const bool half = is_half(kind, q.mt);
      const int row0 = q.mt * TM + (half ? (int)rank * 64 + (quad & 1) * 32 : (int)rank * kBM + quad * 32);
      const int first = group * (half ? kCols / 2 : kCols);
      const int colw = q.nt * BN + first + (half ? (quad >> 1) * (BN / 2) : 0);
      const float4 cf = kind == kGram ? make_float4(0.f, 0.f, 1.f, 0.f) : p.coef[(long long)q.bi * p.steps + q.step];   // b, c, post
      const bool rows_in = row0 < rows;                  // else this warp's quarter lies below the matrix
      // make the staging buffer free and ask for the unit of the previous X or A that unit `u` needs
      auto fetch = [&](int u) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        if (!has_res) return;
        mbar_expect_tx(res_bar, res ? 2 * kUnit : kUnit);
        tma_load_3d(set, r0, colw + u * 32, row0, q.bi, res_bar);
        if (res) tma_load_3d(set + kUnit, r1, colw + u * 32, row0, q.bi, res_bar);
      };
      int units = rows_in ? (cols - colw + 31) / 32 : 0;   // units with any column of the matrix
      units = units < 0 ? 0 : min(units, half ? kUnits / 2 : kUnits);
      if (units > 0 && elect_one()) {
        if (PAIR && has_res) fence_async();              // the leader's does not cover this CTA's loads
        fetch(0);
      }
      __syncwarp();
      if (!wait(&acc_full[acc], acc_phase)) { give_up(); break; }
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN + first);
#pragma unroll 1
      for (int u = 0; u < units; ++u) {
        const int col0 = colw + u * 32;
        uint32_t v[32];
        tmem_ld_32x32(taddr + (uint32_t)(u * 32), v);
        if (u > 0) {
          if (elect_one()) fetch(u);
          __syncwarp();
        }
        if (has_res) {
          if (!wait(res_bar, fetch_phase)) give_up();
          fetch_phase ^= 1;
        }
        tmem_ld_wait();
        // a unit below the diagonal whose mirror image no tile computes is stored there as well
        const bool mirror = kind != kUpdate && row0 > col0 && row0 / BN >= sym_cols<BN, TM>(col0 / TM, p.p);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          // 64-byte swizzle: 16-byte piece index xor bits 1-2 of the row
          const uint32_t off = (uint32_t)lane * 64 + ((((uint32_t)j >> 3) ^ (((uint32_t)lane >> 1) & 3)) << 4);
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(v[j + e]);
          if (kind == kPoly) {
            const uint4 r = *reinterpret_cast<const uint4*>(set + off);
            const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = unpack_h(rr[e]);
              x[2 * e] = fmaf(cf.y, x[2 * e], cf.x * f.x);
              x[2 * e + 1] = fmaf(cf.y, x[2 * e + 1], cf.x * f.y);
            }
            if (row0 + lane >= col0 + j && row0 + lane < col0 + j + 8) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (row0 + lane == col0 + j + e) x[e] += diag;
            }
          }
          if (res) {
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
          if (kind == kUpdate) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= cf.z;
          }
          uint32_t o[4];
          if (bf16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack_b(x[2 * e], x[2 * e + 1]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack_h(x[2 * e], x[2 * e + 1]);
          }
          *reinterpret_cast<uint4*>(set + off) = make_uint4(o[0], o[1], o[2], o[3]);
          if (write_lo) {
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
        if (elect_one()) {
          tma_store_3d(o0, set, col0, row0, q.bi);
          if (write_lo) tma_store_3d(o1, set + kUnit, col0, row0, q.bi);
          if (mirror) tma_store_3d(o0, set + kUnit, row0, col0, q.bi);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      tc_fence_before();
      __syncwarp();
      if (elect_one()) {
        arrive_leader(&acc_empty[acc]);
        for (int u = units; u < kUnits; ++u) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group %0;" ::"n"(kUnits) : "memory");   // all but this tile's
      }
      __syncwarp();
      if (pending >= 0) report(pending);
      pending = q.bi;
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (elect_one()) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
    if (!aborted()) {
      if (pending >= 0) report(pending);
      report(-1);
    }
  }

  tc_fence_before();
  __syncthreads();
  // After a wait that ran out, copies into this CTA's shared memory and products may still be in flight: give them
  // 20 ms to land before the memory is handed back.
  if (*abort_flag)
    for (int i = 0; i < 20000; ++i) __nanosleep(1000);
  if (PAIR) cluster_sync();          // nobody reaches into a CTA that has left
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    else tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------- whole matrices in one CTA

constexpr int kSmallP = 128, kSmallQ = 256;
constexpr int kSmallThreads = 256;
constexpr int kBlock = 128 * 64 * 2;           // 128 rows x 64 columns of fp16: one swizzled column block

struct SmallParams {
  const void* x;
  void* out;
  int m, n, p, q, tall;
  int steps, keep;
  float a, b, c, eps;
  int tmem_cols, acc_col;      // tensor memory: X (fp32) from column 0, the accumulator from acc_col
  int* status;
};

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Where 16-byte piece `piece` of row `row` lies in a column block (128-byte swizzle).
__device__ __forceinline__ uint32_t block_at(int row, int piece) {
  return (uint32_t)row * 128 + (uint32_t)((piece ^ (row & 7)) << 4);
}
// 32 consecutive columns (from c0, a multiple of 32) of a thread's row into a matrix of column blocks, as fp16.
__device__ __forceinline__ void put_row(unsigned char* mat, int row, int c0, const float (&v)[32]) {
  unsigned char* blk = mat + (c0 >> 6) * kBlock;
#pragma unroll
  for (int j = 0; j < 32; j += 8)
    *reinterpret_cast<uint4*>(blk + block_at(row, ((c0 & 63) + j) >> 3)) =
        make_uint4(pack_h(v[j], v[j + 1]), pack_h(v[j + 2], v[j + 3]), pack_h(v[j + 4], v[j + 5]), pack_h(v[j + 6], v[j + 7]));
}

// X is kept wide, (p, q), whatever the matrix' own orientation: element (r, c) is x[r][c] or, for tall ones, x[c][r].  A
// thread owns a row (as tensor memory is read) and one half of the columns.
template <typename T>
__global__ void __launch_bounds__(kSmallThreads, 1) ns_small_kernel(const SmallParams p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t bar;
  __shared__ uint32_t tmem_slot;
  __shared__ double part[kSmallThreads / 32];
  unsigned char* sx = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int qb = (p.q + 63) / 64, pb = (p.p + 63) / 64;    // column blocks
  unsigned char* sa = sx + qb * kBlock;
  unsigned char* sb = sa + pb * kBlock;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3, half = warp >> 2;
  const int row = quad * 32 + lane;
  const int n_gram = (p.p + 15) / 16 * 16, n_upd = (p.q + 15) / 16 * 16;
  if (threadIdx.x == 0) { mbar_init(&bar, 1); asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
  if (warp == 0) { tmem_alloc(&tmem_slot, (uint32_t)p.tmem_cols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now: a dependent's block that took tensor memory while this one still waits for its own would hold it until this
  // kernel's end
  pdl_trigger();
  const uint32_t tx = tmem_slot + ((uint32_t)(quad * 32) << 16), ta = tx + (uint32_t)p.acc_col;
  const uint32_t acc = tmem_slot + (uint32_t)p.acc_col;
  pdl_wait();
  // chunks of 32 columns that this thread's half covers
  const int xc0 = half ? (qb * 64 / 2 + 31) / 32 * 32 : 0, xc1 = half ? qb * 64 : (qb * 64 / 2 + 31) / 32 * 32;
  const int ac0 = half ? (pb * 64 / 2 + 31) / 32 * 32 : 0, ac1 = half ? pb * 64 : (pb * 64 / 2 + 31) / 32 * 32;

  // the matrix into tensor memory, and its norm
  const T* src = static_cast<const T*>(p.x) + (long long)blockIdx.x * p.m * p.n;
  const long long row_step = p.tall ? 1 : p.n, col_step = p.tall ? p.n : 1;
  double sum = 0.0;
  for (int c0 = xc0; c0 < xc1; c0 += 32) {
    uint32_t v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const bool in = row < p.p && c0 + j < p.q;
      const float f = in ? to_f32(src[row * row_step + (c0 + j) * col_step]) : 0.f;
      v[j] = __float_as_uint(f);
      sum = fma((double)f, (double)f, sum);
    }
    tmem_st_32x32(tx + (uint32_t)c0, v);
  }
  tmem_st_wait();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < kSmallThreads / 32; ++i) sum += part[i];
  const Scaling scaling(sum, p.eps);
  float bound = scaling.s;
  int k = scaling.k;
  for (int c0 = xc0; c0 < xc1; c0 += 32) {
    uint32_t v[32];
    float f[32];
    tmem_ld_32x32(tx + (uint32_t)c0, v);
    tmem_ld_wait();
    if (scaling.wide) {
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] = scaling.operator()<true>(__uint_as_float(v[j]));
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] = scaling.operator()<false>(__uint_as_float(v[j]));
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(f[j]);
    tmem_st_32x32(tx + (uint32_t)c0, v);
    put_row(sx, row, c0, f);
  }
  tmem_st_wait();

  uint32_t phase = 0;
  // every thread's operand writes are visible, the product runs ...
  auto begin = [&](const unsigned char* ma, const unsigned char* mb, bool b_mn, int n, int k) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0 && elect_one()) {
      const uint32_t idesc = instr_desc<__half>(n) | ((uint32_t)b_mn << 16);
      for (int i = 0; i < k; i += 16) {
        const uint64_t da = smem_desc_sw128(ma + (i >> 6) * kBlock) + (uint64_t)((i & 63) * 2 / 16);
        // as MN-major: 16 rows of K are 2048 bytes, the next 64 columns one block further
        uint64_t db = smem_desc_sw128(mb + (b_mn ? i * 128 : (i >> 6) * kBlock)) + (uint64_t)(b_mn ? 0 : (i & 63) * 2 / 16);
        if (b_mn) db = (db & ~((uint64_t)0x3fff << 16)) | (uint64_t)(kBlock >> 4) << 16;
        tc_mma_f16(acc, da, db, idesc, i != 0);
      }
      tc_commit(&bar);
    }
    __syncwarp();
  };
  // ... and every thread sees the accumulator
  auto finish = [&] {
    if (!mbar_wait_bounded(&bar, phase)) atomicExch(p.status, kStatusStageTimeout);
    phase ^= 1;
    tc_fence_after();
  };
  auto product = [&](const unsigned char* ma, const unsigned char* mb, bool b_mn, int n, int k) { begin(ma, mb, b_mn, n, k); finish(); };
  for (int step = 0; step < p.steps; ++step) {
    const bool pair = step < p.keep, last = step == p.steps - 1;
    begin(sx, sx, false, n_gram, n_upd);                         // A = X X^T
    const StepCoef cf = step_coef(p.a, p.b, p.c, bound, k, last);
    finish();
    for (int c0 = ac0; c0 < ac1; c0 += 32) {
      uint32_t v[32];
      float f[32];
      tmem_ld_32x32(ta + (uint32_t)c0, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] = row < p.p && c0 + j < p.p ? __uint_as_float(v[j]) : 0.f;
      put_row(sa, row, c0, f);
    }
    product(sa, sa, false, n_gram, n_gram);                      // A A
    for (int c0 = ac0; c0 < ac1; c0 += 32) {                     // B = b A + c A A (+ a on the diagonal)
      uint32_t v[32];
      float f[32];
      tmem_ld_32x32(ta + (uint32_t)c0, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        const uint4 r = *reinterpret_cast<const uint4*>(sa + (c0 >> 6) * kBlock + block_at(row, ((c0 & 63) + j) >> 3));
        const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 h = unpack_h(rr[e >> 1]);
          const bool in = row < p.p && c0 + j + e < p.p;
          f[j + e] = in ? fmaf(cf.c, __uint_as_float(v[j + e]), cf.b * (e & 1 ? h.y : h.x)) : 0.f;
          if (!pair && in && row == c0 + j + e) f[j + e] += p.a;
        }
      }
      put_row(sb, row, c0, f);
    }
    product(sb, sx, true, n_upd, n_gram);                        // B X
    for (int c0 = xc0; c0 < xc1; c0 += 32) {
      uint32_t v[32], w[32];
      float f[32];
      tmem_ld_32x32(ta + (uint32_t)c0, v);
      if (pair) tmem_ld_32x32(tx + (uint32_t)c0, w);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        f[j] = row < p.p && c0 + j < p.q ? __uint_as_float(v[j]) : 0.f;
        if (pair) f[j] = row < p.p && c0 + j < p.q ? fmaf(p.a, __uint_as_float(w[j]), f[j]) : 0.f;
      }
      if (cf.post != 1.f) {
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] *= cf.post;
      }
      if (last) {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + (long long)blockIdx.x * p.m * p.n;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (row < p.p && c0 + j < p.q) dst[row * row_step + (c0 + j) * col_step] = __float2bfloat16_rn(f[j]);
      } else {
        put_row(sx, row, c0, f);
        if (step + 1 < p.keep) {
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(f[j]);
          tmem_st_32x32(tx + (uint32_t)c0, w);
        }
      }
    }
    tmem_st_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_slot, (uint32_t)p.tmem_cols);
  }
}

// ------------------------------------------------------------------- norm and scaling

constexpr int kNormThreads = 256;
constexpr int kMaxChunks = 64;   // partial sums of squares of one matrix
constexpr int kMaxSteps = 100;   // the entry point's limit: the workspace has room for the coefficients of so many

template <typename T> __device__ __forceinline__ float load1(const T* p) { return to_f32(*p); }

// Sum of squares of one slice of one matrix, in 64 bits (fp32 squares of large gradients would overflow).
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
ns_square_kernel(const T* __restrict__ x, double* __restrict__ partial, long long per, long long chunk, int vec,
                 unsigned* __restrict__ done, unsigned* __restrict__ ticket) {
  __shared__ double part[kNormThreads / 32];
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) {   // the counters of the kernel after next
    done[blockIdx.y] = 0;
    if (blockIdx.y == 0) *ticket = 0;
  }
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

// One matrix' share of a block: 2^k X_0 as the fp16 pair, rows padded to `ld` elements (the padding is never read).
template <bool WIDE, typename T>
__device__ __forceinline__ void scale_matrix(const T* __restrict__ src, __half* __restrict__ dh, __half* __restrict__ dl,
                                             int rows, int cols, int ld, const Scaling& scaling, int vec) {
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
        const float x0 = scaling.template operator()<WIDE>(v[2 * e]), x1 = scaling.template operator()<WIDE>(v[2 * e + 1]);
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
      const float v = scaling.template operator()<WIDE>(load1(src + i));
      const __half h = __float2half_rn(v);
      dh[r * ld + c] = h;
      dl[r * ld + c] = __float2half_rn((v - __half2float(h)) * kLoScale);
    }
  }
}
// 2^k X_0 of every matrix, and the coefficients of its steps.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
ns_scale_kernel(const T* __restrict__ x, const double* __restrict__ partial, __half* __restrict__ hi,
                __half* __restrict__ lo, float4* __restrict__ coef, int rows, int cols, int ld, int n_chunks, int steps,
                float a, float b, float c, float eps, int vec) {
  pdl_trigger();
  pdl_wait();
  const int bi = blockIdx.y;
  // every warp adds the partial sums for itself: one thread's chain of loads would hold up the block
  double t = 0.0;
  for (int i = threadIdx.x & 31; i < n_chunks; i += 32) t += partial[(long long)bi * kMaxChunks + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const Scaling scaling(t, eps);
  const T* src = x + (long long)bi * rows * cols;
  __half* dh = hi + (long long)bi * rows * ld;
  __half* dl = lo + (long long)bi * rows * ld;
  if (scaling.wide) scale_matrix<true>(src, dh, dl, rows, cols, ld, scaling, vec);
  else scale_matrix<false>(src, dh, dl, rows, cols, ld, scaling, vec);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    float s = scaling.s;
    int k = scaling.k;
    for (int i = 0; i < steps; ++i) {
      const StepCoef cf = step_coef(a, b, c, s, k, i == steps - 1);
      coef[(long long)bi * steps + i] = make_float4(cf.b, cf.c, cf.post, 0.f);
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

inline long long pad8(long long v) { return (v + 7) / 8 * 8; }
inline size_t pad1k(size_t v) { return (v + 1023) / 1024 * 1024; }

struct Layout {
  size_t x[2], l[2], a, b, norm, coef, done, ticket, total;
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
  w.coef = at; at += pad1k((size_t)batch * kMaxSteps * sizeof(float4));
  w.ticket = at;                   // 8 bytes, the per-matrix counts behind them
  w.done = at + 8; at += pad1k(8 + (size_t)batch * sizeof(unsigned));
  w.total = at;
  return w;
}

template <int BN, bool PAIR>
cudaError_t launch_ns(const NsMaps& maps, NsParams p, int sms, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  constexpr int TM = tile_m<PAIR>();
  int dev = 0;
  cudaGetDevice(&dev);
  dev = dev < 0 || dev >= 64 ? 0 : dev;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(ns_kernel<BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ns_smem<BN, PAIR>());
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  p.sym_tiles = 0;
  for (int i = 0; i < (p.p + TM - 1) / TM; ++i) p.sym_tiles += sym_cols<BN, TM>(i, p.p);
  p.upd_n = (p.n + BN - 1) / BN;
  p.upd_tiles = (p.m + TM - 1) / TM * p.upd_n;
  const long long total = (long long)p.batch * p.steps * (2LL * p.sym_tiles + p.upd_tiles);
  if (total >= (1LL << 31)) return cudaErrorInvalidValue;
  p.total = (unsigned)total;
  const int workers = PAIR ? sms / 2 : sms;
  // the matrices whose A fits one wave, in two halves; the rest are the third group
  const int wave = workers / p.sym_tiles < p.batch ? workers / p.sym_tiles : p.batch;
  p.group1 = (wave + 1) / 2;
  p.group2 = wave - p.group1;
  // more workers than a product has tiles would only wait
  const long long most = (long long)p.batch * (p.sym_tiles > p.upd_tiles ? p.sym_tiles : p.upd_tiles);
  const unsigned grid = (unsigned)(most < workers ? most : workers) * (PAIR ? 2 : 1);
  if (!PAIR) return launch_overlapped(ns_kernel<BN, PAIR>, dim3(grid), dim3(ns_threads<BN>()), ns_smem<BN, PAIR>(), s, maps, p);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(ns_threads<BN>());
  cfg.dynamicSmemBytes = ns_smem<BN, PAIR>();
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, ns_kernel<BN, PAIR>, maps, p);
}

template <typename T>
cudaError_t prepare(const void* x, const Layout& w, unsigned char* ws, long long batch, int m, int n, int steps, float a,
                    float b, float c, float eps, int sms, cudaStream_t s) {
  const long long per = (long long)m * n;
  const bool vec = n % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  // slices of a matrix: four blocks per SM over the stack, at most 64 to a matrix (a single one leaves SMs idle here), each a
  // whole number of vector rounds
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
                                    src, partial, per, chunk, (int)vec, reinterpret_cast<unsigned*>(ws + w.done),
                                    reinterpret_cast<unsigned*>(ws + w.ticket));
  if (e != cudaSuccess) return e;
  long long blocks = (8LL * sms + batch - 1) / batch;
  if (blocks > most) blocks = most;
  return launch_overlapped(ns_scale_kernel<T>, dim3((unsigned)blocks, (unsigned)batch), dim3(kNormThreads), 0, s, src,
                           (const double*)partial, reinterpret_cast<__half*>(ws + w.x[0]),
                           reinterpret_cast<__half*>(ws + w.l[0]), reinterpret_cast<float4*>(ws + w.coef), m, n, w.ldn,
                           (int)chunks, steps, a, b, c, eps, (int)vec);
}

bool small(int m, int n) { return (m < n ? m : n) <= kSmallP && (m < n ? n : m) <= kSmallQ; }

template <typename T>
cudaError_t launch_small(SmallParams p, long long batch, size_t smem, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaGetDevice(&dev);
  dev = dev < 0 || dev >= 64 ? 0 : dev;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(ns_small_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (kSmallQ / 64 + 2 * kSmallP / 64) * kBlock + 1024);
  });
  if (attr_err[dev] != cudaSuccess) return attr_err[dev];
  return launch_overlapped(ns_small_kernel<T>, dim3((unsigned)batch), dim3(kSmallThreads), smem, s, p);
}

}  // namespace

size_t ns_workspace_bytes(long long batch, int m, int n) { return small(m, n) ? 0 : layout_of(batch, m, n).total; }

// dtype: 0 fp32, 1 fp16, 2 bf16 of x; out is bf16.
cudaError_t launch_newton_schulz(int dtype, const void* x, void* out, void* workspace, long long batch, int m, int n,
                                 int steps, float a, float b, float c, float eps, int sms, int* status, cudaStream_t s) {
  if (small(m, n)) {
    SmallParams p = {};
    p.x = x; p.out = out; p.m = m; p.n = n; p.tall = m > n;
    p.p = p.tall ? n : m; p.q = p.tall ? m : n;
    p.steps = steps; p.keep = steps - 2;
    p.a = a; p.b = b; p.c = c; p.eps = eps; p.status = status;
    const int qb = (p.q + 63) / 64, pb = (p.p + 63) / 64;
    p.acc_col = qb * 64;
    p.tmem_cols = 128;
    while (p.tmem_cols < 2 * qb * 64) p.tmem_cols *= 2;       // X, and an accumulator as wide (p <= q)
    const size_t smem = (size_t)(qb + 2 * pb) * kBlock + 1024;
    return dtype == 0 ? launch_small<float>(p, batch, smem, s)
           : dtype == 1 ? launch_small<__half>(p, batch, smem, s) : launch_small<__nv_bfloat16>(p, batch, smem, s);
  }
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Layout w = layout_of(batch, m, n);
  cudaError_t e = dtype == 0   ? prepare<float>(x, w, ws, batch, m, n, steps, a, b, c, eps, sms, s)
                  : dtype == 1 ? prepare<__half>(x, w, ws, batch, m, n, steps, a, b, c, eps, sms, s)
                               : prepare<__nv_bfloat16>(x, w, ws, batch, m, n, steps, a, b, c, eps, sms, s);
  if (e != cudaSuccess) return e;
  const bool direct = n % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  NsParams p = {};
  p.m = m; p.n = n; p.tall = m > n;
  p.p = p.tall ? n : m; p.q = p.tall ? m : n;
  p.steps = steps; p.keep = steps - 2;
  p.batch = (int)batch;
  p.a = a;
  p.coef = reinterpret_cast<const float4*>(ws + w.coef);
  p.done = reinterpret_cast<unsigned*>(ws + w.done);
  p.ticket = reinterpret_cast<unsigned*>(ws + w.ticket);
  p.status = status;
  NsMaps maps;
  bool ok = true;
  for (int i = 0; i < 2; ++i) {
    ok = ok && map3(&maps.x[i], false, ws + w.x[i], batch, m, n, w.ldn, 64, 64);
    ok = ok && map3(&maps.xs[i], false, ws + w.x[i], batch, m, n, w.ldn, 32, 32);
    ok = ok && map3(&maps.ls[i], false, ws + w.l[i], batch, m, n, w.ldn, 32, 32);
  }
  ok = ok && map3(&maps.a, false, ws + w.a, batch, p.p, p.p, w.ldp, 64, 64) &&
       map3(&maps.b, false, ws + w.b, batch, p.p, p.p, w.ldp, 64, 64) &&
       map3(&maps.as, false, ws + w.a, batch, p.p, p.p, w.ldp, 32, 32) &&
       map3(&maps.bs, false, ws + w.b, batch, p.p, p.p, w.ldp, 32, 32);
  // a result whose rows 16-byte stores cannot address goes through the padded buffer the last step does not read
  ok = ok && (direct ? map3(&maps.out, true, out, batch, m, n, n, 32, 32)
                     : map3(&maps.out, true, ws + w.x[steps & 1], batch, m, n, w.ldn, 32, 32));
  if (!ok) return cudaErrorNotSupported;
  // Tile width: the widest whose update still gives every SM a tile.  The widest also goes to pairs of CTAs where products
  // are long enough to gain from their smaller traffic (pairs over single CTAs: 1 x 4000x6000 0.81, 3 x 896x7000 0.76,
  // 5 x 5120x1280 0.91); in short ones the hand-over between two CTAs costs as much (30 x 768x768 1.05, 22 x 640x2560 1.01,
  // 18 x 512x2048 1.00, 40 x 320x1280 1.12).
  const long long rows = (m + kBM - 1) / kBM;
  if (batch * rows * ((n + 255) / 256) >= sms)
    e = p.p > 768 ? launch_ns<256, true>(maps, p, sms, s) : launch_ns<256, false>(maps, p, sms, s);
  else
    e = batch * rows * ((n + 127) / 128) >= sms ? launch_ns<128, false>(maps, p, sms, s) : launch_ns<64, false>(maps, p, sms, s);
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
