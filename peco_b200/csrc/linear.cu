// Linear layers of a transformer block with their epilogue, and their gradient.
//
//   out[m, n] = residual[m, n] + gate[sample(m), n] * act(sum_k x[m, k] W[n, k] + bias[n])
//
// x may be given as two inputs side by side (the attention rows and the MLP
// hidden of a single-stream block), which replaces their concatenation.
// Gradient, with z the pre-activation and g the gradient of out:
//   dz = g * gate * act'(z);  dx = dz W;  dW = dz^T x;  dbias = sum_m dz;
//   dgate[b, n] = sum over the sample's rows of g * act(z).
//
// All three products run through one tcgen05 kernel, D[M, N] = sum_k A[m, k]
// B[n, k], whose operands are read in place by TMA whichever of their two
// dimensions is contiguous (K-major, or MN-major for W in dx and for both
// operands of dW).  Operands that TMA cannot address (a base or row stride
// that is not a multiple of 16 bytes) are first copied to rows that it can.
#include "common.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"
#include "rows.cuh"

#include <atomic>
#include <type_traits>

namespace peco {
namespace {

enum Activation : int { kActNone = 0, kActGeluTanh = 1, kActGelu = 2, kActSilu = 3 };

constexpr int kTileM = 128;
constexpr int kTileK = 64;   // one 128-byte swizzle panel of 16-bit elements
constexpr int kEpilogueWarps = 8;
constexpr int kGemmThreads = 96 + 32 * kEpilogueWarps;  // TMA warp for A, MMA warp, epilogue warps, TMA warp for B

struct GemmArgs {
  CUtensorMap a[2], b[2];    // K segments (x and x2; the second unused otherwise)
  int kblocks[2];            // 64-wide K blocks of each segment
  int m, n, tiles_m, tiles_n;
  int bn;                    // columns of an accumulator, a multiple of 32
  int band;                  // m tiles walked together
  int a_panels, b_panels;    // 64-wide panels of an MN-major operand per CTA
  int a_joined, b_joined;    // ... all of them in one copy (the operand's width is a multiple of 64)
  int stages;                // of the ring in shared memory
  uint32_t a_bytes, b_bytes; // one operand tile in a stage; B's once per accumulator
  uint32_t stage_bytes;      // what one CTA loads per K block, and a stage's size
  void* out;
  long long out_stride;
  // epilogue operands (null where absent)
  const void* bias;          // [n]
  const void* gate;          // [samples, n], rows gate_stride apart
  long long gate_stride;
  int rows_per_sample;
  const void* residual;
  long long res_stride;
  void* preact;              // [m, n] rounded copy of the pre-activation
  int act;
  int vec;                   // every row of every [m, n] operand starts on 16 bytes and n % 8 == 0
  unsigned* status;
};

// ---- activations -------------------------------------------------------------
// Evaluated in fp32.  gelu_tanh is written as z * sigmoid(2u), u = sqrt(2/pi)
// (z + 0.044715 z^3): the exponential keeps full relative precision in the
// negative tail, where 1 + tanh(u) would cancel.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGelu1 = 2.0f * 0.7978845608028654f;  // 2u = z (kGelu1 + kGelu3 z^2)
constexpr float kGelu3 = kGelu1 * 0.044715f;

// 1 / x from the hardware's approximate reciprocal (within an ulp; infinity gives 0)
__device__ __forceinline__ float recip_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(z) of a pair, the normal distribution's integral, and exp(-z^2 / 2).  With
// t = 1 / (1 + 0.36 |z|), Phi(-|z|) exp(z^2 / 2) / t is smooth in t down to its
// limit at t = 0, so a polynomial (fitted for the least relative error over
// 0 <= |z| <= 13.2: 2^-20.4) times the exponential keeps its relative precision
// in the negative tail, where 1 + erf would cancel.  In fp32 the exponential's
// argument rounds too: about 2^-18 of the value down to z = -8, 2^-17 down to -12.8,
// where the exponential nears the smallest normal number.
__device__ __forceinline__ float2 normal_integral_pair(float2 z, float2& bell) {
  auto both = [](float x) { return make_float2(x, x); };
  const float2 d = ffma2(make_float2(fabsf(z.x), fabsf(z.y)), both(0.36f), both(1.0f));
  const float2 t = make_float2(recip_approx(d.x), recip_approx(d.y));
  float2 poly = ffma2(t, both(0.04752533882856369f), both(-0.18137013912200928f));
  poly = ffma2(t, poly, both(0.1831398457288742f));
  poly = ffma2(t, poly, both(0.025042641907930374f));
  poly = ffma2(t, poly, both(0.14027050137519836f));
  poly = ffma2(t, poly, both(0.1416715383529663f));
  poly = ffma2(t, poly, both(0.14372023940086365f));
  const float2 w = fmul2(fmul2(z, z), both(-0.5f * kLog2e));
  bell = make_float2(exp2_approx(w.x), exp2_approx(w.y));
  const float2 tail = fmul2(fmul2(poly, t), bell);
  return make_float2(z.x > 0.0f ? 1.0f - tail.x : tail.x, z.y > 0.0f ? 1.0f - tail.y : tail.y);
}

// (act(z), act'(z)) of a pair; the value only where ``value`` is set.  A saved
// pre-activation may be infinite where its 16-bit type ended (fp16: past 65504):
// in products, where a factor vanishes or meets a zero gradient, it is held
// finite (a NaN comes back through the other factor).
template <int ACT, bool VALUE>
__device__ __forceinline__ void activate_slope2(float2 z, float2& value, float2& slope) {
  auto both = [](float x) { return make_float2(x, x); };
  auto held = [](float x) { return fminf(fmaxf(x, -1e30f), 1e30f); };
  const float2 f = make_float2(held(z.x), held(z.y));
  if constexpr (ACT == kActGeluTanh) {
    const float2 z2 = fmul2(z, z);
    const float2 w = fmul2(z, ffma2(z2, both(-kLog2e * kGelu3), both(-kLog2e * kGelu1)));
    const float2 e = fadd2(make_float2(exp2_approx(w.x), exp2_approx(w.y)), both(1.0f));
    const float2 s = make_float2(recip_approx(e.x), recip_approx(e.y));
    // s + z s (1 - s) d(2u)/dz
    float2 d = fmul2(z, ffma2(z2, both(3.0f * kGelu3), both(kGelu1)));
    d = make_float2(held(d.x), held(d.y));
    const float2 rest = ffma2(make_float2(-s.x, -s.y), d, d);
    slope = ffma2(s, rest, s);
    if (VALUE) value = fmul2(f, s);
  } else if constexpr (ACT == kActGelu) {
    float2 bell;
    const float2 p = normal_integral_pair(z, bell);
    slope = ffma2(fmul2(f, both(0.3989422804014327f)), bell, p);
    if (VALUE) value = fmul2(f, p);
  } else if constexpr (ACT == kActSilu) {
    const float2 w = fmul2(z, both(-kLog2e));
    const float2 e = fadd2(make_float2(exp2_approx(w.x), exp2_approx(w.y)), both(1.0f));
    const float2 s = make_float2(recip_approx(e.x), recip_approx(e.y));
    const float2 rest = ffma2(make_float2(-s.x, -s.y), f, f);  // z (1 - s)
    slope = ffma2(s, rest, s);
    if (VALUE) value = fmul2(f, s);
  } else {
    value = z;
    slope = both(1.0f);
  }
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// Bounded wait of a whole warp: one try by every lane, then as mbar_wait_warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t phase, volatile int* abort_flag, unsigned* status) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, phase))) return true;
  return mbar_wait_warp(bar, phase, abort_flag, status);
}

// ---- CTA pairs -------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same shared-memory location in CTA ``rank`` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Arrive on a barrier of another CTA of the cluster.  What it orders is the TMEM
// reads before it (waited for, with the tcgen05 fence); a release at cluster
// scope would also wait for all the warp's global stores.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <int CG>
__device__ __forceinline__ void tile_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {  // the barrier may be the pair's first CTA's
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void tile_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void product_step(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1) {
    umma_ss(d, a, b, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Two products of a pair with one A operand, into two accumulators: the second
// takes A from the collector that the first filled, not from shared memory again.
__device__ __forceinline__ void product_step_twice(uint32_t d0, uint32_t d1, uint64_t a, uint64_t b0, uint64_t b1,
                                                   uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16.collector::a::fill [%0], %2, %3, %5, p;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16.collector::a::lastuse [%1], %2, %4, %5, p;\n\t}" ::"r"(d0),
      "r"(d1), "l"(a), "l"(b0), "l"(b1), "r"(idesc)
      : "memory");
}

// Arrive on ``bar`` (of both CTAs of a pair, whose first has rank ``lead``) once
// the products issued so far are done.
template <int CG>
__device__ __forceinline__ void product_commit(uint64_t* bar, uint32_t lead) {
  if constexpr (CG == 1) {
    umma_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3u << lead))
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_take(uint32_t* slot, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 1) tmem_dealloc(addr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}

// ---- the product -----------------------------------------------------------------
// Output tiles of (128 CG) x bn, walked by persistent groups of CG CTAs.  Two
// warps of every CTA stream its 64-wide K blocks of A (128 rows) and B (bn / CG
// rows) through a ring of shared-memory stages; warp 1 of the group's first
// CTA issues the MMAs into one of two TMEM accumulators; warps 2-9 read the
// other one back, apply the epilogue and store, so the epilogue of a tile runs
// under the MMAs of the next.
//
// CG = 2 pairs two SMs on one tile: each CTA stages half of A's rows and half
// of B's, so a 256 x 256 tile costs 32 KB of shared memory and of TMA traffic
// per SM and K block, for twice the products of a 128 x 128 tile.
//
// WIDE (with CG = 2): the tile is 256 x 2 bn, both accumulators hold one half of
// it and share A's stage (and A's trip from shared memory).  At the tensor
// core's full rate a 256 x 256 tile draws 64 bytes per clock and SM from L2, a
// 256 x 512 one 48, and long products run at the board's power limit, where
// traffic costs time.  The price is that a tile's epilogue no longer hides
// entirely: the first K blocks' products go to the half that is drained first,
// the last ones' finish that half first.  Back to back for half a second each:
// 6750 x 12288 x 3072 387 us wide and 426 not, the weight gradient of 6750 x
// 3072 x 12288 372 and 400; but 6750 x 3072 x 12288, with four times as many
// epilogues per product, 414 and 397.
//
// SPLIT: one tile per cluster of S groups, each taking a range of the K
// blocks and finishing a share of the tile's columns: the groups store their
// fp32 partials of a share into its group's drained ring, which adds them in a
// fixed order to its own.
//
// What it measured (B200, cold weights): 1 x 3072 x 18432 23 us (4.9 TB/s of
// weights; bound by HBM and the start of the kernel), 256 x 3072 x 12288 with
// gelu 23 us, 256 x 12288 x 3072 26 us (split), 6750 x 3072 x 12288 with gelu 378
// us (1.35 PFLOP/s at the power limit, 335 us and 1.52 PFLOP/s in short runs),
// 7006 x 15360 x 3072 with gate and residual 543 us; the large ones are bound by
// the tensor core and the power limit.
constexpr int kRingBytes = 192 * 1024;
constexpr int kMaxStages = 24;                  // stages hold what a tile needs: small ones have many in flight
constexpr int kStageRow = 32;                    // columns an epilogue warp finishes at a time
constexpr int kStagingBytes = kEpilogueWarps * 32 * kStageRow * 2;
constexpr int kVectorBytes = 2 * 2 * 256 * 4;    // bias and gate of two accumulators' columns, fp32
constexpr int kGemmSmem = kRingBytes + kStagingBytes + kVectorBytes + 1024;  // + alignment slack

struct GemmShared {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem;
  int abort_flag;
};

// (m tile, n tile) of a linear tile number: bands of ``band`` m tiles, walked
// down first.
__device__ __forceinline__ void tile_coords(const GemmArgs& args, int t, int& tm, int& tn) {
  const int per_band = args.band * args.tiles_n;
  const int band = t / per_band;
  const int first = band * args.band;
  const int height = min(args.band, args.tiles_m - first);
  const int in = t - band * per_band;
  tn = in / height;
  tm = first + in - tn * height;
}

// Operand rows x 64 into shared memory: K-major rows of 128 bytes (one box), or
// MN-major panels of 64 elements x 64 K rows, in one copy of a [panel][K][64]
// view where the operand's width allows it
template <int CG, bool MN>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int row0, int panels, int joined, int k0,
                                          uint32_t bar) {
  if constexpr (!MN) {
    tile_load_2d<CG>(dst, map, k0, row0, bar);
  } else if (joined) {
    tile_load_3d<CG>(dst, map, 0, k0, row0 >> 6, bar);
  } else {
    for (int p = 0; p < panels; ++p) tile_load_2d<CG>(dst + p * 8192, map, row0 + p * 64, k0, bar);
  }
}

// what the k-th 16-wide K step of a tile adds to its descriptor's address (16-byte units)
template <bool MN>
__device__ __forceinline__ constexpr uint32_t step_offset(int k) { return MN ? k * 128 : k * 2; }
template <bool MN>
__device__ __forceinline__ uint64_t tile_desc(uint32_t base) {
  return MN ? smem_desc(base, 8192, 1024) : smem_desc(base, 16, 1024);
}

// Position in the ring: stage and the phase of its barriers.
struct RingPos {
  int s;
  uint32_t phase;
  __device__ __forceinline__ void step(int stages) {
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
};

template <typename T, bool EPI>
__device__ __forceinline__ const T* gate_row(const GemmArgs& args, long long row) {
  if (!EPI || !args.gate || row >= args.m) return nullptr;
  return static_cast<const T*>(args.gate) + (args.gate_stride ? (row / args.rows_per_sample) * args.gate_stride : 0);
}

// Waits for the TMEM loads in flight and ties ``r`` to the wait, so that no use
// of it is scheduled earlier.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(addr) : "memory");
  return f;
}
// to another CTA's shared memory (``addr`` from map_rank)
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// act of 16 pairs
template <int ACT>
__device__ __forceinline__ void activate_pairs(float2 (&v)[16]) {
  auto both = [](float x) { return make_float2(x, x); };
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (ACT == kActGelu) {
      float2 bell;
      v[j] = fmul2(v[j], normal_integral_pair(v[j], bell));
    } else {
      // z / (1 + 2^w), each element by itself: a NaN stays in its column
      float2 w;
      if constexpr (ACT == kActGeluTanh) w = fmul2(v[j], ffma2(fmul2(v[j], v[j]), both(-kLog2e * kGelu3), both(-kLog2e * kGelu1)));
      else w = fmul2(v[j], both(-kLog2e));
      const float2 e = fadd2(make_float2(exp2_approx(w.x), exp2_approx(w.y)), both(1.0f));
      v[j] = fmul2(v[j], make_float2(recip_approx(e.x), recip_approx(e.y)));
    }
  }
}

__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 2, %0;" ::"n"(32 * kEpilogueWarps) : "memory"); }

// One chunk of 32 x 32 results (``lane`` holds row ``lane``) to ``out`` through
// the warp's staging block: 64-byte rows whose 16-byte pieces are XORed with the
// row, free of bank conflicts both ways, so that stores cover whole sectors.
__device__ __forceinline__ uint32_t staging_offset(int row, int piece) { return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); }

template <typename T>
__device__ __forceinline__ void store_chunk(const GemmArgs& args, uint32_t staging, const float2 (&v)[16], T* out,
                                            long long stride, long long row0, int col, int col_end, int lane) {
#pragma unroll
  for (int p = 0; p < 4; ++p)
    st_shared_v4(staging + staging_offset(lane, p), pack2<T>(v[4 * p].x, v[4 * p].y), pack2<T>(v[4 * p + 1].x, v[4 * p + 1].y),
                 pack2<T>(v[4 * p + 2].x, v[4 * p + 2].y), pack2<T>(v[4 * p + 3].x, v[4 * p + 3].y));
  __syncwarp();
  if (args.vec) {
    const int piece = lane & 3;
    if (col + piece * 8 < col_end) {
      T* p = out + (row0 + (lane >> 2)) * stride + col + piece * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2);
        const float4 f = ld_shared_v4(staging + staging_offset(r, piece));
        if (row0 + r < args.m) *reinterpret_cast<float4*>(p + i * 8 * stride) = f;
      }
    }
  } else if (col + lane < col_end) {
    // a column per lane, one row at a time
    const int rows = static_cast<int>(min(32LL, args.m - row0));
    uint16_t* p = reinterpret_cast<uint16_t*>(out) + row0 * stride + col + lane;
#pragma unroll 4
    for (int r = 0; r < rows; ++r, p += stride) {
      uint16_t u;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(staging + staging_offset(r, lane >> 3) + (lane & 7) * 2));
      *p = u;
    }
  }
  __syncwarp();
}

// The residual's chunk, in the layout of the results, added to them.
template <typename T>
__device__ __forceinline__ void fetch_residual(const GemmArgs& args, uint4 (&held)[4], long long row0, int col, int col_end,
                                               int lane) {
  const int piece = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + i * 8 + (lane >> 2);
    held[i] = make_uint4(0, 0, 0, 0);
    if (row < args.m && col + piece * 8 < col_end)
      held[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(args.residual) + row * args.res_stride + col + piece * 8);
  }
}
template <typename T>
__device__ __forceinline__ void add_residual(const GemmArgs& args, uint32_t staging, const uint4 (&held)[4], float2 (&v)[16],
                                             long long row0, int col, int col_end, int lane) {
  if (args.vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      st_shared_v4(staging + staging_offset(i * 8 + (lane >> 2), lane & 3), held[i].x, held[i].y, held[i].z, held[i].w);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(args.residual) + row0 * args.res_stride + col + lane;
    const int rows = col + lane < col_end ? static_cast<int>(min(32LL, args.m - row0)) : 0;
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 16) {  // sixteen loads in flight
      uint16_t u[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) u[r] = r0 + r < rows ? p[(r0 + r) * args.res_stride] : static_cast<uint16_t>(0);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(staging + staging_offset(r0 + r, lane >> 3) + (lane & 7) * 2), "h"(u[r]) : "memory");
    }
  }
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float4 f = ld_shared_v4(staging + staging_offset(lane, p));
    const uint32_t w[4] = {__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * p + i] = fadd2(v[4 * p + i], unpack2<T>(w[i]));
  }
  __syncwarp();
}

// bias (0: none) and gate of ``cols`` columns into ``vectors``, where the whole
// tile has one gate row; every epilogue thread takes one column
template <typename T>
__device__ __forceinline__ void stage_vectors(const GemmArgs& args, float* vectors, const T* gate, int col0, int cols,
                                              int thread) {
  const int col = col0 + thread;
  const bool inside = thread < cols && col < args.n;
  vectors[thread] = inside && args.bias ? to_f32<T>(static_cast<const T*>(args.bias)[col]) : 0.0f;
  vectors[256 + thread] = inside && gate ? to_f32<T>(gate[col]) : 1.0f;
}

// The epilogue of one accumulator by one of its 8 warps: TMEM lanes of its
// quarter (a row per lane), every other chunk of 32 columns.  A chunk's results
// are computed in pairs where they lie, rounded, and leave through the staging
// block; the next chunk's TMEM load is in flight meanwhile.
template <typename T, bool EPI>
__device__ __forceinline__ void finish_chunk(const GemmArgs& args, float2 (&v)[16], uint32_t staging,
                                             const float* vectors, const T* own_gate, long long row0, int col0, int c,
                                             int col_end, int lane) {
  const int col = col0 + c * kStageRow;
  if (col >= col_end) return;  // uniform over the warp
  if constexpr (EPI) {
    uint4 held[4];
    if (args.residual && args.vec) fetch_residual<T>(args, held, row0, col, col_end, lane);
    if (args.bias) {
      const float4* b = reinterpret_cast<const float4*>(vectors + c * kStageRow);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 f = b[j];
        v[2 * j] = fadd2(v[2 * j], make_float2(f.x, f.y));
        v[2 * j + 1] = fadd2(v[2 * j + 1], make_float2(f.z, f.w));
      }
    }
    if (args.preact) store_chunk<T>(args, staging, v, static_cast<T*>(args.preact), args.n, row0, col, col_end, lane);
    switch (args.act) {
      case kActGeluTanh: activate_pairs<kActGeluTanh>(v); break;
      case kActGelu: activate_pairs<kActGelu>(v); break;
      case kActSilu: activate_pairs<kActSilu>(v); break;
      default: break;
    }
    if (own_gate) {  // rows of several samples: each lane reads its own row's gate
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float g[8];
        const int count = min(8, col_end - col - 8 * p);
        if (count <= 0) continue;
        load8(own_gate + col + 8 * p, args.vec, count, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * p + i] = fmul2(v[4 * p + i], make_float2(g[2 * i], g[2 * i + 1]));
      }
    } else if (args.gate) {
      const float4* g = reinterpret_cast<const float4*>(vectors + 256 + c * kStageRow);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 f = g[j];
        v[2 * j] = fmul2(v[2 * j], make_float2(f.x, f.y));
        v[2 * j + 1] = fmul2(v[2 * j + 1], make_float2(f.z, f.w));
      }
    }
    if (args.residual) add_residual<T>(args, staging, held, v, row0, col, col_end, lane);
  }
  store_chunk<T>(args, staging, v, static_cast<T*>(args.out), args.out_stride, row0, col, col_end, lane);
}

template <typename T, bool EPI>
__device__ __forceinline__ void finish_tile(const GemmArgs& args, uint32_t tmem, uint32_t staging, const float* vectors,
                                            const T* own_gate, long long row0, int col0, int lane, int half) {
  const int col_end = min(args.n, col0 + args.bn);
  const int chunks = args.bn / kStageRow;
  uint32_t acc[32];
  if (half < chunks) tmem_ld32(tmem + half * kStageRow, acc);
#pragma unroll 1
  for (int c = half; c < chunks; c += 2) {
    tmem_ld_wait_for(acc);
    float2 v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = make_float2(__uint_as_float(acc[2 * j]), __uint_as_float(acc[2 * j + 1]));
    if (c + 2 < chunks) tmem_ld32(tmem + (c + 2) * kStageRow, acc);
    finish_chunk<T, EPI>(args, v, staging, vectors, own_gate, row0, col0, c, col_end, lane);
  }
}

// The column chunks of a split tile that one of its groups finishes.
struct OwnChunks {
  int begin, end;
};
__device__ __forceinline__ OwnChunks own_chunks(int chunks, int part, int splits) {
  return OwnChunks{chunks * part / splits, chunks * (part + 1) / splits};
}
constexpr int kChunkBytes = kTileM * kStageRow * 4;  // fp32 partial of a chunk: [4 columns][128 rows][16 bytes]

template <typename T, int CG, bool SPLIT, bool WIDE, bool AMN, bool BMN, bool EPI>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs args, int splits) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ GemmShared sh;
  const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = CG == 1 && !SPLIT ? 0 : cluster_rank();
  const uint32_t rank = CG == 1 ? 0 : cta & 1, lead = cta - rank;  // within the pair; the pair's first CTA
  volatile int* abort_flag = &sh.abort_flag;
  constexpr uint32_t kAccumulator = CG == 1 ? 128 : 256;  // columns between the two accumulators
  const int stages = args.stages;
  constexpr int kHalves = WIDE ? 2 : 1;  // accumulators per tile
  if (lane == 0 && (warp == 0 || warp == kEpilogueWarps + 2)) {
    prefetch_tensormap(warp == 0 ? &args.a[0] : &args.b[0]);
    if (args.kblocks[1]) prefetch_tensormap(warp == 0 ? &args.a[1] : &args.b[1]);
  }
  if (threadIdx.x == 64) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh.acc_full[b], 1);
      mbar_init(&sh.acc_empty[b], CG * kEpilogueWarps);
    }
    sh.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_take<CG>(&sh.tmem, 2 * kAccumulator);
  tc_fence_before();
  __syncthreads();
  if (CG > 1) cluster_sync();  // the pair's barriers are ready before either CTA signals the other
  tc_fence_after();
  wait_for_prior();
  let_next_start();
  const uint32_t tmem = sh.tmem;
  const int tiles = args.tiles_m * args.tiles_n;
  const int kb0 = args.kblocks[0], kblocks = kb0 + args.kblocks[1];
  // persistent: tiles group, group + groups, ...; split: this cluster's one tile
  const int group = SPLIT ? blockIdx.x / (CG * splits) : blockIdx.x / CG;
  const int groups = SPLIT ? tiles : gridDim.x / CG;
  const int part = SPLIT ? static_cast<int>(cta) / CG : 0;
  const int kb_begin = SPLIT ? static_cast<int>(static_cast<long long>(kblocks) * part / splits) : 0;
  const int kb_end = SPLIT ? static_cast<int>(static_cast<long long>(kblocks) * (part + 1) / splits) : kblocks;

  // The feeding and issuing warps run their loops whole, so that addresses and
  // descriptors stay in uniform registers, and one elected lane issues.
  if (warp == 0 || warp == kEpilogueWarps + 2) {
    // ------------------------------------------- TMA: one warp for A, one for B
    const bool is_a = warp == 0, issuer = elect_one();
    bool ok = true;
    RingPos pos{0, 0};
    // the pair's stages fill one barrier, the first CTA's, which expects both CTAs' bytes
    const uint32_t bar0 = CG > 1 ? map_rank(smem_u32(&sh.full[0]), lead) : smem_u32(&sh.full[0]);
    for (int t = group; t < tiles && ok; t += groups) {
      int tm, tn;
      tile_coords(args, t, tm, tn);
      const int row0 = is_a ? (tm * CG + rank) * kTileM : tn * kHalves * args.bn + rank * (args.bn / CG);
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        ok = warp_wait(&sh.empty[pos.s], pos.phase ^ 1, abort_flag, args.status);
        if (!ok) break;
        const uint32_t st = ring + pos.s * args.stage_bytes, bar = bar0 + pos.s * 8;
        const int seg = kb >= kb0 ? 1 : 0;
        const int k0 = (kb - (seg ? kb0 : 0)) * kTileK;
        if (issuer) {
          if (is_a) {
            if (rank == 0) mbar_arrive_expect_tx(&sh.full[pos.s], CG * args.stage_bytes);
            load_tile<CG, AMN>(st, &args.a[seg], row0, args.a_panels, args.a_joined, k0, bar);
          } else {
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
              load_tile<CG, BMN>(st + args.a_bytes + h * args.b_bytes, &args.b[seg], row0 + h * args.bn, args.b_panels,
                                 args.b_joined, k0, bar);
          }
        }
        __syncwarp();
        pos.step(stages);
      }
    }
    // after an expired wait: time for the copies still in flight to land before the CTA ends
    if (!ok) {
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (rank == 0) {
      constexpr int ab = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      const bool issuer = elect_one();
      const uint32_t idesc = instr_desc(kTileM * CG, args.bn, ab, AMN, BMN);
      const uint64_t desc_a = tile_desc<AMN>(ring), desc_b = tile_desc<BMN>(ring + args.a_bytes);
      const uint32_t stage_step = args.stage_bytes >> 4, half_step = args.b_bytes >> 4;
      bool ok = true;
      RingPos pos{0, 0};
      uint32_t local = 0;
      // one K block's products for one accumulator (``accumulate`` 0: overwriting it)
      auto products = [&](int s, int half, uint32_t acc, uint32_t accumulate) {
        const uint32_t at = s * stage_step, at_b = at + half * half_step;
        product_step<CG>(acc, desc_a + at, desc_b + at_b, idesc, accumulate);
#pragma unroll
        for (int k = 1; k < kTileK / 16; ++k)
          product_step<CG>(acc, desc_a + (at + step_offset<AMN>(k)), desc_b + (at_b + step_offset<BMN>(k)), idesc, 1);
      };
      auto wait_full = [&](const RingPos& p) {
        ok = warp_wait(&sh.full[p.s], p.phase, abort_flag, args.status);
        if (ok) tc_fence_after();
        return ok;
      };
      for (int t = group; t < tiles && ok; t += groups, ++local) {
        if constexpr (!WIDE) {
          const int b = local & 1;
          ok = warp_wait(&sh.acc_empty[b], ((local >> 1) & 1) ^ 1, abort_flag, args.status);
          if (!ok) break;
          tc_fence_after();
          for (int kb = kb_begin; kb < kb_end; ++kb) {
            if (!wait_full(pos)) break;
            if (issuer) {
              products(pos.s, 0, tmem + b * kAccumulator, kb > kb_begin);
              product_commit<CG>(&sh.empty[pos.s], lead);
            }
            __syncwarp();
            pos.step(stages);
          }
          if (ok && issuer) product_commit<CG>(&sh.acc_full[b], lead);
          __syncwarp();
        } else {
          // K blocks in order for each half; the second half trails the first by
          // up to a ring of stages at the tile's start and at its end
          const uint32_t free_phase = (local & 1) ^ 1;
          const int skew = min(stages, kblocks), last = max(skew, kblocks - stages);
          ok = warp_wait(&sh.acc_empty[0], free_phase, abort_flag, args.status);
          if (!ok) break;
          tc_fence_after();
          RingPos ahead = pos;
          auto first_half = [&](int kb) {
            if (!wait_full(ahead)) return;
            if (issuer) products(ahead.s, 0, tmem, kb > 0);
            __syncwarp();
            ahead.step(stages);
          };
          auto second_half = [&](int kb) {
            if (issuer) {
              products(pos.s, 1, tmem + kAccumulator, kb > 0);
              product_commit<CG>(&sh.empty[pos.s], lead);
            }
            __syncwarp();
            pos.step(stages);
          };
          for (int kb = 0; kb < skew && ok; ++kb) first_half(kb);
          if (!ok) break;
          if (skew == kblocks && issuer) product_commit<CG>(&sh.acc_full[0], lead);
          __syncwarp();
          ok = warp_wait(&sh.acc_empty[1], free_phase, abort_flag, args.status);
          if (!ok) break;
          tc_fence_after();
          for (int kb = 0; kb < skew; ++kb) second_half(kb);
          for (int kb = skew; kb < last; ++kb) {
            if (!wait_full(pos)) break;
            if (issuer) {
              const uint32_t at = pos.s * stage_step;
#pragma unroll
              for (int k = 0; k < kTileK / 16; ++k) {
                const uint64_t b0 = desc_b + (at + step_offset<BMN>(k));
                product_step_twice(tmem, tmem + kAccumulator, desc_a + (at + step_offset<AMN>(k)), b0, b0 + half_step, idesc);
              }
              product_commit<CG>(&sh.empty[pos.s], lead);
            }
            __syncwarp();
            pos.step(stages);
          }
          if (!ok) break;
          ahead = pos;
          if (last < kblocks) {
            for (int kb = last; kb < kblocks && ok; ++kb) first_half(kb);
            if (!ok) break;
            if (issuer) product_commit<CG>(&sh.acc_full[0], lead);
            __syncwarp();
            for (int kb = last; kb < kblocks; ++kb) second_half(kb);
          }
          if (issuer) product_commit<CG>(&sh.acc_full[1], lead);
          __syncwarp();
        }
      }
    }
  } else {
    // ----------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;  // the TMEM lanes this warp may read; its column chunks
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int thread = threadIdx.x - 64;
    float* vectors = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)) + kRingBytes + kStagingBytes);
    uint32_t turn = 0;  // accumulators finished
    for (int t = group; t < tiles; t += groups) {
      int tm, tn;
      tile_coords(args, t, tm, tn);
      const long long tile_row = static_cast<long long>(tm * CG + static_cast<int>(rank)) * kTileM;
      const long long row0 = tile_row + quarter * 32;
      // one gate row for all of the CTA's rows, or each row's own
      const T* gate = gate_row<T, EPI>(args, tile_row);
      const T* own_gate = nullptr;
      if (gate && gate != gate_row<T, EPI>(args, min(tile_row + kTileM, static_cast<long long>(args.m)) - 1))
        own_gate = gate_row<T, EPI>(args, min(row0 + lane, static_cast<long long>(args.m) - 1));
#pragma unroll 1
      for (int h = 0; h < kHalves; ++h, ++turn) {
        const int b = turn & 1;
        const int col0 = (tn * kHalves + h) * args.bn;
        float* vec = vectors + b * 512;
        // the same for every tile, also where this CTA's rows lie past the matrix and it has no gate row: the
        // barrier is what keeps a tile's vectors from being overwritten while a slower warp still reads them
        if (EPI && (args.bias || args.gate)) {
          if constexpr (SPLIT) {  // the columns that this group finishes; read after the barriers below
            const OwnChunks own = own_chunks(args.bn / kStageRow, part, splits);
            stage_vectors<T>(args, vec, gate, col0 + own.begin * kStageRow, (own.end - own.begin) * kStageRow, thread);
          } else {
            stage_vectors<T>(args, vec, gate, col0, args.bn, thread);
            epilogue_barrier();
          }
        }
        // after an expired wait the warp still meets the others at the barriers above
        if (!mbar_wait_warp(&sh.acc_full[b], (turn >> 1) & 1, abort_flag, args.status)) continue;
        tc_fence_after();
        if constexpr (!SPLIT) {
          finish_tile<T, EPI>(args, tmem + b * kAccumulator + lanes, ring + kRingBytes + (warp - 2) * 2048, vec, own_gate,
                              row0, col0, lane, half);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 1) mbar_arrive(&sh.acc_empty[b]);
            else arrive_cluster(map_rank(smem_u32(&sh.acc_empty[b]), lead));
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // split: every group's ring is drained; otherwise neither CTA of a pair leaves while the other may still signal it
  if (CG > 1 || SPLIT) cluster_sync();
  if constexpr (SPLIT) {
    int tm, tn;
    tile_coords(args, group, tm, tn);
    const bool works = warp >= 2 && warp < 2 + kEpilogueWarps && !sh.abort_flag;
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const long long tile_row = static_cast<long long>(tm * CG + static_cast<int>(rank)) * kTileM, row0 = tile_row + quarter * 32;
    const int chunks = args.bn / kStageRow;
    const uint32_t at_lane = (quarter * 32 + lane) * 16;
    tc_fence_after();
    if (works) {  // the other groups' columns, each to its group; groups in turn from the next one on
      for (int d = 1; d < splits; ++d) {
        const int to = (part + d) % splits, slot = splits - 1 - d;  // this group is number ``slot`` after ``to``
        const OwnChunks theirs = own_chunks(chunks, to, splits);
        const uint32_t base = map_rank(ring, to * CG + rank) + slot * (theirs.end - theirs.begin) * kChunkBytes + at_lane;
        for (int c = theirs.begin + half; c < theirs.end; c += 2) {
          uint32_t acc[32];
          tmem_ld32_sync(tmem + lanes + c * kStageRow, acc);
          if (row0 + lane < args.m) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              st_cluster_v4(base + (c - theirs.begin) * kChunkBytes + j * kTileM * 16, acc + 4 * j);
          }
          __syncwarp();  // the next TMEM load wants the whole warp
        }
      }
    }
    __syncwarp();
    cluster_sync();  // every partial has arrived
    if (works) {
      const OwnChunks own = own_chunks(chunks, part, splits);
      const int col0 = tn * args.bn + own.begin * kStageRow, count = own.end - own.begin;
      const int col_end = min(args.n, col0 + count * kStageRow);
      const float* vectors = reinterpret_cast<const float*>(smem_raw + (ring - smem_u32(smem_raw)) + kRingBytes + kStagingBytes);
      const T* gate = gate_row<T, EPI>(args, tile_row);
      const T* own_gate = nullptr;
      if (gate && gate != gate_row<T, EPI>(args, min(tile_row + kTileM, static_cast<long long>(args.m)) - 1))
        own_gate = gate_row<T, EPI>(args, min(row0 + lane, static_cast<long long>(args.m) - 1));
      for (int c = half; c < count; c += 2) {
        uint32_t acc[32];
        tmem_ld32_sync(tmem + lanes + (own.begin + c) * kStageRow, acc);
        float2 v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = make_float2(__uint_as_float(acc[2 * j]), __uint_as_float(acc[2 * j + 1]));
        for (int p = 0; p < splits - 1; ++p) {
          const uint32_t from = ring + (p * count + c) * kChunkBytes + at_lane;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 f = ld_shared_v4(from + j * kTileM * 16);
            v[2 * j] = fadd2(v[2 * j], make_float2(f.x, f.y));
            v[2 * j + 1] = fadd2(v[2 * j + 1], make_float2(f.z, f.w));
          }
        }
        finish_chunk<T, EPI>(args, v, ring + kRingBytes + (warp - 2) * 2048, vectors, own_gate, row0, col0, c, col_end, lane);
      }
    }
    __syncwarp();
    tc_fence_before();
    if (CG > 1) cluster_sync();  // the pair frees its TMEM together
    else __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_free<CG>(tmem, 2 * kAccumulator);
  }
}

// ---- unaligned operands ------------------------------------------------------------
// Rows [rows, cols] of 2-byte elements, any stride and alignment, to rows ld
// elements apart (16-byte aligned), up to four operands in one launch: blocks
// stride over an operand's rows, threads over columns.
struct PackArgs {
  const uint16_t* src[4];
  uint16_t* dst[4];
  long long stride[4];
  int ld[4], rows[4], cols[4];
};
__global__ void __launch_bounds__(256) pack_rows_kernel(const __grid_constant__ PackArgs a) {
  wait_for_prior();
  let_next_start();
  const int k = blockIdx.y, cols = a.cols[k];
  for (long long r = blockIdx.x; r < a.rows[k]; r += gridDim.x) {
    const uint16_t* src = a.src[k] + r * a.stride[k];
    uint16_t* dst = a.dst[k] + r * a.ld[k];
    for (int c0 = threadIdx.x; c0 < cols; c0 += 8 * 256) {
      uint16_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c0 + i * 256 < cols ? src[c0 + i * 256] : static_cast<uint16_t>(0);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i * 256 < cols) dst[c0 + i * 256] = v[i];
    }
  }
}

// ---- gradient of the epilogue --------------------------------------------------------
// Bound by HBM with the arithmetic close behind: 6750 x 12288 with gelu (tanh form)
// reads g and z, writes dz: 498 MB in 93 us (5.4 TB/s); for the bias gradient
// alone 68 us, 80 us in the erf form.
// One block per (256 columns, chunk of one sample's rows): lane l of every
// warp owns 8 columns, the 8 warps take every eighth row.  Writes dz and the
// chunk's column sums of dz and of g * act(z); a second kernel adds the
// chunks in order, so the sums do not depend on the launch.
struct ActBackwardArgs {
  const void* grad;
  long long grad_stride;
  const void* preact;        // [rows, n] (null: act' = 1 and no gate gradient)
  const void* gate;
  long long gate_stride;
  void* dz;                  // [rows, dz_stride] (null: not written)
  int dz_stride;
  float* part_bias;          // [samples * chunks, n] (null: no sums)
  float* part_gate;
  int samples, rows_per_sample, n, chunks, chunk_rows;
  int act, vec;
};

// 8 neighbouring elements as they lie in memory (past ``count``: 0), and as four pairs
template <bool VEC>
__device__ __forceinline__ uint4 load_raw(const void* at, int count) {
  if constexpr (VEC) return *static_cast<const uint4*>(at);
  const uint16_t* p = static_cast<const uint16_t*>(at);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (2 * i < count ? p[2 * i] : 0u) | (2 * i + 1 < count ? static_cast<uint32_t>(p[2 * i + 1]) << 16 : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void widen(const uint4& u, float2 (&v)[4]) {
  v[0] = unpack2<T>(u.x), v[1] = unpack2<T>(u.y), v[2] = unpack2<T>(u.z), v[3] = unpack2<T>(u.w);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_pairs(T* p, int count, const float2 (&v)[4]) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(v[0].x, v[0].y), pack2<T>(v[1].x, v[1].y), pack2<T>(v[2].x, v[2].y), pack2<T>(v[3].x, v[3].y));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i < count) p[2 * i] = from_f32<T>(v[i].x);
      if (2 * i + 1 < count) p[2 * i + 1] = from_f32<T>(v[i].y);
    }
  }
}

template <typename T, int ACT, bool GATE, bool VEC>
__global__ void __launch_bounds__(256, GATE ? 3 : 4) act_backward_kernel(const __grid_constant__ ActBackwardArgs a) {
  __shared__ float red[GATE ? 2 : 1][8][256];
  wait_for_prior();
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a one-dimensional grid, the column blocks of a chunk side by side: as many samples as there are rows
  const unsigned col_blocks = (static_cast<unsigned>(a.n) + 255) / 256;
  const int piece = blockIdx.x / col_blocks, col0 = (blockIdx.x - piece * col_blocks) * 256;
  const int sample = piece / a.chunks, chunk = piece - sample * a.chunks;
  const int col = col0 + lane * 8;
  const int count = min(8, a.n - col);
  constexpr bool kValue = ACT != kActNone || GATE;  // the pre-activation is read
  float2 gate[4], sum_dz[4], sum_ga[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sum_dz[i] = sum_ga[i] = gate[i] = make_float2(0.0f, 0.0f);
  if (count > 0) {
    if (GATE) widen<T>(load_raw<VEC>(static_cast<const T*>(a.gate) + sample * a.gate_stride + col, count), gate);
    const int begin = chunk * a.chunk_rows + warp, end = min((chunk + 1) * a.chunk_rows, a.rows_per_sample);
    const long long row0 = static_cast<long long>(sample) * a.rows_per_sample + begin;
    const T* gp = static_cast<const T*>(a.grad) + row0 * a.grad_stride + col;
    const T* zp = static_cast<const T*>(a.preact) + row0 * a.n + col;
    T* dp = static_cast<T*>(a.dz) + row0 * a.dz_stride + col;
    const long long g_step = 8 * a.grad_stride, z_step = 8LL * a.n, d_step = 8LL * a.dz_stride;
    const bool read_z = kValue && a.preact, write = a.dz != nullptr;
    // the next two of the warp's rows are in flight while one is computed
    uint4 g_raw[2], z_raw[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      g_raw[j] = z_raw[j] = make_uint4(0, 0, 0, 0);
      if (begin + 8 * j < end) {
        g_raw[j] = load_raw<VEC>(gp, count);
        if (read_z) z_raw[j] = load_raw<VEC>(zp, count);
      }
      gp += g_step;
      zp += z_step;
    }
    for (int r = begin; r < end; r += 16) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (r + 8 * j < end) {
          float2 g[4], z[4], dz[4];
          widen<T>(g_raw[j], g);
          widen<T>(z_raw[j], z);
          if (r + 8 * j + 16 < end) {
            g_raw[j] = load_raw<VEC>(gp, count);
            if (read_z) z_raw[j] = load_raw<VEC>(zp, count);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dz[i] = GATE ? fmul2(g[i], gate[i]) : g[i];
            if (read_z) {
              float2 value = z[i], slope;
              if constexpr (ACT != kActNone) {
                activate_slope2<ACT, GATE>(z[i], value, slope);
                dz[i] = fmul2(dz[i], slope);
              }
              if (GATE) sum_ga[i] = ffma2(g[i], value, sum_ga[i]);
            }
            sum_dz[i] = fadd2(sum_dz[i], dz[i]);
          }
          // dz is rounded to the operands' type, its sums are not: the 16-bit tensor-core kind takes both operands
          // in one type, and carrying dz's remainder as a second operand would double the products (a relative
          // error of 0.0023 of dx and dW in bf16 against 0.0017 of their own rounding).  In fp16 the rounding has
          // that type's range too: |dz| past 65504 becomes infinite and below 6e-8 zero, as the products of
          // unfused fp16 layers do; the loss scale has to allow for it
          if (write) store_pairs<T, VEC>(dp, count, dz);
        }
        gp += g_step;
        zp += z_step;
        dp += d_step;
      }
    }
  }
  if (!a.part_bias && !a.part_gate) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *reinterpret_cast<float2*>(&red[0][warp][lane * 8 + 2 * i]) = sum_dz[i];
    if (GATE) *reinterpret_cast<float2*>(&red[GATE ? 1 : 0][warp][lane * 8 + 2 * i]) = sum_ga[i];
  }
  __syncthreads();
  const int c = col0 + threadIdx.x;
  if (c < a.n) {
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      s0 += red[0][w][threadIdx.x];
      if (GATE) s1 += red[GATE ? 1 : 0][w][threadIdx.x];
    }
    const long long at = static_cast<long long>(piece) * a.n + c;
    if (a.part_bias) a.part_bias[at] = s0;
    if (GATE && a.part_gate) a.part_gate[at] = s1;
  }
}

// Sums of the chunks: 32 columns x 8 lanes of chunks per block, the lanes'
// sums added in order, sample after sample.
template <typename T>
__global__ void __launch_bounds__(256) act_backward_sums_kernel(const float* part_bias, const float* part_gate,
                                                                T* dbias, T* dgate, int samples, int chunks, int n) {
  __shared__ float red[2][8][33];
  wait_for_prior();
  let_next_start();
  const int cx = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  float total = 0.0f;
  for (int b = 0; b < samples; ++b) {
    float s[2] = {0.0f, 0.0f};
    if (c < n) {
#pragma unroll 4
      for (int i = y; i < chunks; i += 8) {
        const long long at = (static_cast<long long>(b) * chunks + i) * n + c;
        if (part_bias) s[0] += part_bias[at];
        if (part_gate) s[1] += part_gate[at];
      }
    }
    red[0][y][cx] = s[0];
    red[1][y][cx] = s[1];
    __syncthreads();
    if (y == 0 && c < n) {
      float g = 0.0f;
      for (int i = 0; i < 8; ++i) {
        total += red[0][i][cx];
        g += red[1][i][cx];
      }
      if (dgate) dgate[static_cast<long long>(b) * n + c] = from_f32<T>(g);
    }
    __syncthreads();
  }
  if (dbias && y == 0 && c < n) dbias[c] = from_f32<T>(total);
}

// ---- host side --------------------------------------------------------------------------
constexpr long long kAlign = 256;
long long align_up(long long v, long long a) { return (v + a - 1) / a * a; }

// A matrix operand of a product in memory: ``rows`` rows of ``cols`` elements.
struct Operand {
  const void* ptr;
  long long stride;  // elements between rows
  int rows, cols;
  bool aligned() const { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && (stride & 7) == 0; }
  long long pack_bytes() const { return aligned() ? 0 : align_up(2LL * rows * align_up(cols, 8), kAlign); }
};

// Consecutive pieces of the caller's workspace.
struct Carver {
  unsigned char* base;
  long long used;
  void* take(long long bytes) {
    void* p = base ? base + used : nullptr;
    used += align_up(bytes, kAlign);
    return p;
  }
};

// Operands that TMA cannot read become copies in the workspace, in one launch.
int prepare_operands(Operand* const* list, int n, Carver& ws, cudaStream_t stream) {
  PackArgs p{};
  int jobs = 0, most = 0;
  for (int i = 0; i < n; ++i) {
    Operand& o = *list[i];
    if (o.aligned()) continue;
    p.src[jobs] = static_cast<const uint16_t*>(o.ptr);
    p.stride[jobs] = o.stride;
    p.dst[jobs] = static_cast<uint16_t*>(ws.take(o.pack_bytes()));
    p.ld[jobs] = static_cast<int>(align_up(o.cols, 8));
    p.rows[jobs] = o.rows;
    p.cols[jobs] = o.cols;
    if (o.rows > most) most = o.rows;
    o.ptr = p.dst[jobs];
    o.stride = p.ld[jobs];
    ++jobs;
  }
  if (!jobs) return kOk;
  return launch_overlapped(pack_rows_kernel, dim3(most < 8 * kNumSMs ? most : 8 * kNumSMs, jobs), dim3(256), 0, 0, stream, p);
}

bool operand_map(CUtensorMap* map, const Operand& o, bool mn, int tile_rows, int joined_panels, int dtype) {
  const CUtensorMapDataType type = dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (joined_panels) {  // [width / 64][K][64]
    const uint64_t dims[3] = {64, static_cast<uint64_t>(o.rows), static_cast<uint64_t>(o.cols / 64)};
    const uint64_t strides[2] = {static_cast<uint64_t>(o.stride) * 2, 128};
    const uint32_t box[3] = {64, 64, static_cast<uint32_t>(joined_panels)};
    return encode_tensor_map(map, type, 3, o.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const uint64_t dims[2] = {static_cast<uint64_t>(o.cols), static_cast<uint64_t>(o.rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(o.stride) * 2};
  // K-major: 64 K columns of tile_rows rows; MN-major: 64 columns of 64 K rows
  const uint32_t box[2] = {64, static_cast<uint32_t>(mn ? 64 : tile_rows)};
  return encode_tensor_map(map, type, 2, o.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// How a product is cut: CTAs per group, columns per accumulator, accumulators
// per tile, K splits.
struct TileChoice {
  int cg, bn, halves, splits;
};

// Estimated clocks of a choice, from what one SM does per 64-wide K block: 2
// clocks of MMA per column of its tile (128 rows x 16 take half a clock a
// column), or its operand rows' 128 bytes at 50 bytes a clock (the traffic that
// measured equal to it), whichever is longer; plus what a tile adds: little where
// the epilogue hides under the next tile, ``exposed`` clocks a column where it
// does not (wide), the partials at 8 bytes a clock between SMs and the meeting
// (split).  Of all the choices for a shape this takes the fastest or one within
// 3% of it: 256 x 12288 x 3072 25.7 us (224 columns, 4 splits; 128 and 2: 28.1),
// 128 x 12288 x 3072 21.3 us (96 and 4; 64 and 2: 27.6), 256 x 3072 x 12288 22.9
// us (192, no split; 256: 25.5).
TileChoice choose_tiles(int m, int n, int kblocks, bool amn, double exposed) {
  TileChoice best{1, 128, 1, 1};
  double least = 1e300;
  const int cg = m > kTileM ? 2 : 1;
  const int valid = m < kTileM ? m : kTileM;
  const int a_rows = amn ? (m > 64 ? 128 : 64) : (valid + 7) / 8 * 8;
  const long long tiles_m = (m + kTileM * cg - 1) / (kTileM * cg);
  auto consider = [&](int bn, int halves, int splits) {
    const int cols = bn * halves, size = splits * cg;
    const long long tiles = tiles_m * ((n + cols - 1) / cols);
    // clusters of one CTA per SM that the GPU holds at a time
    const int fit = size == 1 ? kNumSMs : size == 2 ? kNumSMs / 2 : size == 4 ? 33 : 15;
    const long long waves = (tiles + fit - 1) / fit;
    if (splits > 1 && waves > 1) return;
    const double mma = 2.0 * cols, load = 128.0 / 50.0 * (a_rows + cols / cg);
    const double cost = waves * (static_cast<double>(kblocks) / splits * (mma > load ? mma : load) +
                                 (halves > 1 ? exposed * bn : 200.0)) +
                        (splits > 1 ? 3500.0 + 0.5 * valid * cols * (splits - 1) / splits : 6.0 * cols);
    if (cost < least) {
      least = cost;
      best = TileChoice{cg, bn, halves, splits};
    }
  };
  for (int splits = 1; splits * cg <= 8; splits *= 2) {
    if (splits > 1 && kblocks < 4 * splits) break;
    const int most = splits == 1 && cg == 1 ? 128 : 256;  // a CTA's accumulators are 128 columns apart, a pair's 256
    for (int bn = 32 * cg; bn <= most; bn += 32) consider(bn, 1, splits);
  }
  if (cg == 2)
    for (int bn = 160; bn <= 256; bn += 32) consider(bn, 2, 1);
  return best;
}

template <typename T, int CG, bool SPLIT, bool WIDE, bool AMN, bool BMN, bool EPI>
int launch_tiles(const GemmArgs& g, int splits, cudaStream_t stream) {
  auto kernel = gemm_kernel<T, CG, SPLIT, WIDE, AMN, BMN, EPI>;
  static std::atomic<unsigned long long> opened{0};  // devices whose kernel has its shared memory granted
  cudaError_t e = grant_smem(reinterpret_cast<const void*>(kernel), kGemmSmem, opened);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int tiles = g.tiles_m * g.tiles_n, most = kNumSMs / CG;
  const unsigned grid = SPLIT ? tiles * CG * splits : (tiles < most ? tiles : most) * CG;
  return launch_overlapped(kernel, dim3(grid), dim3(kGemmThreads), kGemmSmem, CG * splits, stream, g, splits);
}

// Everything of a product's cut that does not need its operands: g.m, g.n and g.act are set.
template <bool AMN, bool BMN, bool EPI>
TileChoice plan_tiles(GemmArgs& g, int kblocks) {
  const TileChoice c = choose_tiles(g.m, g.n, kblocks, AMN, !EPI ? 24.0 : g.act == kActNone ? 72.0 : 88.0);
  g.bn = c.bn;
  g.tiles_m = (g.m + c.cg * kTileM - 1) / (c.cg * kTileM);
  g.tiles_n = (g.n + c.bn * c.halves - 1) / (c.bn * c.halves);
  // The smaller operand stays in L2 while the larger passes once: A smaller, all
  // m tiles under every column of tiles; B smaller, two m tiles across all
  // columns.  The SMs are at their power limit in long products, so DRAM traffic
  // costs time (6750 x 3072 x 12288: 374 us with all m tiles, 400 with bands of
  // eight; 6750 x 12288 x 3072: 378 us with four, 394 with all).
  const double a_all = 128.0 * g.m * kblocks, b_all = 128.0 * g.n * kblocks;
  g.band = (a_all < b_all ? a_all : b_all) > 96e6 ? 8 : a_all <= b_all ? g.tiles_m : 2;
  if (g.band > g.tiles_m) g.band = g.tiles_m;
  // rows (or panels) of the operands one CTA stages per K block; a single tile
  // of few rows loads only those, the others' results are never stored
  const int a_rows = g.m < kTileM ? (g.m + 7) / 8 * 8 : kTileM, b_rows = c.bn / c.cg;
  g.a_panels = g.m > 64 ? 2 : 1;
  g.b_panels = (b_rows + 63) / 64;
  g.a_bytes = AMN ? g.a_panels * 8192 : a_rows * 128;
  g.b_bytes = BMN ? g.b_panels * 8192 : b_rows * 128;
  g.stage_bytes = g.a_bytes + c.halves * g.b_bytes;
  g.stages = kRingBytes / static_cast<int>(g.stage_bytes);
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  // a joined copy starts on a whole panel
  g.a_joined = AMN && g.m % 64 == 0;
  g.b_joined = BMN && g.n % 64 == 0 && b_rows % 64 == 0;
  return c;
}

template <typename T, bool AMN, bool BMN, bool EPI>
int launch_gemm(GemmArgs& g, const Operand* a, const Operand* b, int segments, int dtype, cudaStream_t stream) {
  int kblocks = 0;
  for (int s = 0; s < segments; ++s) {
    g.kblocks[s] = ((AMN ? a[s].rows : a[s].cols) + kTileK - 1) / kTileK;
    kblocks += g.kblocks[s];
  }
  const TileChoice c = plan_tiles<AMN, BMN, EPI>(g, kblocks);
  if (static_cast<long long>(g.tiles_m) * g.tiles_n > 0x0fffffffLL) return kErrUnsupported;
  const int a_rows = g.m < kTileM ? (g.m + 7) / 8 * 8 : kTileM, b_rows = c.bn / c.cg;
  for (int s = 0; s < segments; ++s)
    if (!operand_map(&g.a[s], a[s], AMN, a_rows, g.a_joined ? g.a_panels : 0, dtype) ||
        !operand_map(&g.b[s], b[s], BMN, b_rows, g.b_joined ? g.b_panels : 0, dtype))
      return kErrTensorMap;
  g.status = device_status_ptr();
  if (c.splits > 1)
    return c.cg == 2 ? launch_tiles<T, 2, true, false, AMN, BMN, EPI>(g, c.splits, stream)
                     : launch_tiles<T, 1, true, false, AMN, BMN, EPI>(g, c.splits, stream);
  if (c.halves > 1) return launch_tiles<T, 2, false, true, AMN, BMN, EPI>(g, 1, stream);
  return c.cg == 2 ? launch_tiles<T, 2, false, false, AMN, BMN, EPI>(g, 1, stream)
                   : launch_tiles<T, 1, false, false, AMN, BMN, EPI>(g, 1, stream);
}

bool aligned16(const void* p, long long stride) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride & 7) == 0);
}

struct LinearShape {
  int samples, rows_per_sample, k, k2, n, act, dtype;
  long long rows() const { return static_cast<long long>(samples) * rows_per_sample; }
  bool valid() const {
    return samples >= 0 && rows_per_sample >= 0 && k >= 1 && k2 >= 0 && n >= 1 && act >= kActNone && act <= kActSilu &&
           (dtype == 0 || dtype == 1) && rows() <= 0x7fffff00LL &&
           static_cast<long long>(k) + k2 <= 0x7fffff00LL && n <= 0x7fffff00;
  }
};

const void* offset16(const void* p, long long elements) { return static_cast<const uint16_t*>(p) + elements; }

template <typename T>
int forward(const LinearShape& s, Operand (&a)[2], Operand (&b)[2], GemmArgs& g, Carver& ws, cudaStream_t stream) {
  const int segments = s.k2 > 0 ? 2 : 1;
  Operand* list[4] = {&a[0], &b[0], &a[1], &b[1]};
  if (int st = prepare_operands(list, 2 * segments, ws, stream)) return st;
  return launch_gemm<T, false, false, true>(g, a, b, segments, s.dtype, stream);
}

// Row chunks per sample of the epilogue's gradient: as many as fill the GPU's
// resident blocks once, or two to four times where that leaves fewer idle, and
// no shorter than two rows a warp.  6750 x 12288: 68 us for one or three rounds
// of blocks, 72 us for chunks of 64 rows, 81 for 32 (without writing dz).
int backward_chunks(const LinearShape& s, bool gate) {
  if (s.samples < 1) return 1;
  const long long blocks = static_cast<long long>((s.n + 255) / 256) * s.samples;
  const long long resident = (gate ? 3LL : 4LL) * kNumSMs;  // act_backward_kernel's launch bounds
  long long chunks = 1;
  double most = 0.0;  // share of the rounds' places that have a block
  for (int rounds = 1; rounds <= 4 && most < 0.95; ++rounds) {
    const long long c = rounds * resident / blocks;
    const double used = static_cast<double>(c * blocks) / static_cast<double>(rounds * resident);
    if (used > most) {
      most = used;
      chunks = c;
    }
  }
  const long long shortest = (s.rows_per_sample + 15) / 16;
  if (chunks > shortest) chunks = shortest;
  return chunks < 1 ? 1 : static_cast<int>(chunks);
}

struct BackwardPlan {
  bool elementwise;   // dz differs from grad, or grad cannot be read in place
  bool sums;
  int chunks;
  long long dz_bytes, part_bytes;
};

BackwardPlan plan_backward(const LinearShape& s, const Operand& grad, bool has_gate, bool need_product, bool need_bias,
                           bool need_gate) {
  BackwardPlan p;
  p.elementwise = need_product && (s.act != kActNone || has_gate || !grad.aligned());
  p.sums = need_bias || need_gate;
  p.chunks = backward_chunks(s, has_gate);
  p.dz_bytes = p.elementwise ? 2 * s.rows() * align_up(s.n, 8) : 0;
  p.part_bytes = 4LL * s.samples * p.chunks * s.n;
  return p;
}

template <typename T, int ACT>
int launch_act_backward(const ActBackwardArgs& a, dim3 grid, cudaStream_t stream) {
  if (a.gate && a.vec) return launch_overlapped(act_backward_kernel<T, ACT, true, true>, grid, dim3(256), 0, 0, stream, a);
  if (a.gate) return launch_overlapped(act_backward_kernel<T, ACT, true, false>, grid, dim3(256), 0, 0, stream, a);
  if (a.vec) return launch_overlapped(act_backward_kernel<T, ACT, false, true>, grid, dim3(256), 0, 0, stream, a);
  return launch_overlapped(act_backward_kernel<T, ACT, false, false>, grid, dim3(256), 0, 0, stream, a);
}

template <typename T>
int backward(const LinearShape& s, Operand grad, const void* preact, Operand (&x)[2], Operand (&w)[2],
             const void* gate, long long gate_stride, void* (&dx)[2], void* dweight, void* dbias, void* dgate,
             Carver& ws, cudaStream_t stream) {
  const int segments = s.k2 > 0 ? 2 : 1;
  const bool need_product = dx[0] || dx[1] || dweight;
  const BackwardPlan p = plan_backward(s, grad, gate != nullptr, need_product, dbias != nullptr, dgate != nullptr);
  Operand dz = grad;
  if (p.elementwise || p.sums) {
    ActBackwardArgs a{};
    a.grad = grad.ptr;
    a.grad_stride = grad.stride;
    a.preact = (s.act != kActNone || dgate) ? preact : nullptr;
    a.gate = gate;
    a.gate_stride = gate_stride;
    a.dz_stride = static_cast<int>(align_up(s.n, 8));
    a.dz = p.elementwise ? ws.take(p.dz_bytes) : nullptr;
    if (p.elementwise) dz = Operand{a.dz, a.dz_stride, static_cast<int>(s.rows()), s.n};
    a.part_bias = dbias ? static_cast<float*>(ws.take(p.part_bytes)) : nullptr;
    a.part_gate = dgate ? static_cast<float*>(ws.take(p.part_bytes)) : nullptr;
    a.samples = s.samples;
    a.rows_per_sample = s.rows_per_sample;
    a.n = s.n;
    a.chunks = p.chunks;
    a.chunk_rows = (s.rows_per_sample + p.chunks - 1) / p.chunks;
    a.act = s.act;
    a.vec = s.n % 8 == 0 && aligned16(grad.ptr, grad.stride) && aligned16(a.preact, s.n) && aligned16(gate, gate_stride);
    const long long blocks = (s.n + 255LL) / 256 * s.samples * p.chunks;
    if (blocks > 0x7fffffffLL) return kErrUnsupported;
    const dim3 grid(static_cast<unsigned>(blocks));
    const int st = s.act == kActGeluTanh ? launch_act_backward<T, kActGeluTanh>(a, grid, stream)
                   : s.act == kActGelu   ? launch_act_backward<T, kActGelu>(a, grid, stream)
                   : s.act == kActSilu   ? launch_act_backward<T, kActSilu>(a, grid, stream)
                                         : launch_act_backward<T, kActNone>(a, grid, stream);
    if (st) return st;
    if (p.sums) {
      const int sums = launch_overlapped(act_backward_sums_kernel<T>, dim3((s.n + 31) / 32), dim3(256), 0, 0, stream,
                                         a.part_bias, a.part_gate, static_cast<T*>(dbias), static_cast<T*>(dgate),
                                         s.samples, p.chunks, s.n);
      if (sums) return sums;
    }
  }
  Operand* list[4];
  int wanted = 0;
  for (int i = 0; i < segments; ++i) {
    if (dx[i]) list[wanted++] = &w[i];
    if (dweight) list[wanted++] = &x[i];
  }
  if (int st = prepare_operands(list, wanted, ws, stream)) return st;
  for (int i = 0; i < segments; ++i) {
    const int cols = i ? s.k2 : s.k;
    if (dx[i]) {
      // dx[m, c] = sum_n dz[m, n] W[n, c]: W's rows run along the output's columns
      GemmArgs g{};
      g.m = static_cast<int>(s.rows());
      g.n = cols;
      g.out = dx[i];
      g.out_stride = cols;
      g.vec = cols % 8 == 0 && aligned16(dx[i], cols);
      if (int st = launch_gemm<T, false, true, false>(g, &dz, &w[i], 1, s.dtype, stream)) return st;
    }
    if (dweight) {
      // dW[n, c] = sum_m dz[m, n] x[m, c]: both operands run along the outputs
      GemmArgs g{};
      g.m = s.n;
      g.n = cols;
      g.out = static_cast<T*>(dweight) + (i ? s.k : 0);
      g.out_stride = static_cast<long long>(s.k) + s.k2;
      g.vec = cols % 8 == 0 && aligned16(g.out, g.out_stride);
      if (int st = launch_gemm<T, true, true, false>(g, &dz, &x[i], 1, s.dtype, stream)) return st;
    }
  }
  return kOk;
}

void make_operands(const LinearShape& s, const void* x, long long x_stride, const void* x2, long long x2_stride,
                   const void* weight, long long w_stride, Operand (&a)[2], Operand (&b)[2]) {
  const int rows = static_cast<int>(s.rows());
  // the stride of a single row is never walked; TMA wants it aligned all the same
  if (rows == 1) {
    x_stride = align_up(s.k, 8);
    x2_stride = align_up(s.k2, 8);
  }
  if (s.n == 1 && s.k2 == 0) w_stride = align_up(s.k, 8);
  a[0] = Operand{x, x_stride, rows, s.k};
  a[1] = Operand{x2, x2_stride, rows, s.k2};
  b[0] = Operand{weight, w_stride, s.n, s.k};
  b[1] = Operand{offset16(weight, s.k), w_stride, s.n, s.k2};
}

}  // namespace
}  // namespace peco

using namespace peco;

extern "C" long long peco_linear_forward_workspace(const void* x, long long x_stride, const void* x2,
                                                   long long x2_stride, const void* weight, long long w_stride,
                                                   int samples, int rows_per_sample, int k, int k2, int n) {
  const LinearShape s{samples, rows_per_sample, k, k2, n, 0, 0};
  if (!s.valid()) return -1;
  Operand a[2], b[2];
  make_operands(s, x, x_stride, x2, x2_stride, weight, w_stride, a, b);
  long long bytes = a[0].pack_bytes() + b[0].pack_bytes();
  if (k2) bytes += a[1].pack_bytes() + b[1].pack_bytes();
  return bytes;
}

extern "C" int peco_linear_forward(const void* x, long long x_stride, const void* x2, long long x2_stride,
                                   const void* weight, long long w_stride, const void* bias, const void* gate,
                                   long long gate_stride, const void* residual, long long res_stride, void* out,
                                   long long out_stride, void* preact, int samples, int rows_per_sample, int k, int k2,
                                   int n, int activation, int dtype, void* workspace, long long workspace_bytes,
                                   void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const LinearShape s{samples, rows_per_sample, k, k2, n, activation, dtype};
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (!s.valid()) return kErrInvalidValue;
  if (s.rows() == 0) return kOk;
  if (!x || !weight || !out || (k2 > 0 && !x2)) return kErrInvalidValue;
  // gate_stride is free: a row shared by all samples has stride 0
  if (x_stride < k || (k2 > 0 && x2_stride < k2) || w_stride < static_cast<long long>(k) + k2 || out_stride < n ||
      (residual && res_stride < n) || gate_stride < 0)
    return kErrInvalidValue;
  const long long need =
      peco_linear_forward_workspace(x, x_stride, x2, x2_stride, weight, w_stride, samples, rows_per_sample, k, k2, n);
  if (need > 0 && !usable_workspace(workspace, workspace_bytes, need)) return kErrWorkspace;
  Operand a[2], b[2];
  make_operands(s, x, x_stride, x2, x2_stride, weight, w_stride, a, b);
  GemmArgs g{};
  g.m = static_cast<int>(s.rows());
  g.n = n;
  g.out = out;
  g.out_stride = out_stride;
  g.bias = bias;
  g.gate = gate;
  g.gate_stride = gate_stride;
  g.rows_per_sample = rows_per_sample;
  g.residual = residual;
  g.res_stride = res_stride;
  g.preact = preact;
  g.act = activation;
  g.vec = n % 8 == 0 && aligned16(out, out_stride) && aligned16(bias, 8) && aligned16(gate, gate_stride) &&
          aligned16(residual, res_stride) && aligned16(preact, n);
  Carver ws{static_cast<unsigned char*>(workspace), 0};
  return dtype == 1 ? forward<__nv_bfloat16>(s, a, b, g, ws, stream) : forward<__half>(s, a, b, g, ws, stream);
}

extern "C" long long peco_linear_backward_workspace(const void* grad, long long grad_stride, const void* x,
                                                    long long x_stride, const void* x2, long long x2_stride,
                                                    const void* weight, long long w_stride, int samples,
                                                    int rows_per_sample, int k, int k2, int n, int activation,
                                                    int has_gate) {
  const LinearShape s{samples, rows_per_sample, k, k2, n, activation, 0};
  if (!s.valid()) return -1;
  Operand a[2], b[2];
  make_operands(s, x, x_stride, x2, x2_stride, weight, w_stride, a, b);
  const Operand g{grad, grad_stride, static_cast<int>(s.rows()), n};
  const BackwardPlan p = plan_backward(s, g, has_gate != 0, true, true, true);
  long long bytes = align_up(p.dz_bytes, kAlign) + 2 * align_up(p.part_bytes, kAlign) + a[0].pack_bytes() + b[0].pack_bytes();
  if (k2) bytes += a[1].pack_bytes() + b[1].pack_bytes();
  return bytes;
}

extern "C" int peco_linear_backward(const void* grad, long long grad_stride, const void* preact, const void* x,
                                    long long x_stride, const void* x2, long long x2_stride, const void* weight,
                                    long long w_stride, const void* gate, long long gate_stride, void* dx, void* dx2,
                                    void* dweight, void* dbias, void* dgate, int samples, int rows_per_sample, int k,
                                    int k2, int n, int activation, int dtype, void* workspace,
                                    long long workspace_bytes, void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const LinearShape s{samples, rows_per_sample, k, k2, n, activation, dtype};
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (!s.valid()) return kErrInvalidValue;
  if (s.rows() == 0) return kErrInvalidValue;  // the sums over no rows are the caller's zeros
  if (!grad || grad_stride < n || gate_stride < 0) return kErrInvalidValue;
  if ((dx || dx2) && (!weight || w_stride < static_cast<long long>(k) + k2)) return kErrInvalidValue;
  if (dweight && (!x || x_stride < k || (k2 > 0 && (!x2 || x2_stride < k2)))) return kErrInvalidValue;
  if ((dx2 && k2 == 0) || (dgate && !gate)) return kErrInvalidValue;
  if ((activation != kActNone || dgate) && !preact) return kErrInvalidValue;
  const long long need = peco_linear_backward_workspace(grad, grad_stride, x, x_stride, x2, x2_stride, weight, w_stride,
                                                        samples, rows_per_sample, k, k2, n, activation, gate != nullptr);
  if (need > 0 && !usable_workspace(workspace, workspace_bytes, need)) return kErrWorkspace;
  Operand a[2], b[2];
  make_operands(s, x, x_stride, x2, x2_stride, weight, w_stride, a, b);
  const Operand g{grad, grad_stride, static_cast<int>(s.rows()), n};
  void* dxs[2] = {dx, dx2};
  Carver ws{static_cast<unsigned char*>(workspace), 0};
  return dtype == 1 ? backward<__nv_bfloat16>(s, g, preact, a, b, gate, gate_stride, dxs, dweight, dbias, dgate, ws, stream)
                    : backward<__half>(s, g, preact, a, b, gate, gate_stride, dxs, dweight, dbias, dgate, ws, stream);
}

extern "C" int peco_linear_tiles(int m, int n, int k_blocks, int product, int activation, int* plan) {
  if (m < 1 || n < 1 || k_blocks < 1 || product < 0 || product > 2 || activation < kActNone || activation > kActSilu || !plan)
    return kErrInvalidValue;
  GemmArgs g{};
  g.m = m;
  g.n = n;
  g.act = activation;
  const TileChoice c = product == 0   ? plan_tiles<false, false, true>(g, k_blocks)
                       : product == 1 ? plan_tiles<false, true, false>(g, k_blocks)
                                      : plan_tiles<true, true, false>(g, k_blocks);
  const int values[8] = {c.cg, c.bn, c.halves, c.splits, g.stages, g.tiles_m, g.tiles_n, g.band};
  for (int i = 0; i < 8; ++i) plan[i] = values[i];
  return kOk;
}
