// Gated residual and norm between the parts of a transformer block, and its
// gradient.  Per row (one token of one sample):
//
//   b = post_norm(branch) * post_weight        (or the branch as it is)
//   r = residual_scale * x + gate * b
//   n = norm(r),  y = n * weight,  h = y * (1 + scale) + shift
//
// norm is (r - mean) * rstd (layer) or r * rstd (rms), rstd = rsqrt(mean of
// squares + eps); gate, scale and shift are vectors of the row's sample.  r
// and h are each rounded once: h comes from the fp32 r, not from its rounding.
//
// Gradient, from dh and the gradient e of r as an output:
//   dn = dh (1 + scale) weight
//   dr = e + rstd (dn - [mean dn] - n mean(dn n))      [layer only]
//   dx = residual_scale dr;  db = gate dr;  the post norm's gradient likewise.
// All vector gradients follow from three column sums over a sample's rows,
//   A0 = sum dh, A1 = sum dh n, G = sum dr pn   (pn: the post norm's output
//   before its weight, or the branch)
//   dshift = A0, dscale = weight A1, dweight = sum_samples (1 + scale) A1,
//   dgate = post_weight G, dpost_weight = sum_samples gate G.
//
// Both directions move bytes: the floor is each input read once and each
// output written once at the copy bandwidth.  A row is read once into
// registers of the threads that share it, and every statistic is taken from
// there in fp32, squares around the mean.  The backward kernel recomputes r
// from x and the branch, so nothing has to be saved.  Measured at 3072 bf16
// columns with branch, gate and modulation: forward 34680 rows 133 us (6.4 TB/s;
// 138 us over two sets of inputs back to back), backward 7006 rows 57 us (4.5
// TB/s, of it 6 us for the second kernel), 34680 rows 235 us (5.4 TB/s); the
// backward is bound by the latency of a row's reduction at the 12 warps per SM
// that its registers allow.
#include "common.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"
#include "rows.cuh"

#include <atomic>
#include <type_traits>

namespace peco {
namespace {

enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

// Rows [samples, rows, width] and vectors [samples, width] of one call; a
// vector shared by the samples has batch stride 0.
struct RowTensor {
  const void* p;
  long long sb, sn;
};
struct VecTensor {
  const void* p;
  long long sb;
};

struct NormArgs {
  RowTensor x, branch, grad_h, grad_r;
  VecTensor gate, scale, shift;
  const void* weight;
  const void* post_weight;
  void* out_r;      // forward: r; backward: d branch
  void* out_h;      // forward: h; backward: d x
  float* partial;   // backward: [samples * chunks][3][width]
  int samples, rows, width, vec;
  int norm, post;
  float eps, post_eps, residual_scale;
  int chunks;       // backward: row chunks per sample
  int stages, stage_bytes;  // ring of rows in shared memory
  unsigned* status;
};

// ---- a row in registers ----------------------------------------------------------
// A row is shared by 32 * WARPS threads, each with NCH chunks of 8 columns held
// as four fp32 pairs (the pairs' arithmetic takes one instruction for two).
// Aligned rows: chunk i of a thread is 8 neighbouring columns, one 16-byte
// access.  Other rows: its 8 columns lie a row of threads apart, so that single
// elements are still read side by side.  Columns past the width hold 0.
constexpr int kChunk = 8;

// Full rows are aligned rows that fill every thread's chunks.
enum RowMode : int { kUnaligned = 0, kAligned = 1, kFull = 2 };

template <int WARPS, int NCH, int MODE>
struct Span {
  static constexpr int kThreads = 32 * WARPS;
  static constexpr bool kIsAligned = MODE != kUnaligned;
  int thread, width;
  __device__ __forceinline__ int column(int i, int e) const {
    return kIsAligned ? (i * kThreads + thread) * kChunk + e : (i * kChunk + e) * kThreads + thread;
  }
  __device__ __forceinline__ bool inside(int i, int e) const {
    return MODE == kFull || column(i, kIsAligned ? 0 : e) < width;
  }
  // columns that warp w of the row's threads holds
  __device__ __forceinline__ float held_by(int w) const {
    if (MODE == kFull) return static_cast<float>(32 * kChunk * NCH);
    int n = 0;
    if (kIsAligned) {
      for (int i = 0; i < NCH; ++i) n += max(0, min(32 * kChunk, width - (i * kThreads + w * 32) * kChunk));
    } else {
      for (int i = 0; i < NCH * kChunk; ++i) n += max(0, min(32, width - i * kThreads - w * 32));
    }
    return static_cast<float>(n);
  }
};

// The 8 elements of a chunk as they lie in memory, two to a register.
struct RawChunk {
  uint32_t w[4];
};

template <typename T, int WARPS, int NCH, int MODE>
__device__ __forceinline__ void fetch(const Span<WARPS, NCH, MODE>& sp, const T* row, int i, RawChunk& r) {
  r.w[0] = r.w[1] = r.w[2] = r.w[3] = 0;
  if constexpr (MODE != kUnaligned) {
    if (sp.inside(i, 0)) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + sp.column(i, 0));
      r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int e = 0; e < kChunk; ++e)
      if (sp.inside(i, e)) r.w[e >> 1] |= static_cast<uint32_t>(p[sp.column(i, e)]) << (16 * (e & 1));
  }
}

template <typename T>
__device__ __forceinline__ void widen(const RawChunk& r, float2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = unpack2<T>(r.w[j]);
}

// The same with a register for each element of an unaligned row: joining two
// loads in one would wait for them where they are issued.
struct RawElements {
  uint32_t w[kChunk];
};
template <typename T, int WARPS, int NCH>
__device__ __forceinline__ void fetch(const Span<WARPS, NCH, kUnaligned>& sp, const T* row, int i, RawElements& r) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
  for (int e = 0; e < kChunk; ++e) r.w[e] = sp.inside(i, e) ? p[sp.column(i, e)] : 0u;
}
template <typename T>
__device__ __forceinline__ void widen(const RawElements& r, float2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = unpack2<T>(r.w[2 * j] | r.w[2 * j + 1] << 16);
}

// a vector's (gate, scale, ...) part of chunk i
template <typename T, typename SP>
__device__ __forceinline__ void load_part(const SP& sp, const void* p, long long at, int i, float2 (&v)[4]) {
  RawChunk r;
  fetch<T>(sp, static_cast<const T*>(p) + at, i, r);
  widen<T>(r, v);
}

template <typename T, int WARPS, int NCH, int MODE>
__device__ __forceinline__ void store(const Span<WARPS, NCH, MODE>& sp, void* p, long long at, int i, const float2 (&v)[4]) {
  T* row = static_cast<T*>(p) + at;
  if constexpr (MODE != kUnaligned) {
    if (sp.inside(i, 0))
      *reinterpret_cast<uint4*>(row + sp.column(i, 0)) =
          make_uint4(pack2<T>(v[0].x, v[0].y), pack2<T>(v[1].x, v[1].y), pack2<T>(v[2].x, v[2].y), pack2<T>(v[3].x, v[3].y));
  } else {
#pragma unroll
    for (int e = 0; e < kChunk; ++e)
      if (sp.inside(i, e)) row[sp.column(i, e)] = from_f32<T>(e & 1 ? v[e >> 1].y : v[e >> 1].x);
  }
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// A sample's vectors, in registers while its rows pass: a load between a row's
// prefetch and its use would make the warp wait for the prefetch as well (loads
// share few scoreboards).
// gate * post_weight of chunk i
template <typename T, typename SP>
__device__ __forceinline__ void load_gate(const NormArgs& a, const SP& sp, unsigned sample, int i, float2 (&g)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = both(1.0f);
  if (a.gate.p) load_part<T>(sp, a.gate.p, sample * a.gate.sb, i, g);
  if (a.post_weight) {
    float2 w[4];
    load_part<T>(sp, a.post_weight, 0, i, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = fmul2(g[j], w[j]);
  }
}
// (1 + scale) * weight of chunk i
template <typename T, typename SP>
__device__ __forceinline__ void load_factor(const NormArgs& a, const SP& sp, unsigned sample, int i, float2 (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = both(1.0f);
  if (a.weight) load_part<T>(sp, a.weight, 0, i, f);
  if (a.scale.p) {
    float2 s[4];
    load_part<T>(sp, a.scale.p, sample * a.scale.sb, i, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = ffma2(f[j], s[j], f[j]);
  }
}

// v with the columns past the width set to 0
template <int WARPS, int NCH, int MODE>
__device__ __forceinline__ float2 only_inside(const Span<WARPS, NCH, MODE>& sp, int i, int j, float2 v) {
  if (MODE == kFull) return v;
  if (!sp.inside(i, 2 * j)) v.x = 0.0f;
  if (!sp.inside(i, 2 * j + 1)) v.y = 0.0f;
  return v;
}

// ---- rows through shared memory ---------------------------------------------------
// Aligned rows shared by several warps arrive by bulk copies into a ring of
// stages, a row of every input each, a few rows ahead of the one in work: the
// copies hold no registers, so enough of them are in flight to cover HBM's
// latency (as loads into registers, a row's prefetch and its vectors' loads
// waited for one another).  Thread 0 refills the stage of the row before once
// the block has passed the current row's barrier, where nobody reads that stage
// any more.
constexpr int kMaxStages = 6;

struct RowRing {
  unsigned char* base;
  uint64_t* full;
  volatile int* abort_flag;
  unsigned* status;
  int stages, stage_bytes, row_bytes;
  int take_s, take_p;    // stage and phase of the next row to take
  int start_s;           // stage of the next row to start

  __device__ __forceinline__ void open() {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
      *abort_flag = 0;
      fence_barrier_init();
    }
    __syncthreads();
    take_s = take_p = start_s = 0;
  }
  // thread 0: start the block's next row, whose inputs are ``src``
  __device__ __forceinline__ void start(const void* const (&src)[4]) {
    if (*abort_flag) return;
    int present = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) present += src[k] != nullptr;
    mbar_arrive_expect_tx(&full[start_s], present * row_bytes);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (src[k]) bulk_load(base + start_s * stage_bytes + k * row_bytes, src[k], row_bytes, &full[start_s]);
    start_s = start_s + 1 == stages ? 0 : start_s + 1;
  }
  // wait for the next row; its stage
  __device__ __forceinline__ const unsigned char* next() {
    const unsigned char* stage = base + take_s * stage_bytes;
    if (!mbar_try_wait(&full[take_s], take_p) && !*abort_flag) mbar_wait(&full[take_s], take_p, abort_flag, status);
    if (++take_s == stages) {
      take_s = 0;
      take_p ^= 1;
    }
    return stage;
  }
  // after an expired wait: time for the copies still in flight to land before the block ends
  __device__ __forceinline__ void close() {
    if (*abort_flag && threadIdx.x == 0) {
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) {
      }
    }
  }
};

// chunk i of input k in a stage
template <typename SP>
__device__ __forceinline__ RawChunk staged(const SP& sp, const unsigned char* stage, int k, int row_bytes, int i) {
  RawChunk r;
  r.w[0] = r.w[1] = r.w[2] = r.w[3] = 0;
  if (sp.inside(i, 0)) {
    const uint4 u = *reinterpret_cast<const uint4*>(stage + k * row_bytes + sp.column(i, 0) * 2);
    r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
  }
  return r;
}

// ---- moments of a row ---------------------------------------------------------
// mean and sum of squared deviations of the row's values, and the sums of a
// second row d and of d times the deviations, on every thread of the row.  Each
// warp takes its own mean first and all its sums around that mean; the warps'
// results (one float4 each in ``buf``) are then moved to the common mean, so one
// barrier per row is enough and nothing cancels where the mean is far from zero.
struct Moments {
  float mean, squares, sum_d, sum_dv;
};

// What a thread has to know of the row's division among warps.
struct Shares {
  float own_inv;  // 1 / columns of this warp (0: none)
  float lane_n;   // columns of the warp that this lane reads in the second step
};

constexpr int warp_levels(int warps) { return warps <= 4 ? 2 : warps <= 8 ? 3 : warps <= 16 ? 4 : 5; }

template <int WARPS, int NCH, int MODE>
__device__ __forceinline__ Shares shares_of(const Span<WARPS, NCH, MODE>& sp) {
  const float own = sp.held_by(sp.thread >> 5);
  const int w = sp.thread & ((1 << warp_levels(WARPS)) - 1);
  return Shares{own > 0.0f ? 1.0f / own : 0.0f, WARPS > 1 && w < WARPS ? sp.held_by(w) : 0.0f};
}

template <int LEVELS>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1 << (LEVELS - 1); o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <bool WITH_D, int WARPS, int NCH, int MODE>
__device__ __forceinline__ Moments row_moments(const Span<WARPS, NCH, MODE>& sp, const Shares& share,
                                               const float2 (&v)[NCH][4], const float2 (&d)[NCH][4], bool centred,
                                               float inv_width, float4* buf) {
  Moments m{0.0f, 0.0f, 0.0f, 0.0f};
  if (centred) {
    float2 s = both(0.0f);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fadd2(s, v[i][j]);
    m.mean = warp_sum(s.x + s.y) * share.own_inv;
  }
  float2 q = both(0.0f), sd = both(0.0f), sv = both(0.0f);
  const float2 minus = both(-m.mean);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (MODE == kAligned && !sp.inside(i, 0)) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 dev = fadd2(v[i][j], minus);
      if (MODE == kUnaligned) dev = only_inside(sp, i, j, dev);
      q = ffma2(dev, dev, q);
      if (WITH_D) {
        sd = fadd2(sd, d[i][j]);
        sv = ffma2(d[i][j], dev, sv);
      }
    }
  }
  m.squares = warp_sum(q.x + q.y);
  if (WITH_D) {
    m.sum_d = warp_sum(sd.x + sd.y);
    m.sum_dv = warp_sum(sv.x + sv.y);
  }
  if constexpr (WARPS > 1) {
    constexpr int kLevels = warp_levels(WARPS);
    const int warp = sp.thread >> 5, lane = sp.thread & 31;
    if (lane == 0) buf[warp] = make_float4(m.mean, m.squares, m.sum_d, m.sum_dv);
    __syncthreads();
    const int w = lane & ((1 << kLevels) - 1);
    const float4 f = w < WARPS ? buf[w] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    m.mean = centred ? group_sum<kLevels>(share.lane_n * f.x) * inv_width : 0.0f;
    const float shift = f.x - m.mean;  // unused warps: no columns and sums of 0
    m.squares = group_sum<kLevels>(fmaf(share.lane_n * shift, shift, f.y));
    if (WITH_D) {
      m.sum_d = group_sum<kLevels>(f.z);
      m.sum_dv = group_sum<kLevels>(fmaf(shift, f.z, f.w));
    }
  }
  return m;
}

// ---- forward --------------------------------------------------------------------
// Blocks stay and walk the rows: WARPS warps per row (a block of four warps
// holds four rows when one warp is enough).  The next row's loads are issued as
// soon as the current row is in fp32 registers, before its reduction.
template <typename T, int WARPS, int NCH, int MODE, bool POST>
__global__ void __launch_bounds__(WARPS < 4 ? 128 : 32 * WARPS) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  static_assert(WARPS == 1 || WARPS >= 4, "rows of two warps would share block barriers");
  constexpr int kThreads = 32 * WARPS;
  constexpr unsigned kRows = WARPS < 4 ? 4 / WARPS : 1;
  wait_for_prior();
  let_next_start();
  __shared__ float4 buf[2][2][WARPS];  // alternates between rows: a row's last read may meet the next one's write
  const int slot = threadIdx.x / kThreads;
  const Span<WARPS, NCH, MODE> sp{static_cast<int>(threadIdx.x) - slot * kThreads, a.width};
  const Shares share = shares_of(sp);
  const float inv = 1.0f / static_cast<float>(a.width);
  const unsigned total = static_cast<unsigned>(a.samples) * a.rows, step = gridDim.x * kRows;  // below 2^31
  unsigned row = blockIdx.x * kRows + slot;
  if (row >= total) return;  // whole warps only: kRows > 1 means one warp per row
  unsigned sample = row / a.rows, at = row - sample * a.rows, loaded = 0xffffffffu;
  auto row_of = [&](const RowTensor& t) { return static_cast<const T*>(t.p) + sample * t.sb + at * t.sn; };
  constexpr bool kRing = MODE != kUnaligned && WARPS > 1;
  extern __shared__ __align__(128) unsigned char ring_bytes[];
  __shared__ uint64_t ring_full[kMaxStages];
  __shared__ int ring_abort;
  RowRing ring{ring_bytes, ring_full, &ring_abort, a.status, a.stages, a.stage_bytes, a.width * 2, 0, 0, 0};
  unsigned ahead = row;  // thread 0: the next row to start
  auto start = [&]() {
    const unsigned sm = ahead / a.rows, t = ahead - sm * a.rows;
    const void* src[4] = {static_cast<const T*>(a.x.p) + sm * a.x.sb + t * a.x.sn,
                          a.branch.p ? static_cast<const T*>(a.branch.p) + sm * a.branch.sb + t * a.branch.sn : nullptr,
                          nullptr, nullptr};
    ring.start(src);
    ahead = ahead + step < ahead ? 0xffffffffu : ahead + step;
  };
  std::conditional_t<MODE == kUnaligned, RawElements, RawChunk> raw_x[NCH], raw_b[NCH];
  if constexpr (kRing) {
    ring.open();
    if (threadIdx.x == 0)
      for (int n = 0; n + 1 < a.stages && ahead < total; ++n) start();
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      fetch(sp, row_of(a.x), i, raw_x[i]);
      if (a.branch.p) fetch(sp, row_of(a.branch), i, raw_b[i]);
    }
  }
  const float2 rs = both(a.residual_scale);
  float2 gate[NCH][4], factor[NCH][4], shift[NCH][4];
  int turn = 0;
  while (row < total) {
    if (sample != loaded) {
      loaded = sample;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        load_gate<T>(a, sp, sample, i, gate[i]);
        load_factor<T>(a, sp, sample, i, factor[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) shift[i][j] = both(0.0f);
        if (a.shift.p) load_part<T>(sp, a.shift.p, sample * a.shift.sb, i, shift[i]);
      }
    }
    float2 r[NCH][4];
    const long long out = static_cast<long long>(row) * a.width;
    if constexpr (kRing) {
      const unsigned char* stage = ring.next();
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        raw_x[i] = staged(sp, stage, 0, a.width * 2, i);
        if (a.branch.p) raw_b[i] = staged(sp, stage, 1, a.width * 2, i);
      }
    }
    float2 pscale = both(1.0f), pshift = both(0.0f);  // post norm: b * rstd - mean * rstd
    if constexpr (POST) {
      float2 b[NCH][4];
#pragma unroll
      for (int i = 0; i < NCH; ++i) widen<T>(raw_b[i], b[i]);
      const Moments m = row_moments<false>(sp, share, b, b, a.post == kNormLayer, inv, buf[turn][1]);
      const float rstd = rsqrtf(m.squares * inv + a.post_eps);
      pscale = both(rstd);
      pshift = both(-m.mean * rstd);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      widen<T>(raw_x[i], r[i]);
      if (a.branch.p) {
        float2 b[4];
        widen<T>(raw_b[i], b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (POST) b[j] = only_inside(sp, i, j, ffma2(b[j], pscale, pshift));  // the shift of columns past the width
          r[i][j] = ffma2(rs, r[i][j], fmul2(gate[i][j], b[j]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[i][j] = fmul2(rs, r[i][j]);
      }
    }
    row += step;
    if (row < total) {
      sample = row / a.rows;
      if constexpr (!kRing) {
        at = row - sample * a.rows;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          fetch(sp, row_of(a.x), i, raw_x[i]);
          if (a.branch.p) fetch(sp, row_of(a.branch), i, raw_b[i]);
        }
      }
    }
    if (a.out_r) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) store<T>(sp, a.out_r, out, i, r[i]);
    }
    const Moments m = row_moments<false>(sp, share, r, r, a.norm == kNormLayer, inv, buf[turn][0]);
    if (kRing && threadIdx.x == 0 && ahead < total) start();  // every thread is done with the rows before this one
    turn ^= 1;
    const float2 minus = both(-m.mean), times = both(rsqrtf(m.squares * inv + a.eps));
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[i][j] = ffma2(fmul2(fadd2(r[i][j], minus), times), factor[i][j], shift[i][j]);
      store<T>(sp, a.out_h, out, i, r[i]);
    }
  }
  if constexpr (kRing) ring.close();
}

// ---- backward ---------------------------------------------------------------------
// A block takes every chunks-th row of one sample and keeps its column sums,
// each with the thread that owns the column, in registers or (more than three
// chunks a thread) in shared memory; a second kernel adds the blocks' sums in
// order.  A register that held a piece of the row takes the next row's piece as
// soon as it is free.
template <typename T, int WARPS, int NCH, int BLOCKS, int MODE, bool POST>
__global__ void __launch_bounds__(32 * WARPS, BLOCKS) norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kThreads = 32 * WARPS;
  wait_for_prior();
  let_next_start();
  __shared__ float4 buf[2][3][WARPS];  // alternates between rows: a row's last read may meet the next one's write
  const unsigned sample = blockIdx.x / a.chunks, chunk = blockIdx.x - sample * a.chunks;
  const Span<WARPS, NCH, MODE> sp{static_cast<int>(threadIdx.x), a.width};
  const Shares share = shares_of(sp);
  const float inv = 1.0f / static_cast<float>(a.width);
  constexpr bool kShared = NCH > 3;
  // column sums [3][NCH * 8][threads], a thread's own entries bank by bank; or the ring of rows
  extern __shared__ __align__(128) float shared_sums[];
  constexpr int kR = kShared ? 1 : NCH;
  float2 a0[kR][4], a1[kR][4], g0[kR][4];
#pragma unroll
  for (int i = 0; i < kR; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) a0[i][j] = a1[i][j] = g0[i][j] = both(0.0f);
  auto shared_at = [&](int k, int i, int j) {
    return reinterpret_cast<float2*>(shared_sums) + ((k * NCH + i) * 4 + j) * kThreads + threadIdx.x;
  };
  if (kShared) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      for (int j = 0; j < 4; ++j)
        for (int k = 0; k < 3; ++k) *shared_at(k, i, j) = both(0.0f);
  }
  float2 gate[NCH][4], factor[NCH][4];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    load_gate<T>(a, sp, sample, i, gate[i]);
    load_factor<T>(a, sp, sample, i, factor[i]);
  }
  auto row_of = [&](const RowTensor& t, unsigned at) { return static_cast<const T*>(t.p) + sample * t.sb + at * t.sn; };
  constexpr bool kRing = MODE != kUnaligned && WARPS > 1 && !kShared;
  __shared__ uint64_t ring_full[kMaxStages];
  __shared__ int ring_abort;
  RowRing ring{reinterpret_cast<unsigned char*>(shared_sums), ring_full, &ring_abort, a.status, a.stages, a.stage_bytes,
               a.width * 2, 0, 0, 0};
  const unsigned rows = a.rows, stride = a.chunks;
  unsigned ahead = chunk;  // thread 0: the next row to start
  auto start = [&]() {
    const void* src[4] = {row_of(a.x, ahead), row_of(a.grad_h, ahead), a.branch.p ? row_of(a.branch, ahead) : nullptr,
                          a.grad_r.p ? row_of(a.grad_r, ahead) : nullptr};
    ring.start(src);
    ahead = ahead + stride < ahead ? 0xffffffffu : ahead + stride;
  };
  using Raw = std::conditional_t<MODE == kUnaligned && NCH == 1, RawElements, RawChunk>;  // two chunks' would spill
  Raw raw_x[NCH], raw_d[NCH], raw_b[NCH], raw_e[NCH];
  if constexpr (kRing) {
    ring.open();
    if (threadIdx.x == 0)
      for (int n = 0; n + 1 < a.stages && ahead < rows; ++n) start();
  } else if (chunk < rows) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      fetch(sp, row_of(a.x, chunk), i, raw_x[i]);
      fetch(sp, row_of(a.grad_h, chunk), i, raw_d[i]);
      if (a.branch.p) fetch(sp, row_of(a.branch, chunk), i, raw_b[i]);
      if (a.grad_r.p) fetch(sp, row_of(a.grad_r, chunk), i, raw_e[i]);
    }
  }
  const float2 rs = both(a.residual_scale);
  int turn = 0;
  for (unsigned at = chunk; at < rows; at += stride, turn ^= 1) {
    const long long out = (static_cast<long long>(sample) * rows + at) * a.width;
    const unsigned next = at + stride;
    float2 r[NCH][4], dn[NCH][4];
    const unsigned char* stage = nullptr;
    if constexpr (kRing) stage = ring.next();
    // a piece of an input: from the stage, as often as it is needed, or from its register
    auto piece = [&](int k, int i, const Raw& held) {
      if constexpr (kRing) return staged(sp, stage, k, a.width * 2, i);
      else return held;
    };
    float2 pscale = both(1.0f), pshift = both(0.0f);  // post norm: b * rstd - mean * rstd
    float prstd = 1.0f;
    if constexpr (POST) {
      float2 b[NCH][4];
#pragma unroll
      for (int i = 0; i < NCH; ++i) widen<T>(piece(2, i, raw_b[i]), b[i]);
      const Moments m = row_moments<false>(sp, share, b, b, a.post == kNormLayer, inv, buf[turn][1]);
      prstd = rsqrtf(m.squares * inv + a.post_eps);
      pscale = both(prstd);
      pshift = both(-m.mean * prstd);
    }
    // r and dn = dh (1 + scale) weight
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      widen<T>(piece(0, i, raw_x[i]), r[i]);
      if (!kRing && next < rows) fetch(sp, row_of(a.x, next), i, raw_x[i]);
      float2 d[4];
      widen<T>(piece(1, i, raw_d[i]), d);
#pragma unroll
      for (int j = 0; j < 4; ++j) dn[i][j] = fmul2(d[j], factor[i][j]);
      if (a.branch.p) {
        float2 b[4];
        widen<T>(piece(2, i, raw_b[i]), b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (POST) b[j] = only_inside(sp, i, j, ffma2(b[j], pscale, pshift));  // the shift of columns past the width
          r[i][j] = ffma2(rs, r[i][j], fmul2(gate[i][j], b[j]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[i][j] = fmul2(rs, r[i][j]);
      }
    }
    const Moments m = row_moments<true>(sp, share, r, dn, a.norm == kNormLayer, inv, buf[turn][0]);
    if (kRing && threadIdx.x == 0 && ahead < rows) start();  // every thread is done with the rows before this one
    const float rstd = rsqrtf(m.squares * inv + a.eps);
    const float mean_dn = a.norm == kNormLayer ? m.sum_d * inv : 0.0f, mean_dnn = m.sum_dv * rstd * inv;
    const float2 minus = both(-m.mean), times = both(rstd);
    const float2 c_dn = both(-mean_dn * rstd), c_n = both(-mean_dnn * rstd);  // dr = rstd dn + c_dn + c_n n
    float2 v[POST ? NCH : 1][4];  // post norm: the branch's row once more
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float2 d[4], b[4], e4[4];
      widen<T>(piece(1, i, raw_d[i]), d);
      if (a.branch.p) widen<T>(piece(2, i, raw_b[i]), b);
      if (a.grad_r.p) widen<T>(piece(3, i, raw_e[i]), e4);
      if (!kRing && next < rows) {
        fetch(sp, row_of(a.grad_h, next), i, raw_d[i]);
        if (a.branch.p) fetch(sp, row_of(a.branch, next), i, raw_b[i]);
        if (a.grad_r.p) fetch(sp, row_of(a.grad_r, next), i, raw_e[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 n = fmul2(fadd2(r[i][j], minus), times);
        float2 dr = ffma2(dn[i][j], times, ffma2(n, c_n, c_dn));
        if (a.grad_r.p) dr = fadd2(dr, e4[j]);
        float2 pn = both(0.0f);
        if (a.branch.p) {
          pn = b[j];
          if constexpr (POST) {
            v[i][j] = b[j];
            pn = ffma2(b[j], pscale, pshift);
          }
          float2 db = fmul2(dr, gate[i][j]);
          if (POST) db = only_inside(sp, i, j, db);
          dn[i][j] = db;
        }
        if constexpr (kShared) {
          *shared_at(0, i, j) = fadd2(*shared_at(0, i, j), d[j]);
          *shared_at(1, i, j) = ffma2(d[j], n, *shared_at(1, i, j));
          *shared_at(2, i, j) = ffma2(dr, pn, *shared_at(2, i, j));
        } else {
          a0[i][j] = fadd2(a0[i][j], d[j]);
          a1[i][j] = ffma2(d[j], n, a1[i][j]);
          g0[i][j] = ffma2(dr, pn, g0[i][j]);
        }
        r[i][j] = fmul2(rs, dr);
      }
      if (a.out_h) store<T>(sp, a.out_h, out, i, r[i]);
      if (!POST && a.out_r) store<T>(sp, a.out_r, out, i, dn[i]);
    }
    if constexpr (POST) {
      // through the post norm: dn holds the gradient of its output, whose sums
      // with the branch's deviations are taken here (their squares are known)
      const Moments q = row_moments<true>(sp, share, v, dn, a.post == kNormLayer, inv, buf[turn][2]);
      const float pmean_d = a.post == kNormLayer ? q.sum_d * inv : 0.0f, pmean_dn = q.sum_dv * prstd * inv;
      const float2 c_d = both(-pmean_d * prstd), c_pn = both(-pmean_dn * prstd);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          dn[i][j] = ffma2(dn[i][j], pscale, ffma2(ffma2(v[i][j], pscale, pshift), c_pn, c_d));
        if (a.out_r) store<T>(sp, a.out_r, out, i, dn[i]);
      }
    }
  }
  if constexpr (kRing) ring.close();
  if (a.partial) {
    float* part = a.partial + static_cast<long long>(blockIdx.x) * 3 * a.width;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        float* to = part + static_cast<long long>(k) * a.width;
        float2 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kShared) s[j] = *shared_at(k, i, j);
          else s[j] = k == 0 ? a0[i][j] : k == 1 ? a1[i][j] : g0[i][j];
        }
        if constexpr (MODE != kUnaligned) {
          if (sp.inside(i, 0)) {
            float4* p = reinterpret_cast<float4*>(to + sp.column(i, 0));
            p[0] = make_float4(s[0].x, s[0].y, s[1].x, s[1].y);
            p[1] = make_float4(s[2].x, s[2].y, s[3].x, s[3].y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < kChunk; ++e)
            if (sp.inside(i, e)) to[sp.column(i, e)] = e & 1 ? s[e >> 1].y : s[e >> 1].x;
        }
      }
    }
  }
}

struct NormSumsArgs {
  const float* partial;
  VecTensor gate, scale;
  const void* weight;
  const void* post_weight;
  void *dgate, *dscale, *dshift, *dweight, *dpost;
  int gate_shared, scale_shared, shift_shared;  // one vector for all samples: its gradient is summed over them
  int samples, chunks, width;
};

// Column sums of the blocks' partials: 32 columns x 32 lanes of chunks per
// block, lanes added in order, samples one after the other.  blockIdx.y picks
// A0 (dshift), A1 (dscale, dweight) or G (dgate, dpost).
template <typename T>
__global__ void __launch_bounds__(1024) norm_sums_kernel(const __grid_constant__ NormSumsArgs a) {
  __shared__ float red[32][33];
  wait_for_prior();
  let_next_start();
  const int cx = threadIdx.x & 31, y = threadIdx.x >> 5, k = blockIdx.y;
  const int c = blockIdx.x * 32 + cx;
  void* each = k == 0 ? a.dshift : k == 1 ? a.dscale : a.dgate;      // one vector per sample, or their sum
  void* all = k == 0 ? nullptr : k == 1 ? a.dweight : a.dpost;       // summed over the samples
  const int shared = k == 0 ? a.shift_shared : k == 1 ? a.scale_shared : a.gate_shared;
  if (!each && !all) return;
  float sum_each = 0.0f, sum_all = 0.0f;
  for (int b = 0; b < a.samples; ++b) {
    float s = 0.0f;
    if (c < a.width) {
      const float* p = a.partial + static_cast<long long>(b) * a.chunks * 3 * a.width + static_cast<long long>(k) * a.width + c;
#pragma unroll 8
      for (int i = y; i < a.chunks; i += 32) s += p[static_cast<long long>(i) * 3 * a.width];
    }
    red[y][cx] = s;
    __syncthreads();
    if (y == 0 && c < a.width) {
      float t = 0.0f;
      for (int i = 0; i < 32; ++i) t += red[i][cx];
      float factor = 1.0f, other = 1.0f;
      if (k == 1) {
        if (a.weight) factor = to_f32<T>(static_cast<const T*>(a.weight)[c]);
        if (a.scale.p) other = 1.0f + to_f32<T>(static_cast<const T*>(a.scale.p)[b * a.scale.sb + c]);
      } else if (k == 2) {
        if (a.post_weight) factor = to_f32<T>(static_cast<const T*>(a.post_weight)[c]);
        if (a.gate.p) other = to_f32<T>(static_cast<const T*>(a.gate.p)[b * a.gate.sb + c]);
      }
      sum_all = fmaf(other, t, sum_all);
      sum_each = shared ? fmaf(factor, t, sum_each) : factor * t;
      if (each && !shared) static_cast<T*>(each)[static_cast<long long>(b) * a.width + c] = from_f32<T>(sum_each);
    }
    __syncthreads();
  }
  if (y == 0 && c < a.width) {
    if (each && shared) static_cast<T*>(each)[c] = from_f32<T>(sum_each);
    if (all) static_cast<T*>(all)[c] = from_f32<T>(sum_all);
  }
}

// ---- host side -----------------------------------------------------------------------
constexpr int kMaxWidth = 16384;

// Resident blocks of a kernel per SM, asked once.
int blocks_per_sm(const void* kernel, int threads, std::atomic<int>& known) {
  int n = known.load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n < 1) return 1;
  known.store(n, std::memory_order_relaxed);
  return n;
}

// Stages of a ring with ``blocks`` blocks per SM: as many as fit beside each
// block's static arrays and the system's part, two at least.
constexpr int kRingBudget = 220 * 1024;  // of one block alone
int ring_bytes_of(int blocks) { return (kRingBudget + 4096) / blocks - 4096; }
int ring_stages(int stage_bytes, int blocks) {
  const int n = ring_bytes_of(blocks) / stage_bytes;
  return n < 2 ? 2 : n > kMaxStages ? kMaxStages : n;
}

template <typename T, int WARPS, int NCH, int BLOCKS, int MODE, bool POST>
int launch_backward_mode(NormArgs a, cudaStream_t stream) {
  auto kernel = norm_backward_kernel<T, WARPS, NCH, BLOCKS, MODE, POST>;
  int smem = NCH > 3 ? 3 * NCH * kChunk * 32 * WARPS * 4 : 0;  // the column sums
  if (MODE != kUnaligned && WARPS > 1 && NCH <= 3) {
    a.stage_bytes = a.width * 2 * (a.grad_r.p ? 4 : a.branch.p ? 3 : 2);
    a.stages = ring_stages(a.stage_bytes, BLOCKS);
    smem = a.stages * a.stage_bytes;
  }
  if (smem > 0) {
    static std::atomic<unsigned long long> opened;
    const cudaError_t e = grant_smem(reinterpret_cast<const void*>(kernel), kRingBudget, opened);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return launch_overlapped(kernel, dim3(a.samples * a.chunks), dim3(32 * WARPS), smem, 0, stream, a);
}

template <typename T, int WARPS, int NCH, int BLOCKS, bool POST>
int launch_backward_aligned(const NormArgs& a, cudaStream_t stream) {
  if (a.width == 32 * kChunk * WARPS * NCH) return launch_backward_mode<T, WARPS, NCH, BLOCKS, kFull, POST>(a, stream);
  return launch_backward_mode<T, WARPS, NCH, BLOCKS, kAligned, POST>(a, stream);
}
template <typename T, int WARPS, int NCH, int BLOCKS, bool POST>
int launch_backward(const NormArgs& a, cudaStream_t stream) {
  if (!a.vec) return launch_backward_mode<T, WARPS, NCH, BLOCKS, kUnaligned, POST>(a, stream);
  return launch_backward_aligned<T, WARPS, NCH, BLOCKS, POST>(a, stream);
}

template <typename T, int WARPS, int NCH, int MODE, bool POST>
int launch_forward_mode(NormArgs a, cudaStream_t stream) {
  constexpr int kRows = WARPS < 4 ? 4 / WARPS : 1, kBlock = WARPS < 4 ? 128 : 32 * WARPS;
  auto kernel = norm_forward_kernel<T, WARPS, NCH, MODE, POST>;
  static std::atomic<int> resident;
  int blocks = blocks_per_sm(reinterpret_cast<const void*>(kernel), kBlock, resident), smem = 0;
  if (MODE != kUnaligned && WARPS > 1) {
    a.stage_bytes = a.width * 2 * (a.branch.p ? 2 : 1);
    while (blocks > 1 && ring_bytes_of(blocks) < 2 * a.stage_bytes) --blocks;
    // three stages: deeper rings read further ahead of the writes and measured
    // slower (34680 gated rows of 3072: 138 us with three, 156 with four)
    a.stages = ring_stages(a.stage_bytes, blocks) < 3 ? 2 : 3;
    smem = a.stages * a.stage_bytes;
    static std::atomic<unsigned long long> opened;
    const cudaError_t e = grant_smem(reinterpret_cast<const void*>(kernel), kRingBudget, opened);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const long long want = (static_cast<long long>(a.samples) * a.rows + kRows - 1) / kRows;
  const long long most = static_cast<long long>(kNumSMs) * blocks;
  return launch_overlapped(kernel, dim3(static_cast<unsigned>(want < most ? want : most)), dim3(kBlock), smem, 0, stream, a);
}

template <typename T, int WARPS, int NCH, bool POST>
int launch_forward_aligned(const NormArgs& a, cudaStream_t stream) {
  if (a.width == 32 * kChunk * WARPS * NCH) return launch_forward_mode<T, WARPS, NCH, kFull, POST>(a, stream);
  return launch_forward_mode<T, WARPS, NCH, kAligned, POST>(a, stream);
}
template <typename T, int WARPS, int NCH, bool POST>
int launch_forward(const NormArgs& a, cudaStream_t stream) {
  if (!a.vec) return launch_forward_mode<T, WARPS, NCH, kUnaligned, POST>(a, stream);
  return launch_forward_aligned<T, WARPS, NCH, POST>(a, stream);
}

// Threads per row.  Few warps keep a row's reduction cheap, few columns per
// thread its registers; measured at 34680 x 3072 with branch, gate and modulation:
// backward 235 us with 6 warps x 2 chunks, 318 with 12 x 1, 407 with 4 x 3 (three
// blocks of it per SM spill); forward 138 us with 4 x 3, 140 with 12 x 1, 174 with
// 8 x 2.  Unaligned rows hold a register per element ahead and take fewer of them
// (fp16 with branch, gate and weight): 14769 x 2241 backward 168 us with 12 x 1
// (348 with 6 x 2, two elements to a register), forward 68 us with 4 x 3, 90 with
// 8 x 2; 8000 x 6001 forward 104 us with 16 x 2, 151 with 8 x 3.
// The widest forms do not fit their registers: the forward above 8192 columns and
// the gradient above 6144 (unaligned 4096), and of 257 to 512, spill; with a post
// norm the gradient's other forms do too, by 0.1 to 0.2 KB a thread.  bf16 with
// branch, gate and modulation, floors in brackets: 8192 x 12288 forward 274 us
// (125), gradient 990 (188); 8192 x 8192 gradient 256 us (125); 8192 x 16383
// forward 1314 us (167).
template <typename T, bool POST>
int launch_norm(const NormArgs& a, bool backward, cudaStream_t stream) {
  const int w = a.width;
  if (backward) {
    if (w <= 256) return launch_backward<T, 1, 1, 12, POST>(a, stream);
    if (w <= 512) return launch_backward<T, 1, 2, 12, POST>(a, stream);
    if (w <= 1024) return launch_backward<T, 4, 1, 4, POST>(a, stream);
    if (!a.vec && w <= 4096) {
      if (w <= 2048) return launch_backward_mode<T, 8, 1, 2, kUnaligned, POST>(a, stream);
      if (w <= 3072) return launch_backward_mode<T, 12, 1, 1, kUnaligned, POST>(a, stream);
      return launch_backward_mode<T, 16, 1, 1, kUnaligned, POST>(a, stream);
    }
    if (w <= 2048) return launch_backward_aligned<T, 4, 2, 3, POST>(a, stream);
    if (w <= 3072) return launch_backward_aligned<T, 6, 2, 2, POST>(a, stream);
    if (w <= 4096) return launch_backward_aligned<T, 8, 2, 1, POST>(a, stream);
    if (w <= 6144) return launch_backward<T, 12, 2, 1, POST>(a, stream);
    if (w <= 8192) return launch_backward<T, 16, 2, 1, POST>(a, stream);
    return launch_backward<T, 16, 4, 1, POST>(a, stream);
  }
  if (w <= 256) return launch_forward<T, 1, 1, POST>(a, stream);
  if (w <= 768) return launch_forward<T, 1, 3, POST>(a, stream);
  if (w <= 1024) return launch_forward<T, 4, 1, POST>(a, stream);
  if (w <= 2048) return launch_forward<T, 4, 2, POST>(a, stream);
  if (w <= 3072) return launch_forward<T, 4, 3, POST>(a, stream);
  if (w <= 4096) return launch_forward<T, 8, 2, POST>(a, stream);
  if (a.vec && w <= 6144) return launch_forward_aligned<T, 8, 3, POST>(a, stream);
  if (w <= 8192) return launch_forward<T, 16, 2, POST>(a, stream);
  return launch_forward<T, 16, 4, POST>(a, stream);
}

int launch_any(const NormArgs& a, int dtype, bool backward, cudaStream_t stream) {
  if (a.post)
    return dtype == 1 ? launch_norm<__nv_bfloat16, true>(a, backward, stream) : launch_norm<__half, true>(a, backward, stream);
  return dtype == 1 ? launch_norm<__nv_bfloat16, false>(a, backward, stream) : launch_norm<__half, false>(a, backward, stream);
}

// Row chunks per sample of the backward kernel, one block each, but no more than
// there are rows: the resident blocks of launch_norm's aligned forms.  The
// unaligned forms of 1025 to 3072 columns hold fewer (two blocks per SM to 2048,
// one to 3072), so that theirs run in more than one round.
int norm_chunks(int samples, int rows, int width) {
  if (samples < 1) return 1;
  const long long per_sm = width <= 512 ? 12 : width <= 1024 ? 4 : width <= 2048 ? 3 : width <= 3072 ? 2 : 1;
  long long chunks = (per_sm * kNumSMs + samples - 1) / samples;
  if (chunks > rows) chunks = rows;
  return chunks < 1 ? 1 : static_cast<int>(chunks);
}

bool aligned(const void* p, long long s0, long long s1) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0);
}

bool valid_shape(int samples, int rows, int width, int norm, int post, float residual_scale) {
  return samples >= 0 && rows >= 0 && width >= 1 && (norm == kNormLayer || norm == kNormRms) && post >= kNormNone &&
         post <= kNormRms && residual_scale == residual_scale;
}

}  // namespace
}  // namespace peco

using namespace peco;

extern "C" int peco_gated_norm(const void* x, long long x_batch, long long x_row, const void* branch,
                               long long branch_batch, long long branch_row, const void* gate, long long gate_batch,
                               const void* scale, long long scale_batch, const void* shift, long long shift_batch,
                               const void* weight, const void* post_weight, void* residual, void* normed, int samples,
                               int rows, int width, int norm, int post_norm, float eps, float post_eps,
                               float residual_scale, int dtype, void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (!valid_shape(samples, rows, width, norm, post_norm, residual_scale)) return kErrInvalidValue;
  if (width > kMaxWidth || static_cast<long long>(samples) * rows > 0x7fffffffLL) return kErrUnsupported;
  if ((gate || post_norm || residual) && !branch) return kErrInvalidValue;
  if (post_weight && !post_norm) return kErrInvalidValue;
  if (samples == 0 || rows == 0) return kOk;
  if (!x || !normed) return kErrInvalidValue;
  NormArgs a{};
  a.x = RowTensor{x, x_batch, x_row};
  a.branch = RowTensor{branch, branch_batch, branch_row};
  a.gate = VecTensor{gate, gate_batch};
  a.scale = VecTensor{scale, scale_batch};
  a.shift = VecTensor{shift, shift_batch};
  a.weight = weight;
  a.post_weight = post_weight;
  a.out_r = residual;
  a.out_h = normed;
  a.samples = samples;
  a.rows = rows;
  a.width = width;
  a.vec = width % 8 == 0 && aligned(x, x_batch, x_row) && aligned(branch, branch_batch, branch_row) &&
          aligned(gate, gate_batch, 0) && aligned(scale, scale_batch, 0) && aligned(shift, shift_batch, 0) &&
          aligned(weight, 0, 0) && aligned(post_weight, 0, 0) && aligned(residual, 0, 0) && aligned(normed, 0, 0);
  a.norm = norm;
  a.post = post_norm;
  a.eps = eps;
  a.post_eps = post_eps;
  a.residual_scale = residual_scale;
  a.status = device_status_ptr();
  return launch_any(a, dtype, false, stream);
}

extern "C" long long peco_gated_norm_backward_workspace(int samples, int rows, int width) {
  if (samples < 0 || rows < 0 || width < 1) return -1;
  return 12LL * samples * norm_chunks(samples, rows, width) * width;
}

extern "C" int peco_gated_norm_backward(
    const void* grad_normed, long long gh_batch, long long gh_row, const void* grad_residual, long long gr_batch,
    long long gr_row, const void* x, long long x_batch, long long x_row, const void* branch, long long branch_batch,
    long long branch_row, const void* gate, long long gate_batch, const void* scale, long long scale_batch,
    const void* weight, const void* post_weight, void* dx, void* dbranch, void* dgate, void* dscale, void* dshift,
    int shared, void* dweight, void* dpost_weight, int samples, int rows, int width, int norm, int post_norm,
    float eps, float post_eps, float residual_scale, int dtype, void* workspace, long long workspace_bytes,
    void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (!valid_shape(samples, rows, width, norm, post_norm, residual_scale)) return kErrInvalidValue;
  if (width > kMaxWidth || static_cast<long long>(samples) * rows > 0x7fffffffLL) return kErrUnsupported;
  if (samples == 0 || rows == 0) return kErrInvalidValue;  // the sums over no rows are the caller's zeros
  if (!x || !grad_normed) return kErrInvalidValue;
  if ((gate || post_norm || grad_residual || dbranch) && !branch) return kErrInvalidValue;
  if ((post_weight && !post_norm) || (dgate && !gate) || (dscale && !scale) || (dweight && !weight) ||
      (dpost_weight && !post_weight))
    return kErrInvalidValue;
  const bool sums = dgate || dscale || dshift || dweight || dpost_weight;
  if (sums && !usable_workspace(workspace, workspace_bytes, peco_gated_norm_backward_workspace(samples, rows, width)))
    return kErrWorkspace;
  NormArgs a{};
  a.x = RowTensor{x, x_batch, x_row};
  a.branch = RowTensor{branch, branch_batch, branch_row};
  a.grad_h = RowTensor{grad_normed, gh_batch, gh_row};
  a.grad_r = RowTensor{grad_residual, gr_batch, gr_row};
  a.gate = VecTensor{gate, gate_batch};
  a.scale = VecTensor{scale, scale_batch};
  a.weight = weight;
  a.post_weight = post_weight;
  a.out_h = dx;
  a.out_r = dbranch;
  a.partial = sums ? static_cast<float*>(workspace) : nullptr;
  a.samples = samples;
  a.rows = rows;
  a.width = width;
  a.vec = width % 8 == 0 && aligned(x, x_batch, x_row) && aligned(branch, branch_batch, branch_row) &&
          aligned(grad_normed, gh_batch, gh_row) && aligned(grad_residual, gr_batch, gr_row) &&
          aligned(gate, gate_batch, 0) && aligned(scale, scale_batch, 0) && aligned(weight, 0, 0) &&
          aligned(post_weight, 0, 0) && aligned(dx, 0, 0) && aligned(dbranch, 0, 0);
  a.norm = norm;
  a.post = post_norm;
  a.eps = eps;
  a.post_eps = post_eps;
  a.residual_scale = residual_scale;
  a.status = device_status_ptr();
  a.chunks = norm_chunks(samples, rows, width);
  int st = launch_any(a, dtype, true, stream);
  if (st || !sums) return st;
  NormSumsArgs s{};
  s.partial = a.partial;
  s.gate = a.gate;
  s.scale = a.scale;
  s.weight = weight;
  s.post_weight = post_weight;
  s.dgate = dgate;
  s.dscale = dscale;
  s.dshift = dshift;
  s.dweight = dweight;
  s.dpost = dpost_weight;
  s.gate_shared = shared & 1;
  s.scale_shared = shared & 2;
  s.shift_shared = shared & 4;
  s.samples = samples;
  s.chunks = a.chunks;
  s.width = width;
  const dim3 grid((width + 31) / 32, 3);
  return dtype == 1 ? launch_overlapped(norm_sums_kernel<__nv_bfloat16>, grid, dim3(1024), 0, 0, stream, s)
                    : launch_overlapped(norm_sums_kernel<__half>, grid, dim3(1024), 0, 0, stream, s);
}
