// Gradient of attention over key spans on sm_100a tensor cores (see
// span_attention.cuh).  With p_ij = exp(z_ij - lse_i), delta_i = sum_d g_id out_id
// and s' = dz/d(scale q.k), 1 or 1 - tanh^2:
//   ds_ij = p_ij (g_i.v_j - delta_i) s'_ij
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij g_i
// A row that sees one key has ds 0; rows of few keys take delta_i = sum_j p_ij (g_i.v_j).
//
// One launch holds two kinds of CTAs.  Those of 128 keys walk the query tiles (of
// all the heads that share the keys) and keep dk and dv in TMEM; those of 128
// query rows walk the keys and keep dq.  Scores and g.v are computed in both,
// seven products instead of five; in exchange no sum crosses a CTA: there are no
// atomics, no fp32 copy of dq in memory, and results do not depend on the launch.
//
// What it measured (B200, bf16): 24 heads x 7006 rows x 128 dims, every key: 1580 us (0.92
// PFLOP/s of five products, 1.28 of the seven; 1.8 ms at the power limit after 300
// calls in a row), the CTAs of keys alone 950, those of rows 655; tensor pipe 64%. In the
// CTAs of keys every product waits for the one whose operand it overwrites, and so
// for the softmax between; issuing S right behind dv's product (1640 us), or the two
// chains by a warp each (1680 us), was slower, although both wait less.
// Capped scores 2660 us (two more special functions a pair: 1580 us of that unit in all),
// under a cap above 64 2960 us, a bias by distance 2120 us; their slopes go into p before g.v is read (after it, which
// held three rows of registers at once: 4090 and 2790 us).
// Under two documents 1570 us: a warp reads each step's statistics and spans while the
// place for them is still in use (read after it was free: 1890 us).
#include "span_attention.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"

namespace peco {
namespace {

constexpr int kGradThreads = 384;  // eight softmax warps, then TMA, MMA, MMA and statistics warps
// Tiles that stream past a CTA's own two: of Q (under a tile of keys) or K (under a
// tile of rows), used by its step's first and last product, and of g or V.
constexpr int kSecond = 2;
template <bool RICH>
constexpr int kFirst = RICH ? 2 : 3;  // (capped or biased scores keep the rows' positions there)

struct GradArgs {
  ScoreArgs s;
  HeadRows out, grad, q, k, v;  // of the statistics
  const float* lse;
  float2* stats;             // [batch, heads, padded rows]: lse in log2 units (none: infinity) and delta
  int padded;                // rows, a multiple of 128
  void *dq, *dk, *dv;
  long long q_batch, q_head, q_row, k_batch, k_head, k_row, v_batch, v_head, v_row;
  int key_units, query_units;
  Turns turns;               // of heads and their query tiles
  Divisor blocks, by_parts, kv;  // tiles of keys, parts, key heads
  int parts;                 // CTAs that share a tile of keys, each some of the heads on them
  float* part;               // with several: dv, then dk, [parts, batch, key heads, keys, dims] each
};

// fp16's small probabilities would lose bits below 2^-14: they are held 2^10
// times larger (at most 2^10), and dv is scaled back.
template <int AB>
struct Held {
  static constexpr float kShift = AB == 1 ? 0.0f : 10.0f, kBack = AB == 1 ? 1.0f : 1.0f / 1024.0f;
};

// Rows of up to this many keys take delta from their probabilities.  The rounding of
// ``out`` is one error in every ds of a row, and the fewer the keys, the more of ds it
// is: relative error of dq over 2 keys 0.0038 (bf16) with it and 0.0023 without, 4
// keys 0.0030, 8 keys 0.0027, 128 keys 0.0024.  The statistics of 24 heads x 16000 rows
// of 7 keys each take 232 us with it (39 without), of 24 x 4096 rows in causal order 15 (12).
constexpr int kFewKeys = 8;

// sum_j p_j (g.v_j) over a row's ``count`` keys from ``lo`` on, 16 lanes a row with 8 dims
// each, two keys at a time.  By whole warps.
template <int AB>
__device__ __noinline__ float few_keys_delta(const GradArgs& a, int b, int h, int i, int lo, int pos, int count, float lse,
                                             int lane) {
  using T = Element<AB>;
  const int most = __reduce_max_sync(0xffffffffu, count), kv = a.s.group(h), at = lane >> 3 & 1;
  const float slope = a.s.slopes ? a.s.slopes[h] * kLog2E : 0.0f;
  const Cap cap(a.s);
  float q[8] = {}, g[8] = {}, delta = 0.0f;
  if (lane * 8 >= a.s.d) count = 0;  // (of what this lane reads)
  const int reads = count;
  count = __shfl_sync(0xffffffffu, count, threadIdx.x & 16);
  if (reads > 0) {
    load8(static_cast<const T*>(a.grad.ptr) + b * a.grad.batch + h * a.grad.head + static_cast<long long>(i) * a.grad.row + lane * 8, 1, 8, g);
    load8(static_cast<const T*>(a.q.ptr) + b * a.q.batch + h * a.q.head + static_cast<long long>(i) * a.q.row + lane * 8, 1, 8, q);
  }
  const T* k = static_cast<const T*>(a.k.ptr) + b * a.k.batch + kv * a.k.head + lo * a.k.row + lane * 8;
  const T* v = static_cast<const T*>(a.v.ptr) + b * a.v.batch + kv * a.v.head + lo * a.v.row + lane * 8;
  for (int n = 0; n < most; n += 2) {
    float score[2] = {}, gv[2] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (n + u < reads) {
        float x[8];
        load8(k, 1, 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) score[u] = fmaf(q[e], x[e], score[u]);
        load8(v, 1, 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) gv[u] = fmaf(g[e], x[e], gv[u]);
      }
      k += a.k.row;
      v += a.v.row;
    }
    // sums over the lanes: half of them take one key, and of those half the score
    const bool second = lane & 8, value = lane & 4;
    float s = second ? score[1] : score[0], y = second ? gv[1] : gv[0];
    s += __shfl_xor_sync(0xffffffffu, second ? score[0] : score[1], 8);
    y += __shfl_xor_sync(0xffffffffu, second ? gv[0] : gv[1], 8);
    float sum = value ? y : s;
    sum += __shfl_xor_sync(0xffffffffu, value ? s : y, 4);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    const float other = __shfl_xor_sync(0xffffffffu, sum, 4);
    s = value ? other : sum;
    y = value ? sum : other;
    float z = a.s.cap > 0.0f ? cap.value(s, cap.recip(s)) : s * a.s.scale * kLog2E;
    if (a.s.slopes) z = fmaf(-slope, fabsf(static_cast<float>(pos - lo - n - at)), z);
    if (n + at < count) delta = fmaf(exp2_approx(z - lse), y, delta);
  }
  return delta + __shfl_xor_sync(0xffffffffu, delta, 8);
}

// stats of every row; 16 lanes a row.  FEW: some row may see few keys.
template <int AB, bool FEW>
__global__ void __launch_bounds__(256, 8) grad_stats_kernel(const __grid_constant__ GradArgs a) {
  using T = Element<AB>;
  wait_for_prior();
  let_next_start();
  // the first rows of all heads first: in causal order they are those of few keys, which take longer
  const unsigned all = static_cast<unsigned>(a.s.batch) * static_cast<unsigned>(a.s.heads), rows = blockIdx.x / all;
  const unsigned heads = blockIdx.x - rows * all;  // head of all samples
  const int i = static_cast<int>(rows * 16 + (threadIdx.x >> 4)), lane = threadIdx.x & 15;
  const int b = static_cast<int>(heads / a.s.heads), h = static_cast<int>(heads % a.s.heads);
  const long long at = static_cast<long long>(heads) * a.padded + i;
  bool few = false;
  float l = -INFINITY, sum = 0.0f;
  if (i < a.s.sq) l = a.lse[static_cast<long long>(heads) * a.s.sq + i];
  if constexpr (FEW) {
    // a row of the tile sees at least the keys from the largest first to the least last
    const int4 bounds = tile_span(a.s, b, static_cast<int>(rows / (kTile / 16)));
    if (bounds.w <= kFewKeys || bounds.z >= bounds.w - kFewKeys) {
      int4 span = make_int4(0, 0, 0, 0);
      if (i < a.s.sq) span = span_of(a.s, b, i);
      few = span.x >= 0 && span.y <= a.s.sk && span.y - span.x <= kFewKeys && span.y > span.x;
      if (__any_sync(0xffffffffu, few)) sum = few_keys_delta<AB>(a, b, h, i, span.x, span.z, few ? span.y - span.x : 0, l * kLog2E, lane);
    }
  }
  if (!few) {
    sum = 0.0f;
    if (i < a.s.sq && lane * 8 < a.s.d) {
      float x[8], y[8];
      load8(static_cast<const T*>(a.out.ptr) + b * a.out.batch + h * a.out.head + static_cast<long long>(i) * a.out.row + lane * 8, 1, 8, x);
      load8(static_cast<const T*>(a.grad.ptr) + b * a.grad.batch + h * a.grad.head + static_cast<long long>(i) * a.grad.row + lane * 8, 1, 8, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e], y[e], sum);
    }
  }
  float all16 = sum;
#pragma unroll
  for (int o = 8; o; o >>= 1) all16 += __shfl_xor_sync(0xffffffffu, all16, o);
  if (!few) sum = all16;
  if (lane == 0)
    a.stats[at] = l == -INFINITY ? make_float2(INFINITY, 0.0f) : make_float2(l * kLog2E - Held<AB>::kShift, sum * Held<AB>::kBack);
}

// One step of a CTA of keys: a query tile of one head, as the statistics warp lays it out.
template <bool RICH>
struct Step {
  float lse[kTile], delta[kTile];
  uint32_t range[kTile / 2];  // 16 bits a row: first key of the tile that it sees (0 to 127), kOneKey, the key behind the last << 8
  float pos[RICH ? kTile : 4];
  int masked, clear, end, head;  // masked: 1, or 2 with rows of one key
};
// A row that sees one key has p = 1 whatever its score, so its ds are 0: the difference
// of g.v and delta, sums of different orders, would be what is left of their rounding.
constexpr uint32_t kOneKey = 0x80, kBlind = 0xff;  // a row that sees nothing: kOneKey, from 127 to 0

template <bool RICH>
struct __align__(16) GradShared {
  Step<RICH> step[2];
  uint64_t own_full;                              // the CTA's own two tiles
  uint64_t first_full[3], first_empty[3], second_full[2], second_empty[2], step_full[2], step_empty[2];
  uint64_t s_full[2], p_full, dp_full, dp_free, ds_full[2], dq_done[2], p_read, ds_read, done;
  uint32_t tmem;
  int first, last, abort_flag;
};

template <int D, bool RICH>
constexpr int tiles_bytes() { return (2 + kFirst<RICH> + kSecond) * kTile * D * 2; }
template <int D, bool RICH>
constexpr int grad_smem() {
  constexpr int need = tiles_bytes<D, RICH>() + static_cast<int>(sizeof(GradShared<RICH>));
  return need + 1024 < 227 * 1024 ? need + 1024 : 227 * 1024;  // room to start on 1024 bytes
}
static_assert(tiles_bytes<128, false>() + sizeof(GradShared<false>) <= 227 * 1024 &&
                  tiles_bytes<128, true>() + sizeof(GradShared<true>) <= 226 * 1024, "shared memory of a CTA");

struct Roles {
  int warp, lane;
  bool ok;
  volatile int* abort_flag;
  unsigned* status;
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t phase) {
    if (ok) ok = warp_wait(bar, phase & 1, abort_flag, status);
    if (ok) tc_fence_after();
    return ok;
  }
  __device__ __forceinline__ void arrive(uint64_t* bar) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  }
  __device__ __forceinline__ void land() {  // copies in flight land before the CTA ends
    if (ok) return;
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) {
    }
  }
};

// 64 columns of TMEM as fp32
__device__ __forceinline__ void load_half(uint32_t at, float (&v)[64]) {
  uint32_t raw[64];
  tmem_ld64_sync(at, raw);
#pragma unroll
  for (int e = 0; e < 64; ++e) v[e] = __uint_as_float(raw[e]);
}
template <typename T>
__device__ __forceinline__ void store_half(uint32_t at, const float (&v)[64]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t packed[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) packed[e] = pack2<T>(v[c * 32 + 2 * e], v[c * 32 + 2 * e + 1]);
    tmem_st16(at + c * 16, packed);
  }
  tmem_st_wait();
}

// Rows of an accumulator, scaled, to memory (zeros without one) by way of ``stage``
template <typename T, int D>
__device__ __forceinline__ void store_row(T* out, uint32_t at, float scale, int d, bool any, const RowsOut<D>& stage) {
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    uint32_t raw[32];
    if (any) tmem_ld32_sync(at + c * 32, raw);
    else
#pragma unroll
      for (int e = 0; e < 32; ++e) raw[e] = 0u;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        u[e] = pack2<T>(__uint_as_float(raw[g * 8 + 2 * e]) * scale, __uint_as_float(raw[g * 8 + 2 * e + 1]) * scale);
      stage.put(c * 4 + g, make_uint4(u[0], u[1], u[2], u[3]));
    }
  }
  stage.store(out, d);
}

// The same in fp32, for the sum over the parts
template <int D>
__device__ __forceinline__ void store_part(float* out, uint32_t at, float scale, int d, bool any) {
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    uint32_t raw[32];
    if (any) tmem_ld32_sync(at + c * 32, raw);
    else
#pragma unroll
      for (int e = 0; e < 32; ++e) raw[e] = 0u;
    if (out) {
#pragma unroll
      for (int g = 0; g < 8; ++g)
        if (c * 32 + g * 4 < d)
          *reinterpret_cast<float4*>(out + c * 32 + g * 4) =
              make_float4(__uint_as_float(raw[g * 4]) * scale, __uint_as_float(raw[g * 4 + 1]) * scale,
                          __uint_as_float(raw[g * 4 + 2]) * scale, __uint_as_float(raw[g * 4 + 3]) * scale);
    }
  }
}

// Zeros in the rows of a tile of keys that no row of a tile of query rows sees (they may
// hold anything, and 0 times that would reach dq), by one warp; visible to the tensor
// core.  ``spans``: four query rows' a lane; j0: the tile's first key.
template <int PANELS>
__device__ __forceinline__ void clear_unseen(unsigned char* tile, const int4 (&spans)[kTile / 32], int j0, int lane) {
  uint32_t seen[kTile / 32] = {};  // a bit a key
  bool whole = false;              // a row that sees all
#pragma unroll
  for (int i = 0; i < kTile / 32; ++i) {
    const int from = max(spans[i].x - j0, 0), to = min(spans[i].y - j0, kTile);
    whole = whole || to - from == kTile;
#pragma unroll
    for (int w = 0; w < kTile / 32; ++w) {
      const int lo = max(from - 32 * w, 0), hi = min(to - 32 * w, 32);
      if (lo < hi) seen[w] |= 0xffffffffu >> (32 - (hi - lo)) << lo;
    }
  }
  if (__any_sync(0xffffffffu, whole)) return;
#pragma unroll
  for (int w = 0; w < kTile / 32; ++w) {
    const bool blind = !(__reduce_or_sync(0xffffffffu, seen[w]) >> lane & 1u);
    if (blind)
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(tile + p * kPanelBytes + (32 * w + lane) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncwarp();
}

// The steps of a CTA of keys: heads of the group, query tiles that see one of its keys.
struct StepWalk {
  int head, tile;
  __device__ __forceinline__ bool next(const ScoreArgs& s, int b, int j0, int first, int last, int end_head) {
    for (;;) {
      if (++tile >= last) {
        tile = first - 1;
        if (++head >= end_head) return false;
        continue;
      }
      if (!s.spans) return true;
      const int4 t = tile_span(s, b, tile);
      if (t.x < j0 + kTile && t.y > j0) return true;
    }
  }
};

template <int AB, int D, bool RICH, bool WIDE>
__global__ void __launch_bounds__(kGradThreads, 1)
    span_attention_grad_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                               const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap gmap,
                               const __grid_constant__ GradArgs a) {
  using T = Element<AB>;
  constexpr int kPanels = D / 64, kTileBytes = kPanels * kPanelBytes;
  constexpr uint32_t kDims = instr_desc(kTile, kTile, AB, false, false), kRows = instr_desc(kTile, D, AB, false, true);
  constexpr int kFirsts = kFirst<RICH>;
  constexpr uint32_t kTileStep = kTileBytes >> 4;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* firsts = base + 2 * kTileBytes;
  unsigned char* seconds = firsts + kFirsts * kTileBytes;
  GradShared<RICH>& sh = *reinterpret_cast<GradShared<RICH>*>(base + tiles_bytes<D, RICH>());
  if (base - smem_raw + tiles_bytes<D, RICH>() + static_cast<int>(sizeof(sh)) > grad_smem<D, RICH>()) {
    record_status(a.s.status, kDevBadIndex);  // (dynamic shared memory starts on 1024 bytes where nothing else is in front)
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Roles me{warp, lane, true, &sh.abort_flag, a.s.status};
  const bool of_keys = static_cast<int>(blockIdx.x) < a.key_units;
  if (threadIdx.x == 0) {
    mbar_init(&sh.own_full, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&sh.first_full[i], 1);
      mbar_init(&sh.first_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.second_full[i], 1);
      mbar_init(&sh.second_empty[i], 1);
      mbar_init(&sh.step_full[i], 1);
      mbar_init(&sh.step_empty[i], 1);
      mbar_init(&sh.dq_done[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.ds_full[i], 8);
    }
    mbar_init(&sh.p_full, 8);
    mbar_init(&sh.dp_full, 1);
    mbar_init(&sh.dp_free, 8);
    mbar_init(&sh.p_read, 1);
    mbar_init(&sh.ds_read, 1);
    mbar_init(&sh.done, 1);
    sh.abort_flag = 0;
    sh.first = 0x7fffffff;
    sh.last = 0;
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    prefetch_tensormap(&gmap);
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_prior();
  let_next_start();
  const uint32_t tmem = sh.tmem;
  const int group = a.s.group.by;
  const int half = (warp >> 2) & 1;  // of a softmax warp: its 64 columns
  const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const int r = (warp & 3) * 32 + lane;
  const float scale_log2 = a.s.scale * kLog2E;
  const RowsOut<D> stage{base + warp * (32 * D * 2), lane};  // of a softmax warp, where the CTA's own tiles are read no more

  if (of_keys) {
    // ================================================================ dk and dv of 128 keys
    const int unit = a.blocks(blockIdx.x), j0 = (static_cast<int>(blockIdx.x) - unit * a.blocks.by) * kTile;
    const int heads = a.by_parts(unit), part = unit - heads * a.parts, b = a.kv(heads), kv = heads - b * a.s.kv_heads;
    const int head0 = kv * group + a.by_parts(part * group), head_end = kv * group + a.by_parts((part + 1) * group);
    const int tiles = row_tiles(a.s);
    if (a.s.spans) {  // the query tiles between the first and the last that see one of the keys
      for (int t = threadIdx.x; t < tiles; t += kGradThreads) {
        const int4 sp = tile_span(a.s, b, t);
        if (sp.x < j0 + kTile && sp.y > j0) {
          atomicMin(&sh.first, t);
          atomicMax(&sh.last, t + 1);
        }
      }
    } else if (threadIdx.x == 0) {
      sh.first = 0;
      sh.last = tiles;
    }
    __syncthreads();
    const int first = sh.first, last = sh.last;
    const bool any = first < last;
    const uint32_t s_at = tmem, dp_at = tmem + kTile, dv_at = tmem + 2 * kTile, dk_at = tmem + 3 * kTile;
    StepWalk walk{head0, first - 1};
    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (any && warp == 8) {
        // ------------------------------------------------------------ TMA
        const bool issuer = elect_one();
        if (issuer) {
          mbar_arrive_expect_tx(&sh.own_full, 2 * kTileBytes);
          load_rows<kPanels>(base, &kmap, j0, kv, b, &sh.own_full);
          load_rows<kPanels>(base + kTileBytes, &vmap, j0, kv, b, &sh.own_full);
        }
        __syncwarp();
        RingPos f{0, 0}, s{0, 0};
        while (me.ok && walk.next(a.s, b, j0, first, last, head_end)) {
          if (!me.wait(&sh.first_empty[f.s], f.phase ^ 1)) break;
          if (issuer) {
            mbar_arrive_expect_tx(&sh.first_full[f.s], kTileBytes);
            load_rows<kPanels>(firsts + f.s * kTileBytes, &qmap, walk.tile * kTile, walk.head, b, &sh.first_full[f.s]);
          }
          __syncwarp();
          if (!me.wait(&sh.second_empty[s.s], s.phase ^ 1)) break;
          if (issuer) {
            mbar_arrive_expect_tx(&sh.second_full[s.s], kTileBytes);
            load_rows<kPanels>(seconds + s.s * kTileBytes, &gmap, walk.tile * kTile, walk.head, b, &sh.second_full[s.s]);
          }
          __syncwarp();
          f.step(kFirsts);
          s.step(kSecond);
        }
        me.land();
      } else if (any && warp == 11) {
        // ------------------------------------------------------------ statistics of each step
        for (int n = 0;; ++n) {
          const bool more = walk.next(a.s, b, j0, first, last, head_end);
          // read before the place is free, so that only the stores follow the step before
          constexpr int kEach = kTile / 32;
          float2 stat[kEach];
          int4 span[kEach];
          bool full = true, blind = false, ones = false;
          if (more) {
            const int i0 = walk.tile * kTile;
            const int4 t = tile_span(a.s, b, walk.tile);
            // (a row that sees the last key alone would pass for one that sees the whole tile)
            full = t.z <= j0 && t.w >= min(j0 + kTile, a.s.sk) && t.z < a.s.sk - 1 && i0 + kTile <= a.s.sq;
            blind = t.z == 0x7fffffff;  // some row sees nothing
            const float2* stats = a.stats + (static_cast<long long>(b) * a.s.heads + walk.head) * a.padded + i0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
              const int i = i0 + e * 32 + lane;
              stat[e] = stats[e * 32 + lane];
              span[e] = (RICH || !full) && i < a.s.sq ? span_of(a.s, b, i) : make_int4(0, 0, 0, 0);
              ones = ones || span[e].y - span[e].x == 1;
            }
            ones = __any_sync(0xffffffffu, ones);
          }
          Step<RICH>& step = sh.step[n & 1];
          if (!me.wait(&sh.step_empty[n & 1], (n >> 1) + 1)) break;
          if (more) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
              const int i = e * 32 + lane;
              step.lse[i] = stat[e].x;
              step.delta[i] = stat[e].y;
              if (RICH || !full) {
                const int from = min(max(span[e].x - j0, 0), kTile), to = min(max(span[e].y - j0, 0), kTile);
                const uint32_t seen = (from < to ? from | to << 8 : 0) | (span[e].y - span[e].x == 1 ? kOneKey : 0);
                reinterpret_cast<uint16_t*>(step.range)[i] = static_cast<uint16_t>(span[e].y > span[e].x ? seen : kBlind);
                if constexpr (RICH) step.pos[i] = static_cast<float>(span[e].z - j0);  // from the tile's first key
              }
            }
            if (lane == 0) {
              step.head = walk.head;
              step.masked = full ? 0 : ones ? 2 : 1;
              step.clear = blind ? 1 : 0;
            }
          }
          if (lane == 0) step.end = more ? 0 : 1;
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.step_full[n & 1]);
          if (!more) break;
        }
      } else if (any && warp == 9) {
        // ------------------------------------------------------------ MMA
        const bool issuer = elect_one();
        const uint32_t at = uniform(tmem), s_to = at, dp_to = at + kTile, dv_to = at + 2 * kTile, dk_to = at + 3 * kTile;
        const uint32_t k = uniform(desc_dims(smem_u32(base))), v = k + kTileStep;
        const uint32_t q_dims = k + 2 * kTileStep, g_dims = q_dims + kFirsts * kTileStep;
        const uint32_t q_rows = uniform(desc_rows(smem_u32(firsts))), g_rows = q_rows + kFirsts * kTileStep;
        // the step's rows are there, those that see nothing zeroed (they may hold anything); false at the end
        auto ready = [&](int n, const RingPos& f, const RingPos& s) {
          const Step<RICH>& step = sh.step[n & 1];
          if (!me.wait(&sh.step_full[n & 1], n >> 1) || step.end || !me.wait(&sh.first_full[f.s], f.phase)) return false;
          if (step.clear) {
            if (!me.wait(&sh.second_full[s.s], s.phase)) return false;
            for (int row = lane; row < kTile; row += 32)
              if (reinterpret_cast<const uint16_t*>(step.range)[row] == kBlind)
                for (int p = 0; p < kPanels; ++p)
                  for (int c = 0; c < 8; ++c) {
                    *reinterpret_cast<uint4*>(firsts + f.s * kTileBytes + p * kPanelBytes + row * 128 + c * 16) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(seconds + s.s * kTileBytes + p * kPanelBytes + row * 128 + c * 16) = make_uint4(0, 0, 0, 0);
                  }
            fence_async_smem();
            __syncwarp();
          }
          return true;
        };
        RingPos f{0, 0}, s{0, 0};
        auto scores = [&]() {
          if (issuer) {
            product_dims<D>(s_to, k, q_dims + f.s * kTileStep, kDims);
            umma_commit(&sh.s_full[0]);
          }
          __syncwarp();
        };
        auto values = [&]() {
          if (!me.wait(&sh.second_full[s.s], s.phase)) return;
          if (issuer) {
            product_dims<D>(dp_to, v, g_dims + s.s * kTileStep, kDims);
            umma_commit(&sh.dp_full);
          }
          __syncwarp();
        };
        me.wait(&sh.own_full, 0);
        bool more = me.ok && ready(0, f, s);
        if (more) {
          scores();
          values();
        }
        for (int n = 0; more && me.ok; ++n) {
          const int q_slot = f.s, g_slot = s.s;
          if (!me.wait(&sh.p_full, n)) break;
          if (issuer) {
            product_rows<kTile>(dv_to, s_to, g_rows + g_slot * kTileStep, kRows, n > 0);
            umma_commit(&sh.second_empty[g_slot]);
            umma_commit(&sh.p_read);
          }
          __syncwarp();
          f.step(kFirsts);
          s.step(kSecond);
          more = ready(n + 1, f, s);
          if (more && !me.wait(&sh.p_read, n)) break;  // S goes where the probabilities were
          if (more) scores();
          if (!me.wait(&sh.ds_full[0], n)) break;
          if (issuer) {
            product_rows<kTile>(dk_to, dp_to, q_rows + q_slot * kTileStep, kRows, n > 0);
            umma_commit(&sh.first_empty[q_slot]);
            umma_commit(&sh.step_empty[n & 1]);
            umma_commit(more ? &sh.ds_read : &sh.done);
          }
          __syncwarp();
          if (more && !me.wait(&sh.ds_read, n)) break;  // g.v goes where ds was
          if (more) values();
        }
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      // -------------------------------------------------------------- probabilities; a key a thread
      const int j = j0 + r;
      const Cap cap(a.s);
      const float at_key = static_cast<float>(r);
      const uint32_t s_own = s_at + lanes + half * 64, dp_own = dp_at + lanes + half * 64;
      int n = 0;
      for (; any; ++n) {
        const Step<RICH>& step = sh.step[n & 1];
        if (!me.wait(&sh.step_full[n & 1], n >> 1) || step.end) break;
        if (!me.wait(&sh.s_full[0], n)) break;
        const int c0 = half * 64;
        float p[64], slopes[RICH ? 64 : 1];
        load_half(s_own, p);
        if constexpr (RICH) {
          scaled_scores<WIDE>(a.s, cap, p, slopes);
          if (a.s.slopes) {
            const float bias = a.s.slopes[step.head] * kLog2E;
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
              const float4 pos = *reinterpret_cast<const float4*>(step.pos + c0 + e);
              const float2 x = fadd2(make_float2(pos.x, pos.y), make_float2(-at_key, -at_key));
              const float2 y = fadd2(make_float2(pos.z, pos.w), make_float2(-at_key, -at_key));
              p[e] = fmaf(-bias, fabsf(x.x), p[e]);
              p[e + 1] = fmaf(-bias, fabsf(x.y), p[e + 1]);
              p[e + 2] = fmaf(-bias, fabsf(y.x), p[e + 2]);
              p[e + 3] = fmaf(-bias, fabsf(y.y), p[e + 3]);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const float4 l = *reinterpret_cast<const float4*>(step.lse + c0 + e);
          if constexpr (RICH) {
            const float2 x = fadd2(make_float2(p[e], p[e + 1]), make_float2(-l.x, -l.y));
            const float2 y = fadd2(make_float2(p[e + 2], p[e + 3]), make_float2(-l.z, -l.w));
            p[e] = x.x;
            p[e + 1] = x.y;
            p[e + 2] = y.x;
            p[e + 3] = y.y;
          } else {
            const float2 sc = make_float2(scale_log2, scale_log2);
            const float2 x = ffma2(make_float2(p[e], p[e + 1]), sc, make_float2(-l.x, -l.y));
            const float2 y = ffma2(make_float2(p[e + 2], p[e + 3]), sc, make_float2(-l.z, -l.w));
            p[e] = x.x;
            p[e + 1] = x.y;
            p[e + 2] = y.x;
            p[e + 3] = y.y;
          }
        }
#pragma unroll
        for (int e = 0; e < 64; ++e) p[e] = exp2_approx(p[e]);
        const int masked = step.masked;
        if (masked) {
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            const uint32_t two = step.range[(c0 + e) >> 1];
            p[e] = r >= static_cast<int>(two & 127u) && r < static_cast<int>(two >> 8 & 255u) ? p[e] : 0.0f;
            p[e + 1] = r >= static_cast<int>(two >> 16 & 127u) && r < static_cast<int>(two >> 24) ? p[e + 1] : 0.0f;
          }
        }
        store_half<T>(s_own, p);
        me.arrive(&sh.p_full);
        if constexpr (RICH) {
          if (a.s.cap > 0.0f) {
            if (masked) {  // a score of NaN has a slope of NaN: 0 in its place, for the 0 of a masked pair (a seen one's p is NaN)
#pragma unroll
              for (int e = 0; e < 64; ++e) slopes[e] = fmaxf(slopes[e], 0.0f);
            }
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const float2 x = fmul2(make_float2(p[e], p[e + 1]), make_float2(slopes[e], slopes[e + 1]));
              p[e] = x.x;
              p[e + 1] = x.y;
            }
          }
        }
        if (!me.wait(&sh.dp_full, n)) break;
        float ds[64];
        load_half(dp_own, ds);
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const float4 l = *reinterpret_cast<const float4*>(step.delta + c0 + e);
          const float2 back = make_float2(Held<AB>::kBack, Held<AB>::kBack);
          const float2 x = ffma2(make_float2(ds[e], ds[e + 1]), back, make_float2(-l.x, -l.y));
          const float2 y = ffma2(make_float2(ds[e + 2], ds[e + 3]), back, make_float2(-l.z, -l.w));
          ds[e] = p[e] * x.x;
          ds[e + 1] = p[e + 1] * x.y;
          ds[e + 2] = p[e + 2] * y.x;
          ds[e + 3] = p[e + 3] * y.y;
        }
        if (masked) {  // a masked pair's g.v may be anything
#pragma unroll
          for (int e = 0; e < 64; ++e) ds[e] = p[e] == 0.0f ? 0.0f : ds[e];
          if (masked > 1) {  // (a NaN stays)
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const uint32_t two = step.range[(c0 + e) >> 1];
              if (two & kOneKey) ds[e] *= 0.0f;
              if (two & kOneKey << 16) ds[e + 1] *= 0.0f;
            }
          }
        }
        store_half<T>(dp_own, ds);
        me.arrive(&sh.ds_full[0]);
      }
      if (any) me.wait(&sh.done, 0);
      if (me.ok) {  // the first warps store dv, the others dk
        const uint32_t at = (half ? dk_at : dv_at) + lanes;
        const float back = half ? a.s.scale : Held<AB>::kBack;
        const bool wanted = j < a.s.sk && (half ? a.dk : a.dv);
        if (a.parts > 1) {
          const long long rows = static_cast<long long>(a.s.batch) * a.s.kv_heads * a.s.sk;
          const long long row = (static_cast<long long>(b) * a.s.kv_heads + kv) * a.s.sk + j;
          store_part<D>(wanted ? a.part + ((half * a.parts + part) * rows + row) * a.s.d : nullptr, at, back, a.s.d, any);
        } else {
          T* out = nullptr;
          if (wanted)
            out = half ? static_cast<T*>(a.dk) + b * a.k_batch + kv * a.k_head + static_cast<long long>(j) * a.k_row
                       : static_cast<T*>(a.dv) + b * a.v_batch + kv * a.v_head + static_cast<long long>(j) * a.v_row;
          store_row<T, D>(out, at, back, a.s.d, any, stage);
        }
      }
    }
  } else {
    // ================================================================ dq of 128 query rows
    const int tiles = row_tiles(a.s), unit = static_cast<int>(blockIdx.x) - a.key_units;
    int b, head, rank;
    a.turns.at(unit, b, head, rank);
    const int tile = ranked_tile(a.s, b, rank, tiles), i0 = tile * kTile, kv = a.s.group(head);
    const int4 seen = tile_span(a.s, b, tile);
    const int key0 = max(seen.x, 0), key_end = min(seen.y, a.s.sk);
    const int ntiles = key_end > key0 ? (key_end - key0 + kTile - 1) / kTile : 0;
    const uint32_t dp_at = tmem + 2 * kTile, dq_at = tmem + 3 * kTile;
    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (ntiles > 0 && warp == 8) {
        // ------------------------------------------------------------ TMA
        const bool issuer = elect_one();
        if (issuer) {
          mbar_arrive_expect_tx(&sh.own_full, 2 * kTileBytes);
          load_rows<kPanels>(base, &qmap, i0, head, b, &sh.own_full);
          load_rows<kPanels>(base + kTileBytes, &gmap, i0, head, b, &sh.own_full);
        }
        __syncwarp();
        RingPos f{0, 0}, s{0, 0};
        for (int t = 0; t < ntiles; ++t) {
          if (!me.wait(&sh.first_empty[f.s], f.phase ^ 1)) break;
          if (issuer) {
            mbar_arrive_expect_tx(&sh.first_full[f.s], kTileBytes);
            load_rows<kPanels>(firsts + f.s * kTileBytes, &kmap, key0 + t * kTile, kv, b, &sh.first_full[f.s]);
          }
          __syncwarp();
          if (!me.wait(&sh.second_empty[s.s], s.phase ^ 1)) break;
          if (issuer) {
            mbar_arrive_expect_tx(&sh.second_full[s.s], kTileBytes);
            load_rows<kPanels>(seconds + s.s * kTileBytes, &vmap, key0 + t * kTile, kv, b, &sh.second_full[s.s]);
          }
          __syncwarp();
          f.step(kFirsts);
          s.step(kSecond);
        }
        me.land();
      } else if (ntiles > 0 && warp == 9) {
        // ------------------------------------------------------------ MMA: scores
        const bool issuer = elect_one();
        const uint32_t at = uniform(tmem);
        const uint32_t q = uniform(desc_dims(smem_u32(base))), k = uniform(desc_dims(smem_u32(firsts)));
        const int last = static_cast<int>(uniform(ntiles)) - 1;
        // Spans that share a key or meet leave none out between them: all of them (the
        // largest first key is not behind the least last), or every row's and the next one's
        // (packed documents, windows: 15 keys a row, 24 heads x 16000 rows 584 and 554 us).
        bool gaps = seen.z > seen.w;
        int4 spans[kTile / 32];
        if (gaps) {
#pragma unroll
          for (int i = 0; i < kTile / 32; ++i)
            spans[i] = i0 + i * 32 + lane < a.s.sq ? span_of(a.s, b, i0 + i * 32 + lane) : make_int4(0, 0, 0, 0);
          bool meet = true;
#pragma unroll
          for (int i = 0; i < kTile / 32; ++i) {
            const int after = min(i + 1, kTile / 32 - 1);  // (the tile's last row has no next)
            const int lo = __shfl_sync(0xffffffffu, lane == 0 ? spans[after].x : spans[i].x, lane + 1);
            const int hi = __shfl_sync(0xffffffffu, lane == 0 ? spans[after].y : spans[i].y, lane + 1);
            const int row = i * 32 + lane + 1;
            if (row < kTile && i0 + row < a.s.sq)
              meet = meet && spans[i].x < spans[i].y && lo < hi && lo <= spans[i].y && spans[i].x <= hi;
          }
          gaps = !__all_sync(0xffffffffu, meet);
        }
        RingPos f{0, 0};
        me.wait(&sh.own_full, 0);
        for (int t = 0; t <= last && me.ok; ++t) {
          if (!me.wait(&sh.first_full[f.s], f.phase)) break;
          if (gaps) clear_unseen<kPanels>(firsts + f.s * kTileBytes, spans, key0 + t * kTile, lane);
          const int left = key_end - (key0 + t * kTile);  // keys past these are nobody's and may hold anything
          if (left < kTile) clear_rows<kPanels>(firsts + f.s * kTileBytes, left, kTile, lane);
          // dq's product two tiles before has read the buffer
          if (t > 1 && !me.wait(&sh.dq_done[t & 1], (t >> 1) - 1)) break;
          if (issuer) {
            product_dims<D>(at + (t & 1) * kTile, q, k + f.s * kTileStep, kDims);
            umma_commit(&sh.s_full[t & 1]);
          }
          __syncwarp();
          f.step(kFirsts);
        }
      } else if (ntiles > 0 && warp == 10) {
        // ------------------------------------------------------------ MMA: g.v and dq
        const bool issuer = elect_one();
        const uint32_t at = uniform(tmem), dp_to = at + 2 * kTile, dq_to = at + 3 * kTile;
        const uint32_t g = uniform(desc_dims(smem_u32(base) + kTileBytes)), v = uniform(desc_dims(smem_u32(seconds)));
        const uint32_t k_rows = uniform(desc_rows(smem_u32(firsts)));
        const int last = static_cast<int>(uniform(ntiles)) - 1;
        RingPos f{0, 0}, s{0, 0};
        auto values = [&]() {
          if (!me.wait(&sh.second_full[s.s], s.phase)) return;
          if (issuer) {
            product_dims<D>(dp_to, g, v + s.s * kTileStep, kDims);
            umma_commit(&sh.dp_full);
            umma_commit(&sh.second_empty[s.s]);
          }
          __syncwarp();
          s.step(kSecond);
        };
        me.wait(&sh.own_full, 0);
        if (me.ok) values();
        for (int t = 0; t <= last && me.ok; ++t) {
          if (t < last && me.wait(&sh.dp_free, t)) values();
          if (!me.wait(&sh.first_full[f.s], f.phase) || !me.wait(&sh.ds_full[t & 1], t >> 1)) break;
          if (issuer) {
            product_rows<kTile>(dq_to, at + (t & 1) * kTile, k_rows + f.s * kTileStep, kRows, t > 0);
            umma_commit(&sh.first_empty[f.s]);
            umma_commit(t == last ? &sh.done : &sh.dq_done[t & 1]);
          }
          __syncwarp();
          f.step(kFirsts);
        }
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      // -------------------------------------------------------------- a query row a thread, 64 of the keys
      const int i = i0 + r;
      const bool real = i < a.s.sq;
      const int4 span = real ? span_of(a.s, b, i) : make_int4(0, 0, 0, 0);
      const float2 stat = a.stats[(static_cast<long long>(b) * a.s.heads + head) * a.padded + i];
      const Cap cap(a.s);
      const float bias = RICH && a.s.slopes ? a.s.slopes[head] * kLog2E : 0.0f;
      const bool one = span.y - span.x == 1, ones = __any_sync(0xffffffffu, one);
      const float2 neg2 = make_float2(-stat.x, -stat.x), scale2 = make_float2(scale_log2, scale_log2);
      const float2 back = make_float2(Held<AB>::kBack, Held<AB>::kBack), delta2 = make_float2(-stat.y, -stat.y);
      for (int t = 0; t < ntiles; ++t) {
        const uint32_t s_own = tmem + (t & 1) * kTile + lanes + half * 64;
        if (!me.wait(&sh.s_full[t & 1], t >> 1)) break;
        const int j0 = key0 + t * kTile + half * 64;
        float p[64], slopes[RICH ? 64 : 1];
        load_half(s_own, p);
        if constexpr (RICH) {
          scaled_scores<WIDE>(a.s, cap, p, slopes);
          if (a.s.slopes) less_distance(bias, static_cast<float>(span.z - j0), p);
        }
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 z = make_float2(p[e], p[e + 1]);
          const float2 x = RICH ? fadd2(z, neg2) : ffma2(z, scale2, neg2);
          p[e] = exp2_approx(x.x);
          p[e + 1] = exp2_approx(x.y);
        }
        const bool masked = !__all_sync(0xffffffffu, !real || (span.x <= j0 && span.y >= j0 + 64));
        const int from = span.x - j0, to = span.y - j0;
        if (masked) {
#pragma unroll
          for (int e = 0; e < 64; ++e) p[e] = e >= from && e < to ? p[e] : 0.0f;
        }
        if constexpr (RICH) {
          if (a.s.cap > 0.0f) {
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const float2 x = fmul2(make_float2(p[e], p[e + 1]), make_float2(slopes[e], slopes[e + 1]));
              p[e] = x.x;
              p[e + 1] = x.y;
            }
          }
        }
        if (!me.wait(&sh.dp_full, t)) break;
        float ds[64];
        load_half(dp_at + lanes + half * 64, ds);
        me.arrive(&sh.dp_free);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 x = fmul2(make_float2(p[e], p[e + 1]), ffma2(make_float2(ds[e], ds[e + 1]), back, delta2));
          ds[e] = x.x;
          ds[e + 1] = x.y;
        }
        if (masked) {  // a masked pair's g.v may be anything
#pragma unroll
          for (int e = 0; e < 64; ++e) ds[e] = e >= from && e < to ? ds[e] : 0.0f;
          if (ones) {  // (rows of one key are never whole)
            const float2 keep = one ? make_float2(0.0f, 0.0f) : make_float2(1.0f, 1.0f);
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const float2 x = fmul2(make_float2(ds[e], ds[e + 1]), keep);
              ds[e] = x.x;
              ds[e + 1] = x.y;
            }
          }
        }
        store_half<T>(s_own, ds);
        me.arrive(&sh.ds_full[t & 1]);  // two barriers: a fast warp may be through the next step before a slow one is here
      }
      if (ntiles > 0) me.wait(&sh.done, 0);
      if (me.ok && half == 0) {
        // (a row that sees nothing: its g may hold anything)
        T* out = real ? static_cast<T*>(a.dq) + b * a.q_batch + head * a.q_head + static_cast<long long>(i) * a.q_row : nullptr;
        store_row<T, D>(out, dq_at + lanes, a.s.scale, a.s.d, ntiles > 0, stage);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dv and dk from their parts, added in order; 8 dims a thread
template <int AB>
__global__ void __launch_bounds__(256) join_grad_kernel(const __grid_constant__ GradArgs a) {
  using T = Element<AB>;
  wait_for_prior();
  let_next_start();
  const int eights = a.s.d >> 3;
  const long long rows = static_cast<long long>(a.s.batch) * a.s.kv_heads * a.s.sk;
  const long long n = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, row = n / eights;
  const bool of_k = blockIdx.y == 1;
  if (row >= rows || !(of_k ? a.dk : a.dv)) return;
  const float4* from = reinterpret_cast<const float4*>(a.part + of_k * a.parts * rows * a.s.d) + 2 * n;
  const long long step = rows * a.s.d >> 2;
  float4 x = from[0], y = from[1];
#pragma unroll 4
  for (int p = 1; p < a.parts; ++p) {
    const float4 u = from[p * step], v = from[p * step + 1];
    x = make_float4(x.x + u.x, x.y + u.y, x.z + u.z, x.w + u.w);
    y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
  }
  const long long heads = row / a.s.sk, b = heads / a.s.kv_heads, h = heads % a.s.kv_heads, j = row % a.s.sk;
  T* out = (of_k ? static_cast<T*>(a.dk) + b * a.k_batch + h * a.k_head + j * a.k_row
                 : static_cast<T*>(a.dv) + b * a.v_batch + h * a.v_head + j * a.v_row) + n % eights * 8;
  *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w), pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
}

// ---- host ---------------------------------------------------------------------------------
long long padded_rows(int sq) { return round_up(sq, kTile); }

// CTAs that share a tile of keys, each some of the query heads on them.  Their sums
// pass through memory (about 15 us for 148 tiles of 128 dims), so only where a CTA a
// tile would leave SMs idle.  Measured (us, one CTA a tile and several): 24 heads on
// one, 2048 rows 712 and 184; 8 on 2, 2000 rows, 64 dims 114 and 60; 12 on 2, 256
// rows 30 and 18.  Up to 148 tiles under spans (in causal order the first tile's CTA is
// the last to end): 24 on 4, 4096 rows 455 and 351, but 8 on 4, 4 x 1024 rows 56 and 72;
// without spans 564 and 581.
int key_parts(int batch, int heads, int kv_heads, int sq, int sk, bool spans) {
  const long long units = static_cast<long long>(batch) * kv_heads * ((sk + kTile - 1) / kTile), group = heads / kv_heads;
  const long long steps = group * (padded_rows(sq) / kTile);  // of a CTA, at most
  if (units == 0 || steps < (2 * units <= kNumSMs ? 6 : spans ? 64 : steps + 1)) return 1;
  const long long parts = (kNumSMs + units - 1) / units;
  return static_cast<int>(parts < group ? parts : group);
}

long long stats_bytes(int batch, int heads, int sq) { return 8LL * batch * heads * padded_rows(sq); }

template <int AB, int D>
int launch_grad(const GradArgs& a, const CUtensorMap (&maps)[4], cudaStream_t stream) {
  const int form = score_form(a.s);
  auto kernel = form == 2 ? span_attention_grad_kernel<AB, D, true, true>
                : form == 1 ? span_attention_grad_kernel<AB, D, true, false> : span_attention_grad_kernel<AB, D, false, false>;
  const int smem = form ? grad_smem<D, true>() : grad_smem<D, false>();
  static std::atomic<unsigned long long> granted[3] = {};
  if (cudaError_t e = grant_smem(reinterpret_cast<const void*>(kernel), smem, granted[form])) return static_cast<int>(e);
  if (a.s.sq > 0) {
    const long long rows = static_cast<long long>(a.s.batch) * a.s.heads * a.padded;
    auto stats = a.s.spans || a.s.sk <= kFewKeys ? grad_stats_kernel<AB, true> : grad_stats_kernel<AB, false>;
    if (int st = launch_overlapped(stats, dim3(static_cast<unsigned>(rows / 16)), dim3(256), 0, 0, stream, a)) return st;
  }
  if (int st = launch_overlapped(kernel, dim3(a.key_units + a.query_units), dim3(kGradThreads), smem, 0, stream, maps[0],
                                 maps[1], maps[2], maps[3], a))
    return st;
  if (a.key_units == 0 || a.parts == 1) return kOk;
  const long long eights = static_cast<long long>(a.s.batch) * a.s.kv_heads * a.s.sk * (a.s.d / 8);
  return launch_overlapped(join_grad_kernel<AB>, dim3(static_cast<unsigned>((eights + 255) / 256), 2), dim3(256), 0, 0, stream, a);
}

}  // namespace
}  // namespace peco

using namespace peco;

extern "C" long long peco_span_attention_backward_workspace(int batch, int heads, int kv_heads, int sq, int sk, int d, int spans) {
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || sq < 0 || sk < 0 || sq > 0x7ffffe00 || sk > 0x7ffffe00 ||
      d < 8 || d > 128 || d % 8)
    return -1;
  const long long parts = key_parts(batch, heads, kv_heads, sq, sk, spans != 0);
  return stats_bytes(batch, heads, sq) + (parts > 1 ? 8 * parts * batch * kv_heads * sk * d : 0);
}

extern "C" int peco_span_attention_backward(const void* grad, const void* q, const void* k, const void* v, const void* out,
                                            const float* lse, const long long* strides, const int* span_rows,
                                            const int* span_tiles, int spans_batched, const float* slopes, float scale,
                                            float cap, void* dq, void* dk, void* dv, int batch, int heads, int kv_heads,
                                            int sq, int sk, int d, int dtype, void* workspace, long long workspace_bytes,
                                            void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || sq < 0 || sk < 0 || sq > 0x7ffffe00 || sk > 0x7ffffe00 ||
      d < 8 || d > 128 || d % 8 || !valid_scores(scale, cap) || !strides)
    return kErrInvalidValue;
  const bool keys = (dk || dv) && batch > 0 && sk > 0, rows = dq && batch > 0 && sq > 0;
  if (!keys && !rows) return kOk;
  if (!valid_plan(span_rows, span_tiles)) return kErrInvalidValue;
  HeadRows t[8];  // grad, q, k, v, out, dq, dk, dv
  const void* at[8] = {grad, q, k, v, out, dq, dk, dv};
  for (int i = 0; i < 8; ++i) {
    const bool of_keys = i == 2 || i == 3 || i == 6 || i == 7;
    t[i] = HeadRows{at[i], strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
    const int n = of_keys ? sk : sq;
    if (n == 0 || (i > 4 && !at[i])) continue;
    if (!readable(t[i], batch, of_keys ? kv_heads : heads, n)) return kErrInvalidValue;
  }
  if (sq > 0 && !lse) return kErrInvalidValue;
  if (sq > 0 && !usable_workspace(workspace, workspace_bytes, peco_span_attention_backward_workspace(batch, heads, kv_heads, sq, sk, d, span_rows ? 1 : 0)))
    return kErrWorkspace;
  GradArgs a{};
  a.s.spans = reinterpret_cast<const int4*>(span_rows);
  a.s.span_tiles = reinterpret_cast<const int4*>(span_tiles);
  a.s.spans_batched = spans_batched;
  a.s.slopes = slopes;
  a.s.batch = batch;
  a.s.heads = heads;
  a.s.kv_heads = kv_heads;
  a.s.sq = sq;
  a.s.sk = sk;
  a.s.d = d;
  a.s.scale = scale;
  a.s.cap = cap;
  a.s.status = device_status_ptr();
  a.grad = t[0];
  a.q = t[1];
  a.k = t[2];
  a.v = t[3];
  a.out = t[4];
  a.lse = lse;
  a.stats = static_cast<float2*>(workspace);
  a.padded = static_cast<int>(padded_rows(sq));
  a.parts = key_parts(batch, heads, kv_heads, sq, sk, span_rows != nullptr);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(batch, heads, sq));
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.q_batch = t[5].batch;
  a.q_head = t[5].head;
  a.q_row = t[5].row;
  a.k_batch = t[6].batch;
  a.k_head = t[6].head;
  a.k_row = t[6].row;
  a.v_batch = t[7].batch;
  a.v_head = t[7].head;
  a.v_row = t[7].row;
  const long long key_units = keys ? static_cast<long long>(batch) * kv_heads * ((sk + kTile - 1) / kTile) * a.parts : 0;
  const long long query_units = rows ? static_cast<long long>(batch) * heads * (a.padded / kTile) : 0;
  const long long stat_blocks = static_cast<long long>(batch) * heads * a.padded / 16;
  if (key_units + query_units > 0x7fffffffLL || stat_blocks > 0x7fffffffLL) return kErrUnsupported;
  if (query_units > 0) a.turns = turns(a.s, a.padded / kTile, heads);
  if (key_units > 0) a.blocks = divisor((sk + kTile - 1) / kTile);
  a.by_parts = divisor(a.parts);
  a.kv = divisor(kv_heads);
  a.s.group = divisor(heads / kv_heads);
  a.key_units = static_cast<int>(key_units);
  a.query_units = static_cast<int>(query_units);
  // an empty side is never loaded: its maps stand on the other's rows
  CUtensorMap maps[4];
  const int order[4] = {1, 2, 3, 0};
  for (int i = 0; i < 4; ++i) {
    const bool of_keys = i == 1 || i == 2;
    const bool empty = of_keys ? sk == 0 : sq == 0;
    const HeadRows& from = !empty ? t[order[i]] : sk == 0 ? t[1] : t[2];
    const bool as_keys = empty ? sk != 0 : of_keys;
    // whole tiles: rows past the end read as zeros, as the products over rows need them
    if (!head_map(&maps[i], from, batch, as_keys ? kv_heads : heads, as_keys ? sk : sq, d, kTile, 1, dtype)) return kErrTensorMap;
  }
  if (d <= 64) return dtype == 1 ? launch_grad<1, 64>(a, maps, stream) : launch_grad<0, 64>(a, maps, stream);
  return dtype == 1 ? launch_grad<1, 128>(a, maps, stream) : launch_grad<0, 128>(a, maps, stream);
}
