// Attention over key spans on sm_100a tensor cores (see span_attention.cuh for the
// mathematics): softmax(z) v with its logarithmic sums, for any lengths, shared
// key heads, capped scores and a bias by distance.
//
//  * key_spans_kernel writes every query row's span of keys (documents of a packed
//    sequence, a causal order with a prefix, a window, lengths) and, for every 128
//    rows, the bounds that decide which key tiles are walked and which need masks;
//  * span_attention_kernel walks them; split_attention_kernel joins the parts of
//    calls with few rows, whose keys are split over CTAs.
//
// A CTA takes a tile of 128 query rows of one head (or rows of several heads that
// share their keys, side by side); two warpgroups take its even and its odd key
// tiles.  Per tile of 128 keys:
//   S = Q K^T        tcgen05.mma, both in shared memory, into one of three buffers in TMEM
//   P = 2^(z - m)    a query row a thread; m, the row's running maximum, goes from
//                    tile to tile through shared memory and is raised only when it
//                    grows by more than 2^8, O rescaled then
//   O += P V         tcgen05.mma, P from TMEM (over S, as 16-bit pairs)
// Scores run two tiles ahead of the softmax, issued by a warp of their own; a
// second one issues the products with V.  K and V stream through three
// shared-memory slots each by TMA.  Whatever is written over is waited for.
//
// What it measured (B200, bf16): 24 heads x 7006 rows x 128 dims, every key: 490 us
// (1.18 PFLOP/s; 535 us at the power limit after 300 calls in a row), 64 dims 423 us;
// causal, 24 query heads on 4, 4096 rows 116 us; one row of 24 heads on 4, four samples of
// up to 16384 keys 32 us.  Tensor core and special-function unit are both 62% busy:
// the two warps of a scheduler do not hide all of each other's maxima, TMEM loads
// and hand-offs, and the 128 scores of a thread leave some registers in local memory
// (16 loads and 7 stores a warp and tile, 3% of its instructions).  Capped 1010 us, under
// a cap above 64 1150 us, by distance 830 us.  Before, with a maximum, sum and accumulator for each warpgroup
// 563 us, and with one warp that issued all products 536 us; two tiles of rows a
// CTA in place of two of keys, which halves the traffic from L2, took as long on full
// masks and more on others (clips packed in causal order 102 us against 89).
#include "span_attention.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"

namespace peco {
namespace {

// ---- spans ------------------------------------------------------------------------------
struct SpanArgs {
  const int* q_ends;        // [batch or 1, documents + 1] first rows of the documents, then the end (null: one document)
  const int* k_ends;
  long long q_stride, k_stride;
  int documents;
  const int* lengths;       // [batch] keys of each sample (without documents; null: all)
  const int* prefix;        // [batch or 1, documents or 1] (null: prefix_all)
  long long prefix_batch;   // elements between samples and between documents
  int prefix_doc, prefix_all;
  int causal, window;       // window 0: none
  int batch, queries, keys;
  int4* rows;
  int4* tiles;
};

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return min(max(v, lo), hi); }

// (first key, key behind the last, position) of a row
__device__ int3 row_span(const SpanArgs& a, int b, int i) {
  int lo = 0, hi = 0, pos = 0;
  int q0 = 0, q1 = a.queries, k0 = 0, k1 = a.keys, doc = 0;
  bool inside = true;
  if (a.documents > 0) {
    const int* qe = a.q_ends + b * a.q_stride;
    const int* ke = a.k_ends + b * a.k_stride;
    int l = -1, h = a.documents + 1;  // the last entry not behind the row
    while (h - l > 1) {
      const int mid = (l + h) >> 1;
      if (qe[mid] <= i) l = mid;
      else h = mid;
    }
    inside = l >= 0 && l < a.documents;
    doc = clamped(l, 0, a.documents - 1);
    q0 = clamped(qe[doc], 0, a.queries);
    q1 = clamped(qe[doc + 1], q0, a.queries);
    k0 = clamped(ke[doc], 0, a.keys);
    k1 = clamped(ke[doc + 1], k0, a.keys);
    inside = inside && i >= q0 && i < q1;
  } else if (a.lengths) {
    k1 = clamped(a.lengths[b], 0, a.keys);
  }
  pos = k0 + (i - q0) + (k1 - k0) - (q1 - q0);
  lo = k0;
  hi = inside ? k1 : k0;
  if (a.causal) {
    const int prefix = a.prefix ? a.prefix[b * a.prefix_batch + doc * a.prefix_doc] : a.prefix_all;
    hi = min(hi, max(pos + 1, k0 + clamped(prefix, 0, a.keys - k0)));
  }
  if (a.window > 0) {
    lo = max(lo, static_cast<int>(max(static_cast<long long>(pos) - a.window + 1, 0LL)));
    hi = static_cast<int>(min(static_cast<long long>(hi), static_cast<long long>(pos) + a.window));
  }
  if (hi <= lo) lo = hi = 0;
  return make_int3(lo, hi, pos);
}

// A block per 128 rows of a sample, a row per thread.  Each also ranks its tile by
// the keys that its first and last row see, for the attention's CTAs to take the
// longest tiles first (among more than kRanked tiles: the later ones).
constexpr int kRanked = 1024;
__global__ void __launch_bounds__(kTile) key_spans_kernel(const SpanArgs a) {
  __shared__ int4 part[4];
  __shared__ int sizes[kRanked];
  __shared__ int ahead;
  wait_for_prior();
  let_next_start();
  const int b = blockIdx.y, i = blockIdx.x * kTile + threadIdx.x, tiles = gridDim.x, mine = blockIdx.x;
  if (threadIdx.x == 0) ahead = 0;
  int lo = 0, hi = 0;
  if (i < a.queries) {
    const int3 s = row_span(a, b, i);
    lo = s.x;
    hi = s.y;
    int* row = reinterpret_cast<int*>(a.rows + static_cast<long long>(b) * a.queries + i);
    *reinterpret_cast<int2*>(row) = make_int2(lo, hi);
    row[2] = s.z;
    if (i >= tiles) row[3] = 0;  // (the others' by rank below)
  }
  if (tiles <= kRanked) {
    for (int t = threadIdx.x; t < tiles; t += kTile) {
      const int3 u = row_span(a, b, t * kTile), v = row_span(a, b, min(t * kTile + kTile, a.queries) - 1);
      const int from = min(u.y > u.x ? u.x : 0x7fffffff, v.y > v.x ? v.x : 0x7fffffff), to = max(u.y, v.y);
      sizes[t] = to > from ? (to - from + kTile - 1) / kTile : 0;
    }
    __syncthreads();
    int count = 0;
    for (int t = threadIdx.x; t < tiles; t += kTile) count += sizes[t] > sizes[mine] || (sizes[t] == sizes[mine] && t > mine);
    count = __reduce_add_sync(0xffffffffu, count);
    if ((threadIdx.x & 31) == 0) atomicAdd(&ahead, count);
  } else if (threadIdx.x == 0) {
    ahead = tiles - 1 - mine;
  }
  // rows that see nothing count for the masks only; rows past the end not at all
  const bool real = i < a.queries, sees = hi > lo;
  int4 t = make_int4(sees ? lo : 0x7fffffff, sees ? hi : 0, !real ? 0 : sees ? lo : 0x7fffffff, !real ? 0x7fffffff : hi);
  t.x = __reduce_min_sync(0xffffffffu, t.x);
  t.y = __reduce_max_sync(0xffffffffu, t.y);
  t.z = __reduce_max_sync(0xffffffffu, t.z);
  t.w = __reduce_min_sync(0xffffffffu, t.w);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) {
      t.x = min(t.x, part[w].x);
      t.y = max(t.y, part[w].y);
      t.z = max(t.z, part[w].z);
      t.w = min(t.w, part[w].w);
    }
    a.tiles[static_cast<long long>(b) * tiles + mine] = t;
    a.rows[static_cast<long long>(b) * a.queries + ahead].w = mine;
  }
}

// ---- forward ----------------------------------------------------------------------------
constexpr int kSlots = 3;        // tiles of K, and as many of V
constexpr int kScores = 3;       // S buffers
constexpr int kThreads = 384;    // two softmax warpgroups, one with the TMA warp and the two MMA warps
// A softmax thread holds a tile's 128 scores: the launch's 168 registers a thread
// go 208 to 208 to 88 (256 * 208 + 128 * 88 = 384 * 168).
constexpr uint32_t kTmemCols = 512;  // three tiles' S, then O

struct ForwardArgs {
  ScoreArgs s;
  HeadRows q, k, v;         // for rows whose result is not finite
  void* out;
  long long out_batch, out_head, out_row;
  float* lse;               // [batch, heads, sq]
  int packed;               // heads side by side in a tile (1: consecutive rows of one head)
  Turns turns;              // of heads (packed ones as one) and their tiles
  Divisor splits;           // CTAs along the keys
  Divisor rows;             // query rows
  float* part;              // [unit][split][128][d] unnormalised, then (max, sum) of each row
  float2* part_sums;
};

struct __align__(8) ForwardShared {
  uint64_t q_full, k_full[kSlots], k_empty[kSlots], v_full[kSlots], v_empty[kSlots], s_full[kScores], p_full[kScores], o_done[kScores], o_full, reference[2][4];
  uint32_t tmem;
  int abort_flag, masked;
  float top[kTile];         // the maximum that O's rows stand on
};

template <int D>
constexpr int forward_smem() { return 1024 + (1 + 2 * kSlots) * kTile * D * 2 + 1024; }
static_assert(sizeof(ForwardShared) <= 1024 && forward_smem<128>() <= 227 * 1024, "shared memory of a CTA");

// Which head and query row thread ``r`` of a unit holds.
struct Unit {
  int b, head0, row0;       // first head, first row
  __device__ Unit(const ForwardArgs& a, int unit) {
    int rank;
    a.turns.at(unit, b, head0, rank);
    head0 *= a.packed;
    row0 = ranked_tile(a.s, b, rank, a.turns.tiles) * kTile;
  }
  __device__ __forceinline__ bool row(const ForwardArgs& a, int r, int& head, int& i) const {
    if (a.packed > 1) {
      const int n = a.rows(r);
      head = head0 + n;
      i = r - n * a.s.sq;
      return r < a.packed * a.s.sq;
    }
    head = head0;
    i = row0 + r;
    return i < a.s.sq;
  }
  // keys that a row of the unit sees: [lo, hi)
  __device__ __forceinline__ int2 keys(const ForwardArgs& a) const {
    const int4 t = tile_span(a.s, b, row0 / kTile);
    const int lo = max(t.x, 0), hi = min(t.y, a.s.sk);
    return make_int2(min(lo, hi), hi);
  }
};

// Key tiles of one split: first key, tiles
__device__ __forceinline__ int2 split_keys(int2 keys, int split, const Divisor& splits) {
  const int all = (keys.y - keys.x + kTile - 1) / kTile;
  const int per = splits(all + splits.by - 1);
  const int first = min(all, split * per);
  return make_int2(keys.x + first * kTile, min(all, first + per) - first);
}

// One row's result again, by a warp, without the tensor core: a masked key's
// probability is 0, but 0 times an infinite or NaN value of a key that other rows
// of the tile do see is NaN.  Here masked keys are left out.  Rare (only rows
// whose result is not finite, where masks were at work), so it is not fast.
template <int AB, int D>
__device__ __noinline__ void masked_row(const ForwardArgs& a, int b, int head, int i, int lo, int hi, int pos, int from,
                                        int to, float m, float (&acc)[D / 32]) {
  using T = Element<AB>;
  const int lane = lane_id(), kv = a.s.group(head), d = a.s.d;
  const T* q = static_cast<const T*>(a.q.ptr) + b * a.q.batch + head * a.q.head + static_cast<long long>(i) * a.q.row;
  const T* k = static_cast<const T*>(a.k.ptr) + b * a.k.batch + kv * a.k.head;
  const T* v = static_cast<const T*>(a.v.ptr) + b * a.v.batch + kv * a.v.head;
  const float slope = a.s.slopes ? a.s.slopes[head] * kLog2E : 0.0f;
  const Cap cap(a.s);
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.0f;
  lo = max(lo, from);
  hi = min(hi, min(to, a.s.sk));  // (``to`` is a whole tile's end)
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int j = j0 + lane;
    float p = 0.0f;
    if (j < hi) {
      float raw = 0.0f;
      for (int e = 0; e < d; ++e) raw = fmaf(to_f32<T>(q[e]), to_f32<T>(k[j * a.k.row + e]), raw);
      float z = a.s.cap > 0.0f ? cap.value(raw, cap.recip(raw)) : raw * a.s.scale * kLog2E;
      if (a.s.slopes) z = fmaf(-slope, fabsf(static_cast<float>(pos - j)), z);
      p = exp2_approx(z - m);
    }
    const int count = min(32, hi - j0);
    for (int n = 0; n < count; ++n) {
      const float w = __shfl_sync(0xffffffffu, p, n);
#pragma unroll
      for (int e = 0; e < D / 32; ++e)
        if (lane + 32 * e < d) acc[e] = fmaf(w, to_f32<T>(v[static_cast<long long>(j0 + n) * a.v.row + lane + 32 * e]), acc[e]);
    }
  }
}

// RICH: capped scores or a bias by distance; WIDE: a cap above kWideCap
template <int AB, int D, bool RICH, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1)
    span_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const __grid_constant__ ForwardArgs a) {
  using T = Element<AB>;
  constexpr int kPanels = D / 64, kTileBytes = kPanels * kPanelBytes;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* k_slots = base + kTileBytes;
  unsigned char* v_slots = k_slots + kSlots * kTileBytes;
  ForwardShared& sh = *reinterpret_cast<ForwardShared*>(v_slots + kSlots * kTileBytes);
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < kScores; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_done[i], 1);
    }
    mbar_init(&sh.o_full, 1);
    for (int w = 0; w < 2; ++w) {
      for (int i = 0; i < 4; ++i) mbar_init(&sh.reference[w][i], 1);
    }
    sh.abort_flag = 0;
    sh.masked = 0;
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_prior();
  let_next_start();
  const uint32_t tmem = sh.tmem;
  const int at = a.splits(blockIdx.x), split = static_cast<int>(blockIdx.x) - at * a.splits.by;
  const Unit unit(a, at);
  const int2 all_keys = unit.keys(a);
  const int2 mine = split_keys(all_keys, split, a.splits);
  const int key0 = mine.x, ntiles = mine.y;

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 8) {
    // ---------------------------------------------------------------- TMA
    const bool issuer = elect_one();
    const int kv = a.s.group(unit.head0);
    bool ok = true;
    if (ntiles > 0 && issuer) {
      mbar_arrive_expect_tx(&sh.q_full, static_cast<uint32_t>(a.packed * min(a.s.sq, kTile)) * 128u * kPanels);
      load_rows<kPanels>(base, &qmap, unit.row0, unit.head0, unit.b, &sh.q_full);
    }
    __syncwarp();
    auto load = [&](const CUtensorMap* map, unsigned char* slots, uint64_t* full, uint64_t* empty, RingPos& pos, int t) {
      if (ok) ok = warp_wait(&empty[pos.s], pos.phase ^ 1, abort_flag, a.s.status);
      if (ok && issuer) {
        mbar_arrive_expect_tx(&full[pos.s], kTileBytes);
        load_rows<kPanels>(slots + pos.s * kTileBytes, map, key0 + t * kTile, kv, unit.b, &full[pos.s]);
      }
      __syncwarp();
      pos.step(kSlots);
    };
    RingPos ks{0, 0}, vs{0, 0};
    for (int t = 0; t < 2 && t < ntiles; ++t) load(&kmap, k_slots, sh.k_full, sh.k_empty, ks, t);
    for (int t = 0; t < ntiles && ok; ++t) {
      if (t + 2 < ntiles) load(&kmap, k_slots, sh.k_full, sh.k_empty, ks, t + 2);
      load(&vmap, v_slots, sh.v_full, sh.v_empty, vs, t);
    }
    if (!ok) {  // time for the copies in flight to land before the CTA ends
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 9 || warp == 10) {
    // ---------------------------------------------------------------- MMA
    // One warp issues the scores, the other the products with V, so that neither's waits hold the other up.
    constexpr uint32_t idesc_qk = instr_desc(kTile, kTile, AB, false, false);
    constexpr uint32_t idesc_pv = instr_desc(kTile, D, AB, false, true);
    constexpr uint32_t kSlotStep = kTileBytes >> 4;
    const bool issuer = elect_one();
    const uint32_t s_at = uniform(tmem), o_at = s_at + kScores * kTile;
    const int last = static_cast<int>(uniform(ntiles)) - 1;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      if (ok) ok = warp_wait(bar, phase, abort_flag, a.s.status);
      if (ok) tc_fence_after();
      return ok;
    };
    RingPos slot{0, 0}, buffer{0, 0};
    if (warp == 9) {
      const uint32_t q = uniform(desc_dims(smem_u32(base))), k = uniform(desc_dims(smem_u32(k_slots)));
      if (last >= 0) wait(&sh.q_full, 0);
      for (int t = 0; t <= last && ok; ++t) {
        if (!wait(&sh.k_full[slot.s], slot.phase)) break;
        // the buffer's last P has been read
        if (t >= kScores && !wait(&sh.o_done[buffer.s], buffer.phase ^ 1)) break;
        if (issuer) {
          product_dims<D>(s_at + buffer.s * kTile, q, k + slot.s * kSlotStep, idesc_qk);
          umma_commit(&sh.s_full[buffer.s]);
          umma_commit(&sh.k_empty[slot.s]);
        }
        __syncwarp();
        slot.step(kSlots);
        buffer.step(kScores);
      }
    } else {
      const uint32_t v = uniform(desc_rows(smem_u32(v_slots)));
      for (int t = 0; t <= last && ok; ++t) {
        if (!wait(&sh.v_full[slot.s], slot.phase)) break;
        const int seen = all_keys.y - (key0 + t * kTile);  // keys past a unit's last are nobody's: their values may be anything
        if (seen < kTile) clear_rows<kPanels>(v_slots + slot.s * kTileBytes, seen, kTile, lane);
        if (!wait(&sh.p_full[buffer.s], buffer.phase)) break;
        if (issuer) {
          product_rows<kTile>(o_at, s_at + buffer.s * kTile, v + slot.s * kSlotStep, idesc_pv, t > 0);
          umma_commit(&sh.o_done[buffer.s]);
          umma_commit(&sh.v_empty[slot.s]);
          if (t == last) umma_commit(&sh.o_full);
        }
        __syncwarp();
        slot.step(kSlots);
        buffer.step(kScores);
      }
    }
  }
  } else {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------- softmax, epilogue
    const int w = warp >> 2, r = threadIdx.x & (kTile - 1);
    const int quarter = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t o_at = tmem + kScores * kTile + lanes;
    int head, i;
    const bool real = unit.row(a, r, head, i);
    const int4 span = real ? span_of(a.s, unit.b, i) : make_int4(0, 0, 0, 0);
    const int lo = span.x, hi = span.y;
    const float scale_log2 = a.s.scale * kLog2E;
    const Cap cap(a.s);
    const float slope = RICH && a.s.slopes && real ? a.s.slopes[head] * kLog2E : 0.0f;
    float m = -INFINITY, l = 0.0f;
    bool ok = true, masked = false;
    int buffer = w, phase = 0;  // of the tile's S
    for (int t = w; t < ntiles; t += 2) {
      ok = warp_wait(&sh.s_full[buffer], phase, abort_flag, a.s.status);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_at = tmem + buffer * kTile + lanes;
      const int j0 = key0 + t * kTile;
      float s[kTile];
      {
        uint32_t raw[kTile];
        tmem_ld128_sync(s_at, raw);
#pragma unroll
        for (int e = 0; e < kTile; ++e) s[e] = __uint_as_float(raw[e]);
      }
      if constexpr (RICH) {  // to log2 units
        scaled_scores<WIDE>(a.s, cap, s, nullptr);
        if (a.s.slopes) less_distance(slope, static_cast<float>(span.z - j0), s);
      }
      // rows past the tensor's end are not looked at
      if (!__all_sync(0xffffffffu, !real || (lo <= j0 && hi >= j0 + kTile))) {
        masked = true;
        const int from = lo - j0, to = hi - j0;
#pragma unroll
        for (int e = 0; e < kTile; ++e) s[e] = e >= from && e < to ? s[e] : -INFINITY;
      }
      float mx[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) mx[e] = fmaxf(s[e], s[e + 8]);
#pragma unroll
      for (int e = 16; e < kTile; e += 16)
#pragma unroll
        for (int c = 0; c < 8; ++c) mx[c] = fmaxf(mx[c], fmaxf(s[e + c], s[e + 8 + c]));
#pragma unroll
      for (int c = 4; c > 0; c >>= 1)
#pragma unroll
        for (int e = 0; e < c; ++e) mx[e] = fmaxf(mx[e], mx[e + c]);
      const float top = RICH ? mx[0] : mx[0] * scale_log2;
      // what O stands on so far: the maximum that the tile before left
      float before = -INFINITY;
      if (t > 0) {
        ok = warp_wait(&sh.reference[w ^ 1][quarter], ((t - 1) >> 1) & 1, abort_flag, a.s.status);
        if (!ok) break;
        before = sh.top[r];
      }
      const bool grow = top > before + 8.0f || (before == -INFINITY && top > -INFINITY);
      const float now = grow ? top : before;
      if (__any_sync(0xffffffffu, grow)) {
        const bool rescale = grow && before != -INFINITY;
        if (t > 0 && __any_sync(0xffffffffu, rescale)) {  // with the tile before in it
          // (the phase before is over: S came after it)
          ok = warp_wait(&sh.o_done[(t - 1) % kScores], (t - 1) / kScores & 1, abort_flag, a.s.status);
          if (!ok) break;
          tc_fence_after();
          const float f = rescale ? exp2_approx(before - top) : 1.0f;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t raw[32], part[16];
            tmem_ld32_sync(o_at + c * 32, raw);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int e = 0; e < 16; ++e) part[e] = __float_as_uint(__uint_as_float(raw[h * 16 + e]) * f);
              tmem_st16(o_at + c * 32 + h * 16, part);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
      }
      if (grow || t == 0) sh.top[r] = now;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.reference[w][quarter]);
      if (now != m) l *= m == -INFINITY ? 0.0f : exp2_approx(m - now);
      m = now;
      const float neg = m == -INFINITY ? 0.0f : -m;
      const float2 neg2 = make_float2(neg, neg), scale2 = make_float2(scale_log2, scale_log2);
      float2 sums[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[e] = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < kTile / 32; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 z = make_float2(s[c * 32 + e], s[c * 32 + e + 1]);
          const float2 x = RICH ? fadd2(z, neg2) : ffma2(z, scale2, neg2);
          const float2 p = make_float2(exp2_approx(x.x), exp2_approx(x.y));
          sums[(e >> 1) & 3] = fadd2(sums[(e >> 1) & 3], p);
          packed[e >> 1] = pack2<T>(p.x, p.y);
        }
        tmem_st16(s_at + (c >> 1) * 64 + (c & 1) * 16, packed);
      }
      const float2 sum = fadd2(fadd2(sums[0], sums[1]), fadd2(sums[2], sums[3]));
      l += sum.x + sum.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[buffer]);
      buffer += 2;
      if (buffer >= kScores) {
        buffer -= kScores;
        phase ^= 1;
      }
    }
    if (ok && ntiles > 0) {
      ok = warp_wait(&sh.o_full, 0, abort_flag, a.s.status);
      tc_fence_after();
    }
    float2* sums = reinterpret_cast<float2*>(base);  // (maximum, sum) of each warpgroup, where Q was
    sums[w * kTile + r] = make_float2(m, l);
    if (masked && lane == 0) sh.masked = 1;
    asm volatile("bar.sync 1, 256;" ::: "memory");  // (after an expired wait too)
    if (ok && !*abort_flag) {
      const float2 other = sums[(w ^ 1) * kTile + r];
      const float last = ntiles > 0 ? sh.top[r] : -INFINITY;  // what O stands on
      masked = sh.masked;
      // the two in a fixed order
      const float own = m == -INFINITY ? l : l * exp2_approx(m - last);  // without a maximum: 0, or NaN of NaN scores
      const float its = other.x == -INFINITY ? other.y : other.y * exp2_approx(other.x - last);
      l = w == 0 ? own + its : its + own;
      m = last;
      const bool whole = a.splits.by == 1;
      const float inv = !whole ? 1.0f : l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (a NaN stays)
      // each warpgroup stores half of the columns
      constexpr int kHalf = D / 2;
      T* out = nullptr;
      float* part = nullptr;
      if (real && whole) {
        out = static_cast<T*>(a.out) + unit.b * a.out_batch + head * a.out_head + static_cast<long long>(i) * a.out_row;
        if (w == 0)
          a.lse[(static_cast<long long>(unit.b) * a.s.heads + head) * a.s.sq + i] =
              l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
      } else if (real) {
        const long long at = static_cast<long long>(blockIdx.x) * kTile + r;
        part = a.part + at * a.s.d;
        if (w == 0) a.part_sums[at] = make_float2(m, l);
      }
      // (in K's first tile, whose products are over)
      const RowsOut<kHalf> rows_out{k_slots + warp * (32 * kHalf * 2), lane};
      bool finite = true;
#pragma unroll
      for (int c = w * kHalf; c < (w + 1) * kHalf; c += 32) {
        uint32_t raw[32];
        if (ntiles > 0) tmem_ld32_sync(o_at + c, raw);
        else
#pragma unroll
          for (int e = 0; e < 32; ++e) raw[e] = 0u;
        float2 v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          // a row without a visible key is 0 whatever its masked values were
          v[e] = l == 0.0f ? make_float2(0.0f, 0.0f)
                           : fmul2(make_float2(__uint_as_float(raw[2 * e]), __uint_as_float(raw[2 * e + 1])), make_float2(inv, inv));
          finite = finite && fabsf(v[e].x) < INFINITY && fabsf(v[e].y) < INFINITY;
        }
        if (whole) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            rows_out.put((c - w * kHalf) / 8 + g,
                         make_uint4(pack2<T>(v[4 * g].x, v[4 * g].y), pack2<T>(v[4 * g + 1].x, v[4 * g + 1].y),
                                    pack2<T>(v[4 * g + 2].x, v[4 * g + 2].y), pack2<T>(v[4 * g + 3].x, v[4 * g + 3].y)));
        } else if (part) {
#pragma unroll
          for (int g = 0; g < 8; ++g)
            if (c + g * 4 < a.s.d)
              *reinterpret_cast<float4*>(part + c + g * 4) = make_float4(v[2 * g].x, v[2 * g].y, v[2 * g + 1].x, v[2 * g + 1].y);
        }
      }
      if (whole) rows_out.store(out ? out + w * kHalf : nullptr, a.s.d - w * kHalf);
      // (with a NaN or infinite sum the row sees such scores itself)
      uint32_t again = __ballot_sync(0xffffffffu, masked && real && !finite && l > 0.0f && l < INFINITY);
      while (again) {
        __syncwarp();  // the row's first result is written
        const int from = __ffs(again) - 1;
        again &= again - 1;
        auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, from); };
        const int h2 = of(head), i2 = of(i);
        const float f = __shfl_sync(0xffffffffu, inv, from);
        float acc[D / 32];
        masked_row<AB, D>(a, unit.b, h2, i2, of(lo), of(hi), of(span.z), key0, key0 + ntiles * kTile,
                          __shfl_sync(0xffffffffu, m, from), acc);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const int c = lane + 32 * e;
          if (c >= a.s.d || c / kHalf != w) continue;
          if (whole)
            static_cast<T*>(a.out)[unit.b * a.out_batch + h2 * a.out_head + static_cast<long long>(i2) * a.out_row + c] =
                from_f32<T>(acc[e] * f);
          else
            a.part[(static_cast<long long>(blockIdx.x) * kTile + (r - lane) + from) * a.s.d + c] = acc[e] * f;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// A row's parts joined: out = sum_p O_p 2^(m_p - M) / sum_p l_p 2^(m_p - M).  A block
// a row; each of its warps takes every WARPS-th part, all asked for at once, and their
// sums are added in order.  Latency bounds it: 16 warps for more than 16 parts (74 parts of
// 8 rows, launched cold: 4 warps in turn 13.8 us,
// this 6.1 us), else 4.
template <int AB, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) split_attention_kernel(const __grid_constant__ ForwardArgs a) {
  using T = Element<AB>;
  constexpr int kParts = WARPS == 4 ? 16 : kNumSMs, kEach = (kParts + WARPS - 1) / WARPS, kHeld = (kParts + 31) / 32;
  __shared__ float4 sums[WARPS][kTile / 4];
  wait_for_prior();
  let_next_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = a.packed > 1 ? a.packed * a.s.sq : min(a.s.sq, kTile);  // of a unit that can be there
  const int n = static_cast<int>(blockIdx.x) / rows, r = static_cast<int>(blockIdx.x) - n * rows;
  const Unit unit(a, n);
  int head, i;
  if (!unit.row(a, r, head, i)) return;
  const int parts = a.splits.by, c = lane * 4;
  const long long first = static_cast<long long>(n) * parts * kTile + r;
  float2 of[kHeld];  // (maximum, sum) of parts lane, lane + 32, ...
  float4 v[kEach];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int p = lane + 32 * k;
    of[k] = p < parts ? a.part_sums[first + p * static_cast<long long>(kTile)] : make_float2(-INFINITY, 0.0f);
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int p = warp + WARPS * k;
    v[k] = p < parts && c < a.s.d ? *reinterpret_cast<const float4*>(a.part + (first + p * static_cast<long long>(kTile)) * a.s.d + c)
                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) m = fmaxf(m, of[k].x);
  m = warp_max(m);
  float f[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    f[k] = of[k].y == 0.0f ? 0.0f : exp2_approx(of[k].x - m);
    l = fmaf(of[k].y, f[k], l);
  }
  l = warp_sum(l);
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int p = warp + WARPS * k;
    float w = f[0];
#pragma unroll
    for (int h = 1; h < kHeld; ++h) w = p >> 5 == h ? f[h] : w;
    w = __shfl_sync(0xffffffffu, w, p & 31);
    acc = make_float4(fmaf(v[k].x, w, acc.x), fmaf(v[k].y, w, acc.y), fmaf(v[k].z, w, acc.z), fmaf(v[k].w, w, acc.w));
  }
  sums[warp][lane] = acc;
  __syncthreads();
  const int col = threadIdx.x;
  if (col < a.s.d) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) o += reinterpret_cast<const float*>(sums[w])[col];
    static_cast<T*>(a.out)[unit.b * a.out_batch + head * a.out_head + static_cast<long long>(i) * a.out_row + col] = from_f32<T>(o * inv);
  }
  if (col == 0)
    a.lse[(static_cast<long long>(unit.b) * a.s.heads + head) * a.s.sq + i] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ---- host ---------------------------------------------------------------------------------
// How a call is cut.  Rows of heads that share their keys go side by side into one
// tile where they fit: the keys are then read once for all of them.  Calls that
// leave half of the SMs idle split the keys, four tiles at least to a part.
// (Splitting a last round that leaves many SMs idle gained nothing.)
struct ForwardCut {
  int packed, row_blocks, splits;
  long long units;
};

ForwardCut cut_forward(int batch, int heads, int kv_heads, int sq, int sk) {
  ForwardCut c{1, 1, 1, 0};
  const int group = heads / kv_heads;
  for (int n = 2; n <= group && static_cast<long long>(n) * sq <= kTile; ++n)
    if (group % n == 0) c.packed = n;
  c.row_blocks = (sq + kTile - 1) / kTile;
  c.units = static_cast<long long>(batch) * (heads / c.packed) * c.row_blocks;
  if (c.units > 0 && c.units * 2 <= kNumSMs) {
    const long long most = (static_cast<long long>(sk) + 4 * kTile - 1) / (4 * kTile), fill = kNumSMs / c.units;
    c.splits = static_cast<int>(fill < most ? fill : most);
    if (c.splits < 1) c.splits = 1;
  }
  return c;
}

bool valid_attention(int batch, int heads, int kv_heads, int sq, int sk, int d) {
  return batch >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && sq >= 0 && sk >= 0 && d >= 8 && d <= 128 &&
         d % 8 == 0 && sq <= 0x7ffffe00 && sk <= 0x7ffffe00;
}

long long part_rows(const ForwardCut& c) { return c.splits > 1 ? c.units * c.splits * kTile : 0; }

template <int AB, int D>
int launch_forward(const ForwardArgs& a, const ForwardCut& c, const CUtensorMap (&maps)[3], cudaStream_t stream) {
  const int form = score_form(a.s);
  auto kernel = form == 2 ? span_attention_kernel<AB, D, true, true>
                : form == 1 ? span_attention_kernel<AB, D, true, false> : span_attention_kernel<AB, D, false, false>;
  static std::atomic<unsigned long long> granted[3] = {};
  if (cudaError_t e = grant_smem(reinterpret_cast<const void*>(kernel), forward_smem<D>(), granted[form])) return static_cast<int>(e);
  const dim3 grid(static_cast<unsigned>(c.units * c.splits));
  if (int st = launch_overlapped(kernel, grid, dim3(kThreads), forward_smem<D>(), 0, stream, maps[0], maps[1], maps[2], a)) return st;
  if (c.splits == 1) return kOk;
  const int rows = a.packed > 1 ? a.packed * a.s.sq : a.s.sq < kTile ? a.s.sq : kTile;
  const dim3 joins(static_cast<unsigned>(c.units * rows));
  return c.splits > 16 ? launch_overlapped(split_attention_kernel<AB, 16>, joins, dim3(512), 0, 0, stream, a)
                       : launch_overlapped(split_attention_kernel<AB, 4>, joins, dim3(128), 0, 0, stream, a);
}

}  // namespace
}  // namespace peco

using namespace peco;

extern "C" int peco_key_spans(const int* q_ends, long long q_stride, const int* k_ends, long long k_stride, int documents,
                              const int* lengths, const int* prefix, long long prefix_batch, int prefix_document,
                              int prefix_all, int causal, int window, int batch, int queries, int keys, int* rows,
                              int* tiles, void* stream_ptr) {
  if (batch < 0 || batch > 65535 || queries < 0 || keys < 0 || queries > 0x7ffffe00 || keys > 0x7ffffe00 || documents < 0 ||
      documents > 0x7ffffff0 || window < 0 || (documents > 0 && (!q_ends || !k_ends || lengths)))
    return kErrInvalidValue;
  if (batch == 0 || queries == 0) return kOk;
  if (!rows || !tiles || (reinterpret_cast<uintptr_t>(rows) & 15) || (reinterpret_cast<uintptr_t>(tiles) & 15)) return kErrInvalidValue;
  SpanArgs a{q_ends, k_ends, q_stride, k_stride, documents, lengths, prefix, prefix_batch, prefix_document, prefix_all,
             causal, window, batch, queries, keys, reinterpret_cast<int4*>(rows), reinterpret_cast<int4*>(tiles)};
  return launch_overlapped(key_spans_kernel, dim3((queries + kTile - 1) / kTile, batch), dim3(kTile), 0, 0,
                           static_cast<cudaStream_t>(stream_ptr), a);
}

extern "C" long long peco_span_attention_workspace(int batch, int heads, int kv_heads, int sq, int sk, int d) {
  if (!valid_attention(batch, heads, kv_heads, sq, sk, d)) return -1;
  if (batch == 0 || sq == 0) return 0;
  const ForwardCut c = cut_forward(batch, heads, kv_heads, sq, sk);
  return part_rows(c) * (4LL * d + 8);
}

extern "C" int peco_span_attention(const void* q, const void* k, const void* v, const long long* strides,
                                   const int* span_rows, const int* span_tiles, int spans_batched, const float* slopes,
                                   float scale, float cap, void* out, float* lse, int batch, int heads, int kv_heads, int sq,
                                   int sk, int d, int dtype, void* workspace, long long workspace_bytes,
                                   void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (!valid_attention(batch, heads, kv_heads, sq, sk, d) || !valid_scores(scale, cap) || !strides) return kErrInvalidValue;
  if (batch == 0 || sq == 0) return kOk;
  if (!q || !out || !lse || (sk > 0 && (!k || !v)) || !valid_plan(span_rows, span_tiles)) return kErrInvalidValue;
  ForwardArgs a{};
  a.q = HeadRows{q, strides[0], strides[1], strides[2]};
  a.k = HeadRows{k, strides[3], strides[4], strides[5]};
  a.v = HeadRows{v, strides[6], strides[7], strides[8]};
  const HeadRows o{out, strides[9], strides[10], strides[11]};
  if (!readable(a.q, batch, heads, sq) || !readable(o, batch, heads, sq) ||
      (sk > 0 && (!readable(a.k, batch, kv_heads, sk) || !readable(a.v, batch, kv_heads, sk))))
    return kErrInvalidValue;
  const ForwardCut c = cut_forward(batch, heads, kv_heads, sq, sk);
  if (c.units * c.splits > 0x7fffffffLL) return kErrUnsupported;
  if (c.splits > 1 && !usable_workspace(workspace, workspace_bytes, part_rows(c) * (4LL * d + 8))) return kErrWorkspace;
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
  a.out = out;
  a.out_batch = o.batch;
  a.out_head = o.head;
  a.out_row = o.row;
  a.lse = lse;
  a.packed = c.packed;
  a.turns = turns(a.s, c.row_blocks, heads / c.packed);
  a.splits = divisor(c.splits);
  a.rows = divisor(sq);
  a.s.group = divisor(heads / kv_heads);
  a.part = static_cast<float*>(workspace);
  a.part_sums = reinterpret_cast<float2*>(static_cast<float*>(workspace) + part_rows(c) * d);
  const HeadRows none{q, 0, 0, 0};  // without keys nothing is loaded
  CUtensorMap maps[3];
  const int box_rows = sq < kTile ? sq : kTile, key_rows = sk > 0 ? sk : 1;
  if (!head_map(&maps[0], a.q, batch, heads, sq, d, box_rows, c.packed, dtype) ||
      !head_map(&maps[1], sk > 0 ? a.k : none, sk > 0 ? batch : 1, sk > 0 ? kv_heads : 1, key_rows, d, kTile, 1, dtype) ||
      !head_map(&maps[2], sk > 0 ? a.v : none, sk > 0 ? batch : 1, sk > 0 ? kv_heads : 1, key_rows, d, kTile, 1, dtype))
    return kErrTensorMap;
  if (d <= 64) return dtype == 1 ? launch_forward<1, 64>(a, c, maps, stream) : launch_forward<0, 64>(a, c, maps, stream);
  return dtype == 1 ? launch_forward<1, 128>(a, c, maps, stream) : launch_forward<0, 128>(a, c, maps, stream);
}
