// What the forward and the gradient of attention over key spans share.
//
// Query row i of a sample sees the keys [lo, hi) of its span and stands at key
// position ``pos``:
//   z_ij = cap tanh(scale q_i.k_j / cap) - slope_h |pos_i - j|   (cap, slope optional)
//   p_ij = exp(z_ij - lse_i) for lo_i <= j < hi_i, else 0;  out_i = sum_j p_ij v_j
#pragma once

#include "common.cuh"
#include "rows.cuh"

#include <type_traits>

namespace peco {
namespace {

constexpr int kTile = 128;               // query rows and keys of a tile
constexpr int kPanelBytes = kTile * 128;  // 64 of a tile's dimensions: 128 rows x 128 bytes, 128-byte swizzle
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A [batch, heads, rows, d] tensor with adjacent dims; strides in elements.
struct HeadRows {
  const void* ptr;
  long long batch, head, row;
};

// n / by for 0 <= n < 2^31, without the divide's latency (a CTA's place takes seven of
// them in a row before its first load, 1200 clocks; 592 CTAs of one key tile 24.0 us
// and 22.4).  mul = ceil(2^s / by) with s = 31 +
// ceil(log2 by): mul by - 2^s < by <= 2^(s - 31), so n mul / 2^s is off by less than 1 / by.
struct Divisor {
  unsigned mul;
  int by, shift;
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>(static_cast<unsigned long long>(n) * mul >> shift);
  }
};
inline Divisor divisor(int by) {
  int log = 0;
  while ((1LL << log) < by) ++log;
  const unsigned long long whole = 1ull << (31 + log);
  return Divisor{static_cast<unsigned>((whole + by - 1) / by), by, 31 + log};
}

// Units (heads by tiles of rows, of every sample) in the order in which CTAs take them
struct Turns {
  Divisor sample, chunk, heads, rest;  // units of a sample and of the heads in turn; heads in turn, and of the last ones
  int tiles, all;                      // tiles of rows, heads
  __device__ __forceinline__ void at(int unit, int& b, int& head, int& rank) const {
    b = sample(unit);
    const int n = unit - b * sample.by, first = chunk(n) * heads.by, m = n - first * tiles;
    const Divisor& of = all - first < heads.by ? rest : heads;
    rank = of(m);
    head = first + m - rank * of.by;
  }
};

struct ScoreArgs {
  const int4* spans;        // [batch or 1, sq]: lo, hi, pos, ranked tile (null: every row sees every key, pos = i + sk - sq)
  const int4* span_tiles;   // [batch or 1, ceil(sq / 128)]: least lo, largest hi, largest lo, least hi of the rows
  int spans_batched;
  const float* slopes;      // [heads] or null
  int batch, heads, kv_heads, sq, sk, d;
  Divisor group;            // heads on a key head
  float scale;              // > 0
  float cap;                // 0: none
  unsigned* status;
};

__device__ __forceinline__ int row_tiles(const ScoreArgs& a) { return (a.sq + kTile - 1) / kTile; }
__device__ __forceinline__ int4 span_of(const ScoreArgs& a, int b, int i) {
  if (!a.spans) return make_int4(0, a.sk, i + a.sk - a.sq, 0);
  return a.spans[static_cast<long long>(a.spans_batched ? b : 0) * a.sq + i];
}
// (least lo, largest hi, largest lo, least hi) of a tile of rows; without a visible key: hi <= lo
__device__ __forceinline__ int4 tile_span(const ScoreArgs& a, int b, int tile) {
  if (!a.spans) return make_int4(0, a.sk, 0, a.sk);
  return a.span_tiles[static_cast<long long>(a.spans_batched ? b : 0) * row_tiles(a) + tile];
}

// The n-th tile of query rows to be taken: the longest first, as the plan ranks them.
__device__ __forceinline__ int ranked_tile(const ScoreArgs& a, int b, int n, int tiles) {
  if (!a.spans || tiles == 1) return tiles - 1 - n;
  const int t = a.spans[static_cast<long long>(a.spans_batched ? b : 0) * a.sq + n].w;
  return min(max(t, 0), tiles - 1);
}
// Heads whose tiles are taken in turn, so that the last CTAs to start are short ones
// of every head; no more heads than fill the SMs twice, for their keys to stay in L2.
// With the longest first, 8 heads of 9999 rows in four documents 162 -> 125 us, in
// causal order with 64 dims 98 -> 76 us (a window of 1000 on 16000 rows 448 -> 458 us).
inline Turns turns(const ScoreArgs& a, int tiles, int heads) {
  const int fill = a.spans ? (2 * kNumSMs + tiles - 1) / tiles : 1, together = fill < heads ? fill : heads;
  return Turns{divisor(heads * tiles), divisor(together * tiles), divisor(together),
               divisor(heads % together ? heads % together : together), tiles, heads};
}

// cap tanh(s / cap) in log2 units: with A = cap log2(e) and e = 2^(2 log2(e) s
// scale / cap), A tanh = A - 2A / (1 + e); infinite e gives A, e = 0 gives -A.
// Within a few 2^-23 of A in absolute terms: for caps up to kWideCap 2e-5, a
// probability's rounding to fp16 being 2^-12 of it.  Under larger caps that is all
// that small scores are, so those below a quarter of the cap take the series x (1 -
// x^2/3 + 2 x^4/15 - 17 x^6/315 + 62 x^8/2835), off by 2^-26 of the value (24 heads x 7006
// rows of 128 dims: forward 1009 us without it and 1144 with it, gradient 2667 and
// 3092), in kernels of their own (a branch on the cap cost the others 4%).
constexpr float kWideCap = 64.0f;
struct Cap {
  float a, b, x, unit;
  bool wide;
  __device__ explicit Cap(const ScoreArgs& s)
      : a(s.cap * kLog2E), b(2.0f * kLog2E * s.scale / s.cap), x(s.scale / s.cap), unit(s.scale * kLog2E), wide(s.cap > kWideCap) {}
  __device__ __forceinline__ float recip(float raw) const {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + exp2_approx(raw * b)));
    return y;
  }
  __device__ __forceinline__ float value(float raw, float r) const {
    const float2 twice = make_float2(raw, raw), both = make_float2(r, r);
    return wide ? value<true>(twice, both).x : value<false>(twice, both).x;
  }
  // two scores at a time
  __device__ __forceinline__ float2 recip(float2 raw) const {
    const float2 x = fmul2(raw, make_float2(b, b));
    const float2 y = fadd2(make_float2(exp2_approx(x.x), exp2_approx(x.y)), make_float2(1.0f, 1.0f));
    float2 r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(y.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(y.y));
    return r;
  }
  template <bool WIDE>
  __device__ __forceinline__ float2 value(float2 raw, float2 r) const {
    const float2 whole = ffma2(r, make_float2(-2.0f * a, -2.0f * a), make_float2(a, a));
    if constexpr (!WIDE) return whole;
    auto both = [](float v) { return make_float2(v, v); };
    const float2 y = fmul2(raw, both(x)), t = fmul2(y, y), s = fmul2(raw, both(unit));
    float2 p = ffma2(t, both(62.0f / 2835.0f), both(-17.0f / 315.0f));
    p = ffma2(t, p, both(2.0f / 15.0f));
    p = ffma2(t, p, both(-1.0f / 3.0f));
    p = ffma2(fmul2(t, p), s, s);
    return make_float2(t.x < 0.0625f ? p.x : whole.x, t.y < 0.0625f ? p.y : whole.y);
  }
  // d capped / d raw, without the scale: 1 - tanh^2 = 4 r - 4 r r (r rounded to 2^-24: off by a few 2^-24 in absolute terms)
  static __device__ __forceinline__ float2 slope(float2 r) {
    const float2 f = fmul2(r, make_float2(4.0f, 4.0f));
    return ffma2(f, make_float2(-r.x, -r.y), f);
  }
};

// N scores in log2 units, capped (WIDE: by a cap above kWideCap) or scaled; the slopes of capped ones
template <bool WIDE, int N>
__device__ __forceinline__ void scaled_scores(const ScoreArgs& s, const Cap& cap, float (&z)[N], float* slopes) {
  if (WIDE || s.cap > 0.0f) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 raw = make_float2(z[e], z[e + 1]), r = cap.recip(raw), v = cap.value<WIDE>(raw, r);
      if (slopes) {
        const float2 d = Cap::slope(r);
        slopes[e] = d.x;
        slopes[e + 1] = d.y;
      }
      z[e] = v.x;
      z[e + 1] = v.y;
    }
  } else {
    const float f = s.scale * kLog2E;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 v = fmul2(make_float2(z[e], z[e + 1]), make_float2(f, f));
      z[e] = v.x;
      z[e + 1] = v.y;
    }
  }
}
// less slope |apart - e|, for the keys side by side from a tile's first
template <int N>
__device__ __forceinline__ void less_distance(float slope, float apart, float (&z)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) z[e] = fmaf(-slope, fabsf(apart - static_cast<float>(e)), z[e]);
}

// 16-bit rows that the lanes of a warp hold, on their way to memory through shared
// memory, so that a store writes whole rows: 16 bytes of 32 rows each take the
// store unit eight times as long (24 heads x 16000 rows under a window of 1000: 449
// and 436 us).  ``at``: 32 rows of COLS, the warp's own.
template <int COLS>
struct RowsOut {
  static constexpr int kChunks = COLS / 8, kTurn = 32 / kChunks;  // 16-byte chunks of a row, rows a store writes
  unsigned char* at;
  int lane;
  __device__ __forceinline__ uint4* place(int row, int chunk) const {  // turned, so that eight lanes meet all banks
    return reinterpret_cast<uint4*>(at) + row * kChunks + (chunk ^ (kChunks >= 8 ? row & 7 : row >> 1 & 3));
  }
  __device__ __forceinline__ void put(int chunk, uint4 v) const { *place(lane, chunk) = v; }
  // every lane's row to its ``out`` (null: nowhere), the first ``cols`` columns
  template <typename T>
  __device__ __forceinline__ void store(T* out, int cols) const {
    __syncwarp();
    const int chunk = lane % kChunks;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int row = i * kTurn + lane / kChunks;
      T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), row));
      if (to && chunk * 8 < cols) *reinterpret_cast<uint4*>(to + chunk * 8) = *place(row, chunk);
    }
  }
};

// 128 columns of a TMEM lane: four loads in flight, one wait.
__device__ __forceinline__ void tmem_ld128_sync(uint32_t at, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%129];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95}, [%130];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%131];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
        "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
        "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
        "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
        "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
        "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
        "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(at), "r"(at + 32), "r"(at + 64), "r"(at + 96)
      : "memory");
}

__device__ __forceinline__ void tile_load_4d(void* dst, const CUtensorMap* map, int x, int row, int head, int batch,
                                             uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(batch), "r"(smem_u32(bar))
      : "memory");
}

// All panels of a tile
template <int PANELS>
__device__ __forceinline__ void load_rows(unsigned char* dst, const CUtensorMap* map, int row, int head, int batch,
                                          uint64_t* bar) {
#pragma unroll
  for (int p = 0; p < PANELS; ++p) tile_load_4d(dst + p * kPanelBytes, map, 64 * p, row, head, batch, bar);
}

// Zeros in rows [from, to) of a tile in shared memory, by one warp; visible to the tensor core.
template <int PANELS>
__device__ __forceinline__ void clear_rows(unsigned char* tile, int from, int to, int lane) {
  for (int i = lane; i < (to - from) * 8; i += 32)
#pragma unroll
    for (int p = 0; p < PANELS; ++p)
      *reinterpret_cast<uint4*>(tile + p * kPanelBytes + (from + (i >> 3)) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

// A tile's descriptor for steps of 16 along the dimensions (K-major) or along the
// rows (MN-major): the low word, to which a step adds a constant; the high word is
// the same for all.  The issuing warp runs whole with one elected lane issuing, and
// takes what it computes from warp-uniform values, so that descriptors stay in
// uniform registers: moving each there first made issuing a step slower than the
// tensor core.
__device__ __forceinline__ uint32_t desc_dims(uint32_t tile) { return ((tile >> 4) & 0x3fffu) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_rows(uint32_t tile) {
  return ((tile >> 4) & 0x3fffu) | (static_cast<uint32_t>(kPanelBytes >> 4) << 16);
}
__host__ __device__ constexpr uint32_t dims_step(int i) { return (i >> 2) * (kPanelBytes >> 4) + (i & 3) * 2; }
__host__ __device__ constexpr uint32_t rows_step(int i) { return i * 128; }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8 rows 1024 bytes apart, sm_100 form, 128-byte swizzle

__device__ __forceinline__ uint64_t whole_desc(uint32_t low) { return (static_cast<uint64_t>(kDescHigh) << 32) | low; }

// to = X Y^T over D dimensions
template <int D>
__device__ __forceinline__ void product_dims(uint32_t to, uint32_t x, uint32_t y, uint32_t idesc) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    umma_ss(to, whole_desc(x + dims_step(i)), whole_desc(y + dims_step(i)), idesc, i > 0);
}
// to (+)= A Y over ``ROWS`` rows of a tile, A 16-bit pairs in TMEM, each run of 64 rows
// 64 columns after the one before
template <int ROWS>
__device__ __forceinline__ void product_rows(uint32_t to, uint32_t a, uint32_t y, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int i = 0; i < ROWS / 16; ++i)
    umma_ts(to, a + (i >> 2) * 64 + (i & 3) * 8, whole_desc(y + rows_step(i)), idesc, i > 0 ? 1u : accumulate);
}

// A value that all lanes hold, as the compiler can see
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

template <int AB>
using Element = typename std::conditional<AB == 1, __nv_bfloat16, __half>::type;

// ---- host ----
// Scale, cap (0: none) and their quotient stay well inside fp32.
inline bool valid_scores(float scale, float cap) {
  auto fits = [](float v) { return v >= 0.99e-30f && v <= 1.01e30f; };
  return fits(scale) && (cap == 0.0f || (fits(cap) && scale / cap <= 1.01e30f));
}
// 0: scores as they are, 1: capped or with a bias by distance, 2: under a wide cap
inline int score_form(const ScoreArgs& s) { return s.cap > kWideCap ? 2 : s.cap > 0.0f || s.slopes ? 1 : 0; }
inline long long round_up(long long v, long long a) { return (v + a - 1) / a * a; }

// Rows and tiles of a plan, both or neither; read 16 bytes at a time.
inline bool valid_plan(const int* rows, const int* tiles) {
  return (rows == nullptr) == (tiles == nullptr) && ((reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(tiles)) & 15) == 0;
}

// Whether TMA can read it in place: every row, head and sample on 16 bytes.
inline bool readable(const HeadRows& t, int batch, int heads, int rows) {
  auto fits = [](long long stride, int n) { return n <= 1 || (stride > 0 && (stride & 7) == 0 && stride < (1LL << 38)); };
  return t.ptr && (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0 && fits(t.row, rows) && fits(t.head, heads) &&
         fits(t.batch, batch);
}

// Boxes of 64 dims x box_rows rows x box_heads heads; dims past d and rows past the end read as 0.
inline bool head_map(CUtensorMap* map, const HeadRows& t, int batch, int heads, int rows, int d, int box_rows,
                     int box_heads, int dtype) {
  const uint64_t some = static_cast<uint64_t>(round_up(d, 8)) * 2;  // of an axis that is never walked
  auto bytes = [&](long long stride, int n) { return n > 1 ? static_cast<uint64_t>(stride) * 2 : some; };
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(rows), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {bytes(t.row, rows), bytes(t.head, heads), bytes(t.batch, batch)};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), static_cast<uint32_t>(box_heads), 1};
  return encode_tensor_map(map, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.ptr,
                           dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace
}  // namespace peco
