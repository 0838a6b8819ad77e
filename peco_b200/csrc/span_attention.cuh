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

struct ScoreArgs {
  const int4* spans;        // [batch or 1, sq]: lo, hi, pos, 0 (null: every row sees every key, pos = i + sk - sq)
  const int4* span_tiles;   // [batch or 1, ceil(sq / 128)]: least lo, largest hi, largest lo, least hi of the rows
  int spans_batched;
  const float* slopes;      // [heads] or null
  int batch, heads, kv_heads, sq, sk, d;
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

// cap tanh(s / cap) in log2 units: with A = cap log2(e) and e = 2^(2 log2(e) s
// scale / cap), A tanh = A - 2A / (1 + e); infinite e gives A, e = 0 gives -A.
// Within a few 2^-23 of A in absolute terms.
struct Cap {
  float a, b;
  __device__ explicit Cap(const ScoreArgs& s) : a(s.cap * kLog2E), b(2.0f * kLog2E * s.scale / s.cap) {}
  __device__ __forceinline__ float recip(float raw) const {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + exp2_approx(raw * b)));
    return y;
  }
  __device__ __forceinline__ float value(float r) const { return fmaf(-2.0f * a, r, a); }
  // d capped / d raw, without the scale: 1 - tanh^2 = 4 r (1 - r)
  __device__ __forceinline__ float slope(float r) const { return 4.0f * r * (1.0f - r); }
};

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

// Descriptors of a tile's 16-wide steps along the dimensions (K-major) and along the rows (MN-major).
__device__ __forceinline__ uint64_t desc_dims(uint32_t tile, int step) {
  return smem_desc(tile + (step >> 2) * kPanelBytes + (step & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int step) {
  return smem_desc(tile + step * 2048, kPanelBytes, 1024);
}

template <int AB>
using Element = typename std::conditional<AB == 1, __nv_bfloat16, __half>::type;

// ---- host ----
inline long long round_up(long long v, long long a) { return (v + a - 1) / a * a; }

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
