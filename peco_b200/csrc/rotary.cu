// Rotary embedding by positions on several axes (time, height, width of a
// video token), for Q and K of one attention call together.
//
// Head dimensions are cut into consecutive sections, one per axis, of d_a
// dimensions each.  Pair j of axis a turns by
//   angle = position[a] * theta^(-2 j / d_a),
//   (a, b) -> (a cos - b sin, b cos + a sin),
// where a pair is two neighbouring dimensions, or one from each half of the
// rotated dimensions.  Dimensions past the sections, and rows past the rotated
// ones (the text), are copied.  The inverse turn (the gradient) negates sin.
//
// No tables: the angle is formed in turns, position * (theta^(..) / 2 pi) in
// 64 bits, reduced to [-1/2, 1/2] there and only then rounded to fp32, so its
// error does not grow with the position.
//
// The operator moves bytes: each element is read once and written once, and
// the floor is that traffic at the copy bandwidth.  A thread owns 16 bytes of
// one token's row (of each half in the split pairing of 16-bit types) and walks
// the heads with it, so the sine and cosine are computed once per token and
// head group; the next four heads' loads are in flight while the current four
// are turned and stored.  24 + 24 heads x 119056 tokens x 128 bf16: 452 us, 6.47
// TB/s, the rate of a plain copy (643 us without the loads ahead, 473 / 461 /
// 522 / 489 us with 2 / 3 / 6 / 8 heads at a time).
#include "common.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"
#include "rows.cuh"

#include <math.h>

namespace peco {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 128;  // head dimension up to 256
constexpr int kThreads = 256;

struct RotaryTensor {
  const void* src;
  void* dst;
  long long sb, sh, sn;  // source strides (elements): batch, head, token
  long long db, dh, dn;  // destination strides
  int heads;
};

struct RotaryArgs {
  RotaryTensor t[2];
  int rows, rotated_rows, dims, pairs;
  int units, tokens_per_block, token_blocks, heads_per_block;
  int axes;
  unsigned grid[kMaxAxes];      // token grid (positions == null)
  const void* positions;        // [batch, rotated_rows, axes]
  long long pos_sb, pos_sn;     // strides in elements; the axes are adjacent
  int pos_type;                 // 0 int32, 1 int64, 2 fp32
  int inverse;
  double turns[kMaxPairs];      // turns per unit of position of each pair
  unsigned char axis[kMaxPairs];
};

// Position of a token on every axis.
__device__ __forceinline__ void positions_of(const RotaryArgs& a, int batch, int token, double (&p)[kMaxAxes]) {
  if (a.positions) {
    const long long at = batch * a.pos_sb + token * a.pos_sn;
#pragma unroll
    for (int i = 0; i < kMaxAxes; ++i) {
      p[i] = 0.0;
      if (i >= a.axes) continue;
      if (a.pos_type == 0) p[i] = static_cast<const int*>(a.positions)[at + i];
      else if (a.pos_type == 1) p[i] = static_cast<double>(static_cast<const long long*>(a.positions)[at + i]);
      else p[i] = static_cast<const float*>(a.positions)[at + i];
    }
  } else {
    unsigned rest = token;
#pragma unroll
    for (int i = kMaxAxes - 1; i >= 0; --i) {
      p[i] = 0.0;
      if (i >= a.axes) continue;
      const unsigned up = i ? rest / a.grid[i] : 0;
      p[i] = static_cast<double>(rest - up * a.grid[i]);
      rest = up;
    }
  }
}

// (cos, sin) of ``turns`` full turns, |turns| <= 1/2.  16-bit results hide the
// special-function unit's absolute error of 2^-20; fp32 ones take the library's.
template <typename T>
__device__ __forceinline__ void turn_to(float turns, float& c, float& s) {
  if constexpr (sizeof(T) == 2) {
    const float angle = 6.2831853071795865f * turns;
    c = __cosf(angle);
    s = __sinf(angle);
  } else {
    sincospif(2.0f * turns, &s, &c);
  }
}

// row of head h (Q's heads first, then K's) in the source or the destination
template <typename T>
__device__ __forceinline__ T* row_of(const RotaryArgs& a, int h, int batch, int token, bool destination) {
  const int which = h >= a.t[0].heads ? 1 : 0;
  const RotaryTensor& t = a.t[which];
  const int head = h - (which ? a.t[0].heads : 0);
  return destination ? static_cast<T*>(t.dst) + batch * t.db + head * t.dh + token * t.dn
                     : static_cast<T*>(const_cast<void*>(t.src)) + batch * t.sb + head * t.sh + token * t.sn;
}

// BYTES (2 to 32) between memory and registers in accesses of up to 16 bytes;
// the address is aligned to min(BYTES, 16).
template <int BYTES>
__device__ __forceinline__ void move_bytes(void* to, const void* from) {
  if constexpr (BYTES == 32) {
    reinterpret_cast<uint4*>(to)[0] = reinterpret_cast<const uint4*>(from)[0];
    reinterpret_cast<uint4*>(to)[1] = reinterpret_cast<const uint4*>(from)[1];
  } else if constexpr (BYTES == 16) {
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  } else if constexpr (BYTES == 8) {
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
  } else if constexpr (BYTES == 4) {
    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
  } else {
    *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
  }
}

// The 2V elements a thread moves of one row, as they lie in memory.
template <typename T, int V>
struct alignas(16) Run {
  T e[2 * V];
};

// V pairs per thread.  Interleaved: 2V neighbouring dimensions.  Split: V
// dimensions in each half of the rotated ones; the copied tail is then cut
// into runs of 2V like the interleaved form.  A thread walks its heads HEADS
// at a time with the next ones' loads in flight: source and destination may be
// the same tensor, so the order of loads and stores is written out here (heads
// never share memory).
template <typename T, int V, bool SPLIT, int HEADS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  wait_for_prior();
  let_next_start();
  const int slot = threadIdx.x / a.units, unit = threadIdx.x - slot * a.units;
  const int batch = blockIdx.x / a.token_blocks;
  const int token = (blockIdx.x - batch * a.token_blocks) * a.tokens_per_block + slot;
  if (slot >= a.tokens_per_block || token >= a.rows) return;
  const int pair0 = unit * V;
  // the two runs of V elements this thread moves
  const bool halves = SPLIT && pair0 < a.pairs;
  const int lo = halves ? pair0 : 2 * pair0;
  const int hi = halves ? pair0 + a.pairs : 2 * pair0 + V;
  const int all_heads = a.t[0].heads + a.t[1].heads;
  const int first = blockIdx.y * a.heads_per_block;
  const int last = min(first + a.heads_per_block, all_heads);
  constexpr int kRun = V * sizeof(T);
  // interleaved runs are adjacent: one access (V == 1: element by element, as the rows are not aligned)
  constexpr bool kJoined = !SPLIT && V > 1;

  auto load = [&](int h, Run<T, V>& r) {
    const T* src = row_of<T>(a, h, batch, token, false);
    if constexpr (kJoined) {
      move_bytes<2 * kRun>(r.e, src + lo);
    } else {
      move_bytes<kRun>(r.e, src + lo);
      move_bytes<kRun>(r.e + V, src + hi);
    }
  };
  Run<T, V> next[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
    if (first + h < last) load(first + h, next[h]);

  const int live = token < a.rotated_rows ? min(V, a.pairs - pair0) : 0;  // pairs that turn; the rest is copied
  float c[V], s[V];
  if (live > 0) {
    double p[kMaxAxes];
    positions_of(a, batch, token, p);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i >= live) continue;
      const int axis = a.axis[pair0 + i];
      double t = (axis == 0 ? p[0] : axis == 1 ? p[1] : axis == 2 ? p[2] : p[3]) * a.turns[pair0 + i];
      t -= rint(t);
      turn_to<T>(static_cast<float>(t), c[i], s[i]);
      if (a.inverse) s[i] = -s[i];
    }
  }

  for (int h0 = first; h0 < last; h0 += HEADS) {
    Run<T, V> now[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) now[h] = next[h];
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
      if (h0 + HEADS + h < last) load(h0 + HEADS + h, next[h]);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      if (h0 + h >= last) continue;
      Run<T, V>& r = now[h];
      if (live > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int ia = SPLIT ? i : 2 * i, ib = SPLIT ? V + i : 2 * i + 1;
          const float u = to_f32<T>(r.e[ia]), w = to_f32<T>(r.e[ib]);
          const T x = from_f32<T>(u * c[i] - w * s[i]), y = from_f32<T>(w * c[i] + u * s[i]);
          if (i < live) {
            r.e[ia] = x;
            r.e[ib] = y;
          }
        }
      }
      T* dst = row_of<T>(a, h0 + h, batch, token, true);
      if constexpr (kJoined) {
        move_bytes<2 * kRun>(dst + lo, r.e);
      } else {
        move_bytes<kRun>(dst + lo, r.e);
        move_bytes<kRun>(dst + hi, r.e + V);
      }
    }
  }
}

template <typename T, int V, bool SPLIT, int HEADS>
int launch_form(RotaryArgs& a, int batch, cudaStream_t stream) {
  a.units = a.dims / (2 * V);
  a.tokens_per_block = kThreads / a.units;
  a.token_blocks = (a.rows + a.tokens_per_block - 1) / a.tokens_per_block;
  const long long blocks = static_cast<long long>(batch) * a.token_blocks;
  if (blocks > 0x7fffffffLL) return kErrUnsupported;
  // All heads in one block when the tokens alone fill the GPU (the sines are
  // then computed once per token); otherwise heads are spread over blocks.
  const int heads = a.t[0].heads + a.t[1].heads;
  long long groups = (8LL * kNumSMs + blocks - 1) / blocks;
  if (groups > heads) groups = heads;
  a.heads_per_block = static_cast<int>((heads + groups - 1) / groups);
  const dim3 grid(static_cast<unsigned>(blocks), (heads + a.heads_per_block - 1) / a.heads_per_block);
  return launch_overlapped(rotary_kernel<T, V, SPLIT, HEADS>, grid, dim3(kThreads), 0, 0, stream, a);
}

// Whether every row's runs of V pairs start on the boundaries that V needs.
template <typename T>
bool runs_aligned(const RotaryArgs& a, int v, bool split) {
  if (a.dims % (2 * v) || (split && a.pairs % v)) return false;
  const long long bytes = (split ? v : 2 * v) * sizeof(T), align = bytes < 16 ? bytes : 16;
  for (const RotaryTensor& t : a.t) {
    if (!t.heads) continue;
    const long long step = (t.sb | t.sh | t.sn | t.db | t.dh | t.dn) * static_cast<long long>(sizeof(T));
    if ((step | static_cast<long long>(reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst))) & (align - 1))
      return false;
  }
  return true;
}

template <typename T>
int launch_rotary(RotaryArgs& a, int batch, bool split, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {  // eight pairs: 16 bytes of each half
    if (split && runs_aligned<T>(a, 8, true)) return launch_form<T, 8, true, 2>(a, batch, stream);
  }
  if (runs_aligned<T>(a, 4, split))
    return split ? launch_form<T, 4, true, 4>(a, batch, stream) : launch_form<T, 4, false, 4>(a, batch, stream);
  return split ? launch_form<T, 1, true, 4>(a, batch, stream) : launch_form<T, 1, false, 4>(a, batch, stream);
}

}  // namespace
}  // namespace peco

using namespace peco;

extern "C" int peco_rotary(const void* q, void* q_out, int q_heads, const long long* q_strides, const void* k,
                           void* k_out, int k_heads, const long long* k_strides, int batch, int rows,
                           int rotated_rows, int dims, const int* axes, int n_axes, double theta, const int* grid,
                           const void* positions, long long pos_batch_stride, long long pos_row_stride, int pos_type,
                           int interleaved, int inverse, int dtype, void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype < 0 || dtype > 2 || n_axes < 1 || n_axes > kMaxAxes || dims < 2 || dims > 2 * kMaxPairs || dims % 2)
    return kErrUnsupported;
  if (batch < 0 || rows < 0 || rotated_rows < 0 || rotated_rows > rows || q_heads < 0 || k_heads < 0 || !axes ||
      !(theta > 0.0) || pos_type < 0 || pos_type > 2 || (!grid && !positions))
    return kErrInvalidValue;
  if ((q_heads && !q_strides) || (k_heads && !k_strides) || q_heads > 32767 || k_heads > 32767) return kErrInvalidValue;
  RotaryArgs a{};
  for (int i = 0; i < n_axes; ++i) {
    if (axes[i] < 0 || axes[i] % 2 || 2 * a.pairs + axes[i] > dims) return kErrInvalidValue;
    // theta^(-2 j / d) by repeated multiplication in 64 bits
    const double step = axes[i] ? pow(theta, -2.0 / axes[i]) : 1.0;
    double f = 0.15915494309189533577;  // 1 / (2 pi)
    for (int j = 0; j < axes[i] / 2; ++j, f *= step) {
      a.turns[a.pairs] = f;
      a.axis[a.pairs++] = static_cast<unsigned char>(i);
    }
  }
  if (!positions) {
    long long tokens = 1;
    for (int i = 0; i < n_axes; ++i) {
      if (grid[i] < 0) return kErrInvalidValue;
      a.grid[i] = grid[i] > 0 ? grid[i] : 1;
      tokens *= grid[i];
      if (tokens > rows) return kErrInvalidValue;
    }
    if (tokens != rotated_rows) return kErrInvalidValue;
  }
  if (batch == 0 || rows == 0 || q_heads + k_heads == 0) return kOk;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return kErrInvalidValue;
  const void* src[2] = {q, k};
  void* dst[2] = {q_out, k_out};
  const int heads[2] = {q_heads, k_heads};
  const long long* strides[2] = {q_strides, k_strides};
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    const long long* s = strides[i];
    a.t[i] = RotaryTensor{src[i], dst[i], s[0], s[1], s[2], s[3], s[4], s[5], heads[i]};
  }
  a.rows = rows;
  a.rotated_rows = rotated_rows;
  a.dims = dims;
  a.axes = n_axes;
  a.positions = positions;
  a.pos_sb = pos_batch_stride;
  a.pos_sn = pos_row_stride;
  a.pos_type = pos_type;
  a.inverse = inverse;
  const bool split = !interleaved;
  switch (dtype) {
    case 0: return launch_rotary<__half>(a, batch, split, stream);
    case 1: return launch_rotary<__nv_bfloat16>(a, batch, split, stream);
    default: return launch_rotary<float>(a, batch, split, stream);
  }
}
