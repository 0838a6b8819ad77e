// Linear layers in 8-bit integers: rows quantised with a scale each, weights with
// a scale per output channel, the product of product.cuh.
//
//   X[m, k] = round(127 x[m, k] / max_k |x[m, k]|) (ties to even), row[m] = max / 127
//   out = residual + gate * act(row[m] col[n] sum_k X[m, k] W[n, k] + bias[n])
//
// The integer sums are exact (|sum| <= 128 * 128 * K < 2^31), so the result does
// not depend on how a product is cut.
//
// What the products measured (B200, bf16 results, rows quantised before): 6750 x 3072 x
// 12288 175 us (2.9 POP/s, 359 us in bf16; bound by the tensor core and the power
// limit), with gelu 190; 7006 x 15360 x 3072 241 us (bf16 520); 256 x 3072 x 12288 12 us
// (bf16 17); 1 x 3072 x 18432 10 us (5.7 TB/s of weights, bf16 21).
#include "common.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"
#include "product.cuh"
#include "rows.cuh"

namespace peco {
namespace {

constexpr int kMaxSummands = 131071;

// ---- quantising rows ------------------------------------------------------------------
// What rounding a row needs: x * pre * inv is 127 x / max.  ``pre`` lifts rows so
// small that 127 / max would overflow.
struct RowScale {
  float pre, inv, scale;
};

// From the largest magnitude's bits: magnitudes of 16-bit floats order as integers,
// infinities and NaN (from ``kInfinite`` on) above all numbers.  Such a row has no
// scale: it is NaN, and so is every result of the row; its integers are 0.
template <typename T>
__device__ __forceinline__ RowScale row_scale_of(uint32_t top) {
  constexpr uint32_t kInfinite = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  if (top >= kInfinite) return RowScale{0.0f, 0.0f, __int_as_float(0x7fffffff)};
  if (top == 0) return RowScale{0.0f, 0.0f, 0.0f};
  const unsigned short bits = static_cast<unsigned short>(top);
  const float most = to_f32<T>(*reinterpret_cast<const T*>(&bits));
  const float pre = most < 1e-30f ? 1.2676506e30f : 1.0f;  // 2^100
  return RowScale{pre, __fdiv_rn(127.0f, most * pre), __fdiv_rn(most, 127.0f)};
}

// round(127 x / max) of a pair, ties to even, each as the low byte of a word.
// x inv is within 2^-23 of 127 x / max, relatively.  Where that quotient is not half
// an odd number it is 2^-19 away from it (relatively: x and max have at most 11
// significant bits), so rounding to 20 bits, 2^-20 at most, keeps it on its side
// and puts the quotients that are half an odd number exactly there: the integers
// are those of the exact quotient.  Adding 1.5 * 2^23 rounds to even.
__device__ __forceinline__ uint2 round_pair(float2 x, float2 inv) {
  const float2 t = fmul2(x, inv);
  auto held = [](float v) { return __uint_as_float((__float_as_uint(v) + 8u) & ~15u); };
  const float2 r = fadd2(make_float2(held(t.x), held(t.y)), make_float2(12582912.0f, 12582912.0f));
  return make_uint2(__float_as_uint(r.x), __float_as_uint(r.y));
}
__device__ __forceinline__ uint32_t four_bytes(uint2 a, uint2 b) {
  return __byte_perm(__byte_perm(a.x, a.y, 0x0040), __byte_perm(b.x, b.y, 0x0040), 0x5410);
}
template <typename T>
__device__ __forceinline__ uint2 round_eight(uint4 raw, const RowScale& s) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint2 q[4];
  const float2 inv = make_float2(s.inv, s.inv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = unpack2<T>(w[i]);
    if (s.pre != 1.0f) {  // a tiny row, or one without a scale (infinities times 0 would be NaN)
      if (s.pre == 0.0f) f = make_float2(0.0f, 0.0f);
      f = fmul2(f, make_float2(s.pre, s.pre));
    }
    q[i] = round_pair(f, inv);
  }
  return make_uint2(four_bytes(q[0], q[1]), four_bytes(q[2], q[3]));
}

struct QuantizeArgs {
  const uint16_t* x[2];     // rows of width[0] and width[1] elements side by side
  long long stride[2];
  int width[2];
  int8_t* values;           // rows ld bytes apart
  long long ld;
  float* scales;
  int rows;
};

// The largest magnitude over a row's ``warps`` warps (a power of two) of a block of 8.
__device__ __forceinline__ uint32_t row_top(uint32_t top, int warps, uint32_t* shared) {
  top = __reduce_max_sync(0xffffffffu, top);
  if (warps == 1) return top;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) shared[warp] = top;
  __syncthreads();
  const int first = warp & ~(warps - 1);
  for (int i = 0; i < warps; ++i) top = max(top, shared[first + i]);
  return top;
}

// A row per WARPS warps, in registers between its maximum and its rounding: 8
// elements a thread and chunk, read once.  Blocks walk the rows, the next row's loads in
// flight while one is rounded.  Bound by HBM: 34680 x 3072 59 us (5.4 TB/s; 82 us with a
// block a row pair), 7006 x 15360 53 us (6.1 TB/s).
template <typename T, int WARPS, int CHUNKS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantizeArgs a) {
  __shared__ uint32_t tops[2][8];
  wait_for_prior();
  let_next_start();
  constexpr int kThreads = 32 * WARPS;
  const int at = threadIdx.x % kThreads;
  const int chunks0 = a.width[0] >> 3, chunks = chunks0 + (a.width[1] >> 3);
  auto load = [&](uint4 (&held)[CHUNKS], long long row) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = at + i * kThreads;
      held[i] = make_uint4(0, 0, 0, 0);
      if (row < a.rows && c < chunks)
        held[i] = *reinterpret_cast<const uint4*>(c < chunks0 ? a.x[0] + row * a.stride[0] + c * 8
                                                              : a.x[1] + row * a.stride[1] + (c - chunks0) * 8);
    }
  };
  constexpr int kRows = 8 / WARPS;
  long long row0 = static_cast<long long>(blockIdx.x) * kRows;
  const int own = threadIdx.x / kThreads;
  uint4 held[CHUNKS], next[CHUNKS];
  load(held, row0 + own);
  for (int turn = 0; row0 < a.rows; turn ^= 1) {  // whole blocks: all threads meet in row_top
    const long long row = row0 + own;
    row0 += static_cast<long long>(gridDim.x) * kRows;
    load(next, row0 + own);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const uint32_t m = __vmaxu2(__vmaxu2(held[i].x & 0x7fff7fffu, held[i].y & 0x7fff7fffu),
                                  __vmaxu2(held[i].z & 0x7fff7fffu, held[i].w & 0x7fff7fffu));
      top = max(top, max(m & 0xffffu, m >> 16));
    }
    const RowScale s = row_scale_of<T>(row_top(top, WARPS, tops[turn]));
    if (row < a.rows) {
      if (at == 0) a.scales[row] = s.scale;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int c = at + i * kThreads;
        if (c < chunks) *reinterpret_cast<uint2*>(a.values + row * a.ld + c * 8) = round_eight<T>(held[i], s);
      }
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) held[i] = next[i];
  }
}

// Rows that do not start on 16 bytes, or wider than 16384: a block per row, an
// element at a time, read twice (the second time from the caches; holding them in
// registers instead took as long, 8000 x 1001 16 us).
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const __grid_constant__ QuantizeArgs a) {
  __shared__ uint32_t tops[8];
  wait_for_prior();
  let_next_start();
  const long long row = blockIdx.x;
  uint32_t top = 0;
  for (int s = 0; s < 2; ++s) {
    const uint16_t* x = a.x[s] + row * a.stride[s];
#pragma unroll 4
    for (int c = threadIdx.x; c < a.width[s]; c += 256) top = max(top, x[c] & 0x7fffu);
  }
  const RowScale r = row_scale_of<T>(row_top(top, 8, tops));
  if (threadIdx.x == 0) a.scales[row] = r.scale;
  int8_t* out = a.values + row * a.ld;
  for (int s = 0; s < 2; ++s) {
    const uint16_t* x = a.x[s] + row * a.stride[s];
#pragma unroll 4
    for (int c = threadIdx.x; c < a.width[s]; c += 256) {
      const uint16_t bits = x[c];
      const float f = r.pre == 0.0f ? 0.0f : to_f32<T>(*reinterpret_cast<const T*>(&bits)) * r.pre;
      out[c] = static_cast<int8_t>(round_pair(make_float2(f, 0.0f), make_float2(r.inv, 0.0f)).x);
    }
    out += a.width[s];
  }
}

template <typename T>
int quantize(const QuantizeArgs& a, cudaStream_t stream) {
  const bool vec = ((reinterpret_cast<uintptr_t>(a.x[0]) | reinterpret_cast<uintptr_t>(a.x[1])) & 15) == 0 &&
                   ((a.stride[0] | a.stride[1] | a.width[0] | a.width[1]) & 7) == 0 && (a.ld & 7) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.values) & 7) == 0;
  const int width = a.width[0] + a.width[1];
  const dim3 block(256);
  auto grid = [&](int warps, int resident) {
    const int blocks = (a.rows + 8 / warps - 1) / (8 / warps);
    return dim3(blocks < resident * kNumSMs ? blocks : resident * kNumSMs);
  };
  if (!vec || width > 16384) return launch_overlapped(quantize_rows_any_kernel<T>, dim3(a.rows), block, 0, 0, stream, a);
  // a row stays within one block; the fewer warps, the fewer that wait for each other
  if (width <= 1024) return launch_overlapped(quantize_rows_kernel<T, 1, 4>, grid(1, 4), block, 0, 0, stream, a);
  if (width <= 2048) return launch_overlapped(quantize_rows_kernel<T, 4, 2>, grid(4, 5), block, 0, 0, stream, a);
  if (width <= 4096) return launch_overlapped(quantize_rows_kernel<T, 4, 4>, grid(4, 4), block, 0, 0, stream, a);
  if (width <= 8192) return launch_overlapped(quantize_rows_kernel<T, 8, 4>, grid(8, 4), block, 0, 0, stream, a);
  return launch_overlapped(quantize_rows_kernel<T, 8, 8>, grid(8, 2), block, 0, 0, stream, a);
}

// ---- unaligned operands ------------------------------------------------------------
// Rows of bytes, any stride and alignment, to rows ld bytes apart (a multiple of
// 16).  A thread makes four bytes from the two aligned words that hold them; words
// without a byte of the row are not read.  Blocks stride over the rows, threads
// over the words, eight in flight.
__global__ void __launch_bounds__(256) pack_bytes_kernel(const int8_t* src, long long stride, int8_t* dst, long long ld,
                                                         int rows, int cols) {
  wait_for_prior();
  let_next_start();
  const int words = (cols + 3) >> 2;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(src + r * stride), end = at + cols;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
    const uint32_t shift = static_cast<uint32_t>(at & 3) * 8;
    uint32_t* to = reinterpret_cast<uint32_t*>(dst + r * ld);
    for (int w0 = threadIdx.x; w0 < words; w0 += 8 * 256) {
      uint32_t low[8], high[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int w = w0 + i * 256;
        low[i] = w < words ? from[w] : 0u;
        high[i] = w < words && reinterpret_cast<uintptr_t>(from + w + 1) < end ? from[w + 1] : 0u;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w0 + i * 256 < words) to[w0 + i * 256] = __funnelshift_r(low[i], high[i], shift);
    }
  }
}

bool readable(const Operand& o) { return ((reinterpret_cast<uintptr_t>(o.ptr) | o.stride) & 15) == 0; }
long long copy_bytes(long long rows, long long cols) { return align_up(rows * align_up(cols, 16), kAlign); }

int make_readable(Operand& o, Carver& ws, cudaStream_t stream) {
  if (readable(o)) return kOk;
  int8_t* to = static_cast<int8_t*>(ws.take(copy_bytes(o.rows, o.cols)));
  const long long ld = align_up(o.cols, 16);
  const int st = launch_overlapped(pack_bytes_kernel, dim3(o.rows < 8 * kNumSMs ? o.rows : 8 * kNumSMs), dim3(256), 0, 0,
                                   stream, static_cast<const int8_t*>(o.ptr), o.stride, to, ld, o.rows, o.cols);
  o.ptr = to;
  o.stride = ld;
  return st;
}

// A single row's stride is never walked; TMA wants it aligned all the same.
Operand bytes_operand(const void* p, long long stride, long long rows, int cols) {
  return Operand{p, rows == 1 ? align_up(cols, 16) : stride, static_cast<int>(rows), cols};
}

long long linear_workspace(bool quantizes, const Operand& a, const Operand& b) {
  long long bytes = readable(b) ? 0 : copy_bytes(b.rows, b.cols);
  if (quantizes) bytes += copy_bytes(a.rows, a.cols) + align_up(4LL * a.rows, kAlign);
  else if (!readable(a)) bytes += copy_bytes(a.rows, a.cols);
  return bytes;
}

bool valid_shape(int samples, int rows_per_sample, int k, int k2, int n) {
  return samples >= 0 && rows_per_sample >= 0 && k >= 1 && k2 >= 0 && n >= 1 && n <= 0x7fffff00 &&
         static_cast<long long>(k) + k2 <= kMaxSummands &&
         static_cast<long long>(samples) * rows_per_sample <= 0x7fffff00LL;
}

QuantizeArgs quantize_args(const void* x, long long x_stride, const void* x2, long long x2_stride, void* values,
                           long long ld, float* scales, long long rows, int k, int k2) {
  QuantizeArgs q{};
  q.x[0] = static_cast<const uint16_t*>(x);
  q.x[1] = k2 ? static_cast<const uint16_t*>(x2) : nullptr;
  q.stride[0] = rows == 1 ? 0 : x_stride;
  q.stride[1] = rows == 1 || !k2 ? 0 : x2_stride;
  q.width[0] = k;
  q.width[1] = k2;
  q.values = static_cast<int8_t*>(values);
  q.ld = ld;
  q.scales = scales;
  q.rows = static_cast<int>(rows);
  return q;
}

}  // namespace
}  // namespace peco

using namespace peco;

extern "C" int peco_quantize_rows(const void* x, long long x_stride, const void* x2, long long x2_stride, void* values,
                                  long long v_stride, float* scales, long long rows, int k, int k2, int dtype,
                                  void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (rows < 0 || rows > 0x7fffff00LL || k < 1 || k2 < 0 || static_cast<long long>(k) + k2 > 0x7ffffe00LL) return kErrInvalidValue;
  if (rows == 0) return kOk;
  if (!x || !values || !scales || (k2 > 0 && !x2)) return kErrInvalidValue;
  if (rows > 1 && (x_stride < k || (k2 > 0 && x2_stride < k2) || v_stride < static_cast<long long>(k) + k2)) return kErrInvalidValue;
  const QuantizeArgs q = quantize_args(x, x_stride, x2, x2_stride, values, v_stride, scales, rows, k, k2);
  return dtype == 1 ? quantize<__nv_bfloat16>(q, stream) : quantize<__half>(q, stream);
}

extern "C" long long peco_linear_int8_workspace(int from_16_bits, const void* values, long long v_stride,
                                                const void* weight, long long w_stride, int samples, int rows_per_sample,
                                                int k, int k2, int n) {
  if (!valid_shape(samples, rows_per_sample, k, k2, n)) return -1;
  const long long rows = static_cast<long long>(samples) * rows_per_sample;
  return linear_workspace(from_16_bits != 0, bytes_operand(values, v_stride, rows, k + k2),
                          bytes_operand(weight, w_stride, n, k + k2));
}

extern "C" int peco_linear_int8(const void* x, long long x_stride, const void* x2, long long x2_stride,
                                const void* values, long long v_stride, const float* row_scales, const void* weight,
                                long long w_stride, const float* col_scales, const void* bias, const void* gate,
                                long long gate_stride, const void* residual, long long res_stride, void* out,
                                long long out_stride, int samples, int rows_per_sample, int k, int k2, int n,
                                int activation, int dtype, void* workspace, long long workspace_bytes,
                                void* stream_ptr) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (dtype != 0 && dtype != 1) return kErrUnsupported;
  if (!valid_shape(samples, rows_per_sample, k, k2, n) || activation < kActNone || activation > kActSilu) return kErrInvalidValue;
  const long long rows = static_cast<long long>(samples) * rows_per_sample;
  if (rows == 0) return kOk;
  const bool quantizes = values == nullptr;
  const int wide = k + k2;
  if (!weight || !col_scales || !out || w_stride < wide || out_stride < n || gate_stride < 0 || (residual && res_stride < n))
    return kErrInvalidValue;
  if (quantizes ? !x || (k2 > 0 && !x2) || x_stride < k || (k2 > 0 && x2_stride < k2)
                : !row_scales || v_stride < wide || k2 != 0)
    return kErrInvalidValue;
  Operand a = bytes_operand(values, v_stride, rows, wide), b = bytes_operand(weight, w_stride, n, wide);
  const long long need = linear_workspace(quantizes, a, b);
  if (need > 0 && !usable_workspace(workspace, workspace_bytes, need)) return kErrWorkspace;
  Carver ws{static_cast<unsigned char*>(workspace), 0};
  if (quantizes) {
    const long long ld = align_up(wide, 16);
    void* made = ws.take(copy_bytes(rows, wide));
    float* scales = static_cast<float*>(ws.take(4 * rows));
    const QuantizeArgs q = quantize_args(x, x_stride, x2, x2_stride, made, ld, scales, rows, k, k2);
    if (int st = dtype == 1 ? quantize<__nv_bfloat16>(q, stream) : quantize<__half>(q, stream)) return st;
    a.ptr = made;
    a.stride = ld;
    row_scales = scales;
  } else if (int st = make_readable(a, ws, stream)) {
    return st;
  }
  if (int st = make_readable(b, ws, stream)) return st;
  GemmArgs g{};
  g.m = static_cast<int>(rows);
  g.n = n;
  g.out = out;
  g.out_stride = out_stride;
  g.bias = bias;
  g.gate = gate;
  g.gate_stride = gate_stride;
  g.rows_per_sample = rows_per_sample;
  g.row_scale = row_scales;
  g.col_scale = col_scales;
  g.residual = residual;
  g.res_stride = res_stride;
  g.act = activation;
  g.vec = n % 8 == 0 && aligned16(out, out_stride) && aligned16(bias, 8) && aligned16(gate, gate_stride) &&
          aligned16(residual, res_stride);
  return dtype == 1 ? launch_gemm<__nv_bfloat16, false, false, true, true>(g, &a, &b, 1, dtype, stream)
                    : launch_gemm<__half, false, false, true, true>(g, &a, &b, 1, dtype, stream);
}
