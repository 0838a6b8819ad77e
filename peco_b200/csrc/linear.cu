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
#include "product.cuh"
#include "rows.cuh"

namespace peco {
namespace {

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
