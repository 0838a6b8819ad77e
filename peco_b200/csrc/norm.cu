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
// there in fp32, the variance around the mean already known.  The backward
// kernel recomputes r from x and the branch, so nothing has to be saved.
#include "common.cuh"
#include "../../include/peco_b200.h"
#include "internal.h"
#include "rows.cuh"

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
};

// ---- sums over the threads of one row ---------------------------------------
template <int WARPS>
struct RowGroup {
  static constexpr int kThreads = 32 * WARPS;
};

// Sum of K values over the row's threads, on every thread; ``buf`` is K *
// WARPS floats that no other reduction in flight uses.
template <int WARPS, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* buf) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (WARPS > 1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) buf[k * WARPS + warp] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += buf[k * WARPS + w];
      v[k] = s;
    }
  }
}

// One thread's part of a row: chunk i holds VEC neighbouring elements at
// column (i * threads + thread) * VEC; elements past the width read as 0.
template <int VEC, int NCH, int THREADS>
struct Span {
  int thread, width;
  __device__ __forceinline__ int column(int i) const { return (i * THREADS + thread) * VEC; }
  __device__ __forceinline__ bool inside(int i) const { return column(i) < width; }
};

template <typename T, int VEC, int NCH, int THREADS>
__device__ __forceinline__ void load_row(const Span<VEC, NCH, THREADS>& sp, const T* p, float (&v)[NCH][VEC]) {
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (sp.inside(i)) {
      if constexpr (VEC == 1) v[i][0] = to_f32<T>(p[sp.column(i)]);
      else load_aligned<VEC>(p + sp.column(i), v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void load_chunk(const void* p, long long at, float (&v)[VEC]) {
  if constexpr (VEC == 1) v[0] = to_f32<T>(static_cast<const T*>(p)[at]);
  else load_aligned<VEC>(static_cast<const T*>(p) + at, v);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(void* p, long long at, const float (&v)[VEC]) {
  if constexpr (VEC == 1) static_cast<T*>(p)[at] = from_f32<T>(v[0]);
  else store_aligned<VEC>(static_cast<T*>(p) + at, v);
}

// (mean, rstd) of a row held in registers
template <int WARPS, int VEC, int NCH, int THREADS>
__device__ __forceinline__ void row_stats(const Span<VEC, NCH, THREADS>& sp, const float (&v)[NCH][VEC], int kind,
                                          float eps, float& mean, float& rstd, float* buf) {
  const float inv = 1.0f / static_cast<float>(sp.width);
  mean = 0.0f;
  if (kind == kNormLayer) {
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] += v[i][e];
    row_sum<WARPS>(s, buf);
    mean = s[0] * inv;
  }
  float q[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (sp.inside(i)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) q[0] = fmaf(v[i][e] - mean, v[i][e] - mean, q[0]);
    }
  }
  row_sum<WARPS>(q, buf + WARPS);
  rstd = rsqrtf(q[0] * inv + eps);
}

// ---- forward --------------------------------------------------------------------
// WARPS warps per row; a block of at least four warps holds 4 / WARPS rows
// when a row needs fewer.
template <typename T, int VEC, int WARPS, int NCH, bool POST>
__global__ void __launch_bounds__(WARPS < 4 ? 128 : 32 * WARPS) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  static_assert(WARPS == 1 || WARPS >= 4, "rows of two warps would share block barriers");
  constexpr int kThreads = 32 * WARPS;
  constexpr int kRows = WARPS < 4 ? 4 / WARPS : 1;
  __shared__ float buf[4 * (WARPS < 4 ? 1 : WARPS)];
  const int slot = threadIdx.x / kThreads;
  const long long row = static_cast<long long>(blockIdx.x) * kRows + slot;
  if (row >= static_cast<long long>(a.samples) * a.rows) return;  // whole warps only: kRows > 1 means one warp per row
  const int sample = static_cast<int>(row / a.rows);
  const long long at = row - static_cast<long long>(sample) * a.rows;
  const Span<VEC, NCH, kThreads> sp{static_cast<int>(threadIdx.x) - slot * kThreads, a.width};
  float r[NCH][VEC];
  load_row(sp, static_cast<const T*>(a.x.p) + sample * a.x.sb + at * a.x.sn, r);
  if (a.branch.p) {
    float b[NCH][VEC];
    load_row(sp, static_cast<const T*>(a.branch.p) + sample * a.branch.sb + at * a.branch.sn, b);
    if constexpr (POST) {
      float mean, rstd;
      row_stats<WARPS>(sp, b, a.post, a.post_eps, mean, rstd, buf + 2 * WARPS);
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (!sp.inside(i)) continue;
        float w[VEC];
        if (a.post_weight) load_chunk<T>(a.post_weight, sp.column(i), w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          b[i][e] = (b[i][e] - mean) * rstd;
          if (a.post_weight) b[i][e] *= w[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!sp.inside(i)) continue;
      float g[VEC];
      if (a.gate.p) load_chunk<T>(a.gate.p, sample * a.gate.sb + sp.column(i), g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float gb = a.gate.p ? g[e] * b[i][e] : b[i][e];
        r[i][e] = fmaf(a.residual_scale, r[i][e], gb);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[i][e] *= a.residual_scale;
  }
  const long long out = row * a.width;
  if (a.out_r) {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (sp.inside(i)) store_chunk<T>(a.out_r, out + sp.column(i), r[i]);
  }
  float mean, rstd;
  row_stats<WARPS>(sp, r, a.norm, a.eps, mean, rstd, buf);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (!sp.inside(i)) continue;
    float w[VEC], s[VEC], t[VEC];
    if (a.weight) load_chunk<T>(a.weight, sp.column(i), w);
    if (a.scale.p) load_chunk<T>(a.scale.p, sample * a.scale.sb + sp.column(i), s);
    if (a.shift.p) load_chunk<T>(a.shift.p, sample * a.shift.sb + sp.column(i), t);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float y = (r[i][e] - mean) * rstd;
      if (a.weight) y *= w[e];
      if (a.scale.p) y *= 1.0f + s[e];
      if (a.shift.p) y += t[e];
      r[i][e] = y;
    }
    store_chunk<T>(a.out_h, out + sp.column(i), r[i]);
  }
}

// ---- backward ---------------------------------------------------------------------
// A block takes every chunks-th row of one sample and keeps its threads'
// column sums in registers; a second kernel adds the blocks' sums in order.
template <typename T, int VEC, int WARPS, int NCH, bool POST>
__global__ void __launch_bounds__(32 * WARPS) norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kThreads = 32 * WARPS;
  __shared__ float buf[2][8 * WARPS];  // double-buffered between rows: one row's last read may meet the next one's write
  const int sample = blockIdx.x / a.chunks, chunk = blockIdx.x - sample * a.chunks;
  const Span<VEC, NCH, kThreads> sp{static_cast<int>(threadIdx.x), a.width};
  const float inv = 1.0f / static_cast<float>(a.width);
  float a0[NCH][VEC], a1[NCH][VEC], g0[NCH][VEC];
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) a0[i][e] = a1[i][e] = g0[i][e] = 0.0f;
  int turn = 0;
  for (int at = chunk; at < a.rows; at += a.chunks, turn ^= 1) {
    float* bf = buf[turn];
    const long long out = (static_cast<long long>(sample) * a.rows + at) * a.width;
    float r[NCH][VEC], d[NCH][VEC], b[NCH][VEC];
    load_row(sp, static_cast<const T*>(a.x.p) + sample * a.x.sb + at * a.x.sn, r);
    load_row(sp, static_cast<const T*>(a.grad_h.p) + sample * a.grad_h.sb + at * a.grad_h.sn, d);
    float pmean = 0.0f, prstd = 1.0f;
    if (a.branch.p) {
      load_row(sp, static_cast<const T*>(a.branch.p) + sample * a.branch.sb + at * a.branch.sn, b);
      if constexpr (POST) {
        row_stats<WARPS>(sp, b, a.post, a.post_eps, pmean, prstd, bf);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) b[i][e] = sp.inside(i) ? (b[i][e] - pmean) * prstd : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!sp.inside(i)) continue;
      float g[VEC], w[VEC];
      if (a.gate.p) load_chunk<T>(a.gate.p, sample * a.gate.sb + sp.column(i), g);
      if (POST && a.post_weight) load_chunk<T>(a.post_weight, sp.column(i), w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float gb = 0.0f;
        if (a.branch.p) {
          gb = b[i][e];
          if (POST && a.post_weight) gb *= w[e];
          if (a.gate.p) gb *= g[e];
        }
        r[i][e] = fmaf(a.residual_scale, r[i][e], gb);
      }
    }
    float mean, rstd;
    row_stats<WARPS>(sp, r, a.norm, a.eps, mean, rstd, bf + 2 * WARPS);
    // r -> n, d -> dn, and the two means of the norm's gradient
    float m[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!sp.inside(i)) continue;
      float w[VEC], s[VEC];
      if (a.weight) load_chunk<T>(a.weight, sp.column(i), w);
      if (a.scale.p) load_chunk<T>(a.scale.p, sample * a.scale.sb + sp.column(i), s);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float n = (r[i][e] - mean) * rstd;
        float dn = d[i][e];
        a0[i][e] += dn;
        a1[i][e] = fmaf(dn, n, a1[i][e]);
        if (a.scale.p) dn *= 1.0f + s[e];
        if (a.weight) dn *= w[e];
        m[0] += dn;
        m[1] = fmaf(dn, n, m[1]);
        r[i][e] = n;
        d[i][e] = dn;
      }
    }
    row_sum<WARPS>(m, bf + 4 * WARPS);
    const float mean_dn = a.norm == kNormLayer ? m[0] * inv : 0.0f, mean_dnn = m[1] * inv;
    float pm[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!sp.inside(i)) continue;
      float e4[VEC], g[VEC], w[VEC];
      if (a.grad_r.p) load_chunk<T>(a.grad_r.p, sample * a.grad_r.sb + at * a.grad_r.sn + sp.column(i), e4);
      if (a.gate.p) load_chunk<T>(a.gate.p, sample * a.gate.sb + sp.column(i), g);
      if (POST && a.post_weight) load_chunk<T>(a.post_weight, sp.column(i), w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float dr = rstd * (d[i][e] - mean_dn - r[i][e] * mean_dnn);
        if (a.grad_r.p) dr += e4[e];
        r[i][e] = a.residual_scale * dr;
        if (a.branch.p) {
          g0[i][e] = fmaf(dr, b[i][e], g0[i][e]);
          float db = a.gate.p ? dr * g[e] : dr;
          if (POST && a.post_weight) db *= w[e];
          d[i][e] = db;
          if (POST) {
            pm[0] += db;
            pm[1] = fmaf(db, b[i][e], pm[1]);
          }
        }
      }
      if (a.out_h) store_chunk<T>(a.out_h, out + sp.column(i), r[i]);
      if (!POST && a.out_r) store_chunk<T>(a.out_r, out + sp.column(i), d[i]);
    }
    if constexpr (POST) {
      row_sum<WARPS>(pm, bf + 6 * WARPS);
      const float pmean_d = a.post == kNormLayer ? pm[0] * inv : 0.0f, pmean_dn = pm[1] * inv;
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        if (!sp.inside(i)) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[i][e] = prstd * (d[i][e] - pmean_d - b[i][e] * pmean_dn);
        if (a.out_r) store_chunk<T>(a.out_r, out + sp.column(i), d[i]);
      }
    }
  }
  if (a.partial) {
    float* part = a.partial + static_cast<long long>(blockIdx.x) * 3 * a.width;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (!sp.inside(i)) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int c = sp.column(i) + e;
        part[c] = a0[i][e];
        part[a.width + c] = a1[i][e];
        part[2LL * a.width + c] = g0[i][e];
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

// Column sums of the blocks' partials: 32 columns x 16 lanes of chunks per
// block, lanes added in order, samples one after the other.
template <typename T>
__global__ void __launch_bounds__(512) norm_sums_kernel(const __grid_constant__ NormSumsArgs a) {
  __shared__ float red[3][16][33];
  const int cx = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  float dweight = 0.0f, dpost = 0.0f, dgate = 0.0f, dscale = 0.0f, dshift = 0.0f;
  for (int b = 0; b < a.samples; ++b) {
    float s[3] = {0.0f, 0.0f, 0.0f};
    if (c < a.width) {
#pragma unroll 4
      for (int i = y; i < a.chunks; i += 16) {
        const float* p = a.partial + (static_cast<long long>(b) * a.chunks + i) * 3 * a.width + c;
        s[0] += p[0];
        s[1] += p[a.width];
        s[2] += p[2LL * a.width];
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) red[k][y][cx] = s[k];
    __syncthreads();
    if (y == 0 && c < a.width) {
      float t[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 3; ++k)
        for (int i = 0; i < 16; ++i) t[k] += red[k][i][cx];
      const float gate = a.gate.p ? to_f32<T>(static_cast<const T*>(a.gate.p)[b * a.gate.sb + c]) : 1.0f;
      const float scale = a.scale.p ? to_f32<T>(static_cast<const T*>(a.scale.p)[b * a.scale.sb + c]) : 0.0f;
      const float w = a.weight ? to_f32<T>(static_cast<const T*>(a.weight)[c]) : 1.0f;
      const float pw = a.post_weight ? to_f32<T>(static_cast<const T*>(a.post_weight)[c]) : 1.0f;
      const long long at = static_cast<long long>(b) * a.width + c;
      dweight = fmaf(1.0f + scale, t[1], dweight);
      dpost = fmaf(gate, t[2], dpost);
      dshift = a.shift_shared ? dshift + t[0] : t[0];
      dscale = a.scale_shared ? fmaf(w, t[1], dscale) : w * t[1];
      dgate = a.gate_shared ? fmaf(pw, t[2], dgate) : pw * t[2];
      if (a.dshift && !a.shift_shared) static_cast<T*>(a.dshift)[at] = from_f32<T>(dshift);
      if (a.dscale && !a.scale_shared) static_cast<T*>(a.dscale)[at] = from_f32<T>(dscale);
      if (a.dgate && !a.gate_shared) static_cast<T*>(a.dgate)[at] = from_f32<T>(dgate);
    }
    __syncthreads();
  }
  if (y == 0 && c < a.width) {
    if (a.dshift && a.shift_shared) static_cast<T*>(a.dshift)[c] = from_f32<T>(dshift);
    if (a.dscale && a.scale_shared) static_cast<T*>(a.dscale)[c] = from_f32<T>(dscale);
    if (a.dgate && a.gate_shared) static_cast<T*>(a.dgate)[c] = from_f32<T>(dgate);
    if (a.dweight) static_cast<T*>(a.dweight)[c] = from_f32<T>(dweight);
    if (a.dpost) static_cast<T*>(a.dpost)[c] = from_f32<T>(dpost);
  }
}

// ---- host side -----------------------------------------------------------------------
constexpr int kMaxWidth = 16384;

template <typename T, int VEC, int WARPS, int NCH>
int launch_one(const NormArgs& a, bool backward, cudaStream_t stream) {
  const bool post = a.post != kNormNone;
  if (backward) {
    const int grid = a.samples * a.chunks;
    if (post) norm_backward_kernel<T, VEC, WARPS, NCH, true><<<grid, 32 * WARPS, 0, stream>>>(a);
    else norm_backward_kernel<T, VEC, WARPS, NCH, false><<<grid, 32 * WARPS, 0, stream>>>(a);
  } else {
    constexpr int kRows = WARPS < 4 ? 4 / WARPS : 1;
    const long long rows = static_cast<long long>(a.samples) * a.rows;
    const unsigned grid = static_cast<unsigned>((rows + kRows - 1) / kRows);
    if (post) norm_forward_kernel<T, VEC, WARPS, NCH, true><<<grid, WARPS < 4 ? 128 : 32 * WARPS, 0, stream>>>(a);
    else norm_forward_kernel<T, VEC, WARPS, NCH, false><<<grid, WARPS < 4 ? 128 : 32 * WARPS, 0, stream>>>(a);
  }
  return launch_status();
}

template <typename T>
int launch_norm(const NormArgs& a, bool backward, cudaStream_t stream) {
  const int w = a.width;
  if (a.vec) {
    if (w <= 512) return launch_one<T, 8, 1, 2>(a, backward, stream);
    if (w <= 1024) return launch_one<T, 8, 4, 1>(a, backward, stream);
    if (w <= 2048) return launch_one<T, 8, 4, 2>(a, backward, stream);
    if (w <= 3072) return launch_one<T, 8, 4, 3>(a, backward, stream);
    if (w <= 6144) return launch_one<T, 8, 8, 3>(a, backward, stream);
    return launch_one<T, 8, 16, 4>(a, backward, stream);
  }
  if (w <= 1024) return launch_one<T, 1, 4, 8>(a, backward, stream);
  if (w <= 4096) return launch_one<T, 1, 8, 16>(a, backward, stream);
  return launch_one<T, 1, 16, 32>(a, backward, stream);
}

// Row chunks per sample of the backward kernel: about two blocks per SM
// (their partial sums are a small part of the traffic), fewer for short samples.
int norm_chunks(int samples, int rows) {
  if (samples < 1) return 1;
  long long chunks = (2LL * kNumSMs + samples - 1) / samples;
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
  return dtype == 1 ? launch_norm<__nv_bfloat16>(a, false, stream) : launch_norm<__half>(a, false, stream);
}

extern "C" long long peco_gated_norm_backward_workspace(int samples, int rows, int width) {
  if (samples < 0 || rows < 0 || width < 1) return -1;
  return 12LL * samples * norm_chunks(samples, rows) * width;
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
  if (sums && (!workspace || workspace_bytes < peco_gated_norm_backward_workspace(samples, rows, width)))
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
  a.chunks = norm_chunks(samples, rows);
  int st = dtype == 1 ? launch_norm<__nv_bfloat16>(a, true, stream) : launch_norm<__half>(a, true, stream);
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
  const int grid = (width + 31) / 32;
  if (dtype == 1) norm_sums_kernel<__nv_bfloat16><<<grid, 512, 0, stream>>>(s);
  else norm_sums_kernel<__half><<<grid, 512, 0, stream>>>(s);
  return launch_status();
}
