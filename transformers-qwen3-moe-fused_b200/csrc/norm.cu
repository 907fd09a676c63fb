// The residual stream around a block: s = residual + scale * block output, n = s / rms(s) * gamma, and the gradients.
//
//   s[t] = residual[t] + scale * sum_j weights[t, j] y[inv[t k + j]]      (without inv: s[t] = residual[t] + scale * y[t])
//   n[t] = s[t] * r[t] * gamma,   r[t] = 1 / sqrt(mean(s[t]^2) + eps)
// and, with a = dn gamma and u = s r,
//   ds = dsum + r (a - u mean(a u)),  dresidual = ds,  dgamma = sum_t dn u,
//   dy[inv] = scale * weights * ds,   dweights[t, j] = scale <ds[t], y[inv[t k + j]]>.
//
// Everything between loads and stores is fp32; s and n are each rounded once (n from the sum that has not been rounded).
// The backward pass forms s again from the residual and y, in the order of the forward pass and with its bits: s as it was stored
// is off by its rounding (2.4e-3 in place of 1.7e-3 of a gradient's 2-norm in bf16), or infinite where the sum is past fp16's range
// and n is not.  With k expert rows, which the gradient of the weights reads anyway, no more bytes are moved (residual in place of
// s): 145 us for 139 at 8191 x 2048, k = 8; with one row (add) another T H values are: 78 for 70 at 16001 x 2048.  A caller that
// kept s alone can give that.
//
// Bound by HBM.  A CTA owns a token: its k rows (k H values) are in flight at once, the row stays in registers between the
// sum and the norm, and a decoding step of one token takes one trip to memory instead of k.  dgamma is a sum over all
// tokens: CTAs of the backward pass walk tokens with a fixed stride, keep their columns' sums in registers, write one row
// of partial sums each, and a second launch adds the rows in order, so the result is the same in every run.
#include "vec.cuh"

namespace moe {
namespace {

constexpr int NORM_THREADS = 256;    // most threads of a CTA
constexpr int NORM_MAX_VPT = 4;      // vectors of 16 bytes that a thread keeps of a row
constexpr int NORM_MAX_H = 24576;    // the generic form keeps two fp32 rows in shared memory, or three up to
constexpr int NORM_THREE_ROWS_H = 19200;
constexpr int NORM_BWD_CTAS_PER_SM = 5;  // at most; the rows of partial sums are laid out for that many

struct NormFwd {
  const void* y;
  const int32_t* inv;
  const void* weights;
  const void* residual;
  const void* gamma;
  float scale, eps;
  void* sum;
  void* normed;
  float* rstd;
  int64_t tokens;
  int k, H;
};

struct NormBwd {
  const void* dnormed;
  const void* dsum;
  const void* base;  // the residual (may be null), or s as it was stored
  bool stored;       // base is s
  const float* rstd;
  const void* gamma;
  const void* y;
  const int32_t* inv;
  const void* weights;
  float scale;
  void* dresidual;
  void* dy;
  void* dweights;
  float* partial;  // dgamma: one row of H sums for each CTA
  int64_t tokens;
  int k, H;
  bool u_row;      // the generic form has room for a third fp32 row
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sum over the CTA, the same value in every thread.  `buf` holds one float for each warp and is not reused before another
// __syncthreads has passed (callers alternate between two).
__device__ __forceinline__ float cta_sum(float v, float* buf) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += buf[w];
  return t;
}

// p[0..7] summed over the warp; lane l returns the sum of p[l & 7].
__device__ __forceinline__ float warp_sum8(float (&p)[8], int lane) {
  // halve the number of values a lane carries in each of three steps, then add up the four lanes that hold the same one
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) {
    const bool up = (lane & d) != 0;
#pragma unroll
    for (int i = 0; i < d; ++i) {
      const float send = up ? p[i] : p[i + d];
      const float keep = up ? p[i + d] : p[i];
      p[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
    }
  }
  float v = p[0];
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

template <typename T>
__device__ __forceinline__ void add_scaled(float (&acc)[Vec<T>::N], float w, const Vec<T>& v) {
#pragma unroll
  for (int i = 0; i < Vec<T>::N; ++i) acc[i] = fmaf(w, to_f32(v.v[i]), acc[i]);
}

// ---------------------------------------------------------------------------------------
// forward: rows of whole 16-byte vectors, VPT of them in each thread
// ---------------------------------------------------------------------------------------
template <typename T, int VPT, int KFIX>
__global__ void __launch_bounds__(NORM_THREADS)
norm_fwd_kernel(const NormFwd p) {
  constexpr int V = Vec<T>::N;
  __shared__ float red[NORM_THREADS / 32];
  const int hv = p.H / V;
  const int64_t t = blockIdx.x;
  const T* y = (const T*)p.y;
  const int k = KFIX > 0 ? KFIX : p.k;
  float s[VPT][V];
  int32_t src[KFIX > 0 ? KFIX : 1];
  float wj[KFIX > 0 ? KFIX : 1];
  if constexpr (KFIX > 0) {
#pragma unroll
    for (int j = 0; j < KFIX; ++j) {
      src[j] = p.inv[t * KFIX + j];
      wj[j] = to_f32(((const T*)p.weights)[t * KFIX + j]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c >= hv) continue;
    Vec<T> r;
    if (p.residual) r = load_vec((const T*)p.residual + t * p.H + c * V);
#pragma unroll
    for (int q = 0; q < V; ++q) s[i][q] = 0.f;
    if constexpr (KFIX > 0) {
      Vec<T> v[KFIX];
#pragma unroll
      for (int j = 0; j < KFIX; ++j) *reinterpret_cast<uint4*>(v[j].v) = __ldcs(reinterpret_cast<const uint4*>(y + (int64_t)src[j] * p.H) + c);
#pragma unroll
      for (int j = 0; j < KFIX; ++j) add_scaled<T>(s[i], wj[j], v[j]);
    } else if (p.inv) {
#pragma unroll 4
      for (int j = 0; j < k; ++j)
        add_scaled<T>(s[i], to_f32(((const T*)p.weights)[t * k + j]), load_vec(y + (int64_t)p.inv[t * k + j] * p.H + c * V));
    } else {
      add_scaled<T>(s[i], 1.f, load_vec(y + t * p.H + c * V));
    }
#pragma unroll
    for (int q = 0; q < V; ++q) {
      s[i][q] = p.residual ? fmaf(p.scale, s[i][q], to_f32(r.v[q])) : p.scale * s[i][q];
      ss = fmaf(s[i][q], s[i][q], ss);
    }
    if (p.sum) {
      Vec<T> o;
#pragma unroll
      for (int q = 0; q < V; ++q) o.v[q] = from_f32<T>(s[i][q]);
      store_vec((T*)p.sum + t * p.H + c * V, o);
    }
  }
  if (!p.normed) return;
  const float rstd = rsqrtf(cta_sum(ss, red) / (float)p.H + p.eps);
  if (p.rstd && threadIdx.x == 0) p.rstd[t] = rstd;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c >= hv) continue;
    const Vec<T> g = load_vec((const T*)p.gamma + c * V);
    Vec<T> o;
#pragma unroll
    for (int q = 0; q < V; ++q) o.v[q] = from_f32<T>(s[i][q] * rstd * to_f32(g.v[q]));
    store_vec((T*)p.normed + t * p.H + c * V, o);
  }
}

// Any extent and alignment: the row waits in shared memory for its norm.
template <typename T>
__global__ void __launch_bounds__(NORM_THREADS)
norm_fwd_generic_kernel(const NormFwd p) {
  extern __shared__ float row[];
  __shared__ float red[NORM_THREADS / 32];
  const int64_t t = blockIdx.x;
  const T* y = (const T*)p.y;
  float ss = 0.f;
  for (int c = threadIdx.x; c < p.H; c += NORM_THREADS) {
    float s = 0.f;
    if (p.inv) {
#pragma unroll 4
      for (int j = 0; j < p.k; ++j)
        s = fmaf(to_f32(((const T*)p.weights)[t * p.k + j]), to_f32(y[(int64_t)p.inv[t * p.k + j] * p.H + c]), s);
    } else {
      s = to_f32(y[t * p.H + c]);
    }
    s = p.residual ? fmaf(p.scale, s, to_f32(((const T*)p.residual)[t * p.H + c])) : p.scale * s;
    ss = fmaf(s, s, ss);
    row[c] = s;
    if (p.sum) ((T*)p.sum)[t * p.H + c] = from_f32<T>(s);
  }
  if (!p.normed) return;
  const float rstd = rsqrtf(cta_sum(ss, red) / (float)p.H + p.eps);
  if (p.rstd && threadIdx.x == 0) p.rstd[t] = rstd;
  for (int c = threadIdx.x; c < p.H; c += NORM_THREADS)  // (every thread reads back what it wrote)
    ((T*)p.normed)[t * p.H + c] = from_f32<T>(row[c] * rstd * to_f32(((const T*)p.gamma)[c]));
}

// ---------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------
enum NormBwdForm { BWD_ADD = 0, BWD_COMBINE = 1, BWD_COMBINE8 = 2 };  // no expert rows; any k; k = 8 with one vector in each thread

// CTAs that fit on an SM with the registers their form needs.  BWD_COMBINE8 loads the expert rows together with the gradients,
// ahead of the first sum over the CTA (k = 8, H = 2048, 8191 tokens: 180 us with the rows behind that sum and two CTAs to an SM).
template <int VPT, int FORM>
constexpr int norm_bwd_ctas() { return FORM == BWD_ADD ? (VPT == 1 ? 5 : VPT == 2 ? 3 : 1) : FORM == BWD_COMBINE8 ? 3 : (VPT == 1 ? 2 : 1); }

template <typename T, int VPT, int FORM>
__global__ void __launch_bounds__(NORM_THREADS, norm_bwd_ctas<VPT, FORM>())
norm_bwd_kernel(const NormBwd p) {
  static_assert(FORM != BWD_COMBINE8 || VPT == 1, "the loaded rows stay in registers");
  constexpr int V = Vec<T>::N;
  __shared__ float red[2][NORM_THREADS / 32];
  __shared__ float dots[2][NORM_THREADS / 32][8];
  const int hv = p.H / V;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const T* y = (const T*)p.y;
  float dg[VPT][V];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int q = 0; q < V; ++q) dg[i][q] = 0.f;
  int flip = 0, dflip = 0;
  const bool again = p.dnormed && !p.stored;  // s is formed again
  // dweights of rows j0.. of token t from this thread's products with them
  auto store_dots = [&](float (&dot)[8], int64_t t, int j0, int nj) {
    const float v = warp_sum8(dot, lane);
    if (lane < 8) dots[dflip][warp][lane] = v;
    __syncthreads();
    if ((int)threadIdx.x < nj) {
      float sum = 0.f;
      for (int w = 0; w < warps; ++w) sum += dots[dflip][w][threadIdx.x];
      ((T*)p.dweights)[t * p.k + j0 + threadIdx.x] = from_f32<T>(p.scale * sum);
    }
    dflip ^= 1;  // written again two rounds on, behind the __syncthreads of the round between
  };
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    float ds[VPT][V];  // first a, then the gradient of the sum
    float u[VPT][V];
    Vec<T> d0[VPT];
    Vec<T> rows[FORM == BWD_COMBINE8 ? 8 : 1];
    int32_t idx[FORM == BWD_COMBINE8 ? 8 : 1];
    if constexpr (FORM == BWD_COMBINE8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) idx[j] = p.inv[t * 8 + j];
      if ((p.dweights || again) && (int)threadIdx.x < hv) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(rows[j].v) = __ldcs(reinterpret_cast<const uint4*>(y + (int64_t)idx[j] * p.H) + threadIdx.x);
      }
    }
    const float rstd = p.dnormed ? p.rstd[t] : 0.f;
    float au = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c >= hv) continue;
      if (p.dsum) *reinterpret_cast<uint4*>(d0[i].v) = __ldcs(reinterpret_cast<const uint4*>((const T*)p.dsum + t * p.H) + c);
      if (!p.dnormed) continue;
      Vec<T> dn;
      *reinterpret_cast<uint4*>(dn.v) = __ldcs(reinterpret_cast<const uint4*>((const T*)p.dnormed + t * p.H) + c);
      Vec<T> b, x;
      if (p.base) *reinterpret_cast<uint4*>(b.v) = __ldcs(reinterpret_cast<const uint4*>((const T*)p.base + t * p.H) + c);
      if (FORM == BWD_ADD && again) *reinterpret_cast<uint4*>(x.v) = __ldcs(reinterpret_cast<const uint4*>(y + t * p.H) + c);
      if (!again) {
#pragma unroll
        for (int q = 0; q < V; ++q) u[i][q] = to_f32(b.v[q]);
      } else {
#pragma unroll
        for (int q = 0; q < V; ++q) u[i][q] = 0.f;
        if constexpr (FORM == BWD_ADD) {
          add_scaled<T>(u[i], 1.f, x);
        } else if constexpr (FORM == BWD_COMBINE8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) add_scaled<T>(u[i], to_f32(((const T*)p.weights)[t * 8 + j]), rows[j]);
        } else {
#pragma unroll 4
          for (int j = 0; j < p.k; ++j)
            add_scaled<T>(u[i], to_f32(((const T*)p.weights)[t * p.k + j]), load_vec(y + (int64_t)p.inv[t * p.k + j] * p.H + c * V));
        }
#pragma unroll
        for (int q = 0; q < V; ++q) u[i][q] = p.base ? fmaf(p.scale, u[i][q], to_f32(b.v[q])) : p.scale * u[i][q];
      }
      const Vec<T> g = load_vec((const T*)p.gamma + c * V);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const float d = to_f32(dn.v[q]);
        u[i][q] *= rstd;
        dg[i][q] = fmaf(d, u[i][q], dg[i][q]);
        ds[i][q] = d * to_f32(g.v[q]);
        au = fmaf(ds[i][q], u[i][q], au);
      }
    }
    if (p.dnormed) {
      au = cta_sum(au, red[flip]) / (float)p.H;
      flip ^= 1;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c >= hv) continue;
      Vec<T> o, ox;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        float v = p.dsum ? to_f32(d0[i].v[q]) : 0.f;
        if (p.dnormed) v = fmaf(rstd, ds[i][q] - u[i][q] * au, v);
        ds[i][q] = v;
        o.v[q] = from_f32<T>(v);
        ox.v[q] = from_f32<T>(p.scale * v);
      }
      if (p.dresidual) __stcs(reinterpret_cast<uint4*>((T*)p.dresidual + t * p.H) + c, *reinterpret_cast<const uint4*>(o.v));
      if (FORM == BWD_ADD && p.dy) __stcs(reinterpret_cast<uint4*>((T*)p.dy + t * p.H) + c, *reinterpret_cast<const uint4*>(ox.v));
    }
    if constexpr (FORM == BWD_COMBINE8) {
      if (!p.dy && !p.dweights) continue;
      float dot[8];
      const bool mine = (int)threadIdx.x < hv;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dot[j] = 0.f;
        if (!mine) continue;
        if (p.dweights) {
#pragma unroll
          for (int q = 0; q < V; ++q) dot[j] = fmaf(ds[0][q], to_f32(rows[j].v[q]), dot[j]);
        }
        if (p.dy) {
          const float w = p.scale * to_f32(((const T*)p.weights)[t * 8 + j]);
          Vec<T> o;
#pragma unroll
          for (int q = 0; q < V; ++q) o.v[q] = from_f32<T>(w * ds[0][q]);
          __stcs(reinterpret_cast<uint4*>((T*)p.dy + (int64_t)idx[j] * p.H) + threadIdx.x, *reinterpret_cast<const uint4*>(o.v));
        }
      }
      if (p.dweights) store_dots(dot, t, 0, 8);
    } else if constexpr (FORM == BWD_COMBINE) {
      if (!p.dy && !p.dweights) continue;
      for (int j0 = 0; j0 < p.k; j0 += 8) {
        const int nj = min(8, p.k - j0);
        float dot[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) dot[j] = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int c = threadIdx.x + i * blockDim.x;
          if (c >= hv) continue;
          Vec<T> v[8];
          int32_t r[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            r[j] = j < nj ? p.inv[t * p.k + j0 + j] : 0;
            if (j < nj && p.dweights) *reinterpret_cast<uint4*>(v[j].v) = __ldcs(reinterpret_cast<const uint4*>(y + (int64_t)r[j] * p.H) + c);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j >= nj) continue;
            const float w = p.dy ? p.scale * to_f32(((const T*)p.weights)[t * p.k + j0 + j]) : 0.f;
            Vec<T> o;
#pragma unroll
            for (int q = 0; q < V; ++q) {
              if (p.dweights) dot[j] = fmaf(ds[i][q], to_f32(v[j].v[q]), dot[j]);
              o.v[q] = from_f32<T>(w * ds[i][q]);
            }
            if (p.dy) __stcs(reinterpret_cast<uint4*>((T*)p.dy + (int64_t)r[j] * p.H) + c, *reinterpret_cast<const uint4*>(o.v));
          }
        }
        if (p.dweights) store_dots(dot, t, j0, nj);
      }
    }
  }
  if (p.partial) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c >= hv) continue;
#pragma unroll
      for (int q = 0; q < V; q += 4)
        *reinterpret_cast<float4*>(p.partial + (int64_t)blockIdx.x * p.H + c * V + q) =
            make_float4(dg[i][q], dg[i][q + 1], dg[i][q + 2], dg[i][q + 3]);
    }
  }
}

// (The form of the sum as a parameter: with tests of it between the loads of a column, add took 102 us
// at 8191 x 1001, for 72.)
enum NormBwdSum { SUM_STORED, SUM_ADD, SUM_COMBINE };
template <typename T, int SUM>
__global__ void __launch_bounds__(NORM_THREADS)
norm_bwd_generic_kernel(const NormBwd p) {
  extern __shared__ float rows[];
  float* ds = rows;
  float* dg = rows + p.H;
  float* us = p.u_row ? rows + 2 * p.H : nullptr;  // (the longest rows: formed twice)
  __shared__ float red[2][NORM_THREADS / 32];
  const T* y = (const T*)p.y;
  auto sum_at = [&](int64_t t, int c) {
    const float b = p.base ? to_f32(((const T*)p.base)[t * p.H + c]) : 0.f;
    if constexpr (SUM == SUM_STORED) return b;
    float s = 0.f;
    if constexpr (SUM == SUM_COMBINE) {
#pragma unroll 4
      for (int j = 0; j < p.k; ++j)
        s = fmaf(to_f32(((const T*)p.weights)[t * p.k + j]), to_f32(y[(int64_t)p.inv[t * p.k + j] * p.H + c]), s);
    } else {
      s = to_f32(y[t * p.H + c]);
    }
    return p.base ? fmaf(p.scale, s, b) : p.scale * s;
  };
  // (a thread reads and writes its own columns of the rows only)
  for (int c = threadIdx.x; c < p.H; c += NORM_THREADS) dg[c] = 0.f;
  int flip = 0;
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const float rstd = p.dnormed ? p.rstd[t] : 0.f;
    float au = 0.f;
    if (p.dnormed) {
#pragma unroll 4
      for (int c = threadIdx.x; c < p.H; c += NORM_THREADS) {
        const float d = to_f32(((const T*)p.dnormed)[t * p.H + c]), u = sum_at(t, c) * rstd;
        if (us) us[c] = u;
        const float a = d * to_f32(((const T*)p.gamma)[c]);
        dg[c] = fmaf(d, u, dg[c]);
        ds[c] = a;
        au = fmaf(a, u, au);
      }
      au = cta_sum(au, red[flip]) / (float)p.H;
      flip ^= 1;
    }
    for (int c = threadIdx.x; c < p.H; c += NORM_THREADS) {
      float v = p.dsum ? to_f32(((const T*)p.dsum)[t * p.H + c]) : 0.f;
      if (p.dnormed) v = fmaf(rstd, ds[c] - (us ? us[c] : sum_at(t, c) * rstd) * au, v);
      ds[c] = v;
      if (p.dresidual) ((T*)p.dresidual)[t * p.H + c] = from_f32<T>(v);
      if (!p.inv && p.dy) ((T*)p.dy)[t * p.H + c] = from_f32<T>(p.scale * v);
    }
    if (!p.inv || (!p.dy && !p.dweights)) continue;
    for (int j = 0; j < p.k; ++j) {
      const int64_t r = p.inv[t * p.k + j];
      const float w = p.dy ? p.scale * to_f32(((const T*)p.weights)[t * p.k + j]) : 0.f;
      float dot = 0.f;
      for (int c = threadIdx.x; c < p.H; c += NORM_THREADS) {
        if (p.dweights) dot = fmaf(ds[c], to_f32(y[r * p.H + c]), dot);
        if (p.dy) ((T*)p.dy)[r * p.H + c] = from_f32<T>(w * ds[c]);
      }
      if (p.dweights) {
        dot = cta_sum(dot, red[flip]);
        flip ^= 1;
        if (threadIdx.x == 0) ((T*)p.dweights)[t * p.k + j] = from_f32<T>(p.scale * dot);
      }
    }
  }
  if (p.partial)
    for (int c = threadIdx.x; c < p.H; c += NORM_THREADS) p.partial[(int64_t)blockIdx.x * p.H + c] = dg[c];
}

// dgamma[c] = sum of the CTAs' partial sums, in a fixed order: 32 columns and 32 strided runs of rows for each CTA.
template <typename T>
__global__ void __launch_bounds__(1024)
norm_dgamma_kernel(const float* __restrict__ partial, int rows, int H, T* __restrict__ dgamma) {
  __shared__ float part[32][33];
  const int col = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col;
  float v = 0.f;
  if (c < H) {
#pragma unroll 4
    for (int r = run; r < rows; r += 32) v += partial[(int64_t)r * H + c];
  }
  part[run][col] = v;
  __syncthreads();
  v = warp_sum(part[col][run]);  // warp `run` adds up column `run`
  const int c2 = blockIdx.x * 32 + run;
  if (col == 0 && c2 < H) dgamma[c2] = from_f32<T>(v);
}

// Threads of a CTA and vectors of each thread for a row of hv vectors: whole warps, one vector each as far as that goes.
// (H = 2048 in 16 bits: 256 threads with one vector.)
struct RowShape { int threads, vpt; };
RowShape row_shape(int hv) {
  for (int vpt = 1; vpt <= NORM_MAX_VPT; vpt *= 2)
    if (hv <= NORM_THREADS * vpt) return {((hv + vpt - 1) / vpt + 31) & ~31, vpt};
  return {0, 0};
}

int bwd_grid(int64_t tokens) {
  const int64_t cap = (int64_t)sm_count() * NORM_BWD_CTAS_PER_SM;
  return (int)(tokens < cap ? tokens : cap);
}

template <typename T>
int launch_fwd(const NormFwd& p, bool vec, cudaStream_t stream) {
  const RowShape rs = vec ? row_shape(p.H / Vec<T>::N) : RowShape{0, 0};
  const unsigned grid = (unsigned)p.tokens;
  if (rs.vpt == 1 && p.inv && p.k == 8) norm_fwd_kernel<T, 1, 8><<<grid, rs.threads, 0, stream>>>(p);
  else if (rs.vpt == 2 && p.inv && p.k == 8) norm_fwd_kernel<T, 2, 8><<<grid, rs.threads, 0, stream>>>(p);
  else if (rs.vpt == 1) norm_fwd_kernel<T, 1, 0><<<grid, rs.threads, 0, stream>>>(p);
  else if (rs.vpt == 2) norm_fwd_kernel<T, 2, 0><<<grid, rs.threads, 0, stream>>>(p);
  else if (rs.vpt == 4) norm_fwd_kernel<T, 4, 0><<<grid, rs.threads, 0, stream>>>(p);
  else {
    const int smem = p.H * (int)sizeof(float);
    if (smem > 48 * 1024) {
      const int st = cuda_status(cudaFuncSetAttribute(norm_fwd_generic_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (st != MOE_OK) return st;
    }
    norm_fwd_generic_kernel<T><<<grid, NORM_THREADS, smem, stream>>>(p);
  }
  return launch_status();
}

template <typename T>
int launch_bwd(NormBwd& p, void* dgamma, bool vec, cudaStream_t stream) {
  const RowShape rs = vec ? row_shape(p.H / Vec<T>::N) : RowShape{0, 0};
  int grid = bwd_grid(p.tokens);
  // as many CTAs as are resident at once: each walks several tokens and leaves one row of partial sums
  auto resident = [&](int ctas) { return (int)(p.tokens < (int64_t)sm_count() * ctas ? p.tokens : (int64_t)sm_count() * ctas); };
  if (rs.vpt != 0) {
    const int form = !p.inv ? BWD_ADD : (rs.vpt == 1 && p.k == 8) ? BWD_COMBINE8 : BWD_COMBINE;
#define MOE_NORM_BWD(VPT, FORM)                                       \
  if (rs.vpt == VPT && form == FORM) {                                \
    grid = resident(norm_bwd_ctas<VPT, FORM>());                      \
    norm_bwd_kernel<T, VPT, FORM><<<grid, rs.threads, 0, stream>>>(p); \
  }
    MOE_NORM_BWD(1, BWD_ADD)
    MOE_NORM_BWD(2, BWD_ADD)
    MOE_NORM_BWD(4, BWD_ADD)
    MOE_NORM_BWD(1, BWD_COMBINE8)
    MOE_NORM_BWD(1, BWD_COMBINE)
    MOE_NORM_BWD(2, BWD_COMBINE)
    MOE_NORM_BWD(4, BWD_COMBINE)
#undef MOE_NORM_BWD
  } else {
    p.u_row = !p.stored && p.H <= NORM_THREE_ROWS_H;
    const int smem = (p.u_row ? 3 : 2) * p.H * (int)sizeof(float);
    auto* kernel = p.stored ? norm_bwd_generic_kernel<T, SUM_STORED> : p.inv ? norm_bwd_generic_kernel<T, SUM_COMBINE> : norm_bwd_generic_kernel<T, SUM_ADD>;
    if (smem > 48 * 1024) {
      const int st = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (st != MOE_OK) return st;
    }
    kernel<<<grid, NORM_THREADS, smem, stream>>>(p);
  }
  int st = launch_status();
  if (st != MOE_OK || !p.partial) return st;
  norm_dgamma_kernel<T><<<(p.H + 31) / 32, 1024, 0, stream>>>(p.partial, grid, p.H, (T*)dgamma);
  return launch_status();
}

bool norm_extents_ok(int64_t T, int k, int H, bool combine) {
  combine = combine || T == 0;  // (no tokens: the index may be an address of nothing)
  return T >= 0 && T <= 0x7fffffffLL && H >= 1 && H <= NORM_MAX_H && k >= 1 && (combine || k == 1) && T * k <= 0x7fffffffLL;
}

}  // namespace
}  // namespace moe

using namespace moe;

MOE_API int moe_combine_add_rms_norm(const void* y, const int32_t* inv_sort_idx, const void* weights, const void* residual,
                                     const void* gamma, float scale, float eps, void* sum, void* normed, float* rstd, int64_t T_,
                                     int k, int H, int dtype, void* stream) {
  if (!is_float_dtype(dtype)) return MOE_ERR_DTYPE;
  if (!norm_extents_ok(T_, k, H, inv_sort_idx != nullptr)) return MOE_ERR_SHAPE;
  if (T_ == 0 || (!sum && !normed)) return MOE_OK;
  if (!y || (inv_sort_idx && !weights) || (normed && !gamma)) return MOE_ERR_NULL;
  const NormFwd p{y, inv_sort_idx, weights, residual, gamma, scale, eps, sum, normed, rstd, T_, k, H};
  MOE_DISPATCH_FLOAT(dtype, T, {
    const bool vec = H % Vec<T>::N == 0 && aligned16(y) && aligned16(residual) && aligned16(gamma) && aligned16(sum) && aligned16(normed);
    return launch_fwd<T>(p, vec, (cudaStream_t)stream);
  });
}

MOE_API size_t moe_combine_add_rms_norm_bwd_ws_bytes(int64_t T_, int H) {
  if (T_ <= 0 || H <= 0) return 0;
  return (size_t)bwd_grid(T_) * H * sizeof(float);
}

static int norm_bwd(const void* dnormed, const void* dsum, const void* base, bool stored, const float* rstd, const void* gamma,
                    const void* y, const int32_t* inv_sort_idx, const void* weights, float scale, void* dresidual, void* dy,
                    void* dweights, void* dgamma, int64_t T_, int k, int H, int dtype, void* ws, size_t ws_bytes, void* stream) {
  if (!is_float_dtype(dtype)) return MOE_ERR_DTYPE;
  if (!norm_extents_ok(T_, k, H, inv_sort_idx != nullptr)) return MOE_ERR_SHAPE;
  if (dgamma && (T_ == 0 || !dnormed)) {
    const int st = cuda_status(cudaMemsetAsync(dgamma, 0, (size_t)H * dtype_size(dtype), (cudaStream_t)stream));
    if (st != MOE_OK) return st;
    dgamma = nullptr;
  }
  if (T_ == 0 || (!dresidual && !dy && !dweights && !dgamma)) return MOE_OK;
  if (dnormed && (!rstd || !gamma || (stored ? !base : !y || (inv_sort_idx && !weights)))) return MOE_ERR_NULL;
  if (inv_sort_idx ? (dy && !weights) || (dweights && !y) : dweights != nullptr) return MOE_ERR_NULL;
  if (dgamma && (!ws || ((uintptr_t)ws & 15) || ws_bytes < moe_combine_add_rms_norm_bwd_ws_bytes(T_, H))) return MOE_ERR_WORKSPACE;
  NormBwd p{dnormed, dsum, base, stored, rstd, gamma, y, inv_sort_idx, weights, scale, dresidual, dy, dweights,
            dgamma ? (float*)ws : nullptr, T_, k, H, false};
  MOE_DISPATCH_FLOAT(dtype, T, {
    const bool vec = H % Vec<T>::N == 0 && aligned16(dnormed) && aligned16(dsum) && aligned16(base) && aligned16(gamma) &&
                     aligned16(y) && aligned16(dresidual) && aligned16(dy);
    return launch_bwd<T>(p, dgamma, vec, (cudaStream_t)stream);
  });
}

MOE_API int moe_combine_add_rms_norm_bwd(const void* dnormed, const void* dsum, const void* sum, const float* rstd,
                                         const void* gamma, const void* y, const int32_t* inv_sort_idx, const void* weights,
                                         float scale, void* dresidual, void* dy, void* dweights, void* dgamma, int64_t T_, int k,
                                         int H, int dtype, void* ws, size_t ws_bytes, void* stream) {
  return norm_bwd(dnormed, dsum, sum, true, rstd, gamma, y, inv_sort_idx, weights, scale, dresidual, dy, dweights, dgamma, T_, k, H,
                  dtype, ws, ws_bytes, stream);
}

MOE_API int moe_combine_add_rms_norm_bwd_inputs(const void* dnormed, const void* dsum, const void* residual, const float* rstd,
                                                const void* gamma, const void* y, const int32_t* inv_sort_idx,
                                                const void* weights, float scale, void* dresidual, void* dy, void* dweights,
                                                void* dgamma, int64_t T_, int k, int H, int dtype, void* ws, size_t ws_bytes,
                                                void* stream) {
  return norm_bwd(dnormed, dsum, residual, false, rstd, gamma, y, inv_sort_idx, weights, scale, dresidual, dy, dweights, dgamma, T_,
                  k, H, dtype, ws, ws_bytes, stream);
}
