// Expert products on 8-bit weights: quantisation of activations, the products on CUDA cores for any extents, and the C ABI of
// both these and the tensor-core forms (tc_gemm_fp8.cuh).
//
//   y[t, n] = sum_kb s[kb, t] ws[e, n / 128, kb] * sum_{k in block kb} q[t, k] w[e, n, k]        (which = 0)
//   y[t, n] = sum_kb s[kb, t] ws[e, kb, n / 128] * sum_{k in block kb} q[t, k] w[e, k, n]        (which = 1, the gradient of x)
//
// with q, s from fp8.cuh.  Scales of activations are stored block by block, (ceil(K / 128), M) with rows padded to a
// multiple of 4: the scales that a tile of tokens needs for one block of the contraction are consecutive.
#include "fp8.cuh"
#include "vec.cuh"

namespace moe {

bool tc_fp8_eligible(const void* q, const void* w, const void* q2, const void* w2, const void* out, int64_t M, int N, int K, int E);
int tc_grouped_gemm_fp8(int which, const void* q, const float* s, const void* w, const float* ws, const void* q2, const float* s2,
                        const void* w2, const float* ws2, const void* m_sizes, int ms64, void* out, int64_t M, int N, int K, int E,
                        int dtype_out, int form, cudaStream_t stream);

int tc_gate_up_silu_fp8(const void* q, const float* s, const void* w_gate, const float* ws_gate, const void* w_up,
                        const float* ws_up, const void* m_sizes, int ms64, void* hq, float* hs, void* keep_e, void* keep_g,
                        int64_t M, int I, int K, int E, int dtype, int form, cudaStream_t stream);

namespace {

constexpr int Q_THREADS = 256;

// Half a warp owns 128 values of a row, 8 consecutive ones in each lane (zeros past the row's end): the largest magnitude by
// shuffles, 8 codes stored as one word of 8 bytes.
// `top`: the bits of the lane's largest magnitude.
template <bool VEC>
__device__ __forceinline__ void store_codes(const float (&v)[8], uint32_t top, uint8_t* row, int col, int K, float* scale) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  float inv;
  const float s = fp8_block_scale(top, inv);
  const uint2 codes = make_uint2(fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                                 fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
  if (col < K && (threadIdx.x & 15) == 0) *scale = s;
  if constexpr (VEC) {
    if (col < K) *reinterpret_cast<uint2*>(row + col) = codes;
  } else {
    const uint64_t all = (uint64_t)codes.x | ((uint64_t)codes.y << 32);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < K) row[col + i] = (uint8_t)(all >> (8 * i));
  }
}

// A warp takes UNROLL neighbouring pairs of blocks of a row (blockIdx.x: which of them; a long row has more than the grid's
// second extent could count) and loads all before it works on the first one.
struct RowBlock {
  int64_t row;
  int col, kb;
};
template <int UNROLL, typename Values, typename Load, typename Work>
__device__ __forceinline__ void for_row_blocks(int64_t M, int K, Load load, Work work) {
  const int lane = threadIdx.x & 31;
  const int p0 = blockIdx.x * UNROLL;
  const int64_t step = (int64_t)gridDim.y * (Q_THREADS / 32);
  for (int64_t row = (int64_t)blockIdx.y * (Q_THREADS / 32) + (threadIdx.x >> 5); row < M; row += step) {
    Values v[UNROLL];
    auto at = [&](int u) { return RowBlock{row, (p0 + u) * 2 * FP8_BLOCK + lane * 8, 2 * (p0 + u) + (lane >> 4)}; };
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) load(at(u), v[u]);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if ((p0 + u) * 2 * FP8_BLOCK < K) work(at(u), v[u]);  // (the same for the whole warp)
  }
}

// Eight consecutive values as they are in memory.
template <typename T, bool VEC>
struct alignas(16) Eight {
  T v[8];
  __device__ __forceinline__ void load(const T* row, int col, int K) {
    if constexpr (VEC) {
      constexpr int WORDS = 8 * sizeof(T) / 16;
      uint4* to = reinterpret_cast<uint4*>(v);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) to[i] = col < K ? __ldcs(reinterpret_cast<const uint4*>(row + col) + i) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = col + i < K ? row[col + i] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(v[i]);
  }
  // Bits of the largest magnitude as fp32.  16-bit types: two at a time, as integers (infinity and NaN above all numbers).
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (VEC && sizeof(T) == 2) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
      uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      const uint16_t big = (uint16_t)max(m & 0xffffu, m >> 16);
      T t;
      *reinterpret_cast<uint16_t*>(&t) = big;
      return magnitude_bits(to_f32(t));
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, magnitude_bits(to_f32(v[i])));
      return m;
    }
  }
};

__device__ __forceinline__ uint32_t top_of(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, magnitude_bits(f[i]));
  return m;
}

template <typename T, bool VEC, int UNROLL>
__global__ void __launch_bounds__(Q_THREADS)
quantize_rows_kernel(const T* __restrict__ x, int64_t M, int K, uint8_t* __restrict__ q, float* __restrict__ scale) {
  const int64_t pitch = fp8_scale_pitch(M);
  using Values = Eight<T, VEC>;
  for_row_blocks<UNROLL, Values>(M, K,
    [&](const RowBlock& at, Values& v) { v.load(x + at.row * K, at.col, K); },
    [&](const RowBlock& at, const Values& v) {
      float f[8];
      v.get(f);
      store_codes<VEC>(f, v.top(), q + at.row * K, at.col, K, scale + at.kb * pitch + at.row);
    });
}

// h = silu(e) g of two fp32 products, quantised; e and g are kept in T for a backward pass (keep_e, keep_g, may be null).
template <typename T, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
silu_quantize_kernel(const float* __restrict__ e, const float* __restrict__ g, int64_t M, int I, uint8_t* __restrict__ hq,
                     float* __restrict__ hs, T* __restrict__ keep_e, T* __restrict__ keep_g) {
  const int64_t pitch = fp8_scale_pitch(M);
  struct Values { Eight<float, VEC> e, g; };
  for_row_blocks<1, Values>(M, I,
    [&](const RowBlock& at, Values& v) {
      v.e.load(e + at.row * I, at.col, I);
      v.g.load(g + at.row * I, at.col, I);
    },
    [&](const RowBlock& at, const Values& v) {
      float h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[i] = gated_silu<T>(v.e.v[i], v.g.v[i]);
        if (keep_e && at.col + i < I) {
          keep_e[at.row * I + at.col + i] = from_f32<T>(v.e.v[i]);
          keep_g[at.row * I + at.col + i] = from_f32<T>(v.g.v[i]);
        }
      }
      store_codes<VEC>(h, top_of(h), hq + at.row * I, at.col, I, hs + at.kb * pitch + at.row);
    });
}

// Gradients of e and g from the fp32 gradient of h, quantised.
template <typename T, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
silu_bwd_quantize_kernel(const float* __restrict__ dh, const T* __restrict__ e, const T* __restrict__ g, int64_t M, int I,
                         uint8_t* __restrict__ deq, float* __restrict__ des, uint8_t* __restrict__ dgq, float* __restrict__ dgs) {
  const int64_t pitch = fp8_scale_pitch(M);
  struct Values { Eight<float, VEC> dh; Eight<T, VEC> e, g; };
  for_row_blocks<VEC ? 2 : 1, Values>(M, I,
    [&](const RowBlock& at, Values& v) {
      v.dh.load(dh + at.row * I, at.col, I);
      v.e.load(e + at.row * I, at.col, I);
      v.g.load(g + at.row * I, at.col, I);
    },
    [&](const RowBlock& at, const Values& v) {
      float de[8], dg[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) gated_silu_bwd<T>(v.dh.v[i], to_f32(v.e.v[i]), to_f32(v.g.v[i]), de[i], dg[i]);
      store_codes<VEC>(de, top_of(de), deq + at.row * I, at.col, I, des + at.kb * pitch + at.row);
      store_codes<VEC>(dg, top_of(dg), dgq + at.row * I, at.col, I, dgs + at.kb * pitch + at.row);
    });
}

// ---------------------------------------------------------------------------------------
// products on CUDA cores: any extents.  A CTA owns 64 columns of one expert and walks its rows in tiles of 64.
// ---------------------------------------------------------------------------------------
constexpr int S_TILE = 64, S_K = 16, S_THREADS = 256, S_WORKERS = 8;

// y = q w + q2 w2 (q2 null: one product); both contract K values.
struct Fp8Pairs {
  const uint8_t* q[2];
  const float* s[2];
  const uint8_t* w[2];
  const float* ws[2];
  int n;
};

template <typename T, bool TRANSPOSED>
__global__ void __launch_bounds__(S_THREADS)
simt_gemm_fp8_kernel(const Fp8Pairs ops, const void* m_sizes, int ms64, T* __restrict__ y, int64_t M, int N, int K) {
  __shared__ float xs[S_K][S_TILE + 1], wsm[S_K][S_TILE + 1];
  __shared__ long long first_row[S_THREADS / 32];
  const int e = blockIdx.y, n0 = blockIdx.x * S_TILE;
  long long before = 0;
  for (int i = threadIdx.x; i < e; i += S_THREADS) {
    const int64_t v = load_index(m_sizes, ms64, i);
    before += v < 0 ? 0 : (v > M ? M : v);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
  if ((threadIdx.x & 31) == 0) first_row[threadIdx.x >> 5] = before;
  __syncthreads();
  int64_t row0 = 0;
  for (int i = 0; i < S_THREADS / 32; ++i) row0 += first_row[i];
  int64_t rows = load_index(m_sizes, ms64, e);
  rows = rows < 0 ? 0 : rows;
  row0 = row0 < M ? row0 : M;
  const int64_t row_end = rows < M - row0 ? row0 + rows : M;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int nblocks = (N + FP8_BLOCK - 1) / FP8_BLOCK;
  for (int64_t t0 = row0 + (int64_t)blockIdx.z * S_TILE; t0 < row_end; t0 += (int64_t)S_WORKERS * S_TILE) {
    float acc[4][4] = {};
    for (int i = 0; i < ops.n; ++i) {
      const int kblocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
      const uint8_t* w = ops.w[i] + (int64_t)e * N * K;
      for (int kb = 0; kb < kblocks; ++kb) {
        float part[4][4] = {};
        const int kend = min(K, (kb + 1) * FP8_BLOCK);
        for (int k0 = kb * FP8_BLOCK; k0 < kend; k0 += S_K) {
          for (int j = threadIdx.x; j < S_K * S_TILE; j += S_THREADS) {
            const int kk = j % S_K, r = j / S_K;
            const int64_t t = t0 + r;
            xs[kk][r] = (t < row_end && k0 + kk < kend) ? fp8_value(ops.q[i][t * K + k0 + kk]) : 0.f;
            if constexpr (!TRANSPOSED) {
              const int n = n0 + r;
              wsm[kk][r] = (n < N && k0 + kk < kend) ? fp8_value(w[(int64_t)n * K + k0 + kk]) : 0.f;
            } else {
              const int rr = j % S_TILE, k2 = j / S_TILE, n = n0 + rr;
              wsm[k2][rr] = (n < N && k0 + k2 < kend) ? fp8_value(w[(int64_t)(k0 + k2) * N + n]) : 0.f;
            }
          }
          __syncthreads();
#pragma unroll
          for (int kk = 0; kk < S_K; ++kk) {
            float a[4], b[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) { a[u] = xs[kk][ty * 4 + u]; b[u] = wsm[kk][tx + 16 * u]; }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int v = 0; v < 4; ++v) part[u][v] = fmaf(a[u], b[v], part[u][v]);
          }
          __syncthreads();
        }
        const int nb = n0 / FP8_BLOCK;
        const float sw = TRANSPOSED ? ops.ws[i][((int64_t)e * kblocks + kb) * nblocks + nb]
                                    : ops.ws[i][((int64_t)e * nblocks + nb) * kblocks + kb];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t t = t0 + ty * 4 + u;
          const float sx = t < row_end ? ops.s[i][kb * fp8_scale_pitch(M) + t] * sw : 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(part[u][v], sx, acc[u][v]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t t = t0 + ty * 4 + u;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int n = n0 + tx + 16 * v;
        if (t < row_end && n < N) y[t * N + n] = from_f32<T>(acc[u][v]);
      }
    }
  }
}

dim3 quantize_grid(int64_t M, int K, int unroll) {
  const int64_t pairs = (K + 2 * FP8_BLOCK - 1) / (2 * FP8_BLOCK), groups = (pairs + unroll - 1) / unroll;
  const int64_t want = (M + Q_THREADS / 32 - 1) / (Q_THREADS / 32), cap = (int64_t)sm_count() * 16 / groups + 1;
  return dim3((unsigned)groups, (unsigned)(want < cap ? want : cap));
}

bool aligned8(const void* p) { return ((uintptr_t)p & 7) == 0; }

constexpr int MAX_EXTENT = 1 << 24;  // of N and K: tile and block ends fit in an int

bool rows_ok(int64_t M, int K) { return M >= 0 && M <= 0x7fffffffLL && K >= 1 && K <= MAX_EXTENT; }
bool product_ok(int64_t M, int N, int K) { return M <= 0x7fffffffLL - 1024 && rows_ok(M, K) && N >= 1 && N <= MAX_EXTENT; }

}  // namespace
}  // namespace moe

using namespace moe;

MOE_API int moe_fp8_quantize_rows(const void* x, int dtype, int64_t M, int K, void* q, float* scale, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!is_float_dtype(dtype)) return MOE_ERR_DTYPE;
  if (!rows_ok(M, K)) return MOE_ERR_SHAPE;
  if (M == 0) return MOE_OK;
  if (!x || !q || !scale) return MOE_ERR_NULL;
  const bool vec = K % 8 == 0 && aligned16(x) && aligned8(q);
  MOE_DISPATCH_FLOAT(dtype, T, {
    // four pairs of blocks to a warp, or three where that leaves fewer of them idle (K = 768: 39 us with four, 65536 rows)
    const int pairs = (K + 2 * FP8_BLOCK - 1) / (2 * FP8_BLOCK);
    const int u = !vec ? 1 : (pairs + 2) / 3 * 3 < (pairs + 3) / 4 * 4 ? 3 : 4;
    const dim3 grid = quantize_grid(M, K, u);
    if (u == 4) quantize_rows_kernel<T, true, 4><<<grid, Q_THREADS, 0, stream>>>((const T*)x, M, K, (uint8_t*)q, scale);
    else if (u == 3) quantize_rows_kernel<T, true, 3><<<grid, Q_THREADS, 0, stream>>>((const T*)x, M, K, (uint8_t*)q, scale);
    else quantize_rows_kernel<T, false, 1><<<grid, Q_THREADS, 0, stream>>>((const T*)x, M, K, (uint8_t*)q, scale);
  });
  return launch_status();
}

MOE_API int moe_fp8_silu_quantize(const float* e, const float* g, int64_t M, int I, void* hq, float* hs, void* keep_e,
                                  void* keep_g, int dtype, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!is_float_dtype(dtype)) return MOE_ERR_DTYPE;
  if (!rows_ok(M, I)) return MOE_ERR_SHAPE;
  if (M == 0) return MOE_OK;
  if (!e || !g || !hq || !hs || !keep_e != !keep_g) return MOE_ERR_NULL;
  const bool vec = I % 8 == 0 && aligned16(e) && aligned16(g) && aligned8(hq);
  const dim3 grid = quantize_grid(M, I, 1);
  MOE_DISPATCH_FLOAT(dtype, T, {
    if (vec) silu_quantize_kernel<T, true><<<grid, Q_THREADS, 0, stream>>>(e, g, M, I, (uint8_t*)hq, hs, (T*)keep_e, (T*)keep_g);
    else silu_quantize_kernel<T, false><<<grid, Q_THREADS, 0, stream>>>(e, g, M, I, (uint8_t*)hq, hs, (T*)keep_e, (T*)keep_g);
  });
  return launch_status();
}

MOE_API int moe_fp8_silu_bwd_quantize(const float* dh, const void* e, const void* g, int64_t M, int I, void* deq, float* des,
                                      void* dgq, float* dgs, int dtype, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!is_float_dtype(dtype)) return MOE_ERR_DTYPE;
  if (!rows_ok(M, I)) return MOE_ERR_SHAPE;
  if (M == 0) return MOE_OK;
  if (!dh || !e || !g || !deq || !des || !dgq || !dgs) return MOE_ERR_NULL;
  const bool vec = I % 8 == 0 && aligned16(dh) && aligned16(e) && aligned16(g) && aligned8(deq) && aligned8(dgq);
  const dim3 grid = quantize_grid(M, I, vec ? 2 : 1);
  MOE_DISPATCH_FLOAT(dtype, T, {
    if (vec) silu_bwd_quantize_kernel<T, true><<<grid, Q_THREADS, 0, stream>>>(dh, (const T*)e, (const T*)g, M, I, (uint8_t*)deq, des, (uint8_t*)dgq, dgs);
    else silu_bwd_quantize_kernel<T, false><<<grid, Q_THREADS, 0, stream>>>(dh, (const T*)e, (const T*)g, M, I, (uint8_t*)deq, des, (uint8_t*)dgq, dgs);
  });
  return launch_status();
}

MOE_API int moe_gate_up_silu_fp8(const void* q, const float* s, const void* w_gate, const float* ws_gate, const void* w_up,
                                 const float* ws_up, const void* m_sizes, int msd, void* hq, float* hs, void* keep_e,
                                 void* keep_g, int64_t M, int I, int K, int E, int dtype, void* stream) {
  if (!is_float_dtype(dtype) || !is_int_dtype(msd)) return MOE_ERR_DTYPE;
  if (!product_ok(M, I, K) || E < 1) return MOE_ERR_SHAPE;
  if (M == 0) return MOE_OK;
  if (!q || !s || !w_gate || !ws_gate || !w_up || !ws_up || !m_sizes || !hq || !hs || !keep_e != !keep_g) return MOE_ERR_NULL;
  const int path = moe_get_gemm_path();
  if (path == MOE_PATH_SIMT || dtype == MOE_F32 || !aligned16(keep_e) || !aligned16(keep_g) ||
      !tc_fp8_eligible(q, w_gate, nullptr, w_up, hq, M, I, K, E))
    return MOE_ERR_UNSUPPORTED;
  return tc_gate_up_silu_fp8(q, s, w_gate, ws_gate, w_up, ws_up, m_sizes, msd == MOE_I64, hq, hs, keep_e, keep_g, M, I, K, E, dtype,
                             path, (cudaStream_t)stream);
}

MOE_API int moe_grouped_gemm_fp8(int which, const void* q, const float* s, const void* w, const float* ws, const void* q2,
                                 const float* s2, const void* w2, const float* ws2, const void* m_sizes, int msd, void* y,
                                 int64_t M, int N, int K, int E, int dtype_out, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!is_float_dtype(dtype_out) || !is_int_dtype(msd)) return MOE_ERR_DTYPE;
  if ((which != 0 && which != 1) || !product_ok(M, N, K) || E < 1 || E > 65535) return MOE_ERR_SHAPE;
  if (M == 0) return MOE_OK;
  if (!q || !s || !w || !ws || !m_sizes || !y || (q2 && (!s2 || !w2 || !ws2))) return MOE_ERR_NULL;
  const int ms64 = msd == MOE_I64;
  const int path = moe_get_gemm_path();
  if (path != MOE_PATH_SIMT && tc_fp8_eligible(q, w, q2, w2, y, M, N, K, E))
    return tc_grouped_gemm_fp8(which, q, s, w, ws, q2, s2, w2, ws2, m_sizes, ms64, y, M, N, K, E, dtype_out, path, stream);
  if (path == MOE_PATH_TC || path == MOE_PATH_TC_SINGLE) return MOE_ERR_UNSUPPORTED;
  const Fp8Pairs ops = {{(const uint8_t*)q, (const uint8_t*)q2}, {s, s2}, {(const uint8_t*)w, (const uint8_t*)w2}, {ws, ws2}, q2 ? 2 : 1};
  const dim3 grid((N + S_TILE - 1) / S_TILE, E, S_WORKERS);
  MOE_DISPATCH_FLOAT(dtype_out, T, {
    if (which == 0) simt_gemm_fp8_kernel<T, false><<<grid, S_THREADS, 0, stream>>>(ops, m_sizes, ms64, (T*)y, M, N, K);
    else simt_gemm_fp8_kernel<T, true><<<grid, S_THREADS, 0, stream>>>(ops, m_sizes, ms64, (T*)y, M, N, K);
  });
  return launch_status();
}
