// CTA-pair (tcgen05 cta_group::2) grouped GEMMs on e4m3 operands with scales for blocks of 128.  Included by tc_gemm.cu.
//
//   pair_fp8_kernel<false>: y[t,n] = sum_kb s[kb,t] ws[e,n/128,kb] sum_{k in kb} q[t,k] w[e,n,k]     A = w K-major
//   pair_fp8_kernel<true> : y[t,n] = sum_kb s[kb,t] ws[e,kb,n/128] sum_{k in kb} q[t,k] w[e,k,n]     A = w MN-major
// over one or two operand pairs of the same contraction length into one result.
//
// Tiling as in pair_fwd_kernel: accumulator rows are 256 weight rows (128 per CTA, one scale block each), accumulator columns
// up to 256 tokens.  The scales are arbitrary fp32 numbers, so the tensor cores cannot apply them: every block of 128 of the
// contraction (one stage: 128 rows x 128 bytes of either operand in each CTA) is a sum of its own in TMEM, and 8 epilogue
// warps add it to fp32 sums in registers with its factor, acc += s ws * block.  Two accumulators of 256 columns alternate, so
// the addition of one block runs beside the MMAs of the next: 512 cycles of MMA for a full tile, against 64 packed FMAs, 8 TMEM
// loads and 8 shared-memory loads for each of the 8 warps.
//
// In the accumulator-fragment shape (16x256b) a thread holds 2 of every 8 columns and 4 of the warp's 32 rows: a factor is
// loaded once for 4 values, and two loads of 16 bytes bring the factors of 32 columns (they are stored in that order by the
// warp that multiplies s with ws, `scale_pos`).  A warp owns 32 accumulator rows and every other run of 32 columns: 128 sums
// in each thread, hence the register split (8 epilogue warps 208, the 4 others 88).
//
// A group of r rows is cut into ceil(r / 256) tiles of about equal width (a multiple of 32): the MMAs' cost goes with the columns, the
// weight stream with the number of tiles.
#pragma once

namespace moe {
namespace tc {

constexpr int F8_THREADS = 384;        // TMA, MMA, scales, one idle warp; 8 epilogue warps
constexpr int F8_BK = 128;             // contraction values (bytes) of a stage
constexpr int F8_UMMA_K = 32;
constexpr int F8_HALF_BYTES = 128 * F8_BK;
constexpr int F8_STAGE_BYTES = 2 * F8_HALF_BYTES;
constexpr int F8_STAGES = 5;
constexpr int F8_SLOTS = 8;            // blocks of factors in flight
constexpr int F8_READERS = 21;         // of the tile ring: 2 producers, 2 scale warps, the MMA thread, 16 epilogue warps
constexpr int F8_EPI_REGS = 208, F8_OTHER_REGS = 88;
static_assert(256 * F8_EPI_REGS + 128 * F8_OTHER_REGS <= F8_THREADS * 168, "shares of the registers that the CTA is launched with");

struct Fp8Maps {
  CUtensorMap w[2];   // weights
  CUtensorMap x[2];   // codes of the activations, boxes of 128 rows
  CUtensorMap xs[2];  // the same in boxes of PAIR_SMALL_BOX rows
  CUtensorMap out;    // 16-bit outputs, boxes of 32 rows x 64
};

struct Fp8Params {
  const void* m_sizes;
  int ms64;
  int64_t M;
  int N, E;
  int kb;               // blocks of the contraction
  int n_seg;            // operand pairs
  const float* s[2];    // (kb, M)
  const float* ws[2];
  int64_t ws_e;         // strides of a weight scale: expert, block of rows, block of the contraction
  int ws_n, ws_k;
  void* out;
  int dtype_out;
  uint32_t idesc;
};

struct Fp8Control {
  uint64_t full[F8_STAGES];
  uint64_t empty[F8_STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_free[2];   // 16 warps; the leader CTA's copies are the ones used
  uint64_t sfull[F8_SLOTS];
  uint64_t sempty[F8_SLOTS];
  SchedRing sched;
  uint64_t cancel_bar;
  alignas(16) uint4 cancel_response;
  uint32_t tmem_base;
  int abort_flag;
};

enum Fp8WaitCode { FW_SFULL = 24, FW_SEMPTY = 25 };

constexpr int F8_STAGING_BYTES = 2 * 2 * 2 * PAIR_STAGING_BYTES;  // 2 warpgroups x 2 buffers x 2 halves of the weight rows
static int fp8_smem_bytes(int E) {
  return F8_STAGES * F8_STAGE_BYTES + F8_STAGING_BYTES + F8_SLOTS * 1024 + (int)sizeof(Fp8Control) + 2 * (E + 1) * 4 + 1024;
}

// Where the factor of column `col` of a run of 32 lies: thread t of a warp needs those of columns 8g + 2(t%4) and +1.
__device__ __forceinline__ int scale_pos(int col) { return ((col >> 1) & 3) * 8 + (col >> 3) * 2 + (col & 1); }

struct Fp8Tile {
  int e, t0, n0, n_main, t_end;
};

template <bool W_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8_THREADS, 1)
pair_fp8_kernel(const __grid_constant__ Fp8Maps maps, const Fp8Params p) {
  constexpr int TILE_N = 256;
  constexpr uint32_t TMEM_COLS = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + F8_STAGES * F8_STAGE_BYTES;
  float* factors = reinterpret_cast<float*>(staging + F8_STAGING_BYTES);
  Fp8Control* ctl = reinterpret_cast<Fp8Control*>(factors + F8_SLOTS * 256);
  int* row_start = reinterpret_cast<int*>(ctl + 1);
  int* tt_start = row_start + (p.E + 1);
  volatile int* abort_flag = &ctl->abort_flag;
  using Feed = TileFeed<2, F8_READERS>;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < F8_STAGES; ++s) { mbar_init(&ctl->full[s], 1); mbar_init(&ctl->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&ctl->tmem_full[a], 1); mbar_init(&ctl->tmem_free[a], 16); }
    for (int q = 0; q < F8_SLOTS; ++q) { mbar_init(&ctl->sfull[q], 32); mbar_init(&ctl->sempty[q], 8); }
    Feed::init(&ctl->sched);
    mbar_init(&ctl->cancel_bar, 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.w[0]);
    tma_prefetch_desc(&maps.x[0]);
  }
  if (warp == 1) {
    tmem_alloc_pair(&ctl->tmem_base, TMEM_COLS);
    tmem_relinquish_pair();
  }
  build_group_tables(p.m_sizes, p.ms64, p.E, p.M, PAIR_TOKENS, row_start, tt_start);
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;

  const int n_tiles = (p.N + TILE_N - 1) / TILE_N;
  const int64_t total_tiles = (int64_t)tt_start[p.E] * n_tiles;
  const int steps = p.kb * p.n_seg;  // stages of a tile

  auto decode = [&](int tile) {
    Fp8Tile t;
    const int q = tile / n_tiles;
    t.e = find_group(tt_start, p.E, q);
    const int tt_e = tt_start[t.e + 1] - tt_start[t.e];
    const int j = tile - tt_start[t.e] * n_tiles;
    const int jt = j % tt_e;
    t.t_end = row_start[t.e + 1];
    const int rows = t.t_end - row_start[t.e];
    // (several tiles: whole runs of 32 columns, and every tile has rows, since 256 (tiles - 1) < rows)
    const int width = tt_e == 1 ? (rows + 15) & ~15 : ((rows + tt_e - 1) / tt_e + 31) & ~31;
    t.t0 = row_start[t.e] + jt * width;
    t.n0 = (j / tt_e) * TILE_N;
    t.n_main = min(width, (t.t_end - t.t0 + 15) & ~15);
    return t;
  };
  auto small_boxes = [&](int n_main) {  // of this CTA's half of the tokens; 0: one box of 128 rows
    const int rows = n_main >> 1;
    return rows <= 64 ? (rows + PAIR_SMALL_BOX - 1) / PAIR_SMALL_BOX : 0;
  };

  if (warp < 4) {
    registers_dec<F8_OTHER_REGS>();
    if (warp == 0) {
      // ------------------------------ TMA producer (both CTAs) ------------------------------
      if (elect_one()) {
        Feed feed(&ctl->sched, abort_flag);
        const uint32_t full_leader0 = map_to_cta(smem_u32(&ctl->full[0]), 0);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok) {
          const int tile = feed.take();
          if (tile < 0) break;
          const Fp8Tile t = decode(tile);
          const int w_row = t.n0 + (int)rank * 128;
          const int tok = t.t0 + (int)rank * (t.n_main >> 1);
          const int nsb = small_boxes(t.n_main);
          const uint32_t b_bytes = nsb ? nsb * PAIR_SMALL_BOX * F8_BK : F8_HALF_BYTES;
          for (int i = 0; i < p.n_seg && ok; ++i) {
            for (int kb = 0; kb < p.kb; ++kb) {
              if (!mbar_wait(&ctl->empty[s], ph ^ 1, abort_flag, PW_EMPTY)) { ok = false; break; }
              uint8_t* sa = smem + s * F8_STAGE_BYTES;
              uint8_t* sb = sa + F8_HALF_BYTES;
              const uint32_t bar = full_leader0 + s * 8;
              if (leader) mbar_expect_tx(&ctl->full[s], 2 * (F8_HALF_BYTES + b_bytes));  // both CTAs' bytes
              if constexpr (W_MN) tma_load_3d_pair(sa, &maps.w[i], bar, w_row, kb * F8_BK, t.e);
              else tma_load_3d_pair(sa, &maps.w[i], bar, kb * F8_BK, w_row, t.e);
              if (nsb == 0) {
                tma_load_2d_pair(sb, &maps.x[i], bar, kb * F8_BK, tok);
              } else {
                for (int b = 0; b < nsb; ++b)
                  tma_load_2d_pair(sb + b * (PAIR_SMALL_BOX * F8_BK), &maps.xs[i], bar, kb * F8_BK, tok + b * PAIR_SMALL_BOX);
              }
              if (++s == F8_STAGES) { s = 0; ph ^= 1; }
            }
          }
        }
      }
    } else if (warp == 1) {
      // ------------- MMA issuer (leader CTA); the same warp of the other CTA draws the tiles -------------
      if (!leader) {
        if (elect_one()) {
          Feed feed(&ctl->sched, abort_flag);
          feed.run_cancel(&ctl->cancel_bar, &ctl->cancel_response, (int)total_tiles, (int)(blockIdx.x >> 1));
        }
      } else if (elect_one()) {
        Feed feed(&ctl->sched, abort_flag);
        uint32_t it = 0;  // blocks so far: accumulator it % 2
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok) {
          const int tile = feed.take();
          if (tile < 0) break;
          const Fp8Tile t = decode(tile);
          const uint32_t idesc = p.idesc | ((uint32_t)(t.n_main >> 3) << 17);
          for (int b = 0; b < steps; ++b, ++it) {
            const uint32_t buf = it & 1;
            if (!mbar_wait_cluster(&ctl->tmem_free[buf], ((it >> 1) & 1) ^ 1, abort_flag, PW_TMEM_EMPTY)) { ok = false; break; }
            if (!mbar_wait_cluster(&ctl->full[s], ph, abort_flag, PW_FULL)) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t sa = smem_u32(smem + s * F8_STAGE_BYTES);
            const uint64_t da = make_smem_desc(sa, W_MN ? F8_HALF_BYTES : 16, 1024);
            const uint64_t db = make_smem_desc(sa + F8_HALF_BYTES, 16, 1024);
            const uint32_t d = tmem_base + buf * PAIR_TOKENS;
#pragma unroll
            for (int k = 0; k < F8_BK / F8_UMMA_K; ++k) {
              const uint64_t b_adv = (uint64_t)((k * F8_UMMA_K) >> 4);
              const uint64_t a_adv = W_MN ? (uint64_t)((k * F8_UMMA_K * 128) >> 4) : b_adv;
              umma_f8_pair(d, da + a_adv, db + b_adv, idesc, k != 0);
            }
            umma_commit_pair(&ctl->empty[s], 3);
            umma_commit_pair(&ctl->tmem_full[buf], 3);
            if (++s == F8_STAGES) { s = 0; ph ^= 1; }
          }
        }
      }
    } else if (warp == 2) {
      // ------------------------------ factors (both CTAs) ------------------------------
      // Four blocks' scales are loaded at a time: a block's MMAs take less time than one trip to memory.
      Feed feed(&ctl->sched, abort_flag);
      constexpr int AHEAD = 4;
      uint32_t it = 0;
      bool ok = true;
      const int n_blocks = (p.N + 127) / 128;
      while (ok) {
        const int tile = feed.take_warp(lane);
        if (tile < 0) break;
        const Fp8Tile t = decode(tile);
        const int nb = min(t.n0 / 128 + (int)rank, n_blocks - 1);
        const int64_t ws0 = t.e * p.ws_e + (int64_t)nb * p.ws_n;
        for (int b0 = 0; b0 < steps && ok; b0 += AHEAD) {
          float v[AHEAD][8], w[AHEAD];
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            const int b = b0 + a;
            const int seg = b >= p.kb ? 1 : 0;
            const int kb = b - seg * p.kb;
            if (b < steps) {
              w[a] = __ldg(p.ws[seg] + ws0 + (int64_t)kb * p.ws_k);
              const float* src = p.s[seg] + (int64_t)kb * p.M + t.t0;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int col = i * 32 + lane;
                v[a][i] = col < t.n_main && t.t0 + col < p.M ? __ldg(src + col) : 0.f;
              }
            }
          }
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            if (b0 + a >= steps || !ok) break;
            const uint32_t q = it % F8_SLOTS, ph = (it / F8_SLOTS) & 1;
            if (!mbar_wait(&ctl->sempty[q], ph ^ 1, abort_flag, FW_SEMPTY)) { ok = false; break; }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i * 32 < t.n_main) factors[q * 256 + i * 32 + scale_pos(lane)] = v[a][i] * w[a];
            mbar_arrive(&ctl->sfull[q]);
            ++it;
          }
        }
      }
    }
  } else {
    // ------------------------------ epilogue (both CTAs) ------------------------------
    registers_inc<F8_EPI_REGS>();
    Feed feed(&ctl->sched, abort_flag);
    const int quarter = warp & 3;
    const int wg = (warp >> 2) - 1;
    const int epi_tid = threadIdx.x & 127;
    const uint32_t tmem_free_leader0 = map_to_cta(smem_u32(&ctl->tmem_free[0]), 0);
    uint8_t* const my_staging = staging + wg * (4 * PAIR_STAGING_BYTES);
    const int half = quarter >> 1;
    const int chunk = 4 * (quarter & 1) + (lane >> 3);  // 16-byte chunk of the 128-byte staging row
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const float* my_factors = factors + (lane & 3) * 8;
    uint32_t it = 0, round = 0;
    bool ok = true;
    while (true) {
      const int tile = feed.take_warp(lane);
      // the four warps of a warpgroup leave together; a warp whose wait was abandoned goes on without waiting until here
      if (named_barrier_any(3 + wg, 128, tile < 0 || !ok)) break;
      const Fp8Tile t = decode(tile);
      const int runs = (t.n_main + 31) >> 5;  // of 32 columns; this warp's are wg, wg + 2, ...
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
#pragma unroll 1
      for (int b = 0; b < steps; ++b, ++it) {
        const uint32_t buf = it & 1, q = it % F8_SLOTS;
        if (ok) ok = mbar_wait_cluster(&ctl->tmem_full[buf], (it >> 1) & 1, abort_flag, PW_TMEM_FULL);
        if (ok) ok = mbar_wait(&ctl->sfull[q], (it / F8_SLOTS) & 1, abort_flag, FW_SFULL);
        tc_fence_after_sync();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (2 * i + wg < runs) {
            const int c = (2 * i + wg) * 32;
            uint32_t lo[16], hi[16];
            tmem_ld_16x256b_x4(lane_base + buf * PAIR_TOKENS + c, lo);
            tmem_ld_16x256b_x4(lane_base + buf * PAIR_TOKENS + c + (16u << 16), hi);
            const ulonglong2 f0 = *reinterpret_cast<const ulonglong2*>(my_factors + q * 256 + c);
            const ulonglong2 f1 = *reinterpret_cast<const ulonglong2*>(my_factors + q * 256 + c + 4);
            const uint64_t f[4] = {f0.x, f0.y, f1.x, f1.y};
            tmem_ld_wait();
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint64_t* a = acc + i * 16 + g * 4;
              a[0] = fma_f32x2(pack_f32x2(lo[4 * g], lo[4 * g + 1]), f[g], a[0]);
              a[1] = fma_f32x2(pack_f32x2(lo[4 * g + 2], lo[4 * g + 3]), f[g], a[1]);
              a[2] = fma_f32x2(pack_f32x2(hi[4 * g], hi[4 * g + 1]), f[g], a[2]);
              a[3] = fma_f32x2(pack_f32x2(hi[4 * g + 2], hi[4 * g + 3]), f[g], a[3]);
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_cluster(tmem_free_leader0 + buf * 8);
          mbar_arrive(&ctl->sempty[q]);
        }
      }
      const int n_cta = t.n0 + (int)rank * 128;
      if (p.dtype_out == MOE_F32) {
        float* out = reinterpret_cast<float*>(p.out);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (2 * i + wg < runs) {
            const int tok = t.t0 + (2 * i + wg) * 32 + 2 * (lane & 3);
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int n = n_cta + quarter * 32 + r * 8 + (lane >> 2);
                const uint64_t v = acc[i * 16 + g * 4 + r];
                if (n < p.N && tok + 8 * g < t.t_end) out[(int64_t)(tok + 8 * g) * p.N + n] = lo_f32(v);
                if (n < p.N && tok + 8 * g + 1 < t.t_end) out[(int64_t)(tok + 8 * g + 1) * p.N + n] = hi_f32(v);
              }
          }
        }
      } else {
        const bool is_bf16 = p.dtype_out == MOE_BF16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (2 * i + wg < runs) {
            const int c = (2 * i + wg) * 32;
            uint8_t* buf = my_staging + (round & 1) * (2 * PAIR_STAGING_BYTES);
            ++round;
            if (epi_tid == 0) tma_store_wait_read<1>();  // the stores of two rounds ago have read this buffer
            named_barrier_sync(1 + wg, 128);
            uint8_t* tile_buf = buf + half * PAIR_STAGING_BYTES;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint32_t m[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint64_t v = acc[i * 16 + g * 4 + r];
                m[r] = is_bf16 ? pack2<__nv_bfloat16>(lo_f32(v), hi_f32(v)) : pack2<__half>(lo_f32(v), hi_f32(v));
              }
              const int trow = 8 * g + (lane & 7);
              stmatrix_x4_trans(smem_u32(tile_buf + trow * 128 + ((chunk ^ (trow & 7)) << 4)), m[0], m[1], m[2], m[3]);
            }
            fence_proxy_async_smem();
            named_barrier_sync(1 + wg, 128);
            const bool clip = t.t_end - (t.t0 + c) < 32;
            if (clip) store_clipped_rows<16>(buf, reinterpret_cast<uint8_t*>(p.out), t.t0 + c, t.t_end, n_cta, p.N, epi_tid);
            if (epi_tid == 0) {
              if (!clip && n_cta < p.N) {
                tma_store_2d(&maps.out, buf, n_cta, t.t0 + c);
                if (n_cta + 64 < p.N) tma_store_2d(&maps.out, buf + PAIR_STAGING_BYTES, n_cta + 64, t.t0 + c);
              }
              tma_store_commit();
            }
          }
        }
      }
    }
    if (epi_tid == 0) tma_store_wait_all();
  }

  tc_fence_before_sync();
  cluster_sync_all();  // nobody frees TMEM or exits while the peer may still touch this CTA
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

}  // namespace tc
}  // namespace moe
