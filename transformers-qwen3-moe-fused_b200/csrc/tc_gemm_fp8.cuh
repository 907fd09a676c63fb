// CTA-pair (tcgen05 cta_group::2) grouped GEMMs on e4m3 operands with scales for blocks of 128.  Included by tc_gemm.cu.
//
//   pair_fp8_kernel<false>: y[t,n] = sum_kb s[kb,t] ws[e,n/128,kb] sum_{k in kb} q[t,k] w[e,n,k]     A = w K-major
//   pair_fp8_kernel<true> : y[t,n] = sum_kb s[kb,t] ws[e,kb,n/128] sum_{k in kb} q[t,k] w[e,k,n]     A = w MN-major
// over one or two operand pairs of the same contraction length into one result.
//
// Accumulator rows are up to 256 tokens (128 per CTA), columns up to 256 weight rows, the other way round than in
// pair_fwd_kernel.  The scales are arbitrary fp32 numbers, so the tensor cores cannot apply them: every block of 128 of the
// contraction (one stage: 128 rows x 128 bytes of either operand in each CTA) is a sum of its own in TMEM, and 8 epilogue
// warps add it to fp32 sums in registers with its factor, acc += s ws * block.  A thread owns one token and 128 columns, one
// block of weight rows: its factor is one number for all of them, and nothing crosses threads.  Two accumulators of 256
// columns alternate, so the addition of one block runs beside the MMAs of the next.
// (With weight rows as accumulator rows the factor changes from column to column.  In the fragment shape 16x256b, where a thread
// needs few of them, TMEM loads run at half the rate: 535 cycles for 256 columns against 260 in the shape 32x32b.  Forward /
// dX at 65536 rows, 2048 -> 1536: 401 / 424 us, against 305 / 315 us here.)
//
// What bounds it: the latency of the additions, not the MMAs and no throughput.  A block takes 1250 cycles (65536 rows in even
// groups: 255 us, tensor pipe 41 %), where the MMAs need 512 (with the additions left out it takes 515), the TMEM loads 256 and
// the FMAs 285 on each quarter of the SM, which would be 541 even one after the other.  A quarter's two warps each load 32
// columns, wait, and issue 16 packed FMAs, four times in a row: no warp can issue in 60 % of the cycles, the fp32 pipe is 31 % busy.
// With 128 sums and 32 loaded values a thread has no registers left for loads that run ahead (half the sums: 240 us).  Narrower
// tiles (192 columns, 96 or 64 sums), 16 warps, four accumulators of 128 columns, scales that come by TMA, and loads of 64 columns
// were no faster: 310 to 390 us.
//
// The price of tokens as rows is that a tile costs 256 rows of MMAs whatever it holds (warps without rows skip the additions);
// groups of few rows have a kernel of their own, thin_fp8_kernel.
#pragma once

namespace moe {
namespace tc {

constexpr int F8_THREADS = 384;        // TMA, MMA, tiles, one idle warp; 8 epilogue warps
constexpr int F8_BK = 128;             // contraction values (bytes) of a stage
constexpr int F8_UMMA_K = 32;
constexpr int F8_HALF_BYTES = 128 * F8_BK;
constexpr int F8_STAGE_BYTES = 2 * F8_HALF_BYTES;
constexpr int F8_STAGES = 5;
constexpr int F8_READERS = 5;          // of the pair's tile ring: 2 producers, 2 tile warps, the MMA thread
constexpr int F8_TILES = 2;            // decoded tiles on their way to the epilogue warps
constexpr int F8_EPI_REGS = 192, F8_OTHER_REGS = 120;
static_assert(256 * F8_EPI_REGS + 128 * F8_OTHER_REGS <= F8_THREADS * 168, "shares of the registers that the CTA is launched with");

struct Fp8Maps {
  CUtensorMap w[2];   // weights (GATE_UP: gate, up)
  CUtensorMap x[2];   // codes of the activations, boxes of 128 rows
  CUtensorMap xs[2];  // the same in boxes of PAIR_SMALL_BOX rows
  CUtensorMap out;    // 16-bit outputs, boxes of 32 rows x 64
};

struct Fp8Params {
  const void* m_sizes;
  int ms64;
  int64_t M;
  int N, E;
  int stages;
  int kb;               // blocks of the contraction
  int n_seg;            // operand pairs
  int64_t pitch;        // of s
  const float* s[2];    // (kb, M)
  const float* ws[2];
  int64_t ws_e;         // strides of a weight scale: expert, block of rows, block of the contraction
  int ws_n, ws_k;
  void* out;            // GATE_UP: codes of h
  float* out_s;         // GATE_UP: scales of h
  void* keep_e;         // GATE_UP: the projections in dtype_out, or null
  void* keep_g;
  int dtype_out;
  uint32_t idesc;
};

struct Fp8Control {
  uint64_t full[F8_STAGES];
  uint64_t empty[F8_STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_free[2];   // 16 warps; the leader CTA's copies are the ones used
  uint64_t tile_full[F8_TILES];   // the tile warp
  uint64_t tile_empty[F8_TILES];  // 8 epilogue warps
  SchedRing sched;
  uint64_t cancel_bar;
  alignas(16) uint4 cancel_response;
  int4 tiles[F8_TILES];           // expert (-1: no more tiles), first token, first column, first row past the expert
  uint64_t drain;                 // the MMA thread's last MMAs
  int stages_done[3];             // loaded by the leader's producer, by the other CTA's, multiplied; the same in both CTAs
  uint32_t tmem_base;
  int abort_flag;
};

enum Fp8WaitCode { FW_TILE_FULL = 24, FW_TILE_EMPTY = 25 };

constexpr int F8_ROWS = 256;                       // tokens of a tile
constexpr int F8_WARP_STAGING = 32 * 128;          // 32 tokens x 64 columns x 16 bit, two of them for each epilogue warp
constexpr int F8_STAGING_BYTES = 8 * 2 * F8_WARP_STAGING;
static int fp8_smem_bytes(int stages, int E) {
  return stages * F8_STAGE_BYTES + F8_STAGING_BYTES + (int)sizeof(Fp8Control) + 2 * (E + 1) * 4 + 1024;
}
// Deepest ring that fits (tables of up to 1024 experts leave room for four stages).
static int fp8_stages(int E) { return fp8_smem_bytes(F8_STAGES, E) <= SMEM_LIMIT ? F8_STAGES : F8_STAGES - 1; }

struct Fp8Tile {
  int e, t0, n0;
  int n;      // columns of the MMA, a multiple of 32
  int t_end;  // first row past the expert
};

// W_MN: the weight is (E, K, N), read MN-major (the gradient of x).
// GATE_UP: 128 features of two weights (E, I, K): columns [gate f..f+63][up f..f+63] from the leader's half of the B operand,
// the next 64 features from the other CTA's, so a thread holds gate and up of the same 64 features of its token.  The epilogue
// writes h = silu(gate) * up as codes and scales (the scale's 128 features are those of two threads of one CTA), and the
// projections themselves in 16 bits where a backward pass wants them.
template <bool W_MN, bool GATE_UP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F8_THREADS, 1)
pair_fp8_kernel(const __grid_constant__ Fp8Maps maps, const Fp8Params p) {
  static_assert(!(W_MN && GATE_UP), "gate and up read K-major weights");
  constexpr int TILE_N = GATE_UP ? 128 : 256;  // output columns of a tile
  constexpr uint32_t TMEM_COLS = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + p.stages * F8_STAGE_BYTES;
  Fp8Control* ctl = reinterpret_cast<Fp8Control*>(staging + F8_STAGING_BYTES);
  int* row_start = reinterpret_cast<int*>(ctl + 1);
  int* tt_start = row_start + (p.E + 1);
  volatile int* abort_flag = &ctl->abort_flag;
  using Feed = TileFeed<2, F8_READERS>;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&ctl->full[s], 1); mbar_init(&ctl->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&ctl->tmem_full[a], 1); mbar_init(&ctl->tmem_free[a], 16); }
    for (int q = 0; q < F8_TILES; ++q) { mbar_init(&ctl->tile_full[q], 1); mbar_init(&ctl->tile_empty[q], 8); }
    Feed::init(&ctl->sched);
    mbar_init(&ctl->cancel_bar, 1);
    mbar_init(&ctl->drain, 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.w[0]);
    tma_prefetch_desc(&maps.x[0]);
  }
  if (warp == 1) {
    tmem_alloc_pair(&ctl->tmem_base, TMEM_COLS);
    tmem_relinquish_pair();
  }
  build_group_tables(p.m_sizes, p.ms64, p.E, p.M, F8_ROWS, row_start, tt_start);
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;

  const int n_tiles = (p.N + TILE_N - 1) / TILE_N;
  const int64_t total_tiles = (int64_t)tt_start[p.E] * n_tiles;
  const int steps = p.kb * p.n_seg;  // stages of a tile

  auto report_stages = [&](int who, int n) {
    for (uint32_t c = 0; c < 2; ++c) st_shared_cluster_u32(map_to_cta(smem_u32(&ctl->stages_done[who]), c), (uint32_t)n);
  };

  // Within an expert the token tile varies fastest: neighbouring tiles read the same weight slice.
  auto decode = [&](int tile) {
    Fp8Tile t;
    const int q = tile / n_tiles;
    t.e = find_group(tt_start, p.E, q);
    const int tt_e = tt_start[t.e + 1] - tt_start[t.e];
    const int j = tile - tt_start[t.e] * n_tiles;
    t.t0 = row_start[t.e] + (j % tt_e) * F8_ROWS;
    t.n0 = (j / tt_e) * TILE_N;
    t.n = GATE_UP ? 256 : min(256, (p.N - t.n0 + 31) & ~31);
    t.t_end = row_start[t.e + 1];
    return t;
  };

  if (warp < 4) {
    registers_dec<F8_OTHER_REGS>();
    if (warp == 0) {
      // ------------------------------ TMA producer (both CTAs) ------------------------------
      if (elect_one()) {
        Feed feed(&ctl->sched, abort_flag);
        const uint32_t full_leader0 = map_to_cta(smem_u32(&ctl->full[0]), 0);
        // boxes of a CTA's token rows: one of 128, or as many of 16 as hold rows; rows that are not loaded have sums that
        // nobody reads
        auto small_boxes = [&](int rows) { return rows > 64 ? 0 : rows <= 0 ? -1 : (rows + PAIR_SMALL_BOX - 1) / PAIR_SMALL_BOX; };
        auto box_bytes = [&](int boxes) { return boxes < 0 ? 0 : boxes == 0 ? F8_HALF_BYTES : boxes * PAIR_SMALL_BOX * F8_BK; };
        int s = 0, loaded = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok) {
          const int tile = feed.take();
          if (tile < 0) break;
          const Fp8Tile t = decode(tile);
          const int tok = t.t0 + (int)rank * 128;
          const int nsb = small_boxes(t.t_end - tok);
          const uint32_t bytes = 2 * F8_HALF_BYTES + box_bytes(small_boxes(t.t_end - t.t0)) + box_bytes(small_boxes(t.t_end - t.t0 - 128));
          for (int i = 0; i < p.n_seg && ok; ++i) {
            for (int kb = 0; kb < p.kb; ++kb) {
              if (!mbar_wait(&ctl->empty[s], ph ^ 1, abort_flag, PW_EMPTY)) { ok = false; break; }
              uint8_t* sa = smem + s * F8_STAGE_BYTES;
              uint8_t* sb = sa + F8_HALF_BYTES;
              const uint32_t bar = full_leader0 + s * 8;
              if (leader) mbar_expect_tx(&ctl->full[s], bytes);  // both CTAs' bytes
              if constexpr (GATE_UP) {
                const int feat = t.n0 + (int)rank * 64;
                tma_load_3d_pair(sb, &maps.w[0], bar, kb * F8_BK, feat, t.e);
                tma_load_3d_pair(sb + F8_HALF_BYTES / 2, &maps.w[1], bar, kb * F8_BK, feat, t.e);
              } else {
                const int w_row = t.n0 + (int)rank * (t.n >> 1);
                if constexpr (W_MN) tma_load_3d_pair(sb, &maps.w[i], bar, w_row, kb * F8_BK, t.e);
                else tma_load_3d_pair(sb, &maps.w[i], bar, kb * F8_BK, w_row, t.e);
              }
              if (nsb == 0) tma_load_2d_pair(sa, &maps.x[i], bar, kb * F8_BK, tok);
              for (int b = 0; b < nsb; ++b)
                tma_load_2d_pair(sa + b * (PAIR_SMALL_BOX * F8_BK), &maps.xs[i], bar, kb * F8_BK, tok + b * PAIR_SMALL_BOX);
              ++loaded;
              if (++s == p.stages) { s = 0; ph ^= 1; }
            }
          }
        }
        report_stages((int)rank, loaded);
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
        int tile = feed.take();
        while (ok && tile >= 0) {
          const uint32_t idesc = p.idesc | ((uint32_t)(decode(tile).n >> 3) << 17);
          for (int b = 0; b < steps; ++b, ++it) {
            const uint32_t buf = it & 1;
            if (!mbar_wait(&ctl->full[s], ph, abort_flag, PW_FULL)) { ok = false; break; }
            if (!mbar_wait(&ctl->tmem_free[buf], ((it >> 1) & 1) ^ 1, abort_flag, PW_TMEM_EMPTY)) { ok = false; break; }
            tc_fence_after_sync();
            const uint32_t sa = smem_u32(smem + s * F8_STAGE_BYTES);
            const uint64_t da = make_smem_desc(sa, 16, 1024);
            const uint64_t db = make_smem_desc(sa + F8_HALF_BYTES, W_MN ? F8_HALF_BYTES : 16, 1024);
            const uint32_t d = tmem_base + buf * 256;
#pragma unroll
            for (int k = 0; k < F8_BK / F8_UMMA_K; ++k) {
              const uint64_t a_adv = (uint64_t)((k * F8_UMMA_K) >> 4);
              const uint64_t b_adv = W_MN ? (uint64_t)((k * F8_UMMA_K * 128) >> 4) : a_adv;
              umma_f8_pair(d, da + a_adv, db + b_adv, idesc, k != 0);
            }
            umma_commit_pair(&ctl->empty[s], 3);
            umma_commit_pair(&ctl->tmem_full[buf], 3);
            if (++s == p.stages) { s = 0; ph ^= 1; }
            if (b == 0) tile = feed.take();  // the next one, while this tile's blocks are on their way
          }
        }
        report_stages(2, (int)it);
        umma_commit_pair(&ctl->drain, 1);  // operands and accumulators of both CTAs stay until the last MMA is over
        mbar_wait_through(&ctl->drain, 0);
      }
    } else if (warp == 2) {
      // ---------------- tiles for the epilogue (both CTAs): taken from the pair's ring and decoded ----------------
      // (under the MMAs' operand traffic an access to shared memory takes 100 to 300 cycles, and this chain has a dozen: 3400
      // cycles of a tile when the epilogue warps did it themselves)
      Feed feed(&ctl->sched, abort_flag);
      if (elect_one()) {
        uint32_t n = 0;
        while (true) {
          const int tile = feed.take();
          int4 info = make_int4(-1, 0, 0, 0);
          if (tile >= 0) {
            const Fp8Tile t = decode(tile);
            info = make_int4(t.e, t.t0, t.n0, t.t_end);
          }
          const uint32_t q = n % F8_TILES;
          if (!mbar_wait(&ctl->tile_empty[q], ((n / F8_TILES) & 1) ^ 1, abort_flag, FW_TILE_EMPTY)) break;
          ctl->tiles[q] = info;
          mbar_arrive(&ctl->tile_full[q]);
          if (tile < 0) break;
          ++n;
        }
      }
    }
  } else {
    // ------------------------------ epilogue (both CTAs) ------------------------------
    registers_inc<F8_EPI_REGS>();
    const int quarter = warp & 3;
    const int wg = (warp >> 2) - 1;       // columns wg * 128 ..
    const int row = quarter * 32 + lane;  // of this CTA
    const uint32_t tmem_free_leader0 = map_to_cta(smem_u32(&ctl->tmem_free[0]), 0);
    uint8_t* const my_staging = staging + (warp - 4) * (2 * F8_WARP_STAGING);
    const uint32_t taddr0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + wg * 128;
    uint32_t it = 0, n_tile = 0;
    // A warp with an abandoned wait goes on to the end of the tile without waiting, but lane 0 hands no accumulator back any more
    // (other warps, the other CTA's too, may still have to read it), and no warp of the CTA stores sums.  `sign` is the lane, or 32
    // behind an abandoned wait.
    int sign = lane;
    auto take = [&]() {
      const uint32_t slot = n_tile % F8_TILES;
      const bool there = sign != 32 && mbar_wait(&ctl->tile_full[slot], (n_tile / F8_TILES) & 1, abort_flag, FW_TILE_FULL);
      const int4 info = there ? ctl->tiles[slot] : make_int4(-1, 0, 0, 0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->tile_empty[slot]);
      ++n_tile;
      return info;
    };
    // Factors: s of the thread's token times ws of its columns' block (GATE_UP: of gate and of up).  They are loaded two blocks
    // ahead, a tile's first ones before the tile in front of it is stored: a trip to L2 takes longer than a block.
    struct Raw { float s, w0, w1; };
    const float* sp = p.s[0];
    const float* wp = p.ws[0];
    const int last = p.kb - 1;
    auto start = [&](const int4& t, int seg) {
      const int nb = GATE_UP ? t.z / 128 : min(t.z / 128 + wg, (p.N - 1) / 128);
      sp = p.s[seg] + min(t.y + (int)rank * 128 + row, t.w - 1);
      wp = p.ws[seg] + t.x * p.ws_e + (int64_t)nb * p.ws_n;
    };
    auto fetch = [&](int b) {
      Raw r;
      const uint32_t kb = (uint32_t)min(b, last);  // (past the last block: the last one again, not used)
      r.s = __ldg(sp + (uint64_t)kb * (uint32_t)p.pitch);
      r.w0 = __ldg(wp + kb * (uint32_t)p.ws_k);
      r.w1 = GATE_UP ? __ldg(wp + (p.ws[1] - p.ws[0]) + kb * (uint32_t)p.ws_k) : 0.f;
      return r;
    };
    int4 info = take();
    if (info.x >= 0) start(info, 0);
    Raw r0 = {}, r1 = {};
    if (info.x >= 0) { r0 = fetch(0); r1 = fetch(1); }
    bool ready = false;  // the next block's sums were seen to be there while this one was added
    while (true) {
      const bool leave = __any_sync(0xffffffffu, info.x < 0);
      if constexpr (GATE_UP) {  // the two warps that share tokens leave together
        if (named_barrier_any(1 + quarter, 64, leave)) break;
      } else {
        if (leave) break;
      }
      const int t_n0 = info.z;
      const int tok0 = info.y + (int)rank * 128 + quarter * 32;  // first token of the warp
      const int rows = info.w - tok0;                            // of the warp's 32 that belong to the expert
      const bool live = rows > 0;
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      // The loads of the factors and the test for the next block stand where the thread would wait for TMEM or has additions to
      // issue.
      auto add_block = [&](Raw& r, int ahead) {
        const uint32_t buf = it & 1;
        if (!ready && (sign == 32 || !mbar_wait(&ctl->tmem_full[buf], (it >> 1) & 1, abort_flag, PW_TMEM_FULL))) sign = 32;
        __syncwarp();  // (each lane tests and waits for itself; the TMEM loads, and the arrival behind them, are the whole warp's)
        tc_fence_after_sync();
        ++it;
        const uint32_t taddr = taddr0 + buf * 256;
        uint32_t f0, f1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t v[32];
          tmem_ld_32x32(taddr + i * 32, v);
          if (i == 0) {
            f0 = __float_as_uint(r.s * r.w0);
            f1 = GATE_UP ? __float_as_uint(r.s * r.w1) : f0;
            r = fetch(ahead);
          }
          tmem_ld_wait(v);
          if (i == 3) {
            tc_fence_before_sync();
            arrive_lane0(tmem_free_leader0 + buf * 8, sign);  // (the wait above was the whole warp's)
            ready = mbar_test(&ctl->tmem_full[it & 1], (it >> 1) & 1);
          }
          const uint64_t ff = i < 2 ? pack_f32x2(f0, f0) : pack_f32x2(f1, f1);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[i * 16 + j] = fma_f32x2(pack_f32x2(v[2 * j], v[2 * j + 1]), ff, acc[i * 16 + j]);
        }
      };
      if (live) {
        for (int seg = 0; seg < p.n_seg; ++seg) {
          if (seg > 0) {
            start(info, 1);
            r0 = fetch(0);
            r1 = fetch(1);
          }
#pragma unroll 1
          for (int b = 0; b < p.kb; b += 2) {
            add_block(r0, b + 2);
            if (b + 1 < p.kb) add_block(r1, b + 3);
          }
        }
      } else {
        for (int b = 0; b < steps; ++b, ++it) {
          if (sign == 32 || !mbar_wait(&ctl->tmem_full[it & 1], (it >> 1) & 1, abort_flag, PW_TMEM_FULL)) sign = 32;
          tc_fence_after_sync();
          __syncwarp();
          arrive_lane0(tmem_free_leader0 + (it & 1) * 8, sign);
        }
        ready = false;
      }
      const bool whole = !__any_sync(0xffffffffu, *abort_flag != 0);  // nobody here gave up: every block is in the sums
      info = take();
      if (info.x >= 0) {
        start(info, 0);
        r0 = fetch(0);
        r1 = fetch(1);
      }
      if constexpr (!GATE_UP) {
        if (!live || !whole) continue;
        const int n0 = t_n0 + wg * 128;  // first column
        if (p.dtype_out == MOE_F32) {
          float* out = reinterpret_cast<float*>(p.out) + (int64_t)(tok0 + lane) * p.N + n0;
#pragma unroll
          for (int j = 0; j < 32; ++j)  // columns end at a multiple of 16
            if (lane < rows && n0 + j * 4 < p.N)
              *reinterpret_cast<ulonglong2*>(out + j * 4) = make_ulonglong2(acc[2 * j], acc[2 * j + 1]);
        } else {
          const bool is_bf16 = p.dtype_out == MOE_BF16;
          if (lane == 0) tma_store_wait_read<0>();  // the stores of the tile before have read the buffers
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = n0 + h * 64;
            uint8_t* buf = my_staging + h * F8_WARP_STAGING;
            if (n < p.N) {
#pragma unroll
              for (int c = 0; c < 8; ++c) {  // 16 bytes: 8 columns
                uint32_t m[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const uint64_t a = acc[h * 32 + c * 4 + r];
                  m[r] = is_bf16 ? pack2<__nv_bfloat16>(lo_f32(a), hi_f32(a)) : pack2<__half>(lo_f32(a), hi_f32(a));
                }
                *reinterpret_cast<uint4*>(buf + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(m[0], m[1], m[2], m[3]);
              }
            }
          }
          if (rows >= 32) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (n0 < p.N) tma_store_2d(&maps.out, my_staging, n0, tok0);  // columns past N are clipped
              if (n0 + 64 < p.N) tma_store_2d(&maps.out, my_staging + F8_WARP_STAGING, n0 + 64, tok0);
              tma_store_commit();
            }
          } else {
            __syncwarp();
            uint8_t* out = reinterpret_cast<uint8_t*>(p.out);
            for (int i = lane; i < rows * 16; i += 32) {
              const int r = i >> 4, c = i & 15;
              if (n0 + c * 8 < p.N)
                *reinterpret_cast<uint4*>(out + ((int64_t)(tok0 + r) * p.N + n0 + c * 8) * 2) =
                    *reinterpret_cast<const uint4*>(my_staging + (c >> 3) * F8_WARP_STAGING + r * 128 + (((c & 7) ^ (r & 7)) << 4));
            }
            __syncwarp();
          }
        }
      } else {
        if (!live) continue;  // (the same for the two warps that share the tokens)
        const int tok = tok0 + lane, f0 = t_n0 + wg * 64;
        bool mine = lane < rows && whole;
        if (p.keep_e != nullptr && mine) {
          const bool is_bf16 = p.dtype_out == MOE_BF16;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (f0 + c * 8 < p.N) {  // features end at a multiple of 16
              uint32_t m[8];
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                const uint64_t a = acc[(r >> 2) * 32 + c * 4 + (r & 3)];
                m[r] = is_bf16 ? pack2<__nv_bfloat16>(lo_f32(a), hi_f32(a)) : pack2<__half>(lo_f32(a), hi_f32(a));
              }
              const int64_t at = ((int64_t)tok * p.N + f0 + c * 8) * 2;
              *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.keep_e) + at) = make_uint4(m[0], m[1], m[2], m[3]);
              *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.keep_g) + at) = make_uint4(m[4], m[5], m[6], m[7]);
            }
          }
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {  // (features past the last one have zeros in both)
          const float h0 = gated_silu<__half>(lo_f32(acc[i]), lo_f32(acc[32 + i]));  // (either 16-bit type)
          const float h1 = gated_silu<__half>(hi_f32(acc[i]), hi_f32(acc[32 + i]));
          top = max(top, max(magnitude_bits(h0), magnitude_bits(h1)));
          acc[i] = pack_f32x2(__float_as_uint(h0), __float_as_uint(h1));
        }
        // the scale's other 64 features are with the other warpgroup; the next tile's words are written behind the vote above
        uint32_t* tops = reinterpret_cast<uint32_t*>(staging);
        tops[wg * 128 + row] = whole ? top : 0xffffffffu;  // (above the bits of any magnitude)
        named_barrier_sync(1 + quarter, 64);
        const uint32_t other = tops[(wg ^ 1) * 128 + row];
        mine = mine && other != 0xffffffffu;
        top = max(top, other);
        float inv;
        const float scale = fp8_block_scale(top, inv);
        if (mine) {
          if (wg == 0) p.out_s[(int64_t)(t_n0 / 128) * p.pitch + tok] = scale;
          uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + (int64_t)tok * p.N + f0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (f0 + c * 16 < p.N) {
              uint32_t m[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint64_t a = acc[c * 8 + r * 2], b = acc[c * 8 + r * 2 + 1];
                m[r] = fp8_pack4(lo_f32(a) * inv, hi_f32(a) * inv, lo_f32(b) * inv, hi_f32(b) * inv);
              }
              *reinterpret_cast<uint4*>(out + c * 16) = make_uint4(m[0], m[1], m[2], m[3]);
            }
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }

  tc_fence_before_sync();
  cluster_sync_all();  // nobody frees TMEM or exits while the peer may still touch this CTA
  // A stage that was multiplied had landed.  Where somebody gave up, the ones that were loaded behind it are waited for; one that
  // only one of the CTAs loaded does not become full, and the limit is for all of them together.
  const int* done = ctl->stages_done;
  if (done[0] != done[2] || done[1] != done[2]) {
    if (leader && threadIdx.x == 0) {
      const unsigned long long t0 = global_ns();
      for (int i = done[2], n = max(done[0], done[1]); i < n; ++i)
        while (!mbar_try_wait_cluster(&ctl->full[i % p.stages], (uint32_t)(i / p.stages) & 1) && global_ns() - t0 <= WAIT_LIMIT_NS) {}
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

}  // namespace tc
}  // namespace moe
