// The products of tc_gemm_fp8.cuh for groups of few rows (decoding): one CTA, weight rows as accumulator rows.  Included by
// tc_gemm.cu behind that file, whose formulas, maps and parameters it shares.
//
// Such a product is bound by the weights, each of which is read once for a handful of tokens.  With tokens as accumulator rows
// a block costs 256 rows of MMAs whatever the tile holds, and its trip through two accumulators (MMAs, commit, TMEM loads,
// additions, release) takes 1250 cycles however few rows are added.  Here a tile is 128 weight rows x up to 64 tokens (32 for
// gate and up together, which need two sums for each): MMAs of 16 to 64 columns, four accumulators, and an epilogue thread that
// owns one weight row and adds 16 to 64 numbers per block.  Its factors differ from token to token; lane i loads those of tokens
// i and 32 + i, four blocks ahead, and shuffles hand them round.
// Two CTAs on an SM, 64 KB of weights under way in each, take the tiles in turn; the loads of the next tile are issued while the
// last blocks of one are added and stored (with a CTA to a tile: 97 us for 88).
// 384 rows, 128 experts, 2048 -> 1536, L2 flushed: 82 to 88 us from box to box, 4.4 to 4.7 TB/s of weights, 82 for the gradient
// (pair_fp8_kernel: 121, 128); gate and up of 768 features 86 (129), with 64 tokens to a tile 127; 768 -> 2048 51 (81).
// (A counter of stages that wraps round by a comparison, in place of the low bits of a running one, cost the thread that issues
// the MMAs 12 us of 93 at 4096 rows.)
#pragma once

namespace moe {
namespace tc {

constexpr int F8T_THREADS = 192;       // TMA, MMA, 4 epilogue warps
constexpr int F8T_STAGES = 4;          // and accumulators
constexpr int F8T_AHEAD = 4;           // blocks whose factors are under way
constexpr int F8T_W_BYTES = 128 * F8_BK;
constexpr uint32_t F8T_TMEM_COLS = 256;  // of 512: two CTAs
__host__ __device__ constexpr int fp8_thin_rows(bool gate_up) { return gate_up ? 32 : 64; }  // tokens of a tile
__host__ __device__ constexpr int fp8_thin_stage_bytes(bool gate_up) { return F8T_W_BYTES + fp8_thin_rows(gate_up) * F8_BK; }
static_assert(F8T_STAGES * fp8_thin_rows(false) <= F8T_TMEM_COLS, "an accumulator for each stage");

struct Fp8ThinControl {
  uint64_t full[F8T_STAGES];
  uint64_t empty[F8T_STAGES];
  uint64_t tmem_full[F8T_STAGES];
  uint64_t tmem_free[F8T_STAGES];  // 4 warps
  uint64_t drain;                  // the last MMAs
  alignas(16) uint32_t tops[fp8_thin_rows(true)][4];  // GATE_UP: largest magnitude of a token in each warp's features
  uint32_t tmem_base;
  int abort_flag;
};

static int fp8_thin_smem_bytes(bool gate_up, int E) {
  return F8T_STAGES * fp8_thin_stage_bytes(gate_up) + (int)sizeof(Fp8ThinControl) + 2 * (E + 1) * 4 + 1024;
}

// 16 columns of 32 rows, waited for.
__device__ __forceinline__ void tmem_ld_32x16_wait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

struct Fp8ThinTile {
  int e, t0, n0;
  int rows;   // at least one
  int boxes;  // of 16 rows
};

// W_MN, GATE_UP: as in pair_fp8_kernel.  With GATE_UP a block of the contraction is two stages, the gate's and the up
// projection's 128 features.
template <bool W_MN, bool GATE_UP>
__global__ void __launch_bounds__(F8T_THREADS, 2)
thin_fp8_kernel(const __grid_constant__ Fp8Maps maps, const Fp8Params p) {
  static_assert(!(W_MN && GATE_UP), "gate and up read K-major weights");
  constexpr int WEIGHTS = GATE_UP ? 2 : 1;
  constexpr int ROWS = fp8_thin_rows(GATE_UP), STAGES = F8T_STAGES, STAGE_BYTES = fp8_thin_stage_bytes(GATE_UP), AHEAD = F8T_AHEAD;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Fp8ThinControl* ctl = reinterpret_cast<Fp8ThinControl*>(smem + STAGES * STAGE_BYTES);
  int* row_start = reinterpret_cast<int*>(ctl + 1);
  int* tt_start = row_start + (p.E + 1);
  volatile int* abort_flag = &ctl->abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
      mbar_init(&ctl->tmem_full[s], 1);
      mbar_init(&ctl->tmem_free[s], 4);
    }
    mbar_init(&ctl->drain, 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.w[0]);
    tma_prefetch_desc(&maps.xs[0]);
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, F8T_TMEM_COLS);
    tmem_relinquish();
  }
  build_group_tables(p.m_sizes, p.ms64, p.E, p.M, ROWS, row_start, tt_start);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  const int n_tiles = (p.N + 127) / 128;
  const int total = tt_start[p.E] * n_tiles, stride = (int)gridDim.x;
  const int steps = p.kb * p.n_seg * WEIGHTS;

  // Within an expert the token tile varies fastest: neighbouring CTAs read the same weights.
  auto decode = [&](int tile) {
    Fp8ThinTile t;
    t.e = find_group(tt_start, p.E, tile / n_tiles);
    const int tt_e = tt_start[t.e + 1] - tt_start[t.e];
    const int j = tile - tt_start[t.e] * n_tiles;
    t.t0 = row_start[t.e] + (j % tt_e) * ROWS;
    t.n0 = (j / tt_e) * 128;
    t.rows = min(ROWS, row_start[t.e + 1] - t.t0);
    t.boxes = (t.rows + PAIR_SMALL_BOX - 1) / PAIR_SMALL_BOX;
    return t;
  };

  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < total && ok; tile += stride) {
        const Fp8ThinTile t = decode(tile);
        const uint32_t bytes = F8T_W_BYTES + t.boxes * PAIR_SMALL_BOX * F8_BK;
        for (int seg = 0; seg < p.n_seg && ok; ++seg) {
          for (int b = 0; b < p.kb * WEIGHTS; ++b, ++it) {
            const int s = it % STAGES, kb = b / WEIGHTS, w = GATE_UP ? b % WEIGHTS : seg;
            if (!mbar_wait(&ctl->empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, PW_EMPTY)) { ok = false; break; }
            uint8_t* sa = smem + s * STAGE_BYTES;
            mbar_expect_tx(&ctl->full[s], bytes);
            if constexpr (W_MN) tma_load_3d(sa, &maps.w[w], &ctl->full[s], t.n0, kb * F8_BK, t.e);
            else tma_load_3d(sa, &maps.w[w], &ctl->full[s], kb * F8_BK, t.n0, t.e);
            for (int x = 0; x < t.boxes; ++x)
              tma_load_2d(sa + F8T_W_BYTES + x * (PAIR_SMALL_BOX * F8_BK), &maps.xs[seg], &ctl->full[s], kb * F8_BK,
                          t.t0 + x * PAIR_SMALL_BOX);
          }
        }
      }
      // the copies on their way: an MMA thread that gave up does not wait for them
      for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait_through(&ctl->full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < total && ok; tile += stride) {
        const uint32_t idesc = p.idesc | ((uint32_t)(decode(tile).boxes * PAIR_SMALL_BOX >> 3) << 17);
        for (int b = 0; b < steps; ++b, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(&ctl->full[s], ph, abort_flag, PW_FULL)) { ok = false; break; }
          if (!mbar_wait(&ctl->tmem_free[s], ph ^ 1, abort_flag, PW_TMEM_EMPTY)) { ok = false; break; }
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(smem + s * STAGE_BYTES);
          const uint64_t da = make_smem_desc(sa, W_MN ? F8T_W_BYTES : 16, 1024);
          const uint64_t db = make_smem_desc(sa + F8T_W_BYTES, 16, 1024);
#pragma unroll
          for (int k = 0; k < F8_BK / F8_UMMA_K; ++k) {
            const uint64_t b_adv = (uint64_t)((k * F8_UMMA_K) >> 4);
            const uint64_t a_adv = W_MN ? (uint64_t)((k * F8_UMMA_K * 128) >> 4) : b_adv;
            umma_f8(tmem_base + s * ROWS, da + a_adv, db + b_adv, idesc, k != 0);
          }
          umma_commit(&ctl->empty[s]);
          umma_commit(&ctl->tmem_full[s]);
        }
      }
      umma_commit(&ctl->drain);  // an epilogue warp that gave up does not wait for the last MMAs
      mbar_wait_through(&ctl->drain, 0);
    }
  } else {
    // ------------------------------ epilogue ------------------------------
    const int quarter = warp & 3;  // of TMEM's lanes
    const int row = quarter * 32 + lane;
    const uint32_t taddr0 = tmem_base + ((uint32_t)(quarter * 32) << 16);
    float acc[WEIGHTS][ROWS];
    uint32_t it = 0;  // stages so far
    int boxes = 0;
    bool ok = true;
    struct Raw { float s0, s1, w[WEIGHTS]; };
    const float* sp = nullptr;
    const float* wp = nullptr;
    int off1 = 0;
    auto fetch = [&](int b) {  // (past the last block: the last one again, not used)
      Raw r;
      const uint32_t kb = (uint32_t)min(b, p.kb - 1);
      const float* at = sp + (uint64_t)kb * (uint32_t)p.pitch;
      r.s0 = __ldg(at);
      r.s1 = ROWS > 32 ? __ldg(at + off1) : 0.f;
#pragma unroll
      for (int w = 0; w < WEIGHTS; ++w) r.w[w] = __ldg(wp + (w ? p.ws[1] - p.ws[0] : 0) + kb * (uint32_t)p.ws_k);
      return r;
    };
    auto add_block = [&](Raw& raw, int ahead) {
      const Raw r = raw;
      raw = fetch(ahead);
#pragma unroll
      for (int w = 0; w < WEIGHTS; ++w) {
        const uint32_t s = it % STAGES;
        ok = ok && mbar_wait(&ctl->tmem_full[s], (it / STAGES) & 1, abort_flag, PW_TMEM_FULL);
        __syncwarp();
        tc_fence_after_sync();
        const float f0 = r.s0 * r.w[w], f1 = r.s1 * r.w[w];
#pragma unroll
        for (int g = 0; g < ROWS / 16; ++g) {
          if (g < boxes) {
            uint32_t v[16];
            tmem_ld_32x16_wait(taddr0 + s * ROWS + g * 16, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float f = __shfl_sync(0xffffffffu, g < 2 ? f0 : f1, (g & 1) * 16 + i);
              acc[w][g * 16 + i] = fmaf(__uint_as_float(v[i]), f, acc[w][g * 16 + i]);
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&ctl->tmem_free[s]);  // (not behind an abandoned wait: the other warps may still have to read it)
        ++it;
      }
    };
    Raw r[AHEAD] = {};
    auto fetch_first = [&]() {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) r[i] = fetch(i);
    };
    auto start = [&](const Fp8ThinTile& t, int seg) {
      const int tok = min(lane, t.rows - 1);
      off1 = min(lane + 32, t.rows - 1) - tok;
      sp = p.s[seg] + t.t0 + tok;
      wp = p.ws[seg] + t.e * p.ws_e + (int64_t)(t.n0 / 128) * p.ws_n;
    };
    Fp8ThinTile next = {};
    if ((int)blockIdx.x < total) {
      next = decode(blockIdx.x);
      start(next, 0);
      fetch_first();
    }
    for (int tile = blockIdx.x; tile < total; tile += stride) {
      const int t0 = next.t0, n0 = next.n0, rows = next.rows;
      boxes = next.boxes;
#pragma unroll
      for (int w = 0; w < WEIGHTS; ++w)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) acc[w][i] = 0.f;
      for (int seg = 0; seg < p.n_seg; ++seg) {
        if (seg > 0) {
          start(next, seg);
          fetch_first();
        }
#pragma unroll 1
        for (int b = 0; b < p.kb; b += AHEAD) {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i)
            if (i == 0 || b + i < p.kb) add_block(r[i], b + i + AHEAD);
        }
      }
      if (tile + stride < total) {  // the next tile's first factors, ahead of this one's stores
        next = decode(tile + stride);
        start(next, 0);
        fetch_first();
      }
      const int n = n0 + row;
      const bool mine = n < p.N;
      auto store = [&](void* to, const float (&v)[ROWS]) {
        if (p.dtype_out == MOE_F32) {
          float* out = reinterpret_cast<float*>(to) + (int64_t)t0 * p.N + n;
#pragma unroll
          for (int i = 0; i < ROWS; ++i) if (i < rows && mine) out[(int64_t)i * p.N] = v[i];
        } else if (p.dtype_out == MOE_BF16) {
          __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(to) + (int64_t)t0 * p.N + n;
#pragma unroll
          for (int i = 0; i < ROWS; ++i) if (i < rows && mine) out[(int64_t)i * p.N] = __float2bfloat16_rn(v[i]);
        } else {
          __half* out = reinterpret_cast<__half*>(to) + (int64_t)t0 * p.N + n;
#pragma unroll
          for (int i = 0; i < ROWS; ++i) if (i < rows && mine) out[(int64_t)i * p.N] = __float2half_rn(v[i]);
        }
      };
      // a warp that gave up has sums that nobody may see; those that share a barrier leave together
      const bool leave = __any_sync(0xffffffffu, !ok);
      if constexpr (!GATE_UP) {
        if (leave) break;
        store(p.out, acc[0]);
      } else {
        if (named_barrier_any(1, 128, leave)) break;
        if (p.keep_e != nullptr) {
          store(p.keep_e, acc[0]);
          store(p.keep_g, acc[WEIGHTS - 1]);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          if (i < rows) {  // (features past the last one have zeros in both)
            acc[0][i] = gated_silu<__half>(acc[0][i], acc[WEIGHTS - 1][i]);  // (either 16-bit type)
            const uint32_t top = __reduce_max_sync(0xffffffffu, magnitude_bits(acc[0][i]));
            if (lane == 0) ctl->tops[i][quarter] = top;
          }
        }
        named_barrier_sync(1, 128);
        uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + (int64_t)t0 * p.N + n;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          if (i < rows) {
            const uint4 t = *reinterpret_cast<const uint4*>(ctl->tops[i]);
            float inv;
            const float scale = fp8_block_scale(max(max(t.x, t.y), max(t.z, t.w)), inv);
            if (row == i) p.out_s[(int64_t)(n0 / 128) * p.pitch + t0 + i] = scale;
            if (mine) out[(int64_t)i * p.N] = (uint8_t)fp8_pack4(acc[0][i] * inv, 0.f, 0.f, 0.f);
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, F8T_TMEM_COLS);
  }
}

}  // namespace tc
}  // namespace moe
