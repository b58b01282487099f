// Products in 8-bit integers: Y[t, n] = (sum_k X[t, k] W[n, k]) * sx[t] * sw[n], codes with one scale a row on both sides. The sum of
// code products is exact in 32 bits up to K = 131,072 (127^2 K < 2^31), so it does not matter how it is cut; the two scales and
// the rounding to the output's type follow in float.
//
// For more than a few tokens (those: int8_stream.cu), behind the kernel that quantises them: tcgen05.mma.kind::i8, the codes of both sides
// brought in by TMA, accumulators in TMEM.
#include "quant.cuh"
#include "sm100.cuh"

using namespace rllm;
using namespace sm100;

namespace {

enum : int { EPI_STORE = 0, EPI_STORE_F32 = 1, EPI_ACCUM_F32 = 2, EPI_SWIGLU = 3 };

struct Int8Params {
  const float* sx; const float* sw;
  void* y; long long ldy;
  int vec;                           // rows of y start on 16 bytes, and so do scales of every fourth weight row (N % 4 == 0)
  int T, N, K;                       // N: outputs (of one half with SwiGLU); K: bytes a row, a multiple of 16
  int box;                           // token rows a copy brings
  int splits;                        // ranges of K
  int w_fixed;                       // nothing in front of this kernel writes the weight
  int* err;
};

// D (+)= A B with 8-bit signed operands and 32-bit sums.
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// s8 x s8 -> s32, A and B K-major, M x N tile.
__host__ __device__ constexpr uint32_t umma_idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

constexpr int BM = 128, BK = 128, UMMA_K = 32;      // token rows a tile, bytes of K a stage and an MMA
constexpr int THREADS_TC = 320;

template <int BN> struct TcCfg {                      // BN: weight rows a tile (gate and up rows together)
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES_RAW = 208 * 1024 / STAGE_BYTES;
  static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES;
  static constexpr int TMEM_COLS = 2 * BN <= 64 ? 64 : 2 * BN;
};

// CH neighbouring outputs of one token, in rows that start on 16 bytes.
template <int EPI, typename OUT, int CH>
__device__ __forceinline__ void emit_row(const Int8Params& p, int t, int n, const float (&v)[CH]) {
  OUT* y = (OUT*)p.y + (size_t)t * p.ldy + n;
  if (n + CH > p.N) {                                    // the last ones
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (n + i < p.N) {
        if constexpr (EPI == EPI_ACCUM_F32) atomicAdd(y + i, v[i]);
        else y[i] = from_f32<OUT>(v[i]);
      }
  } else if constexpr (EPI == EPI_ACCUM_F32) {
#pragma unroll
    for (int i = 0; i < CH; i += 4)
      asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(y + i), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]) : "memory");
  } else if constexpr (sizeof(OUT) == 4) {
#pragma unroll
    for (int i = 0; i < CH; i += 4) *reinterpret_cast<float4*>(y + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < CH; i += 8) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[i + 2 * e], v[i + 2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(y + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The same in rows that start anywhere: a warp's block of 32 tokens (one a lane) x 16 outputs is turned first, in four steps of exchanges
// between lanes, so that neighbouring lanes store neighbouring outputs. Number by number from each lane's row, 32 rows an
// instruction, 333 tokens of 1,111 with 1,001 outputs took 14.5 us (the quantising in front included), turned 7.6.
template <int EPI, typename OUT>
__device__ __forceinline__ void emit_turned(const Int8Params& p, int t_warp, int n, float (&v)[16], int lane) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!(i & o)) {
        const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i | o], o);
        if (up) v[i] = got; else v[i | o] = got;
      }
  }
  // v[i] is now output lane % 16 of the half warp's token i
  const int col = n + (lane & 15), first = t_warp + (lane & 16);
  if (col >= p.N) return;
  OUT* y = (OUT*)p.y + (size_t)first * p.ldy + col;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (first + i < p.T) {
      if constexpr (EPI == EPI_ACCUM_F32) atomicAdd(y + (size_t)i * p.ldy, v[i]);
      else y[(size_t)i * p.ldy] = from_f32<OUT>(v[i]);
    }
}

// Scales of the W weight rows from n on (what lies behind the last one is not used). Plain loads: the kernel in front may have written them.
template <int W>
__device__ __forceinline__ void scales(const Int8Params& p, int n, float (&s)[W]) {
  const int end = n < p.N ? p.N : 2 * p.N;               // (with SwiGLU up rows follow the gate rows)
  if (p.vec) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(p.sw + min(n + i, end - 4));
      s[i] = q.x; s[i + 1] = q.y; s[i + 2] = q.z; s[i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) s[i] = p.sw[min(n + i, end - 1)];
  }
}

template <int CH> __device__ __forceinline__ void tmem_cols(uint32_t taddr, uint32_t (&r)[CH]) {
  if constexpr (CH == 16) tmem_ld16(taddr, r); else tmem_ld32(taddr, r);
}

// One tile's accumulator from TMEM to the output, by eight warps: a thread's row is a token; the two warps of a quarter of the lanes take
// half of the features each.
template <int BN, int EPI, typename OUT>
__device__ __forceinline__ void tile_out(const Int8Params& p, uint32_t taddr, int t0, int n0, int warp, int lane) {
  constexpr bool DUAL = EPI == EPI_SWIGLU;
  constexpr int F = DUAL ? BN / 2 : BN;                // features a tile
  constexpr int CH = F / 2 >= 32 ? 32 : 16;
  static_assert(F / 2 >= 16, "a warp takes 16 features or more");
  const int t_warp = t0 + (warp & 3) * 32, t = t_warp + lane;
  if (t_warp >= p.T) return;
  const float sx = t < p.T ? p.sx[t] : 0.f;
  const int grp = (warp - 2) >> 2;
  auto numbers = [&](int c, int n, auto& v) {            // finished outputs c, c + 1 ... of the tile
    constexpr int W = sizeof(v) / sizeof(float);
    uint32_t a[W], b[DUAL ? W : 1];
    tmem_cols<W>(taddr + c, a);
    if constexpr (DUAL) tmem_cols<W>(taddr + F + c, b);
    float sa[W], sb[DUAL ? W : 1];
    scales(p, n, sa);
    if constexpr (DUAL) scales(p, n + p.N, sb);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < W; ++i) {
      v[i] = (float)(int)a[i] * sx * sa[i];
      if constexpr (DUAL) v[i] = silu_gate(v[i], (float)(int)b[i] * sx * sb[i], sizeof(OUT) == 4);
    }
  };
  const int end = min((grp + 1) * (F / 2), p.N - n0);
  if (p.vec) {
#pragma unroll 1
    for (int c = grp * (F / 2); c < end; c += CH) {
      float v[CH];
      numbers(c, n0 + c, v);
      if (t < p.T) emit_row<EPI, OUT, CH>(p, t, n0 + c, v);
    }
  } else {
#pragma unroll 1
    for (int c = grp * (F / 2); c < end; c += 16) {
      float v[16];
      numbers(c, n0 + c, v);
      emit_turned<EPI, OUT>(p, t_warp, n0 + c, v, lane);
    }
  }
}

// Tokens on the accumulator's rows, a tile of 128 tokens x BN weight rows; one CTA an SM walks the tiles, token tiles fastest (a weight tile
// is then read by neighbouring CTAs at once). Warp 0 issues the copies, warp 1 the MMAs, warps 2-9 take the finished
// accumulator out of TMEM while the next tile's is made. Few tokens fill a part of the 128 rows: the copies bring their rows only
// (`box`), the rows behind them hold whatever lay there, and their sums are not read.
template <int BN, int EPI, typename OUT>
__global__ void __launch_bounds__(THREADS_TC, 1)
int8_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Int8Params p) {
  constexpr bool DUAL = EPI == EPI_SWIGLU;
  constexpr int F = DUAL ? BN / 2 : BN;
  typedef TcCfg<BN> C;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ int never_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int t_tiles = (p.T + BM - 1) / BM, n_tiles = (p.N + F - 1) / F;
  const int tiles = t_tiles * n_tiles;
  const int n_kb = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 8); }
    abort_flag = 0;
    never_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) { prefetch_tensormap(&tmap_w); prefetch_tensormap(&tmap_x); }
  if (warp == 1) { tmem_alloc(&tmem_base_slot, C::TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch();
  const uint32_t tmem_base = tmem_base_slot;

  if (warp == 0) {
    if (elect_one()) {
      const uint64_t pol_x = policy_evict_last();    // the token tiles are read by every weight tile
      const uint32_t bytes = (uint32_t)(C::B_BYTES + p.box * BK);
      const uint32_t st0 = smem_u32(smem);
      // the first stages' weights need not wait for the kernel in front, unless it, or one before it, may still write them
      if (!p.w_fixed) pdl_wait();
      const int mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * n_kb;
      const int pre = min(mine, C::STAGES);
      auto weights = [&](int s, int tile, int kb) {
        const uint32_t dst = st0 + s * C::STAGE_BYTES + C::A_BYTES, full = smem_u32(&full_bar[s]);
        const int n0 = tile / t_tiles * F;
        tma_load_2d(dst, &tmap_w, full, kb * BK, n0);
        if (DUAL) tma_load_2d(dst + F * BK, &tmap_w, full, kb * BK, p.N + n0);
      };
      auto tokens = [&](int s, int tile, int kb) {
        tma_load_2d_hint(st0 + s * C::STAGE_BYTES, &tmap_x, smem_u32(&full_bar[s]), kb * BK, tile % t_tiles * BM, pol_x);
      };
      for (int i = 0; i < pre; ++i) {
        mbar_expect_tx(&full_bar[i], bytes);
        weights(i, blockIdx.x + i / n_kb * gridDim.x, i % n_kb);
      }
      pdl_wait();
      for (int i = 0; i < pre; ++i) tokens(i, blockIdx.x + i / n_kb * gridDim.x, i % n_kb);
      int it = pre, tile = blockIdx.x + pre / n_kb * gridDim.x, kb = pre % n_kb;
      for (; it < mine; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&empty_bar[s], (uint32_t)(it / C::STAGES - 1) & 1u, &abort_flag)) {
          abort_flag = 1; record_failure(p.err, 5); break;
        }
        mbar_expect_tx(&full_bar[s], bytes);
        weights(s, tile, kb);
        tokens(s, tile, kb);
        if (++kb == n_kb) { kb = 0; tile += gridDim.x; }
      }
      if (abort_flag)                                // let copies already issued land before the shared memory is given back
        for (int i = max(0, it - C::STAGES); i < it; ++i)
          mbar_wait(&full_bar[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, &never_flag, 200000000LL);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_i8(BM, BN);
      const uint64_t d0 = umma_desc_sw128(smem_u32(smem));
      int it = 0, ti = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++ti) {
        const int buf = ti & 1, use = ti >> 1;
        if (use > 0 && !mbar_wait(&acc_empty[buf], (uint32_t)(use - 1) & 1u, &abort_flag)) {
          abort_flag = 1; record_failure(p.err, 6); ok = false; break;
        }
        tc_fence_after();
        const uint32_t acc = tmem_base + (uint32_t)(buf * BN);
        for (int kb = 0; kb < n_kb; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&full_bar[s], (uint32_t)(it / C::STAGES) & 1u, &abort_flag)) { abort_flag = 1; record_failure(p.err, 2); ok = false; break; }
          tc_fence_after();
          const uint64_t da = d0 + (uint64_t)(s * (C::STAGE_BYTES >> 4)), db = da + (uint64_t)(C::A_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_i8(acc, da + (uint64_t)(k * UMMA_K / 16), db + (uint64_t)(k * UMMA_K / 16), idesc, kb > 0 || k > 0);
          umma_commit(&empty_bar[s]);
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
    }
  } else {
    pdl_wait();
    int ti = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++ti) {
      const int buf = ti & 1, use = ti >> 1;
      bool got = mbar_wait(&acc_full[buf], (uint32_t)use & 1u, &abort_flag);
      if (!got) { abort_flag = 1; record_failure(p.err, 3); }
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(buf * BN);
      tile_out<BN, EPI, OUT>(p, taddr, tile % t_tiles * BM, tile / t_tiles * F, warp, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, C::TMEM_COLS); }
}

// ---------------------------------------------------------------------------- many tokens, two SMs a tile
// The persistent scheme on pairs of CTAs (a cluster of two, cta_group::2): a tile is 256 tokens x 256 weight rows; each CTA of a pair loads its own
// 128 tokens and its own half of the weight rows (SwiGLU: the gate rows in the even CTA, the up rows in the odd one) and keeps the accumulator
// of its own tokens. The even CTA issues the MMAs, which read both CTAs' shared memory. A block of K takes 32 KB into and out of an SM's
// shared memory where a tile of 128 x 256 on one SM takes 48: 0.36 us a block for twice the work of that kernel's 0.45. 512 tokens, 2 x 14,336 x 4,096
// 56.6 -> 48.0 us (2.5 of the 3.3 Pop/s that twice the library's bfloat16 rate would be), 2,048 tokens 3.1 Pop/s with the tokens' quantising; with 16 blocks
// of K a tile's start and end weigh more: 2,048 tokens, 2 x 8,192 x 2,048 51.7 -> 50.4, scales read four at a time 48.
// Hand-overs as on the pairs of tc_gemm.cu: both CTAs' bytes are counted by the even CTA's `full` barrier, commits go to both CTAs' `empty`
// and `acc_full`, both CTAs' epilogue warps arrive at the even CTA's `acc_empty`; both meet before TMEM is freed.
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
struct PairCfg {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BM * BK, STAGE_BYTES = A_BYTES + B_BYTES, STAGES = 6;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES;
};
constexpr long long PAIR_WAIT_CYCLES = 1000000000LL;     // about half a second

template <int EPI, typename OUT>
__global__ void __launch_bounds__(THREADS_TC, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Int8Params p) {
  constexpr bool DUAL = EPI == EPI_SWIGLU;
  constexpr int F = DUAL ? 128 : 256;                    // features a tile
  typedef PairCfg C;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ int never_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int rank = (int)cluster_rank();
  const bool leader = rank == 0;
  const int pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int t_tiles = (p.T + 2 * BM - 1) / (2 * BM), n_tiles = (p.N + F - 1) / F;
  const int tiles = t_tiles * n_tiles;
  const int n_kb = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 16); }
    abort_flag = 0;
    never_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) { prefetch_tensormap(&tmap_w); prefetch_tensormap(&tmap_x); }
  if (warp == 1) { tmem_alloc_pair(&tmem_base_slot, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_sync_all();          // the peer's barriers exist before anything is signalled there
  pdl_launch();
  const uint32_t tmem_base = tmem_base_slot;

  if (warp == 0) {
    if (elect_one()) {
      constexpr uint32_t stage_bytes = 2u * C::STAGE_BYTES;            // of both CTAs
      const int mine = (tiles - pair_id + n_pairs - 1) / n_pairs * n_kb;
      const int pre = min(mine, C::STAGES);
      const uint32_t st0 = smem_u32(smem), even0 = map_to_rank(smem_u32(full_bar), 0);
      auto weights = [&](int s, int tile, int kb) {
        const int n0 = tile / t_tiles * F;
        tma_load_2d_pair(st0 + s * C::STAGE_BYTES + C::A_BYTES, &tmap_w, even0 + 8 * s, kb * BK, DUAL ? n0 + rank * p.N : n0 + rank * BM);
      };
      auto tokens = [&](int s, int tile, int kb) {
        tma_load_2d_pair(st0 + s * C::STAGE_BYTES, &tmap_x, even0 + 8 * s, kb * BK, tile % t_tiles * 2 * BM + rank * BM);
      };
      if (!p.w_fixed) pdl_wait();                        // (see the kernel above)
      for (int i = 0; i < pre; ++i) {
        if (leader) mbar_expect_tx(&full_bar[i], stage_bytes);
        weights(i, pair_id + i / n_kb * n_pairs, i % n_kb);
      }
      pdl_wait();
      for (int i = 0; i < pre; ++i) tokens(i, pair_id + i / n_kb * n_pairs, i % n_kb);
      int it = pre, tile = pair_id + pre / n_kb * n_pairs, kb = pre % n_kb;
      for (; it < mine; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&empty_bar[s], (uint32_t)(it / C::STAGES - 1) & 1u, &abort_flag, PAIR_WAIT_CYCLES)) {
          abort_flag = 1; record_failure(p.err, 5, rank); break;
        }
        if (leader) mbar_expect_tx(&full_bar[s], stage_bytes);
        weights(s, tile, kb);
        tokens(s, tile, kb);
        if (++kb == n_kb) { kb = 0; tile += n_pairs; }
      }
      if (abort_flag && leader)                          // let copies already issued land before the shared memory is given back
        for (int i = max(0, it - C::STAGES); i < it; ++i)
          mbar_wait(&full_bar[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, &never_flag, 200000000LL);
    }
  } else if (warp == 1) {
    if (elect_one() && leader) {
      constexpr uint32_t idesc = umma_idesc_i8(2 * BM, 256);
      const uint64_t d0 = umma_desc_sw128(smem_u32(smem));
      int it = 0, ti = 0;
      bool ok = true;
      for (int tile = pair_id; tile < tiles && ok; tile += n_pairs, ++ti) {
        const int buf = ti & 1, use = ti >> 1;
        if (use > 0 && !mbar_wait(&acc_empty[buf], (uint32_t)(use - 1) & 1u, &abort_flag, PAIR_WAIT_CYCLES)) {
          abort_flag = 1; record_failure(p.err, 6); ok = false; break;
        }
        tc_fence_after();
        const uint32_t acc = tmem_base + (uint32_t)(buf * 256);
        for (int kb = 0; kb < n_kb; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&full_bar[s], (uint32_t)(it / C::STAGES) & 1u, &abort_flag, PAIR_WAIT_CYCLES)) { abort_flag = 1; record_failure(p.err, 2); ok = false; break; }
          tc_fence_after();
          const uint64_t da = d0 + (uint64_t)(s * (C::STAGE_BYTES >> 4)), db = da + (uint64_t)(C::A_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_i8_pair(acc, da + (uint64_t)(k * UMMA_K / 16), db + (uint64_t)(k * UMMA_K / 16), idesc, kb > 0 || k > 0);
          umma_commit_pair_both(smem_u32(&empty_bar[s]));
        }
        if (ok) umma_commit_pair_both(smem_u32(&acc_full[buf]));
      }
    }
  } else {
    const uint32_t drained = map_to_rank(smem_u32(&acc_empty[0]), 0);
    pdl_wait();
    int ti = 0;
    for (int tile = pair_id; tile < tiles; tile += n_pairs, ++ti) {
      const int buf = ti & 1, use = ti >> 1;
      bool got = mbar_wait(&acc_full[buf], (uint32_t)use & 1u, &abort_flag, PAIR_WAIT_CYCLES);
      if (!got) { abort_flag = 1; record_failure(p.err, 3, rank); }
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(buf * 256);
      tile_out<256, EPI, OUT>(p, taddr, tile % t_tiles * 2 * BM + rank * BM, tile / t_tiles * F, warp, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(drained + (uint32_t)(buf * 8));
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // both CTAs are done with each other's shared memory, barriers and TMEM
  if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem_base, 512); }
}

// ---------------------------------------------------------------------------- few tiles: ranges of K
// A CTA's time goes with its blocks of K, 0.22 us each with 64 weight rows and 0.45 with 256, however few its tokens. Where the tiles
// leave most SMs idle and K is long, a tile is shared by the CTAs of a cluster, each with a range of K. The parts are whole numbers, so
// their sum does not depend on the cut. Rank r finishes the r-th part of the tile's features: every rank pushes its accumulator's
// columns to their owners through distributed shared memory, into the stage ring, which is idle once all ranks' products are
// complete (one cluster barrier), and the owners add them up behind a second one. A landing area holds [rank][four columns][128 rows] x 16 bytes,
// a warp's rows side by side (with a column's rows side by side, 4 bytes a push, the exchange alone took 15 us).
template <int BN, int EPI, typename OUT>
__global__ void __launch_bounds__(THREADS_TC, 1)
int8_split_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Int8Params p) {
  constexpr bool DUAL = EPI == EPI_SWIGLU;
  constexpr int F = DUAL ? BN / 2 : BN;
  typedef TcCfg<BN> C;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[C::STAGES];
  __shared__ __align__(8) uint64_t empty_bar[C::STAGES];
  __shared__ __align__(8) uint64_t acc_full;
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ int never_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int splits = p.splits, rank = (int)cluster_rank(), tile = blockIdx.x;
  const int t_tiles = (p.T + BM - 1) / BM;
  const int t0 = tile % t_tiles * BM, n0 = tile / t_tiles * F;
  const int n_kb = (p.K + BK - 1) / BK, kb0 = rank * n_kb / splits, mine = (rank + 1) * n_kb / splits - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(&acc_full, 1);
    abort_flag = 0;
    never_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) { prefetch_tensormap(&tmap_w); prefetch_tensormap(&tmap_x); }
  if (warp == 1) { tmem_alloc(&tmem_base_slot, C::TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch();
  const uint32_t tmem_base = tmem_base_slot;
  bool got = false;

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t bytes = (uint32_t)(C::B_BYTES + p.box * BK), st0 = smem_u32(smem);
      const int pre = min(mine, C::STAGES);
      auto weights = [&](int s, int kb) {
        const uint32_t dst = st0 + s * C::STAGE_BYTES + C::A_BYTES, full = smem_u32(&full_bar[s]);
        tma_load_2d(dst, &tmap_w, full, kb * BK, n0);
        if (DUAL) tma_load_2d(dst + F * BK, &tmap_w, full, kb * BK, p.N + n0);
      };
      if (!p.w_fixed) pdl_wait();
      for (int i = 0; i < pre; ++i) { mbar_expect_tx(&full_bar[i], bytes); weights(i, kb0 + i); }
      pdl_wait();
      for (int i = 0; i < pre; ++i) tma_load_2d(st0 + i * C::STAGE_BYTES, &tmap_x, smem_u32(&full_bar[i]), (kb0 + i) * BK, t0);
      int it = pre;
      for (; it < mine; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&empty_bar[s], (uint32_t)(it / C::STAGES - 1) & 1u, &abort_flag)) {
          abort_flag = 1; record_failure(p.err, 5); break;
        }
        mbar_expect_tx(&full_bar[s], bytes);
        weights(s, kb0 + it);
        tma_load_2d(st0 + s * C::STAGE_BYTES, &tmap_x, smem_u32(&full_bar[s]), (kb0 + it) * BK, t0);
      }
      if (abort_flag)
        for (int i = max(0, it - C::STAGES); i < it; ++i)
          mbar_wait(&full_bar[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, &never_flag, 200000000LL);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_i8(BM, BN);
      const uint64_t d0 = umma_desc_sw128(smem_u32(smem));
      bool ok = true;
      for (int it = 0; it < mine; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&full_bar[s], (uint32_t)(it / C::STAGES) & 1u, &abort_flag)) { abort_flag = 1; record_failure(p.err, 2); ok = false; break; }
        tc_fence_after();
        const uint64_t da = d0 + (uint64_t)(s * (C::STAGE_BYTES >> 4)), db = da + (uint64_t)(C::A_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k)
          umma_i8(tmem_base, da + (uint64_t)(k * UMMA_K / 16), db + (uint64_t)(k * UMMA_K / 16), idesc, it > 0 || k > 0);
        umma_commit(&empty_bar[s]);
      }
      if (ok) umma_commit(&acc_full);
    }
  } else {
    pdl_wait();
    got = mbar_wait(&acc_full, 0u, &abort_flag);
    if (!got) { abort_flag = 1; record_failure(p.err, 3); }
    got = __all_sync(0xffffffffu, got);
    tc_fence_after();
  }
  __syncwarp();
  cluster_sync_all();                                    // every rank's products have read its ring
  const int part = F / splits;                           // features that a rank finishes
  const int row = (warp & 3) * 32 + lane, grp = (warp - 2) >> 2;
  const bool rows_live = warp >= 2 && t0 + (warp & 3) * 32 < p.T;
  const uint32_t land = smem_u32(smem);
  if (rows_live && got) {
    const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
    for (int c = 16 * grp; c < BN; c += 32) {            // 16 columns at a time, dealt out to the two warps of a quarter
      uint32_t a[16];
      tmem_ld16(taddr + c, a);
      tmem_ld_wait();
      const int f = c % F, owner = f / part;
      const int col = rank * (BN / splits) + c / F * part + f % part;
      const uint32_t dst = map_to_rank(land + (uint32_t)((col >> 2) * 128 + row) * 16, (uint32_t)owner);
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 512 * i), "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]) : "memory");
    }
  }
  __syncwarp();
  cluster_sync_all();                                    // every part has landed
  if (rows_live && got) {
    const int t = t0 + row;
    const float sx = t < p.T ? p.sx[t] : 0.f;
    const int4* src = reinterpret_cast<const int4*>(smem) + row;
    auto add_up = [&](int col, int (&a)[16]) {           // 16 columns from `col` of a rank's area on, over the ranks
#pragma unroll
      for (int i = 0; i < 16; ++i) a[i] = 0;
      for (int z = 0; z < splits; ++z) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int4 q = src[((z * (BN / splits) + col) / 4 + i) * 128];
          a[4 * i] += q.x; a[4 * i + 1] += q.y; a[4 * i + 2] += q.z; a[4 * i + 3] += q.w;
        }
      }
    };
#pragma unroll 1
    for (int c = 16 * grp; c < part; c += 32) {
      const int n = n0 + rank * part + c;
      if (n >= p.N) break;
      int a[16], b[DUAL ? 16 : 1];
      add_up(c, a);
      if constexpr (DUAL) add_up(part + c, b);
      float v[16], sa[16], sb[DUAL ? 16 : 1];
      scales(p, n, sa);
      if constexpr (DUAL) scales(p, n + p.N, sb);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = (float)a[i] * sx * sa[i];
        if constexpr (DUAL) v[i] = silu_gate(v[i], (float)b[i] * sx * sb[i], sizeof(OUT) == 4);
      }
      if (!p.vec) emit_turned<EPI, OUT>(p, t - lane, n, v, lane);
      else if (t < p.T) emit_row<EPI, OUT, 16>(p, t, n, v);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, C::TMEM_COLS); }
}

// ------------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return (EncodeTiledFn)f;
  }();
  return fn;
}

// codes [rows, K], a copy brings 128 bytes of `box` rows
int make_map(CUtensorMap* m, const void* ptr, long long rows, int K, int box) {
  const EncodeTiledFn enc = encoder();
  if (!enc) return -5;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K};
  const cuuint32_t b[2] = {(cuuint32_t)BK, (cuuint32_t)box}, one[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -5;
}

template <int BN, int EPI, typename OUT>
int launch_tc(const void* x, const void* w, Int8Params p, int sm_count, cudaStream_t s) {
  typedef TcCfg<BN> C;
  constexpr int F = EPI == EPI_SWIGLU ? BN / 2 : BN;
  static bool configured[64] = {}, configured_split[64] = {};
  p.box = p.T >= BM ? BM : (p.T + 7) / 8 * 8;
  CUtensorMap mx, mw;
  int rc = make_map(&mx, x, p.T, p.K, p.box);
  if (!rc) rc = make_map(&mw, w, EPI == EPI_SWIGLU ? 2ll * p.N : p.N, p.K, F);
  if (rc) return rc;
  const long long tiles = (long long)((p.T + BM - 1) / BM) * ((p.N + F - 1) / F);
  if (tiles > 2147483647LL) return ERR_TOO_LARGE;
  if (p.splits > 1) {
    if (allow_dynamic_smem(int8_split_kernel<BN, EPI, OUT>, C::SMEM_BYTES, configured_split)) return -5;
    return launch_ex(int8_split_kernel<BN, EPI, OUT>, dim3((unsigned)tiles, 1, p.splits), dim3(THREADS_TC), C::SMEM_BYTES, s, p.splits, mx, mw, p);
  }
  if (allow_dynamic_smem(int8_tc_kernel<BN, EPI, OUT>, C::SMEM_BYTES, configured)) return -5;
  return launch_ex(int8_tc_kernel<BN, EPI, OUT>, dim3((unsigned)(tiles < sm_count ? tiles : sm_count)), dim3(THREADS_TC), C::SMEM_BYTES, s, 1, mx, mw, p);
}

template <int EPI, typename OUT>
int launch_pair(const void* x, const void* w, Int8Params p, int sm_count, cudaStream_t s) {
  static bool configured[64] = {};
  if (allow_dynamic_smem(int8_pair_kernel<EPI, OUT>, PairCfg::SMEM_BYTES, configured)) return -5;
  constexpr int F = EPI == EPI_SWIGLU ? 128 : 256;
  CUtensorMap mx, mw;
  int rc = make_map(&mx, x, p.T, p.K, BM);
  if (!rc) rc = make_map(&mw, w, EPI == EPI_SWIGLU ? 2ll * p.N : p.N, p.K, BM);
  if (rc) return rc;
  const long long tiles = (long long)((p.T + 2 * BM - 1) / (2 * BM)) * ((p.N + F - 1) / F);
  if (tiles > 1073741823LL) return ERR_TOO_LARGE;
  const long long pairs = tiles < sm_count / 2 ? tiles : sm_count / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(THREADS_TC);
  cfg.dynamicSmemBytes = PairCfg::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 2; attrs[0].val.clusterDim.y = 1; attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, int8_pair_kernel<EPI, OUT>, mx, mw, p);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return 0;
}

// Weight rows a tile (512: pairs of CTAs, 256 x 256) and ranges of K, by an estimate of the time in us: the blocks of K of the CTA with the most
// of them, `block` each (how many tokens hardly matters, nor how many CTAs are busy), a start and an end, and with ranges the
// exchange of an accumulator. Fitted to 20 sizes of 32 to 2,048 tokens, each timed at every width and number of ranges; the choice was the best of
// them, or within 8 % of it. Best | widths 64, 128, 256, pairs without ranges, us: 64 tokens, 2,048 x 8,192 7.9 (64 rows, 4 ranges) | 15.9, 18.1, 28.9;
// 256 tokens of it 11.0 (128, 4) | 16.5, 19.3, 31.2, 27.0; 2,048 tokens of it 29.4 (pairs) | 55.7, 35.5, 31.1, 29.4; 2,048 tokens, 2 x 8,192 x 2,048
// 50.4 (pairs) | 102, 64.3, 51.7, 50.4; 512 tokens, 2 x 14,336 x 4,096 48.0 (pairs) | 92.3, 60.9, 56.6, 48.0.
void plan(int epi, int T, int N, int K, int sm_count, int& bn, int& splits) {
  const int half = epi == EPI_SWIGLU ? 2 : 1, rows = half * N, box = T >= BM ? BM : (T + 7) / 8 * 8;
  const long long n_kb = (K + BK - 1) / BK;
  double best = 1e30;
  auto offer = [&](int b, int z, long long rounds, double block, double rest) {
    const double cost = (double)(rounds * ((n_kb + z - 1) / z)) * block + rest;
    if (cost < best) { best = cost; bn = b; splits = z; }
  };
  for (int b = 64; b <= 256; b <<= 1)
    for (int z = 1; z <= 4; z <<= 1) {
      const long long tiles = (long long)((T + BM - 1) / BM) * ((rows + b - 1) / b);
      if (z > 1 && (b / half / z < 16 || n_kb < 4 * z || tiles * z > sm_count)) break;
      const double exchange = z > 1 ? 0.5 * z + 1.2e-4 * b * box * (z - 1) / z : 0.0;
      offer(b, z, (tiles * z + sm_count - 1) / sm_count, b == 64 ? 0.215 : b == 128 ? 0.28 : 0.45, 1.8 + 0.005 * b + exchange);
    }
  if (T > BM && sm_count >= 2) {
    const long long tiles = (long long)((T + 2 * BM - 1) / (2 * BM)) * ((rows + 255) / 256), pairs = sm_count / 2;
    offer(512, 1, (tiles + pairs - 1) / pairs, 0.375, 4.5);
  }
}

template <int EPI, typename OUT>
int launch_epi(const void* x, const void* w, Int8Params p, int sm_count, cudaStream_t s) {
  int bn = 64;
  plan(EPI, p.T, p.N, p.K, sm_count, bn, p.splits);
  switch (bn) {
    case 512: return launch_pair<EPI, OUT>(x, w, p, sm_count, s);
    case 256: return launch_tc<256, EPI, OUT>(x, w, p, sm_count, s);
    case 128: return launch_tc<128, EPI, OUT>(x, w, p, sm_count, s);
    default: return launch_tc<64, EPI, OUT>(x, w, p, sm_count, s);
  }
}

}  // namespace

// The tile and the ranges that rllm_int8_gemm takes (for measurement).
RLLM_API int rllm_int8_plan(int epi, int T, int N, int K, int sm_count, int* bn, int* splits) {
  if (epi < 0 || epi > 3 || T <= 0 || N <= 0 || K <= 0 || sm_count <= 0) return ERR_BAD_SIZE;
  *bn = 64; *splits = 1;
  plan(epi, T, N, K, sm_count, *bn, *splits);
  return 0;
}

// x int8 [T, K] with scales sx [T]; w int8 [N, K] (SwiGLU: [2 N, K], gate rows first) with scales sw; K a multiple of 16, both
// 16-byte aligned. y [T, N] in out_dt (epilogues 0 and 3) or float (1, 2: added), row stride ldy. w_fixed: w's codes are not written by work
// that may still be running, so that they are read before the kernel in front has ended.
RLLM_API int rllm_int8_gemm(int epi, int out_dt, const void* x, const float* sx, const void* w, const float* sw, void* y, long long ldy,
                            int T, int N, int K, int w_fixed, int* err, int sm_count, void* stream) {
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 16 || K > 131072 || ldy < N || epi < 0 || epi > 3 || N > (1 << 30)) return ERR_BAD_SIZE;
  if (((uintptr_t)x | (uintptr_t)w) & 15) return ERR_BAD_ALIGN;
  if (out_dt != DT_F32 && out_dt != DT_BF16) return ERR_BAD_DTYPE;
  const int size = epi == EPI_STORE_F32 || epi == EPI_ACCUM_F32 || out_dt == DT_F32 ? 4 : 2;
  const Int8Params p = {sx, sw, y, ldy, !(((uintptr_t)y | (uintptr_t)sw) & 15) && ldy * size % 16 == 0 && N % 4 == 0, T, N, K, 0, 1, w_fixed, err};
  cudaStream_t s = (cudaStream_t)stream;
  if (epi == EPI_STORE_F32) return launch_epi<EPI_STORE_F32, float>(x, w, p, sm_count, s);
  if (epi == EPI_ACCUM_F32) return launch_epi<EPI_ACCUM_F32, float>(x, w, p, sm_count, s);
  if (epi == EPI_STORE) return out_dt == DT_F32 ? launch_epi<EPI_STORE, float>(x, w, p, sm_count, s) : launch_epi<EPI_STORE, bf16>(x, w, p, sm_count, s);
  return out_dt == DT_F32 ? launch_epi<EPI_SWIGLU, float>(x, w, p, sm_count, s) : launch_epi<EPI_SWIGLU, bf16>(x, w, p, sm_count, s);
}

// The two launchers that a product from numbers goes through (quant_rows.cu, int8_stream.cu).
RLLM_API int rllm_quantize_rows(int dt, const void* x, long long ldx, const int* rows, const void* g, int g_dt, float eps, void* codes,
                                long long ldc, float* scales, int T, int K, int early, void* stream);
RLLM_API int rllm_int8_streams(int T, int xk, int x_dt, const void* x, long long ldx, const void* g);
RLLM_API int rllm_int8_stream(int epi, int out_dt, int x_dt, const void* x, long long ldx, const int* rows, const void* g, int g_dt, float eps,
                              const void* w, const float* sw, void* y, long long ldy, int T, int N, int xk, int K, int w_fixed, int sm_count,
                              void* stream);

RLLM_API int rllm_int8_streams_codes(int epi, int T, int N, int K, int sm_count);
RLLM_API int rllm_int8_stream_codes(int epi, int out_dt, const void* x, const float* sx, const void* w, const float* sw, void* y, long long ldy,
                                    int T, int N, int K, int w_fixed, int sm_count, void* stream);

// y = x w^T from numbers x [*, xk] (as rllm_quantize_rows takes them): in one kernel for few tokens, else quantised into codes [T, K] and scales [T]
// first. Without scratch (codes null) a product that wants it is not run: 1000000.
RLLM_API int rllm_int8_linear(int epi, int out_dt, int x_dt, const void* x, long long ldx, const int* rows, const void* g, int g_dt, float eps,
                              void* codes, float* scales, const void* w, const float* sw, void* y, long long ldy, int T, int N, int xk,
                              int K, int w_fixed, int* err, int sm_count, void* stream) {
  if (T <= 0 || N <= 0) return 0;
  if (rllm_int8_streams(T, xk, x_dt, x, ldx, g))
    return rllm_int8_stream(epi, out_dt, x_dt, x, ldx, rows, g, g_dt, eps, w, sw, y, ldy, T, N, xk, K, w_fixed, sm_count, stream);
  if (codes == nullptr) return 1000000;
  const int rc = rllm_quantize_rows(x_dt, x, ldx, rows, g, g_dt, eps, codes, K, scales, T, xk, 1, stream);
  if (!rc && rllm_int8_streams_codes(epi, T, N, K, sm_count))
    return rllm_int8_stream_codes(epi, out_dt, codes, scales, w, sw, y, ldy, T, N, K, w_fixed, sm_count, stream);
  return rc ? rc : rllm_int8_gemm(epi, out_dt, codes, scales, w, sw, y, ldy, T, N, K, w_fixed, err, sm_count, stream);
}
