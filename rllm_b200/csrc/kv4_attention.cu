// Attention over the paged cache held in 4 bits (layout: quant.cuh).
//
// Single tokens, heads of 64 and 128 in bfloat16 (kv4_decode_kernel): one pass over the codes, which stay codes until they are fragments of
// mma.sync. A CTA has one (sequence, kv head, range of keys), a warp tiles of keys of its own, which per-lane
// asynchronous copies bring into a ring; the ranges of a sequence form a cluster and meet in distributed shared memory.
//   * S^T = K Q^T, keys on the rows (16 of them an instruction), 4 query heads of the kv head twice on the 8 columns: columns 0-3 take the
//     first of a block's two groups of 32 dimensions, columns 4-7 the second. A word holds four codes of either group, so a pair of
//     numbers that a fragment's register wants is a word's nibble i of both halves, as it lies there: the queries' fragment holds a
//     zero for the group that is not its column's. Nothing is permuted, every column does work with 4 query heads a kv head, and each
//     lane multiplies by one group's scale; the two groups' sums meet by one shuffle.
//   * Fragments hold codes, exact half numbers: nibbles 0 and 1 of a half word are the last four bits of 1024 + n and four higher ones of 64 + n
//     by one AND-OR each for two numbers, nibbles 2 and 3 the same after a shift by 8; less 1032 and 72 they are the codes. (In bfloat16, with 7 bits
//     behind the first, three of the four nibbles would want a shift; shifts, ANDs and permutations share the kernel's busiest pipe: with
//     those and with pairs put together from two words, 64 sequences of 4,096 keys, 8 x 128, took 115 us, now 85.) Queries are half numbers
//     times a power of two a row, which is exact down to 2^-14 of the row's largest. A group's sum is as exact as float; it is multiplied
//     by the group's scale as a float number. No dequantised key exists.
//   * O^T = V^T P^T, dimensions within a group on the rows; the contraction is over (key, group) pairs, so that a register is again a word's
//     nibble of both halves, and a column's weights are zero for the group that is not its own: columns 0-3 become the
//     output's first 32 dimensions of a block, columns 4-7 the second. The scale of a (key, group) goes onto the weight in float, before its
//     one rounding, to half precision (bfloat16 cost 0.0016 of the output's norm). So that the product stays in half's range whatever the
//     sizes of a group's scales, each group of 32 dimensions has a running maximum of score + log2 of its scale beside the scores' own, and
//     its sums are against that one. movmatrix turns the rounded weights from rows of keys into the columns that the second product takes.
//   * Which key a row of the fragment stands for is free, as long as both products agree, and is chosen so that neither product's reads of
//     shared memory meet a bank twice.
//   * The running maximum moves only when a score passes it by 8 (in the log2 domain): weights reach 256 then, which is as good as 1, and
//     the lanes' maxima meet once in a while instead of in every tile.
// 64 sequences of 2,048 keys, 32 / 8 heads of 128: 52 us, 2.9 TB/s, an instruction issued in 60 % of the cycles, the pipe of shifts, ANDs and permutations
// busy 47 %: nothing is full, 14 of 64 warps wait for their own chains. One sequence of 300 keys 4.1 us, eight of 4,096 (32 / 8 heads of 64) 12.
//
// On the CUDA cores, for any mix of prompt portions and single tokens, both run types and head sizes of 64, 128, 192 and 256: one
// warp per (query token, query head), keys 32 at a time in position order with a running maximum and sum, all arithmetic in
// float, as paged_attention_simt_kernel does over a cache of whole numbers. A lane scores one key: the key's codes times the
// queries of a group of 32 are summed first and multiplied by the group's scale once. The weighted sum of the values takes one
// byte of a row's block a lane, which is two neighbouring dimensions.
#include "quant.cuh"
#include "sm100.cuh"
#include <cuda_fp16.h>

using namespace rllm;
using namespace sm100;

namespace {

struct Kv4Params {
  const void* q; int q_stride;
  const uint8_t* k4; const bf16* ks; const uint8_t* v4; const bf16* vs;
  long long num_pages;
  void* out; int out_stride;
  const int* token_seq; const int* positions;       // CUDA cores: [T]
  const int* kv_lens;                                // single tokens: [S]
  const int* block_table; int bt_stride;
  int rows, nh, nkv, page_size, window;
  float scale;
  int page_shift, splits;
};

constexpr int WARPS = 4;

template <typename T, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32)
kv4_attention_simt_kernel(const Kv4Params p) {
  pdl_launch();
  pdl_wait();
  constexpr int HD = 64 * BLOCKS;
  __shared__ float qs[WARPS][HD];                    // in the order of the codes: [block][word][nibble]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long gw = (long long)blockIdx.x * WARPS + warp;
  if (gw >= (long long)p.rows * p.nh) return;
  const int t = (int)(gw / p.nh), h = (int)(gw % p.nh);
  const int kvh = h / (p.nh / p.nkv);
  const int pos = p.positions[t];
  const int start = (p.window > 0 && pos - p.window + 1 > 0) ? pos - p.window + 1 : 0;
  const int* bt = p.block_table + (size_t)p.token_seq[t] * p.bt_stride;

  const T* qp = (const T*)p.q + (size_t)t * p.q_stride + (size_t)h * HD;
  for (int d = lane; d < HD; d += 32) {
    const int r = d & 63;
    qs[warp][(d & ~63) + ((r & 31) >> 2) * 8 + (r >> 5) * 4 + (r & 3)] = to_f32(qp[d]) * p.scale;
  }
  __syncwarp();
  float acc[2 * BLOCKS];
#pragma unroll
  for (int i = 0; i < 2 * BLOCKS; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int base = start; base <= pos; base += 32) {
    const int j = base + lane;
    const bool valid = j <= pos;
    float s = valid ? 0.f : -INFINITY;
    long long row = -1;
    const int page = valid ? bt[j / p.page_size] : -1;
    if (page >= 0 && page < p.num_pages) {                 // a table entry without a page reads as zeros
      row = ((long long)page * p.nkv + kvh) * p.page_size + j % p.page_size;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const uint4* kp = reinterpret_cast<const uint4*>(p.k4 + row * (HD / 2) + 32 * b);
        const uint4 a = __ldcg(kp), c = __ldcg(kp + 1);
        const uint32_t two = __ldcg(reinterpret_cast<const uint32_t*>(p.ks + row * (HD / 32)) + b);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 q0 = *reinterpret_cast<const float4*>(&qs[warp][64 * b + 8 * i]);
          const float4 q1 = *reinterpret_cast<const float4*>(&qs[warp][64 * b + 8 * i + 4]);
          s0 = fmaf((float)code4(w[i], 0), q0.x, s0); s0 = fmaf((float)code4(w[i], 1), q0.y, s0);
          s0 = fmaf((float)code4(w[i], 2), q0.z, s0); s0 = fmaf((float)code4(w[i], 3), q0.w, s0);
          s1 = fmaf((float)code4(w[i], 4), q1.x, s1); s1 = fmaf((float)code4(w[i], 5), q1.y, s1);
          s1 = fmaf((float)code4(w[i], 6), q1.z, s1); s1 = fmaf((float)code4(w[i], 7), q1.w, s1);
        }
        s = fmaf(s0, bf16_lo(two), fmaf(s1, bf16_hi(two), s));
      }
    }
    const float m_new = fmaxf(m, warp_max(s));
    const bool none = m_new == -INFINITY;                  // no key yet
    const float pr = !valid ? 0.f : none ? s - s : expf(s - m_new);      // (a first chunk of NaN scores gives NaN)
    const float corr = none ? 1.f : expf(m - m_new);
    l = l * corr + warp_sum(pr);
#pragma unroll
    for (int i = 0; i < 2 * BLOCKS; ++i) acc[i] *= corr;
    const int cnt = min(32, pos - base + 1);
    for (int jj = 0; jj < cnt; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, pr, jj);
      const long long rj = __shfl_sync(0xffffffffu, row, jj);
      if (rj < 0) continue;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const uint32_t two = __ldcg(reinterpret_cast<const uint32_t*>(p.vs + rj * (HD / 32)) + b);
        const int byte = __ldcg(p.v4 + rj * (HD / 2) + 32 * b + lane);
        const float f = pj * (lane & 2 ? bf16_hi(two) : bf16_lo(two));
        acc[2 * b] = fmaf(f, (float)((byte & 15) - 8), acc[2 * b]);
        acc[2 * b + 1] = fmaf(f, (float)((byte >> 4) - 8), acc[2 * b + 1]);
      }
    }
    m = m_new;
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);       // no visible key: zeros; a NaN stays one
  T* op = (T*)p.out + (size_t)t * p.out_stride + (size_t)h * HD + (lane >> 2) * 4 + (lane & 2) * 16 + (lane & 1) * 2;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    op[64 * b] = from_f32<T>(acc[2 * b] * inv);
    op[64 * b + 1] = from_f32<T>(acc[2 * b + 1] * inv);
  }
}

// ---------------------------------------------------------------------------- single tokens
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {          // an 8 x 8 matrix of 16-bit numbers, rows to columns
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  const int n = there ? BYTES : 0;                                 // 0 bytes read: the place is filled with zeros
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float fast_exp2(float x) {              // exp2(-inf) = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {     // nothing to add to
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t less(uint32_t v, uint32_t c) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// (a & mask) | bits, one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}
// The codes of the four nibbles of both halves of a word: two half numbers each.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&c)[4]) {
  const uint32_t v = w >> 8;
  c[0] = less(and_or(w, 0x000f000fu, 0x64006400u), 0x64086408u);   // 1024 + n, 1032
  c[1] = less(and_or(w, 0x00f000f0u, 0x54005400u), 0x54805480u);   // 64 + n, 72
  c[2] = less(and_or(v, 0x000f000fu, 0x64006400u), 0x64086408u);
  c[3] = less(and_or(v, 0x00f000f0u, 0x54005400u), 0x54805480u);
}
// floor(log2 x) of a float >= 0, not below -100 (weights then stay below 2^108, and a sum of 2^17 of them below 2^126)
__device__ __forceinline__ float exponent_of(float x) {
  return fmaxf(__int_as_float((__float_as_int(x) >> 23) | 0x4b000000) - 8388735.f, -100.f);
}

// A warp's tile is 4.5 KB whatever the head size, three of them a warp: 108 KB a CTA, two CTAs an SM.
template <int HD> struct DecCfg {
  static constexpr int NW = 8, D = 3, THREADS = NW * 32;
  static constexpr int TILE = HD == 64 ? 64 : 32;                  // keys
  static constexpr int CODES = TILE * HD / 2, SCALES = TILE * HD / 16;
  static constexpr int STAGE = 2 * (CODES + SCALES);               // K codes, V codes, K scales, V scales
  static constexpr int RING = NW * D * STAGE;
  static constexpr int ALONE = 120 * 1024;                         // more than half of an SM's shared memory
  // the warps' parts lie over the ring once it is done with: [NW][queries][HD], then the CTA's [queries][HD], maxima and sums
  static constexpr int parts(int nq) { return (NW + 1) * nq * HD * 4 + (NW + 1) * 16 * 8; }
};
static_assert(DecCfg<128>::RING >= DecCfg<128>::parts(16) && DecCfg<64>::RING >= DecCfg<64>::parts(16), "the parts fit the ring");

// Where 16-byte piece `ch` of key row r lies in a tile of codes.
template <int HD> __device__ __forceinline__ uint32_t code_off(int r, int ch) {
  return HD == 128 ? (uint32_t)(r * 64 + ((ch ^ ((((r >> 1) ^ (r >> 2)) & 1) << 1)) << 4)) : (uint32_t)((r ^ (((r >> 2) & 1) << 1)) * 32 + (ch << 4));
}

// NQ: groups of 4 query heads a CTA
template <int HD, int NQ>
__global__ void __launch_bounds__(256, NQ <= 2 ? 2 : 1)
kv4_decode_kernel(const Kv4Params p) {
  typedef DecCfg<HD> C;
  constexpr int NW = C::NW, D = C::D, TILE = C::TILE, THREADS = C::THREADS;
  constexpr int GR = HD / 32, BL = HD / 64;              // groups and blocks of a row
  constexpr int CPR = HD / 32;                           // 16-byte pieces of a row's codes
  extern __shared__ __align__(128) uint8_t ring_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, qi = lane & 3;
  const int G = p.nh / p.nkv, qgroups = (G + 4 * NQ - 1) / (4 * NQ);
  const int kvh = blockIdx.x / qgroups, seq = blockIdx.y;
  const int h0 = kvh * G + blockIdx.x % qgroups * (4 * NQ);        // first query head
  const int nq = min(4 * NQ, kvh * G + G - h0);
  const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
  pdl_launch();
  pdl_wait();                                            // the kernel in front may have written any of the cache

  const int pos = p.kv_lens[seq] - 1;
  const int lo = (p.window > 0 && pos - p.window + 1 > 0) ? pos - p.window + 1 : 0;
  const int tile_first = lo / TILE, tiles_total = pos >= 0 ? pos / TILE + 1 - tile_first : 0;
  const int per = (tiles_total + p.splits - 1) / p.splits;
  const int tb = tile_first + rank * per;
  const int n_tiles = max(0, min(tile_first + tiles_total, tb + per) - tb);
  const int* bt = p.block_table + (size_t)seq * p.bt_stride;
  const uint32_t base = smem_u32(ring_raw), ring = base + (uint32_t)(warp * D) * C::STAGE;

  // What a lane's copies share is worked out once: piece `lane % CPR` of every (32 / CPR)-th key row, and a key's scales.
  const int ch = lane % CPR;
  const uint8_t* k4 = p.k4 + 16 * ch;
  const uint8_t* v4 = p.v4 + 16 * ch;
  const uint32_t dst0 = ring + code_off<HD>(lane / CPR, ch), dst1 = ring + 2 * C::CODES + lane * (HD / 16);
  // The pages of this lane's keys in tile i, -1 where there is no key; asked for a tile ahead of the copies.
  int page[TILE / 32];
  auto look_up = [&](int i) {
    const int j0 = (tb + i) * TILE;
#pragma unroll
    for (int h = 0; h < TILE / 32; ++h) {
      const int j = j0 + 32 * h + lane;
      page[h] = i < n_tiles && j >= lo && j <= pos ? bt[p.page_shift >= 0 ? j >> p.page_shift : j / p.page_size] : -1;
    }
  };
  // Starts the copies of this warp's tile i and closes a copy group, also when there is no such tile, so that the groups can be counted.
  auto issue = [&](int i, int slot) {
    if (i < n_tiles) {
      const uint32_t st = (uint32_t)slot * C::STAGE;
      const int j0 = (tb + i) * TILE;
      int row[TILE / 32];                                // a lane has the rows of its keys, the others ask it
      bool all = true;
#pragma unroll
      for (int h = 0; h < TILE / 32; ++h) {
        const int j = j0 + 32 * h + lane;
        const int off = p.page_shift >= 0 ? j & (p.page_size - 1) : j % p.page_size;
        row[h] = page[h] >= 0 && page[h] < p.num_pages ? (page[h] * p.nkv + kvh) * p.page_size + off : -1;
        all = all && row[h] >= 0;
      }
      all = __all_sync(0xffffffffu, all);
      // (two loops: in the one that runs the lengths are constants)
      auto copies = [&](bool known) {
#pragma unroll
        for (int h = 0; h < TILE / 32; ++h) {
          const bool there = known || row[h] >= 0;
          const uint32_t r = there ? row[h] : 0;
          copy_async<HD / 16>(dst1 + st + 32 * h * (HD / 16), p.ks + (size_t)r * GR, there);
          copy_async<HD / 16>(dst1 + st + C::SCALES + 32 * h * (HD / 16), p.vs + (size_t)r * GR, there);
        }
#pragma unroll
        for (int c = 0; c < TILE * CPR / 32; ++c) {
          const int r = __shfl_sync(0xffffffffu, row[c * 32 / CPR / 32], (c * 32 / CPR + lane / CPR) & 31);
          const bool there = known || r >= 0;
          const size_t src = (size_t)(uint32_t)(there ? r : 0) * (HD / 2);
          copy_async<16>(dst0 + st + c * 512, k4 + src, there);
          copy_async<16>(dst0 + st + C::CODES + c * 512, v4 + src, there);
        }
      };
      if (all) copies(true); else copies(false);
    }
    copy_commit();
    look_up(i + NW);
  };
  look_up(warp);
#pragma unroll
  for (int d = 0; d < D; ++d) issue(warp + d * NW, d);

  // The queries as fragments: lane (quad, qi) has numbers 8 qi .. 8 qi + 7 of group quad / 4 of each block of query quad % 4; in step t
  // of a block go numbers t and t + 4, in the half of the register that the group's codes have, the other half zero.
  const int hi_cols = quad >> 2;
  uint32_t qf[NQ][BL][4][2];
  float sl[NQ][2];                                       // scale, log2 e and the power of two of the queries of columns 2 qi and 2 qi + 1
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const bool live = 4 * x + (quad & 3) < nq;
    const bf16* qp = (const bf16*)p.q + (size_t)seq * p.q_stride + (size_t)(h0 + (live ? 4 * x + (quad & 3) : 0)) * HD + 32 * hi_cols + 8 * qi;
    uint4 v[BL];
    float big = 0.f;
#pragma unroll
    for (int b = 0; b < BL; ++b) {
      v[b] = live ? __ldcg(reinterpret_cast<const uint4*>(qp + 64 * b)) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t w[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) big = fmaxf(big, fmaxf(fabsf(bf16_lo(w[i])), fabsf(bf16_hi(w[i]))));
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 16));
    const int e = (int)fminf(exponent_of(big), 100.f);
    const float down = __int_as_float((127 - e) << 23), up = __int_as_float((127 + e) << 23) * p.scale * 1.4426950408889634f;
    sl[x][0] = __shfl_sync(0xffffffffu, up, 8 * (qi & 1));
    sl[x][1] = __shfl_sync(0xffffffffu, up, 8 * (qi & 1) + 4);
#pragma unroll
    for (int b = 0; b < BL; ++b) {
      const uint32_t w[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float f = (t & 1 ? bf16_hi(w[2 * u + (t >> 1)]) : bf16_lo(w[2 * u + (t >> 1)])) * down;
          qf[x][b][t][u] = hi_cols ? pack2(0.f, f) : pack2(f, 0.f);
        }
    }
  }

  float o[NQ][2 * BL][4];                                // [block, half of a group]: rows dimensions, columns queries (see below)
  float m[NQ][2], l[NQ][2];
  float top[NQ][2][BL];                                  // what the sums of this lane's columns' group in each block are against (log2)
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
#pragma unroll
    for (int i = 0; i < 2 * BL; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[x][e] = -INFINITY;
      l[x][e] = 0.f;
#pragma unroll
      for (int b = 0; b < BL; ++b) top[x][e][b] = -INFINITY;
    }
  }
  // a scale of this lane's columns' group out of the two, as float; where the weights of the keys 2 qi and 2 qi + 1 go
  const uint32_t pick = qi & 2 ? 0x3244u : 0x1044u, put0 = hi_cols ? 0x1044u : 0x4410u, put1 = hi_cols ? 0x3244u : 0x4432u;
  auto scale_of = [&](uint32_t two) { return __uint_as_float(__byte_perm(two, 0u, pick)); };
  // row r of a fragment is key (r & 7) / 2 + 4 (r & 1) + (r & 8)
  const int krow = (quad >> 1) + 4 * (quad & 1);
  // this lane's places in a stage: both rows' codes (words 2 qi, 2 qi + 1 of a block), the value words of its four keys, the scales. A fragment's
  // keys are 16 rows on from the one before, which changes nothing in where pieces lie within a row.
  uint32_t ka[BL], va[BL], vb[BL];
#pragma unroll
  for (int b = 0; b < BL; ++b) {
    ka[b] = ring + code_off<HD>(krow, 2 * b + (qi >> 1)) + 8 * (qi & 1);
    va[b] = ring + C::CODES + code_off<HD>(qi, 2 * b + (quad >> 2)) + 4 * (quad & 3);
    vb[b] = ring + C::CODES + code_off<HD>(qi + 4, 2 * b + (quad >> 2)) + 4 * (quad & 3);
  }
  constexpr int ROW = HD / 2;
  const uint32_t sa = ring + 2 * C::CODES + krow * (HD / 16);
  int slot = 0;
  for (int i = warp; i < n_tiles; i += NW) {
    copy_wait<D - 1>();                                  // this warp's oldest group, tile i, has landed
    __syncwarp();
    const uint32_t st = (uint32_t)slot * C::STAGE;
    const int j0 = (tb + i) * TILE;
    const bool edge = j0 < lo || j0 + TILE - 1 > pos;
#pragma unroll
    for (int half = 0; half < TILE / 32; ++half) {
      // two fragments of 16 keys go together: their chains of products hide each other, and they share a look at the maximum
      float s[2][NQ][4];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int k0 = 32 * half + 16 * f;
#pragma unroll
        for (int x = 0; x < NQ; ++x) s[f][x][0] = s[f][x][1] = s[f][x][2] = s[f][x][3] = 0.f;
        // ---- scores, block by block
#pragma unroll
        for (int b = 0; b < BL; ++b) {
          const uint2 wa = lds64(ka[b] + st + k0 * ROW), wb = lds64(ka[b] + st + (k0 + 8) * ROW);
          const float d0 = scale_of(lds32(sa + st + k0 * (HD / 16) + 4 * b)), d1 = scale_of(lds32(sa + st + (k0 + 8) * (HD / 16) + 4 * b));
          uint32_t c0[4], c1[4], c2[4], c3[4];
          codes_f16(wa.x, c0); codes_f16(wb.x, c1); codes_f16(wa.y, c2); codes_f16(wb.y, c3);
#pragma unroll
          for (int x = 0; x < NQ; ++x) {
            float c[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint32_t a[4] = {c0[t], c1[t], c2[t], c3[t]};
              if (t == 0) mma16816_first(c, a, qf[x][b][t][0], qf[x][b][t][1]);
              else mma16816(c, a, qf[x][b][t][0], qf[x][b][t][1]);
            }
            s[f][x][0] = fmaf(d0, c[0], s[f][x][0]); s[f][x][1] = fmaf(d0, c[1], s[f][x][1]);
            s[f][x][2] = fmaf(d1, c[2], s[f][x][2]); s[f][x][3] = fmaf(d1, c[3], s[f][x][3]);
          }
        }
#pragma unroll
        for (int x = 0; x < NQ; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {                  // plus the other group's columns
            s[f][x][e] += __shfl_xor_sync(0xffffffffu, s[f][x][e], 2);
            s[f][x][e] *= sl[x][e & 1];
          }
        if (edge) {
          const int ja = j0 + k0 + krow, jb = ja + 8;
#pragma unroll
          for (int x = 0; x < NQ; ++x) {
            if (ja < lo || ja > pos) s[f][x][0] = s[f][x][1] = -INFINITY;
            if (jb < lo || jb > pos) s[f][x][2] = s[f][x][3] = -INFINITY;
          }
        }
      }
      // ---- weights
      float sc[2][2][BL], big[2][2][BL];                 // the value scales of rows quad and quad + 8 in this lane's group, their log2
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int b = 0; b < BL; ++b) {
            sc[f][e][b] = scale_of(lds32(sa + st + C::SCALES + (32 * half + 16 * f + 8 * e) * (HD / 16) + 4 * b));
            big[f][e][b] = exponent_of(fabsf(sc[f][e][b]));
          }
      auto risen = [](float now, float old) { return now == old ? 1.f : fast_exp2(old - now); };
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        float mx[2], tx[2][BL];
        bool rises = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(fmaxf(s[0][x][e], s[0][x][2 + e]), fmaxf(s[1][x][e], s[1][x][2 + e]));
          rises = rises || mx[e] > m[x][e] + 8.f;
#pragma unroll
          for (int b = 0; b < BL; ++b) {
            tx[e][b] = fmaxf(fmaxf(s[0][x][e] + big[0][0][b], s[0][x][2 + e] + big[0][1][b]),
                             fmaxf(s[1][x][e] + big[1][0][b], s[1][x][2 + e] + big[1][1][b]));
            rises = rises || tx[e][b] > top[x][e][b] + 8.f;
          }
        }
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], d));
#pragma unroll
              for (int b = 0; b < BL; ++b) tx[e][b] = fmaxf(tx[e][b], __shfl_xor_sync(0xffffffffu, tx[e][b], d));
            }
            mx[e] = fmaxf(mx[e], m[x][e]);
            l[x][e] *= risen(mx[e], m[x][e]);
            m[x][e] = mx[e];
#pragma unroll
            for (int b = 0; b < BL; ++b) {
              tx[e][b] = fmaxf(tx[e][b], top[x][e][b]);
              const float c = risen(tx[e][b], top[x][e][b]);
              top[x][e][b] = tx[e][b];
#pragma unroll
              for (int u = 0; u < 2; ++u) { o[x][2 * b + u][e] *= c; o[x][2 * b + u][2 + e] *= c; }
            }
          }
        }
        const float u0 = m[x][0] == -INFINITY ? 0.f : m[x][0], u1 = m[x][1] == -INFINITY ? 0.f : m[x][1];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          s[f][x][0] = fast_exp2(s[f][x][0] - u0); s[f][x][1] = fast_exp2(s[f][x][1] - u1);
          s[f][x][2] = fast_exp2(s[f][x][2] - u0); s[f][x][3] = fast_exp2(s[f][x][3] - u1);
          l[x][0] += s[f][x][0] + s[f][x][2];
          l[x][1] += s[f][x][1] + s[f][x][3];
        }
      }
      // from the scores' maximum to the group's (a maximum of -inf: no key yet, or NaN scores only)
      float up[NQ][2][BL];
#pragma unroll
      for (int x = 0; x < NQ; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int b = 0; b < BL; ++b) up[x][e][b] = m[x][e] == -INFINITY ? 1.f : fast_exp2(m[x][e] - top[x][e][b]);
      // ---- values: the keys of weights 2 qi, 2 qi + 1, 2 qi + 8 and 2 qi + 9 are qi, qi + 4, qi + 8 and qi + 12
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int b = 0; b < BL; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {                  // rows 0-7, then 8-15
            const int k0 = 32 * half + 16 * f + 8 * e;
            const float d = sc[f][e][b];
            uint32_t ca[4], cb[4];
            codes_f16(lds32(va[b] + st + k0 * ROW), ca);
            codes_f16(lds32(vb[b] + st + k0 * ROW), cb);
#pragma unroll
            for (int x = 0; x < NQ; ++x) {
              // (the weight times its power first: below 2^8 over the scale, so that nothing overflows on the way)
              const uint32_t w = turn8x8(pack2(s[f][x][2 * e] * up[x][0][b] * d, s[f][x][2 * e + 1] * up[x][1][b] * d));
              const uint32_t b0 = __byte_perm(w, 0u, put0), b1 = __byte_perm(w, 0u, put1);
              // rows quad and quad + 8 are dimensions 4 quad + 2 u and 4 quad + 2 u + 1 of the columns' group
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint32_t a[4] = {ca[2 * u], ca[2 * u + 1], cb[2 * u], cb[2 * u + 1]};
                mma16816(o[x][2 * b + u], a, b0, b1);
              }
            }
          }
    }
    __syncwarp();                                        // every lane has read the stage
    issue(i + D * NW, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
  }
  copy_wait<0>();
  __syncthreads();                                       // the ring is done with: the parts go over it
  float* w_o = reinterpret_cast<float*>(ring_raw);       // [NW][4 NQ][HD]
  float* c_o = w_o + NW * 4 * NQ * HD;                   // [4 NQ][HD]
  float* w_m = c_o + 4 * NQ * HD;                        // [NW][16]
  float* w_l = w_m + NW * 16;
  float* c_m = w_l + NW * 16;                            // [16]
  float* c_l = c_m + 16;
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l[x][0] += __shfl_xor_sync(0xffffffffu, l[x][0], d);
      l[x][1] += __shfl_xor_sync(0xffffffffu, l[x][1], d);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int query = 4 * x + ((2 * qi + e) & 3);
      if (lane < 2) { w_m[warp * 16 + query] = m[x][e]; w_l[warp * 16 + query] = l[x][e]; }
      if (query < nq) {
#pragma unroll
        for (int t = 0; t < 2 * BL; ++t) {
          // the groups' sums against the scores' maximum, in two steps that stay in range where the sums are zero
          const float c = m[x][e] == -INFINITY ? 1.f : fast_exp2(0.5f * (top[x][e][t >> 1] - m[x][e]));
          *reinterpret_cast<float2*>(w_o + ((size_t)warp * 4 * NQ + query) * HD + 64 * (t >> 1) + 32 * (qi >> 1) + 4 * quad + 2 * (t & 1)) =
              make_float2(o[x][t][e] * c * c, o[x][t][2 + e] * c * c);
        }
      }
    }
  }
  __syncthreads();
  bf16* out = (bf16*)p.out + (size_t)seq * p.out_stride + (size_t)h0 * HD;
  auto finish = [](float O, float L) { return L > 0.f ? O / L : (L == L ? 0.f : L); };     // no visible key: zeros; a NaN stays one
  for (int idx = threadIdx.x; idx < nq * HD; idx += THREADS) {
    const int r = idx / HD, d = idx % HD;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, w_m[w * 16 + r]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      // a part whose scores were all NaN has a maximum of -inf and a sum of NaN
      const float mw = w_m[w * 16 + r], f = mw == -INFINITY ? 1.f : exp2f(mw - M);
      L += w_l[w * 16 + r] * f;
      O += w_o[((size_t)w * 4 * NQ + r) * HD + d] * f;
    }
    if (p.splits == 1) out[idx] = __float2bfloat16_rn(finish(O, L));
    else {
      c_o[idx] = O;
      if (d == 0) { c_m[r] = M; c_l[r] = L; }
    }
  }
  if (p.splits > 1) {
    __syncwarp();
    cluster_sync_all();
    const uint32_t ao = smem_u32(c_o), am = smem_u32(c_m), al = smem_u32(c_l);
    // number idx is finished by the rank of its place among the ranges
    for (int idx = threadIdx.x + rank * THREADS; idx < nq * HD; idx += THREADS * p.splits) {
      const int r = idx / HD;
      float M = -INFINITY, L = 0.f, O = 0.f;
      for (int z = 0; z < p.splits; ++z) M = fmaxf(M, ld_cluster_f32(map_to_rank(am, z) + 4 * r));
      for (int z = 0; z < p.splits; ++z) {
        const float mz = ld_cluster_f32(map_to_rank(am, z) + 4 * r), f = mz == -INFINITY ? 1.f : exp2f(mz - M);
        L += ld_cluster_f32(map_to_rank(al, z) + 4 * r) * f;
        O += ld_cluster_f32(map_to_rank(ao, z) + 4 * idx) * f;
      }
      out[idx] = __float2bfloat16_rn(finish(O, L));
    }
    __syncwarp();
    cluster_sync_all();                                  // nobody leaves while its shared memory is still read
  }
}

template <int HD, int NQ>
int launch_decode(const Kv4Params& p, int sm_count, cudaStream_t s) {
  typedef DecCfg<HD> C;
  static bool configured[64] = {}, wide[64] = {};
  if (allow_dynamic_smem(kv4_decode_kernel<HD, NQ>, C::ALONE, configured)) return -5;
  if (p.splits > 8) {                                    // a cluster beyond the portable size needs the kernel's own permission, per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return -5; }
    if (!wide[dev]) {
      if (cudaFuncSetAttribute(kv4_decode_kernel<HD, NQ>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return ERR_BAD_SIZE;
      }
      wide[dev] = true;
    }
  }
  const int G = p.nh / p.nkv;
  const dim3 grid(p.nkv * ((G + 4 * NQ - 1) / (4 * NQ)), p.rows, p.splits);
  if (grid.y > 65535) return ERR_TOO_LARGE;
  // While every CTA can have an SM of its own it takes one: the CTAs of a cluster are otherwise put on SMs in pairs (8 sequences of 4,096
  // keys, 8 kv heads of 64, 2 ranges: 16.1 us, alone 12.8; the 4 ranges that the rule takes, two CTAs an SM, 11.9). Not so clusters of 16, for which too few GPCs have 16 SMs (41 us for one
  // sequence of 60,000 keys of 128, 57 alone).
  const long long ctas = (long long)grid.x * grid.y * grid.z;
  return launch_ex(kv4_decode_kernel<HD, NQ>, grid, dim3(C::THREADS), ctas <= sm_count && p.splits <= 8 ? C::ALONE : C::RING, s, p.splits, p);
}

template <typename T>
int launch_simt(const Kv4Params& p, int hd, cudaStream_t s) {
  const long long blocks = ((long long)p.rows * p.nh + WARPS - 1) / WARPS;
  if (blocks > 2147483647LL) return ERR_TOO_LARGE;
  const dim3 g((unsigned)blocks), b(WARPS * 32);
  switch (hd) {
    case 64: return launch_ex(kv4_attention_simt_kernel<T, 1>, g, b, 0, s, 1, p);
    case 128: return launch_ex(kv4_attention_simt_kernel<T, 2>, g, b, 0, s, 1, p);
    case 192: return launch_ex(kv4_attention_simt_kernel<T, 3>, g, b, 0, s, 1, p);
    case 256: return launch_ex(kv4_attention_simt_kernel<T, 4>, g, b, 0, s, 1, p);
  }
  return ERR_BAD_SIZE;
}

}  // namespace

// q [T, ...] float or bf16 with row stride q_stride, head h at h * hd; out likewise. token_seq, positions int32 [T].
RLLM_API int rllm_kv4_attention_simt(int dt, const void* q, int q_stride, const void* k4, const void* ks, const void* v4,
                                     const void* vs, long long num_pages, void* out, int out_stride, const int* token_seq,
                                     const int* positions, const int* block_table, int bt_stride, int T, int nh, int nkv, int hd,
                                     int page_size, float scale, int window, void* stream) {
  if (T <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || page_size <= 0 || num_pages <= 0) return ERR_BAD_SIZE;
  if (((uintptr_t)k4 | (uintptr_t)ks | (uintptr_t)v4 | (uintptr_t)vs) & 15) return ERR_BAD_ALIGN;
  const Kv4Params p = {q, q_stride, (const uint8_t*)k4, (const bf16*)ks, (const uint8_t*)v4, (const bf16*)vs, num_pages, out, out_stride,
                       token_seq, positions, nullptr, block_table, bt_stride, T, nh, nkv, page_size, window, scale, -1, 1};
  if (dt == DT_F32) return launch_simt<float>(p, hd, (cudaStream_t)stream);
  if (dt == DT_BF16) return launch_simt<bf16>(p, hd, (cudaStream_t)stream);
  return ERR_BAD_DTYPE;
}

// One bf16 query row per sequence: q [S, ...] with row stride q_stride (a multiple of 8, 16-byte aligned), head h at h * hd; out likewise.
// kv_lens int32 [S]: keys that a sequence's token sees, its own included. splits: ranges of keys (1..16, the CTAs of a cluster).
RLLM_API int rllm_kv4_decode(const void* q, int q_stride, const void* k4, const void* ks, const void* v4, const void* vs,
                             long long num_pages, void* out, int out_stride, const int* kv_lens, const int* block_table,
                             int bt_stride, int num_seqs, int nh, int nkv, int hd, int page_size, float scale, int window, int splits,
                             int sm_count, void* stream) {
  if (num_seqs <= 0) return 0;
  if ((hd != 64 && hd != 128) || nkv <= 0 || nh <= 0 || nh % nkv || page_size <= 0 || num_pages <= 0 || splits < 1 || splits > 16 || !(scale > 0.f))
    return ERR_BAD_SIZE;
  if (num_pages * nkv * page_size > 2147483647LL) return ERR_TOO_LARGE;
  if (q_stride % 8 || (((uintptr_t)q | (uintptr_t)k4 | (uintptr_t)ks | (uintptr_t)v4 | (uintptr_t)vs) & 15)) return ERR_BAD_ALIGN;
  int shift = -1;
  for (int b = 0; b < 31; ++b) if ((1 << b) == page_size) shift = b;
  const Kv4Params p = {q, q_stride, (const uint8_t*)k4, (const bf16*)ks, (const uint8_t*)v4, (const bf16*)vs, num_pages, out, out_stride,
                       nullptr, nullptr, kv_lens, block_table, bt_stride, num_seqs, nh, nkv, page_size, window, scale, shift, splits};
  cudaStream_t s = (cudaStream_t)stream;
  const int G = nh / nkv;
  if (hd == 64)
    return G <= 4 ? launch_decode<64, 1>(p, sm_count, s) : G <= 8 ? launch_decode<64, 2>(p, sm_count, s) : launch_decode<64, 4>(p, sm_count, s);
  return G <= 4 ? launch_decode<128, 1>(p, sm_count, s) : G <= 8 ? launch_decode<128, 2>(p, sm_count, s) : launch_decode<128, 4>(p, sm_count, s);
}
