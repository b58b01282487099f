// Products in 8-bit integers for few tokens: Y[t, n] = (sum_k X[t, k] W[n, k]) * sx[t] * sw[n], X quantised on the way.
//
// Up to 8 tokens the product is a read of W. A job is a slab of 16 weight rows (SwiGLU: a gate and an up slab); the warps of a CTA share
// K, every warp copies its own pieces (16 rows x 128 or 256 codes, 2 or 4 KB) with cp.async into a ring of its own and multiplies with mma.sync
// m16n8k16 in half precision: weights are the A operand, tokens the B operand, the contraction index permuted alike on both sides so
// that the 16 bytes that a lane reads are fragments. (The instruction's 8-bit form takes some 200 cycles here: 1 token of 14,336 numbers
// with 4,096 outputs 34 us.) A code is an exact half number, 1024 + (code + 128) by one byte permutation for two of them, less 1152; a piece's
// sum, below 2^22, is exact in float. The warps' sums meet in shared memory in any
// order.
// The tokens are quantised here, by every CTA for itself while its first weights are on their way: a lane's fragments are 16 numbers of
// a token at a time, of which it needs the row's largest; the warps' maxima (and sums of squares, with an RMSNorm in front) meet once in
// shared memory, then the codes are made and stay in registers for all of the CTA's jobs. With a kernel of its own in front 8 tokens
// took 7.2 us with 2,048 x 2,048, so 4.6; 1 token 3.4. Against a gate/up pair of 2 x 8,192 rows of 2,048 8 tokens take 11.4 us, 33.6 MB at
// 2.9 TB/s: every CTA makes the tokens' codes for 2 us before its weights, which have arrived meanwhile, are used.
#include "quant.cuh"
#include "sm100.cuh"
#include <cuda_fp16.h>

using namespace rllm;
using namespace sm100;

namespace {

enum : int { EPI_STORE = 0, EPI_STORE_F32 = 1, EPI_ACCUM_F32 = 2, EPI_SWIGLU = 3 };

struct StreamParams {
  const void* x; long long ldx;
  const int* rows;                   // row of x that token t is made from, or null
  const void* g; int g_is_bf16; float eps;      // norm weight, or null
  const float* sx;                   // CODES: x holds codes, these are their scales
  int xk;                            // numbers of a row of x (K without what pads it)
  const int8_t* w; const float* sw;
  void* y; long long ldy;
  int T, N, K, njobs;
  int epi, out_f32;
  int w_fixed;                       // nothing in front of this kernel writes the weight
};

constexpr int SNT = 8;
constexpr int SUMS = 4;              // slabs' sums that lie in shared memory together
constexpr int WARPS = 16, THREADS = WARPS * 32;
// KB: steps of 64 numbers that a warp's piece of K has, 2 or 4. Rows of up to 2,048 numbers are shared by all 16 warps in pieces of 128.
template <int KB> struct StreamCfg {
  static constexpr int SCK = 64 * KB, CHUNK = 16 * SCK;                  // 128 or 256 codes of each of 16 rows
  static constexpr int RING = 192 * 1024 / (WARPS * CHUNK);              // 192 KB on the way
  static constexpr int RING_BYTES = WARPS * RING * CHUNK;
  static constexpr int SMEM_BYTES = RING_BYTES + SUMS * WARPS * 16 * SNT * 4;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes 0, 1 (hi: 2, 3) of a word of codes + 128 as two half numbers.
__device__ __forceinline__ uint32_t halves(uint32_t w, bool hi) {
  const uint32_t v = __byte_perm(w, 0x64646464u, hi ? 0x4342 : 0x4140), c = 0x64806480u;        // 1024 + byte, 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ int sum_col(int row, int col) { return col ^ (((row >> 2) & 3) << 1); }     // banks: see stream_gemm.cu

// 16 numbers of a row from k on (a multiple of 8 of them lie in it), float ones times the norm's weight; squares added to ss.
template <bool F32>
__device__ __forceinline__ void load16(const StreamParams& p, const void* xrow, int k, float (&v)[16], float& ss) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int kk = k + 8 * h;
    float* o = v + 8 * h;
    if (F32) {
      const bool in = kk < p.xk;
      const float4* src = reinterpret_cast<const float4*>((const float*)xrow + (in ? kk : 0));
      const float4 a = __ldcg(src), b = __ldcg(src + 1);
      o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
      if (p.g) {
        float w[8];
        if (p.g_is_bf16) {
          const uint4 a4 = __ldg(reinterpret_cast<const uint4*>((const bf16*)p.g + (in ? kk : 0)));
          const uint32_t u[4] = {a4.x, a4.y, a4.z, a4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) { w[2 * i] = bf16_lo(u[i]); w[2 * i + 1] = bf16_hi(u[i]); }
        } else {
          const float4* gs = reinterpret_cast<const float4*>((const float*)p.g + (in ? kk : 0));
          const float4 c = __ldg(gs), d = __ldg(gs + 1);
          w[0] = c.x; w[1] = c.y; w[2] = c.z; w[3] = c.w; w[4] = d.x; w[5] = d.y; w[6] = d.z; w[7] = d.w;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (in) ss = fmaf(o[i], o[i], ss);
          o[i] *= w[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = in ? o[i] : 0.f;
    } else {
      const uint4 a = kk < p.xk ? __ldcg(reinterpret_cast<const uint4*>((const bf16*)xrow + kk)) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { o[2 * i] = bf16_lo(w[i]); o[2 * i + 1] = bf16_hi(w[i]); }
    }
  }
}

// IN: bfloat16, float or codes; TILES: 2 with SwiGLU; NCH: pieces of K a warp has (codes only). A warp's sum is exact in float up to 1,024 products
// of codes: 64 KB NCH at most.
enum : int { NUMBERS = 0, FLOATS = 1, CODES = 2 };
template <int IN, int TILES, int KB, int NCH>
__global__ void __launch_bounds__(THREADS, 1)
int8_stream_kernel(const StreamParams p) {
  static_assert(NCH * KB <= 16 && (NCH == 1 || IN == CODES), "sums of a warp are exact; numbers are quantised in one piece");
  typedef StreamCfg<KB> C;
  constexpr bool F32 = IN == FLOATS;
  constexpr int RING = C::RING, SCK = C::SCK, BATCH = SUMS / TILES;
  constexpr int UNITS = SCK / 16, STEP = 32 / UNITS;      // 16-byte units of a row, rows a copy instruction brings
  extern __shared__ __align__(128) uint8_t stream_smem[];
  __shared__ float s_max[WARPS][SNT], s_sq[WARPS][SNT], s_scale[SNT];
  int* red = reinterpret_cast<int*>(stream_smem + C::RING_BYTES);        // [job of batch][tile][warp][row][token]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(stream_smem) + warp * (RING * C::CHUNK);
  const int my_jobs = p.njobs > (int)blockIdx.x ? (p.njobs - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;
  pdl_launch();

  int pj = 0, ptile = 0, pci = 0, pslot = 0;
  const int crow = lane / UNITS, cunit = lane % UNITS;
  auto produce = [&]() {
    if (pj < my_jobs) {
      const int n0 = (blockIdx.x + pj * gridDim.x) * 16;
      const int k = (warp * NCH + pci) * SCK + 16 * cunit;
      const int8_t* src = p.w + (size_t)(n0 + (ptile ? p.N : 0) + crow) * p.K + k;
      const uint32_t dst = ring + pslot * C::CHUNK + crow * SCK + ((cunit ^ ((crow & 1) << 2)) << 4);      // odd rows: units' bit 2 flipped
#pragma unroll
      for (int i = 0; i < 16 / STEP; ++i) {
        const bool there = k < p.K && n0 + crow + STEP * i < p.N;
        copy16(dst + i * 512, there ? src + (size_t)(STEP * i) * p.K : p.w, there);
      }
      if (++pci == NCH) { pci = 0; if (++ptile == TILES) { ptile = 0; ++pj; } }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    pslot = pslot + 1 == RING ? 0 : pslot + 1;
  };
  // the weights need not wait for the kernel in front, unless it, or one before it, may still write them
  if (!p.w_fixed) pdl_wait();
#pragma unroll
  for (int i = 0; i < RING; ++i) produce();
  pdl_wait();

  // ---- the tokens: their rows' largest numbers, then their codes as fragments: b[piece][step] words of codes + 128
  uint32_t b[NCH][KB][4];
  const int tok = min(g, p.T - 1);                        // tokens beyond the last one: its codes again, never stored
  if constexpr (IN == CODES) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int k = (warp * NCH + c) * SCK + 64 * kb + 16 * t;
        const uint4 q = k < p.K ? __ldcg(reinterpret_cast<const uint4*>((const int8_t*)p.x + (size_t)tok * p.ldx + k)) : make_uint4(0u, 0u, 0u, 0u);
        b[c][kb][0] = q.x ^ 0x80808080u; b[c][kb][1] = q.y ^ 0x80808080u; b[c][kb][2] = q.z ^ 0x80808080u; b[c][kb][3] = q.w ^ 0x80808080u;
      }
    if (warp == 0 && t == 0) s_scale[g] = __ldcg(p.sx + tok);
  } else {
    const uint8_t* xr = (const uint8_t*)p.x + (size_t)(p.rows ? p.rows[tok] : tok) * p.ldx * (F32 ? 4 : 2);
    float v[KB][16], mx = 0.f, ss = 0.f, bad = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) load16<F32>(p, xr, warp * SCK + 64 * kb + 16 * t, v[kb], ss);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) { mx = fmaxf(mx, fabsf(v[kb][i])); bad = fmaf(v[kb][i], 0.f, bad); }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      bad += __shfl_xor_sync(0xffffffffu, bad, o);
    }
    if (t == 0) { s_max[warp][g] = bad == 0.f ? mx : INFINITY; s_sq[warp][g] = ss; }
    __syncthreads();
    mx = ss = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      mx = fmaxf(mx, s_max[w][g]);
      ss += s_sq[w][g];
    }
    const float rstd = p.g ? rsqrtf(ss / (float)p.xk + p.eps) : 1.f;
    const float amax = mx * rstd;
    const bool whole = mx <= 3.402823466e38f && amax <= 3.402823466e38f;      // every number finite
    const float s = __fdiv_rn(amax, 127.f);
    const bool codes = whole && s > 0.f;
    const Rounding rd(codes ? s : 1.f);
    if (warp == 0 && t == 0) s_scale[g] = whole ? s : __int_as_float(0x7fc00000);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if (p.g) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[kb][i] *= rstd;
      }
      uint32_t w[4] = {0u, 0u, 0u, 0u};
      if (codes) codes8<16>(v[kb], rd, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) b[0][kb][i] = w[i] ^ 0x80808080u;
    }
  }

  int cslot = 0;
  const uint32_t frag_off = (uint32_t)(g * SCK), frag_key = (uint32_t)((g & 1) << 2);
  for (int batch0 = 0; batch0 < my_jobs; batch0 += BATCH) {
    const int nb = min(BATCH, my_jobs - batch0);
    for (int jb = 0; jb < nb; ++jb) {
#pragma unroll
      for (int tile = 0; tile < TILES; ++tile) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ci = 0; ci < NCH; ++ci) {
          asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
          __syncwarp();
          const uint32_t src = ring + cslot * C::CHUNK + frag_off;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const uint32_t at = src + ((((uint32_t)(4 * kb + t)) ^ frag_key) << 4);
            uint32_t lo[4], hi[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3]) : "r"(at));
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3]) : "r"(at + 8 * SCK));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t u = lo[i] ^ 0x80808080u, v = hi[i] ^ 0x80808080u, c = b[ci][kb][i];
              mma_f16(sum, halves(u, false), halves(v, false), halves(u, true), halves(v, true), halves(c, false), halves(c, true));
            }
          }
          cslot = cslot + 1 == RING ? 0 : cslot + 1;
          __syncwarp();                                   // every lane has read the slot that is refilled now
          produce();
        }
        int* r = red + (size_t)((jb * TILES + tile) * WARPS + warp) * (16 * SNT);
        *reinterpret_cast<int2*>(r + g * SNT + sum_col(g, 2 * t)) = make_int2(__float2int_rn(sum[0]), __float2int_rn(sum[1]));
        *reinterpret_cast<int2*>(r + (g + 8) * SNT + sum_col(g + 8, 2 * t)) = make_int2(__float2int_rn(sum[2]), __float2int_rn(sum[3]));
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nb * (16 * SNT); e += THREADS) {
      const int jb = e / (16 * SNT), tok = (e >> 4) & (SNT - 1), r = e & 15;
      const int n = (blockIdx.x + (batch0 + jb) * gridDim.x) * 16 + r;
      if (tok >= p.T || n >= p.N) continue;
      int s0 = 0, s1 = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const int* part = red + (size_t)(jb * TILES * WARPS + w) * (16 * SNT) + r * SNT + sum_col(r, tok);
        s0 += part[0];
        if (TILES == 2) s1 += part[WARPS * 16 * SNT];
      }
      const float sx = s_scale[tok], v = __fmul_rn((float)s0 * sx, p.sw[n]);      // (rounded before it is added, as in int8_gemm.cu)
      const size_t o = (size_t)tok * p.ldy + n;
      if (p.epi == EPI_ACCUM_F32) { ((float*)p.y)[o] += v; continue; }
      const float out = TILES == 2 ? silu_gate(v, (float)s1 * sx * p.sw[p.N + n], p.out_f32) : v;
      if (p.out_f32) ((float*)p.y)[o] = out; else ((bf16*)p.y)[o] = __float2bfloat16_rn(out);
    }
    if (batch0 + BATCH < my_jobs) __syncthreads();        // the sums are read before the next batch overwrites them
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int IN, int TILES, int KB, int NCH>
int launch_stream(const StreamParams& p, int sm_count, cudaStream_t s) {
  typedef StreamCfg<KB> C;
  static bool configured[64] = {};
  if (allow_dynamic_smem(int8_stream_kernel<IN, TILES, KB, NCH>, C::SMEM_BYTES, configured)) return -5;
  return launch_ex(int8_stream_kernel<IN, TILES, KB, NCH>, dim3(p.njobs < sm_count ? p.njobs : sm_count), dim3(THREADS), C::SMEM_BYTES, s, 1, p);
}

// What the kernel takes: fragments of all of K in registers; rows that 16-byte loads read, a norm in front of float ones only. (Beyond 4,096
// numbers a CTA has too much to quantise: 8 tokens, 8,192 to 2,048 12.9 us, behind a kernel that makes the codes 8.2; 14,336 to 4,096 29 and 17.
// With two groups of 8 tokens every CTA had twice as much to quantise: 16 tokens of 2,048 with a gate/up pair of 8,192 17.7 us, on
// tcgen05 behind a kernel that quantises 11.)
bool streams(int T, int xk, int x_dt, const void* x, long long ldx, const void* g) {
  if (T > SNT || xk % 8 || xk > WARPS * 256 || ((uintptr_t)x & 15) || ((uintptr_t)g & 15)) return false;
  return x_dt == DT_F32 ? ldx % 4 == 0 : ldx % 8 == 0 && !g;
}

template <int IN, int TILES>
int launch_stream_k(const StreamParams& p, int sm_count, cudaStream_t s) {
  return p.K <= WARPS * 128 ? launch_stream<IN, TILES, 2, 1>(p, sm_count, s) : launch_stream<IN, TILES, 4, 1>(p, sm_count, s);
}

}  // namespace

// Does the product quantise its own tokens (rllm_int8_stream), or does it take codes and scales (rllm_quantize_rows, rllm_int8_gemm)?
RLLM_API int rllm_int8_streams(int T, int xk, int x_dt, const void* x, long long ldx, const void* g) { return streams(T, xk, x_dt, x, ldx, g); }

// x [*, xk] float or bf16 (x_dt) with row stride ldx, rows int32 [T] or null, g norm weight [xk] (g_dt) or null; the rest as for
// rllm_int8_gemm, K what xk is padded to.
RLLM_API int rllm_int8_stream(int epi, int out_dt, int x_dt, const void* x, long long ldx, const int* rows, const void* g, int g_dt, float eps,
                              const void* w, const float* sw, void* y, long long ldy, int T, int N, int xk, int K, int w_fixed, int sm_count,
                              void* stream) {
  if (T <= 0 || N <= 0) return 0;
  if ((out_dt != DT_F32 && out_dt != DT_BF16) || (x_dt != DT_F32 && x_dt != DT_BF16)) return ERR_BAD_DTYPE;
  if (xk <= 0 || K % 16 || K < xk || K - xk >= 16 || !streams(T, xk, x_dt, x, ldx, g) || ldy < N || epi < 0 || epi > 3 || N > (1 << 30))
    return ERR_BAD_SIZE;
  if ((uintptr_t)w & 15) return ERR_BAD_ALIGN;
  const bool out_f32 = out_dt == DT_F32 || epi == EPI_STORE_F32;
  const StreamParams p = {x, ldx, rows, g, g_dt == DT_BF16, eps, nullptr, xk, (const int8_t*)w, sw, y, ldy, T, N, K, (N + 15) / 16, epi, out_f32, w_fixed};
  cudaStream_t s = (cudaStream_t)stream;
  if (x_dt == DT_F32) return epi == EPI_SWIGLU ? launch_stream_k<FLOATS, 2>(p, sm_count, s) : launch_stream_k<FLOATS, 1>(p, sm_count, s);
  return epi == EPI_SWIGLU ? launch_stream_k<NUMBERS, 2>(p, sm_count, s) : launch_stream_k<NUMBERS, 1>(p, sm_count, s);
}

// The same from codes x [T, K] and scales sx [T], where every slab of 16 weight rows has an SM of its own: T up to 8, K up to 8,192, no SwiGLU.
// Behind the kernel that makes the codes, on whose time the weights arrive: 8,192 to 2,048, 1 token 8.9 us on tcgen05 with ranges of K,
// here 7.1 (8 tokens 9.2 and 8.2). With more slabs than SMs, or longer rows, tcgen05 is ahead: 14,336 to 4,096 16.3 and 22.5, 8,200 to 8,192 17.7 and 34.7.
RLLM_API int rllm_int8_streams_codes(int epi, int T, int N, int K, int sm_count) {
  return T <= SNT && K <= WARPS * 512 && epi != EPI_SWIGLU && (N + 15) / 16 <= sm_count;
}
RLLM_API int rllm_int8_stream_codes(int epi, int out_dt, const void* x, const float* sx, const void* w, const float* sw, void* y, long long ldy,
                                    int T, int N, int K, int w_fixed, int sm_count, void* stream) {
  if (T <= 0 || N <= 0) return 0;
  if (out_dt != DT_F32 && out_dt != DT_BF16) return ERR_BAD_DTYPE;
  if (K <= 0 || K % 16 || ldy < N || epi < 0 || epi > 3 || !rllm_int8_streams_codes(epi, T, N, K, sm_count)) return ERR_BAD_SIZE;
  if (((uintptr_t)x | (uintptr_t)w) & 15) return ERR_BAD_ALIGN;
  const StreamParams p = {x, K, nullptr, nullptr, 0, 0.f, sx, K, (const int8_t*)w, sw, y, ldy, T, N, K, (N + 15) / 16, epi,
                          out_dt == DT_F32 || epi == EPI_STORE_F32, w_fixed};
  return launch_stream<CODES, 1, 4, 2>(p, sm_count, (cudaStream_t)stream);
}
