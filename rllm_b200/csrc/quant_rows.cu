// Rows in 8 bits with one scale each: codes[t, k] = x[t, k] / s[t] to the nearest integer, s[t] = float(max_k |x[t, k]| / 127); with
// an RMSNorm in front the row is x[t, k] * g[k] * rsqrt(mean(x^2) + eps), in float and not rounded in between. Activations of a
// step and, once at load, the rows of a weight.
//
// The row has to be read before its scale is known, so a CTA holds it: 256 threads with up to VPT groups of 8 numbers in registers
// each (16,384 numbers with eight groups), longer rows are read twice, the second time out of the caches. What it has to do is the
// read of x and the write of the codes; a quotient is a multiplication by 1 / s except next to a border (`codes8`), since
// a division for every number took as long as the memory. 2,048 bfloat16 rows of 8,192 take 13 us (50 MB, floor 7.7): an
// instruction is issued in 63 % of the cycles, the integer pipe busy 57 %.
// Codes lie in rows of a multiple of 16 bytes (`ldc`), the numbers behind K are zeros: the products' copies are whole pieces.
#include "quant.cuh"

using namespace rllm;

namespace {

constexpr int THREADS = 256;

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<bf16>(const bf16* p, float (&v)[8]) {
  const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
}

struct RowArgs {
  const void* x; long long ldx;
  const int* rows;                 // row of x that row t is made from, or null: t itself
  const void* g; int g_is_bf16; float eps;      // norm weight, or null: no norm
  int8_t* codes; long long ldc; float* scales;
  int K;
  int early;                       // the next kernel in the stream may begin before this one ends
};

// VPT: groups of 8 numbers a thread holds; 0: any K, two passes. VEC: rows and weight start on 16 (32) bytes, K is a multiple of 8.
template <typename T, int VPT, bool VEC>
__global__ void __launch_bounds__(THREADS)
quantize_rows_kernel(const RowArgs a) {
  if (a.early) pdl_launch();
  pdl_wait();
  __shared__ float red[32];
  const int t = blockIdx.x, K = a.K;
  const T* x = (const T*)a.x + (size_t)(a.rows ? a.rows[t] : t) * a.ldx;
  auto load = [&](int k, float (&v)[8]) {
    if (VEC) load8<T>(x + k, v);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < K ? to_f32(x[k + e]) : 0.f;
    }
  };
  auto weigh = [&](int k, float (&v)[8]) {               // times the norm's weight
    float g[8];
    if (VEC) {
      if (a.g_is_bf16) load8<bf16>((const bf16*)a.g + k, g); else load8<float>((const float*)a.g + k, g);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        g[e] = k + e >= K ? 0.f : a.g_is_bf16 ? to_f32(((const bf16*)a.g)[k + e]) : ((const float*)a.g)[k + e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= g[e];
  };
  float keep[VPT ? VPT : 1][8];
  float ss = 0.f, mx = 0.f, bad = 0.f;
  auto look = [&](int k, float (&v)[8]) {
    load(k, v);
    if (a.g) {
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
      weigh(k, v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mx = fmaxf(mx, fabsf(v[e]));
      bad = fmaf(v[e], 0.f, bad);                        // 0, or NaN where v is not finite (fmaxf drops a NaN)
    }
  };
  if (VPT) {
#pragma unroll
    for (int i = 0; i < (VPT ? VPT : 1); ++i) {
      const int k = (i * THREADS + threadIdx.x) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) keep[i][e] = 0.f;
      if (k < K) look(k, keep[i]);
    }
  } else {
    for (int k = threadIdx.x * 8; k < K; k += THREADS * 8) look(k, keep[0]);
  }
  mx = block_max(bad == 0.f ? mx : INFINITY, red);
  float rstd = 1.f;
  if (a.g) rstd = rsqrtf(block_sum(ss, red) / (float)K + a.eps);
  // the row's numbers are v * rstd; the largest is the largest v's, as rounding keeps order
  const float amax = mx * rstd;
  const bool whole = mx <= 3.402823466e38f && amax <= 3.402823466e38f;      // every number finite
  const float s = __fdiv_rn(amax, 127.f);
  if (threadIdx.x == 0) a.scales[t] = whole ? s : __int_as_float(0x7fc00000);
  const bool codes = whole && s > 0.f;
  const Rounding rd(codes ? s : 1.f);
  int8_t* row = a.codes + (size_t)t * a.ldc;
  auto put = [&](int k, const float (&v)[8]) {
    uint32_t w[2] = {0u, 0u};
    if (codes) {                                         // (no scale: codes of zero)
      float n[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = a.g ? v[e] * rstd : v[e];
      codes8<8>(n, rd, w);
    }
    *reinterpret_cast<uint2*>(row + k) = make_uint2(w[0], w[1]);
  };
  if (VPT) {
#pragma unroll
    for (int i = 0; i < (VPT ? VPT : 1); ++i) {
      const int k = (i * THREADS + threadIdx.x) * 8;
      if (k < a.ldc) put(k, keep[i]);
    }
  } else {
    for (int k = threadIdx.x * 8; k < a.ldc; k += THREADS * 8) {
      float v[8];
      if (k < K) { load(k, v); if (a.g) weigh(k, v); }
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
      put(k, v);
    }
  }
}

// bfloat16 rows without a norm that 16-byte loads read (activations, weights): the numbers stay packed between the two looks, and the first is an
// integer maximum of two numbers' lower 15 bits at a time, which a NaN or an infinity tops (with floats 2,048 rows of 8,192 took 20 us).
template <int VPT>
__global__ void __launch_bounds__(THREADS)
quantize_bf16_kernel(const RowArgs a) {
  if (a.early) pdl_launch();
  pdl_wait();
  __shared__ float red[32];
  const int t = blockIdx.x, K = a.K;
  const bf16* x = (const bf16*)a.x + (size_t)(a.rows ? a.rows[t] : t) * a.ldx;
  uint4 keep[VPT];
  uint32_t mx2 = 0u;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = (i * THREADS + threadIdx.x) * 8;
    keep[i] = k < K ? __ldcg(reinterpret_cast<const uint4*>(x + k)) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t w[4] = {keep[i].x, keep[i].y, keep[i].z, keep[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("max.u16x2 %0, %0, %1;" : "+r"(mx2) : "r"(w[e] & 0x7fff7fffu));
  }
  const uint32_t top = max(mx2 & 0xffffu, mx2 >> 16);
  const float mx = block_max(top < 0x7f80u ? __uint_as_float(top << 16) : INFINITY, red);
  const bool whole = mx <= 3.402823466e38f;
  const float s = __fdiv_rn(mx, 127.f);
  const bool codes = whole && s > 0.f;
  if (threadIdx.x == 0) a.scales[t] = whole ? s : __int_as_float(0x7fc00000);
  const Rounding rd(codes ? s : 1.f);
  int8_t* row = a.codes + (size_t)t * a.ldc;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int k = (i * THREADS + threadIdx.x) * 8;
    if (k >= a.ldc) break;
    const uint32_t w[4] = {keep[i].x, keep[i].y, keep[i].z, keep[i].w};
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[2 * e] = bf16_lo(w[e]); v[2 * e + 1] = bf16_hi(w[e]); }
    uint32_t c[2] = {0u, 0u};
    if (codes) codes8<8>(v, rd, c);
    *reinterpret_cast<uint2*>(row + k) = make_uint2(c[0], c[1]);
  }
}

template <typename T, bool VEC>
int launch_rows(const RowArgs& a, int T_, cudaStream_t s) {
  const long long groups = (a.ldc + THREADS * 8 - 1) / (THREADS * 8);
  if (sizeof(T) == 2 && VEC && !a.g && groups <= 8) {
    if (groups <= 1) return launch_ex(quantize_bf16_kernel<1>, dim3(T_), dim3(THREADS), 0, s, 1, a);
    if (groups <= 2) return launch_ex(quantize_bf16_kernel<2>, dim3(T_), dim3(THREADS), 0, s, 1, a);
    if (groups <= 4) return launch_ex(quantize_bf16_kernel<4>, dim3(T_), dim3(THREADS), 0, s, 1, a);
    return launch_ex(quantize_bf16_kernel<8>, dim3(T_), dim3(THREADS), 0, s, 1, a);
  }
  if (groups <= 1) return launch_ex(quantize_rows_kernel<T, 1, VEC>, dim3(T_), dim3(THREADS), 0, s, 1, a);
  if (groups <= 2) return launch_ex(quantize_rows_kernel<T, 2, VEC>, dim3(T_), dim3(THREADS), 0, s, 1, a);
  if (groups <= 4) return launch_ex(quantize_rows_kernel<T, 4, VEC>, dim3(T_), dim3(THREADS), 0, s, 1, a);
  if (groups <= 8) return launch_ex(quantize_rows_kernel<T, 8, VEC>, dim3(T_), dim3(THREADS), 0, s, 1, a);
  return launch_ex(quantize_rows_kernel<T, 0, VEC>, dim3(T_), dim3(THREADS), 0, s, 1, a);
}

}  // namespace

// x [*, K] float or bf16 with row stride ldx; rows int32 [T] or null; g norm weight [K] (g_dt) or null. codes int8 [T, ldc], ldc a
// multiple of 16 that holds K, zeros behind K; scales float [T]. early: the next kernel in the stream may begin before this one has ended.
RLLM_API int rllm_quantize_rows(int dt, const void* x, long long ldx, const int* rows, const void* g, int g_dt, float eps,
                                void* codes, long long ldc, float* scales, int T, int K, int early, void* stream) {
  if (T <= 0) return 0;
  if (K <= 0 || ldc < K || ldc % 16 || ldc - K >= 16) return ERR_BAD_SIZE;
  if ((uintptr_t)codes & 15) return ERR_BAD_ALIGN;
  if (dt != DT_F32 && dt != DT_BF16) return ERR_BAD_DTYPE;
  const RowArgs a = {x, ldx, rows, g, g_dt == DT_BF16, eps, (int8_t*)codes, ldc, scales, K, early};
  const int unit = dt == DT_F32 ? 4 : 8;
  const bool vec = K % 8 == 0 && ldx % unit == 0 && !((uintptr_t)x & 15) && !((uintptr_t)g & 15);
  cudaStream_t s = (cudaStream_t)stream;
  if (dt == DT_F32) return vec ? launch_rows<float, true>(a, T, s) : launch_rows<float, false>(a, T, s);
  return vec ? launch_rows<bf16, true>(a, T, s) : launch_rows<bf16, false>(a, T, s);
}
