// Products in 8-bit integers: Y[t, n] = (sum_k X[t, k] W[n, k]) * sx[t] * sw[n], codes with one scale a row on both sides. The sum of
// code products is exact in 32 bits up to K = 131,072 (127^2 K < 2^31).
//
// One thread an output, four products an instruction.
#include "quant.cuh"

using namespace rllm;

namespace {

enum : int { EPI_STORE = 0, EPI_STORE_F32 = 1, EPI_ACCUM_F32 = 2, EPI_SWIGLU = 3 };

struct Int8Params {
  const int8_t* x; const float* sx;
  const int8_t* w; const float* sw;
  void* y; long long ldy;
  int T, N, K;                       // N: outputs (of one half with SwiGLU); K: bytes a row, a multiple of 16
};

__device__ __forceinline__ float silu_gate(float g, float u) { return g / (1.f + expf(-g)) * u; }

template <int EPI, typename OUT>
__global__ void __launch_bounds__(256)
int8_simple_kernel(const Int8Params p) {
  pdl_launch();
  pdl_wait();
  const int n = blockIdx.x * 32 + (threadIdx.x & 31), t = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (n >= p.N || t >= p.T) return;
  float v[2];
#pragma unroll
  for (int half = 0; half < (EPI == EPI_SWIGLU ? 2 : 1); ++half) {
    const int row = n + half * p.N;
    const int* x = reinterpret_cast<const int*>(p.x + (size_t)t * p.K);
    const int* w = reinterpret_cast<const int*>(p.w + (size_t)row * p.K);
    int acc = 0;
    for (int k = 0; k < p.K / 4; ++k) acc = __dp4a(x[k], w[k], acc);
    v[half] = (float)acc * p.sx[t] * p.sw[row];
  }
  const size_t o = (size_t)t * p.ldy + n;
  if (EPI == EPI_ACCUM_F32) ((float*)p.y)[o] += v[0];
  else ((OUT*)p.y)[o] = from_f32<OUT>(EPI == EPI_SWIGLU ? silu_gate(v[0], v[1]) : v[0]);
}

template <int EPI, typename OUT>
int launch_simple(const Int8Params& p, cudaStream_t s) {
  return launch_ex(int8_simple_kernel<EPI, OUT>, dim3((p.N + 31) / 32, (p.T + 7) / 8), dim3(256), 0, s, 1, p);
}

}  // namespace

// x int8 [T, K] with scales sx [T]; w int8 [N, K] (SwiGLU: [2 N, K], gate rows first) with scales sw; K a multiple of 16, both
// 16-byte aligned. y [T, N] in out_dt (epilogues 0 and 3) or float (1, 2: added), row stride ldy.
RLLM_API int rllm_int8_gemm(int epi, int out_dt, const void* x, const float* sx, const void* w, const float* sw, void* y, long long ldy,
                            int T, int N, int K, int* err, int sm_count, void* stream) {
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 16 || K > 131072 || ldy < N || epi < 0 || epi > 3) return ERR_BAD_SIZE;
  if (((uintptr_t)x | (uintptr_t)w) & 15) return ERR_BAD_ALIGN;
  if (out_dt != DT_F32 && out_dt != DT_BF16) return ERR_BAD_DTYPE;
  (void)err; (void)sm_count;
  const Int8Params p = {(const int8_t*)x, sx, (const int8_t*)w, sw, y, ldy, T, N, K};
  cudaStream_t s = (cudaStream_t)stream;
  if (epi == EPI_STORE_F32) return launch_simple<EPI_STORE_F32, float>(p, s);
  if (epi == EPI_ACCUM_F32) return launch_simple<EPI_ACCUM_F32, float>(p, s);
  if (epi == EPI_STORE) return out_dt == DT_F32 ? launch_simple<EPI_STORE, float>(p, s) : launch_simple<EPI_STORE, bf16>(p, s);
  return out_dt == DT_F32 ? launch_simple<EPI_SWIGLU, float>(p, s) : launch_simple<EPI_SWIGLU, bf16>(p, s);
}
