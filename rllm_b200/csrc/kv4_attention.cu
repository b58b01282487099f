// Attention over the paged cache held in 4 bits (layout: quant.cuh).
//
// On the CUDA cores, for any mix of prompt portions and single tokens, both run types and head sizes of 64, 128, 192 and 256: one
// warp per (query token, query head), keys 32 at a time in position order with a running maximum and sum, all arithmetic in
// float, as paged_attention_simt_kernel does over a cache of whole numbers. A lane scores one key: the key's codes times the
// queries of a group of 32 are summed first and multiplied by the group's scale once. The weighted sum of the values takes one
// byte of a row's block a lane, which is two neighbouring dimensions.
#include "quant.cuh"

using namespace rllm;

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
    bool valid = j <= pos;
    float s = -INFINITY;
    long long row = 0;
    const int page = valid ? bt[j / p.page_size] : -1;
    valid = valid && page >= 0 && page < p.num_pages;      // a table entry without a page: not read
    if (valid) {
      row = ((long long)page * p.nkv + kvh) * p.page_size + j % p.page_size;
      s = 0.f;
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
      if (!__shfl_sync(0xffffffffu, (int)valid, jj)) continue;
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
                       token_seq, positions, nullptr, block_table, bt_stride, T, nh, nkv, page_size, window, scale};
  if (dt == DT_F32) return launch_simt<float>(p, hd, (cudaStream_t)stream);
  if (dt == DT_BF16) return launch_simt<bf16>(p, hd, (cudaStream_t)stream);
  return ERR_BAD_DTYPE;
}
