// The cache held in 4 bits: new keys and values stored, stored ones read back (layout and formulas: quant.cuh).
//
// Both kernels are a read and a write with little between. Eight lanes share the 64 dimensions of a row's block, four numbers of
// each of its two groups a lane: the groups' largest numbers meet in three shuffles, a lane's eight codes are one word,
// and the block's 32 bytes and its two scales leave as whole pieces. 2,048 tokens of 8 heads of 128 are stored and read back as floats in 17 us
// (27.5 MB, 1.6 TB/s: instructions a number, a quotient on the one side and a product on the other, bound both: the store issues one in 80 % of its
// cycles, the read in 69 %), 8 of 8 heads of 64 in 4.9.
#include "quant.cuh"
#include <cuda_fp16.h>

using namespace rllm;

namespace {

constexpr int THREADS = 256;

struct Pages {                       // one layer's tensors
  uint8_t* k4; uint8_t* v4; bf16* ks; bf16* vs;
  int nkv, page_size, hd;
};

template <typename T> __device__ __forceinline__ void load4(const T* p, bool vec, float (&v)[4]) {
  if (sizeof(T) == 2 && vec) {
    const uint2 a = __ldcg(reinterpret_cast<const uint2*>(p));
    v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
  } else if (sizeof(T) == 4 && vec) {
    const float4 a = __ldcg(reinterpret_cast<const float4*>(p));
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f32(p[i]);
  }
}

// The codes (as nibbles from bit `shift` of `word` on) and the scale of a group, four numbers of it in each of eight lanes.
__device__ __forceinline__ bf16 quantize_group(const float (&v)[4], int shift, uint32_t& word) {
  float hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), lo = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
  float bad = fmaf(v[0], 0.f, fmaf(v[1], 0.f, fmaf(v[2], 0.f, v[3] * 0.f)));      // 0, or NaN where a number is not finite
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    bad += __shfl_xor_sync(0xffffffffu, bad, o);
  }
  bf16 d = __float2bfloat16_rn((hi >= -lo ? hi : lo) * -0.125f);
  if (bad != 0.f) d = __ushort_as_bfloat16((unsigned short)0x7fc0);
  const float df = __bfloat162float(d);
  const bool codes = df != 0.f && bad == 0.f;
  const Rounding rd(codes ? df : 1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = codes ? rd.code(v[i], -8, 7) : 0;
    word |= (uint32_t)(c + 8) << (shift + 4 * i);
  }
  return d;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
kv4_store_kernel(const T* __restrict__ k, const T* __restrict__ v, long long ldk, long long ldv, bool vec,
                 const int* __restrict__ slots, long long num_slots, Pages c, long long units) {
  pdl_launch();
  pdl_wait();
  const long long idx = (long long)blockIdx.x * THREADS + threadIdx.x;
  const int w = (int)(idx & 7);
  long long u = idx >> 3;                                // (token, keys or values, head, block of 64)
  const bool live = u < units;                           // (the lanes of a warp stay together for the shuffles)
  if (!live) u = units - 1;
  const int blocks = c.hd >> 6;
  const int b = (int)(u % blocks);
  const int h = (int)(u / blocks % c.nkv);
  const long long tv = u / ((long long)blocks * c.nkv);
  const bool is_v = tv & 1;
  const long long t = tv >> 1;
  const int slot = slots[t];
  const T* src = (is_v ? v + t * ldv : k + t * ldk) + (size_t)h * c.hd + 64 * b + 4 * w;
  float x0[4], x1[4];
  load4<T>(src, vec, x0);
  load4<T>(src + 32, vec, x1);
  uint32_t word = 0u;
  const bf16 d0 = quantize_group(x0, 0, word), d1 = quantize_group(x1, 16, word);
  if (!live || slot < 0 || slot >= num_slots) return;    // a slot of -1: the layer must not write this token
  const size_t row = ((size_t)(slot / c.page_size) * c.nkv + h) * c.page_size + slot % c.page_size;
  reinterpret_cast<uint32_t*>((is_v ? c.v4 : c.k4) + row * (c.hd >> 1))[8 * b + w] = word;
  if (w == 0) {
    const uint32_t two = (uint32_t)__bfloat16_as_ushort(d0) | (uint32_t)__bfloat16_as_ushort(d1) << 16;
    reinterpret_cast<uint32_t*>((is_v ? c.vs : c.ks) + row * (c.hd >> 5))[b] = two;
  }
}

__device__ __forceinline__ void store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(bf16* p, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

__device__ __forceinline__ void store4h(void* p, const float (&v)[4]) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {       // of both halves
  asm("max.u16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
__device__ __forceinline__ uint32_t block_max2(uint32_t v) {              // eight neighbouring lanes have the same
  __shared__ uint32_t red[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 4; o >>= 1) v = max2(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) v = max2(v, red[w]);
  return v;
}

// Places i * out_page .. of sequence s go to page s * width + i of the output, in the cache's order [kv head][offset][hd]; places behind
// the sequence's last token are zeros, and so are those in pages it does not hold. A CTA takes one kv head's part of a page. With `cu_q` (attention
// of portions) i counts from the page of the first place that a query of the step sees, and pages that none sees are left out; table_out
// [table_width pages from place 0 on] says where which are, cu_out counts the portions' rows from zero.
// vexp: the values are 16-bit numbers times a power of two a page and kv head (`value_word`). A value has 12 significant bits: half numbers hold 11
// of them, bfloat16 8, but half numbers have few powers of two. So a page whose scales lie within 2^6 of each other is half numbers, its
// largest scale between 1 and 2; any other is bfloat16, its smallest scale (but not less than 2^-40 of its largest) between 1 and 2. The power
// joins the scores where the weights are made: with the smallest scale no group of such a page, be it one a row's weight lies
// wholly on, raises a row's maximum by more than it adds to the sum, so that the other pages' weights, in half precision, keep their bits.
// A page of zeros adds nothing and so has the lowest power; not a lower one still, since its weights, times that power beside
// others', have to stay float numbers for the denominator. vlost: the places of groups whose scale is NaN.
// UNITS: pieces (place, block of 64 dimensions) that a thread has at once, eight lanes together: 8 are a page of 128 places of 128 dimensions.
// (With place after place, each behind its page's number, 2,012 keys of 8 heads of 128 took 11.5 us to read, now 7.6.)
template <typename T, int UNITS>
__global__ void __launch_bounds__(THREADS)
kv4_read_kernel(Pages c, long long num_pages, int page_shift, const int* __restrict__ block_table, int bt_stride, const int* __restrict__ kv_lens,
                const int* __restrict__ cu_q, int window, int num_seqs, int width, int out_page, T* __restrict__ k, T* __restrict__ v,
                int table_width, int* __restrict__ table_out, int* __restrict__ cu_out, int* __restrict__ vexp, uint32_t* __restrict__ vlost) {
  pdl_launch();
  pdl_wait();
  const int i = blockIdx.x, s = blockIdx.y;
  const bool is_v = (int)blockIdx.z >= c.nkv;
  const int kvh = (int)blockIdx.z - (is_v ? c.nkv : 0);
  const int n = kv_lens[s];
  int first = 0;                                         // the first position that a query sees
  if (cu_q != nullptr && window > 0) first = max(0, n - (cu_q[s + 1] - cu_q[s]) - window + 1);
  const int base = first > 0 ? first / out_page : 0, at = base + i, j0 = at * out_page;
  const bool left_out = table_out != nullptr && (j0 >= n || at >= table_width);
  if (table_out != nullptr && i == 0 && blockIdx.z == 0)
    for (int t = threadIdx.x; t < table_width; t += THREADS)
      if (t < base || t >= base + width) table_out[(size_t)s * table_width + t] = -1;
  if (threadIdx.x == 0 && blockIdx.z == 0) {
    if (table_out != nullptr && at < table_width) table_out[(size_t)s * table_width + at] = left_out ? -1 : s * width + i;
    if (cu_out != nullptr && i == 0) {
      cu_out[s] = cu_q[s] - cu_q[0];
      if (s == num_seqs - 1) cu_out[s + 1] = cu_q[s + 1] - cu_q[0];
    }
  }
  if (left_out) return;
  const int blocks = c.hd >> 6, w = threadIdx.x & 7, units = out_page * blocks;
  const uint8_t* src = is_v ? c.v4 : c.k4;
  const bf16* sc = is_v ? c.vs : c.ks;
  T* dst = (is_v ? v : k) + (((size_t)s * width + i) * c.nkv + kvh) * out_page * c.hd;
  const int* bt = block_table + (size_t)s * bt_stride;
  const bool half = sizeof(T) == 2 && is_v && vexp != nullptr;
#pragma unroll 1
  for (int u0 = threadIdx.x >> 3; u0 < units; u0 += UNITS * (THREADS / 8)) {
    // a thread's units (place, block of 64 dimensions), all of its page numbers on their way at once, then all of its words
    int page[UNITS];
    uint32_t word[UNITS], two[UNITS];
    bool there[UNITS];
    auto place = [&](int e, int& r, int& b) { const int u = u0 + e * (THREADS / 8); r = blocks == 1 ? u : blocks == 2 ? u >> 1 : u / blocks; b = u - r * blocks; };
    auto page_of = [&](int j) { return page_shift >= 0 ? j >> page_shift : j / c.page_size; };
#pragma unroll
    for (int e = 0; e < UNITS; ++e) {
      int r, b;
      place(e, r, b);
      page[e] = r < out_page && j0 + r < n ? bt[page_of(j0 + r)] : -1;      // -1: behind the last token, or on a page that is not held
    }
#pragma unroll
    for (int e = 0; e < UNITS; ++e) {
      int r, b;
      place(e, r, b);
      const int j = j0 + r;
      const size_t row = ((size_t)page[e] * c.nkv + kvh) * c.page_size + (j - page_of(j) * c.page_size);
      there[e] = page[e] >= 0 && page[e] < num_pages;
      word[e] = there[e] ? __ldcg(reinterpret_cast<const uint32_t*>(src + row * (c.hd >> 1)) + 8 * b + w) : 0u;
      two[e] = there[e] ? __ldcg(reinterpret_cast<const uint32_t*>(sc + row * (c.hd >> 5)) + b) : 0u;
    }
    float down = 1.f;
    bool wide = false;
    if (half) {                                          // (the page is one turn of the loop)
      // the largest scale's bits, and 0x7fff less the smallest's, as two maxima in a word
      auto both_ends = [&]() {
        uint32_t hi = 0u, lo = 0u;
#pragma unroll
        for (int e = 0; e < UNITS; ++e) {
          const uint32_t m = two[e] & 0x7fff7fffu;
          hi = max2(hi, m);
          lo = max2(lo, there[e] ? 0x7fff7fffu - m : 0u);
        }
        return block_max2(max(hi & 0xffffu, hi >> 16) | max(lo & 0xffffu, lo >> 16) << 16);
      };
      uint32_t ends = both_ends();
      const bool lost = (ends & 0xffffu) >= 0x7f80u;
      if (lost) {                                        // a scale of NaN: zeros (a number times zero), a bit, and the ends of the others
        __shared__ uint32_t bits[4 * 8];                 // [group][32 places]: at most 256 pieces of two groups
        const int words = out_page / 32, all = 2 * blocks * words;
        if (threadIdx.x < 32) bits[threadIdx.x] = 0u;
        __syncthreads();
        uint32_t hi = 0u, lo = 0u;
#pragma unroll
        for (int e = 0; e < UNITS; ++e) {
          int r, b;
          place(e, r, b);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const uint32_t m = two[e] >> (16 * g) & 0x7fffu;
            if (m >= 0x7f80u) {
              two[e] &= g ? 0xffffu : 0xffff0000u;
              if (w == g) atomicOr(&bits[(2 * b + g) * words + (r >> 5)], 1u << (r & 31));
            } else {
              hi = max(hi, m);
              lo = max(lo, there[e] ? 0x7fffu - m : 0u);
            }
          }
        }
        ends = block_max2(hi | lo << 16);
        if ((int)threadIdx.x < all) vlost[(((size_t)s * width + i) * c.nkv + kvh) * all + threadIdx.x] = bits[threadIdx.x];
      }
      const int top = (int)(ends >> 7 & 0xffu) - 127, low = (int)((0x7fffu - (ends >> 16)) >> 7 & 0xffu) - 127;
      const bool zeros = (ends & 0xffffu) == 0u;
      wide = !zeros && (low < top - 6 || top < -VALUE_EXPONENTS || top > VALUE_EXPONENTS);
      const int e = zeros ? ZEROS_EXPONENT : min(max(wide ? max(low, top - 40) : top, -VALUE_EXPONENTS), VALUE_EXPONENTS);
      if (threadIdx.x == 0) vexp[((size_t)s * width + i) * c.nkv + kvh] = value_word(e, wide, lost);
      down = __int_as_float((127 - e) << 23);
    }
#pragma unroll
    for (int e = 0; e < UNITS; ++e) {
      int r, b;
      place(e, r, b);
      if (r >= out_page) break;
      float x0[4] = {0.f, 0.f, 0.f, 0.f}, x1[4] = {0.f, 0.f, 0.f, 0.f};
      if (there[e]) {
        const float d0 = bf16_lo(two[e]) * down, d1 = bf16_hi(two[e]) * down;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) { x0[i4] = (float)code4(word[e], i4) * d0; x1[i4] = (float)code4(word[e], 4 + i4) * d1; }
      }
      T* o = dst + (size_t)r * c.hd + 64 * b + 4 * w;
      if (half && !wide) { store4h(o, x0); store4h(o + 32, x1); }
      else { store4(o, x0); store4(o + 32, x1); }
    }
  }
}

int make_pages(Pages& c, void* k4, void* ks, void* v4, void* vs, int nkv, int page_size, int hd) {
  if (nkv <= 0 || page_size <= 0 || (hd != 64 && hd != 128 && hd != 192 && hd != 256)) return ERR_BAD_SIZE;
  if (((uintptr_t)k4 | (uintptr_t)v4 | (uintptr_t)ks | (uintptr_t)vs) & 15) return ERR_BAD_ALIGN;
  c.k4 = (uint8_t*)k4; c.v4 = (uint8_t*)v4; c.ks = (bf16*)ks; c.vs = (bf16*)vs; c.nkv = nkv; c.page_size = page_size; c.hd = hd;
  return 0;
}

}  // namespace

// k, v [T, nkv * hd] float or bf16 with row strides ldk, ldv; slots int32 [T]: page * page_size + offset, -1 (or beyond the
// num_pages pages): not stored. No slot twice in a call.
RLLM_API int rllm_kv4_store(int dt, const void* k, const void* v, long long ldk, long long ldv, const int* slots, void* k4, void* ks,
                            void* v4, void* vs, long long num_pages, int T, int nkv, int page_size, int hd, void* stream) {
  if (T <= 0) return 0;
  Pages c;
  const int rc = make_pages(c, k4, ks, v4, vs, nkv, page_size, hd);
  if (rc) return rc;
  const long long units = (long long)T * 2 * nkv * (hd >> 6);
  const long long blocks = (units * 8 + THREADS - 1) / THREADS;
  if (blocks > 2147483647LL) return ERR_TOO_LARGE;
  const uintptr_t piece = dt == DT_F32 ? 15 : 7;
  const bool vec = ldk % 4 == 0 && ldv % 4 == 0 && !(((uintptr_t)k | (uintptr_t)v) & piece);
  cudaStream_t s = (cudaStream_t)stream;
  if (dt == DT_F32)
    return launch_ex(kv4_store_kernel<float>, dim3((unsigned)blocks), dim3(THREADS), 0, s, 1, (const float*)k, (const float*)v, ldk, ldv,
                     vec, slots, num_pages * page_size, c, units);
  if (dt == DT_BF16)
    return launch_ex(kv4_store_kernel<bf16>, dim3((unsigned)blocks), dim3(THREADS), 0, s, 1, (const bf16*)k, (const bf16*)v, ldk, ldv,
                     vec, slots, num_pages * page_size, c, units);
  return ERR_BAD_DTYPE;
}

// The sequences' keys and values as numbers: k, v [num_seqs * width, nkv, out_page, hd] float or bf16 (rounded once). kv_lens int32
// [num_seqs], none above width * out_page (with cu_q and a window: no more places seen than `width` pages hold); block_table int32 with an entry
// for each of their pages. cu_q (int32 [num_seqs + 1]), window, table_out [num_seqs, table_width] and cu_out
// [num_seqs + 1], and vexp [num_seqs * width, nkv] with vlost [num_seqs * width, nkv, hd / 32, out_page / 32] (bf16 only: v is then 16-bit
// numbers as `value_word` says; pages of a multiple of 32 places, out_page * hd / 64 between 32 and 256) for attention of portions, or null.
RLLM_API int rllm_kv4_read(int dt, void* k4, void* ks, void* v4, void* vs, long long num_pages, const int* block_table, int bt_stride,
                           const int* kv_lens, const int* cu_q, int window, int num_seqs, int width, int out_page, void* k,
                           void* v, int table_width, int* table_out, int* cu_out, int* vexp, uint32_t* vlost,
                           int nkv, int page_size, int hd, void* stream) {
  if (num_seqs <= 0 || width <= 0) return 0;
  if (out_page <= 0 || 2 * nkv > 65535) return ERR_BAD_SIZE;
  if (vexp != nullptr && (dt != DT_BF16 || (long long)out_page * (hd >> 6) > 8 * (THREADS / 8) || out_page * (hd >> 6) < THREADS / 8 || out_page % 32 || !vlost)) return ERR_BAD_SIZE;
  Pages c;
  const int rc = make_pages(c, k4, ks, v4, vs, nkv, page_size, hd);
  if (rc) return rc;
  if (num_seqs > 65535 || (cu_out != nullptr && cu_q == nullptr) || (long long)num_seqs * width > 2147483647LL || (long long)width * out_page > 2147483647LL || (long long)table_width * out_page > 2147483647LL) return ERR_TOO_LARGE;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return ERR_BAD_ALIGN;
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid(width, num_seqs, 2 * nkv);
  int shift = -1;
  for (int b = 0; b < 31; ++b) if ((1 << b) == page_size) shift = b;
  auto run = [&](auto type, auto kernel) {
    typedef decltype(type) T;
    return launch_ex(kernel, grid, dim3(THREADS), 0, s, 1, c, num_pages, shift, block_table, bt_stride, kv_lens, cu_q, window, num_seqs, width,
                     out_page, (T*)k, (T*)v, table_width, table_out, cu_out, vexp, vlost);
  };
  const long long each = ((long long)out_page * (hd >> 6) + THREADS / 8 - 1) / (THREADS / 8);
  if (dt == DT_F32) return each <= 1 ? run(float(), kv4_read_kernel<float, 1>) : each <= 4 ? run(float(), kv4_read_kernel<float, 4>) : run(float(), kv4_read_kernel<float, 8>);
  if (dt == DT_BF16) return each <= 1 ? run(bf16(), kv4_read_kernel<bf16, 1>) : each <= 4 ? run(bf16(), kv4_read_kernel<bf16, 4>) : run(bf16(), kv4_read_kernel<bf16, 8>);
  return ERR_BAD_DTYPE;
}
