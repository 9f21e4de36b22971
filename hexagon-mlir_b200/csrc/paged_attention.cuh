// Parameters and device helpers shared by the paged-attention kernels.
#pragma once
#include "common.cuh"

namespace hexb {

static __device__ int g_paged_status = 0;  // one word per source file that includes this header

namespace paged {

struct Params {
  const __half *q, *k, *v;
  __half *out;
  int64_t sq_t, sq_h;                 // q [token, head, D]
  int64_t sk_p, sk_s, sk_h;           // k cache [page, slot, head, D]
  int64_t sv_p, sv_s, sv_h;
  int64_t so_t, so_h;
  const int *prefix_pages, *table, *lens, *offsets;
  int64_t table_stride;
  int T, B, Hq, G, D;
  int prefix_len, page_size, num_pages, own_capacity;
  int prefix_parts, prefix_chunk, own_parts;
  float scale_log2;
  float *part_o;                      // [part][T * Hq][D]
  float2 *part_ml;                    // [part][T * Hq]: row maximum (base 2) and sum
};

// Tokens [tok0, tok0 + n) of sequence b.  Offsets are data on the device: whatever they hold, the rows
// stay inside the tensors.
__device__ __forceinline__ void seq_range(const Params &p, int b, int &tok0, int &n) {
  if (!p.offsets) {
    tok0 = b;
    n = 1;
    return;
  }
  tok0 = min(max(p.offsets[b], 0), p.T);
  n = min(max(p.offsets[b + 1], tok0), p.T) - tok0;
}
__device__ __forceinline__ int tokens_used(const Params &p) {
  return p.offsets ? min(max(p.offsets[p.B], 0), p.T) : p.T;
}
// Own length of sequence b; more than its pages hold is cut and recorded.
__device__ __forceinline__ int seq_len(const Params &p, int b) {
  const int n = p.lens[b];
  if (n > p.own_capacity) atomicExch(&g_paged_status, (int)HEXB_ERR_BAD_ARG);
  return min(max(n, 0), p.own_capacity);
}

// Results of a part, or the output itself when the call has one part.  l == 0 marks a part in which the row saw
// no key: its O is neither stored nor read.
__device__ __forceinline__ void store4(const Params &p, int part, int t, int hd, int d, const float (&f)[4], float m, float l) {
  if (p.part_o) {
    const int64_t i = (int64_t)part * p.T * p.Hq + (int64_t)t * p.Hq + hd;
    if (d == 0) p.part_ml[i] = make_float2(m, l);
    if (l != 0.f) *reinterpret_cast<float4 *>(p.part_o + i * p.D + d) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    __half2 *o = reinterpret_cast<__half2 *>(p.out + (int64_t)t * p.so_t + (int64_t)hd * p.so_h + d);
    o[0] = __floats2half2_rn(f[0] * inv, f[1] * inv);
    o[1] = __floats2half2_rn(f[2] * inv, f[3] * inv);
  }
}
__device__ __forceinline__ void store2(const Params &p, int part, int t, int hd, int d, float a, float b, float m, float l) {
  if (p.part_o) {
    const int64_t i = (int64_t)part * p.T * p.Hq + (int64_t)t * p.Hq + hd;
    if (d == 0) p.part_ml[i] = make_float2(m, l);
    if (l != 0.f) *reinterpret_cast<float2 *>(p.part_o + i * p.D + d) = make_float2(a, b);
  } else {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<__half2 *>(p.out + (int64_t)t * p.so_t + (int64_t)hd * p.so_h + d) = __floats2half2_rn(a * inv, b * inv);
  }
}

}  // namespace paged
}  // namespace hexb
