// Parameters and device helpers shared by the paged-attention kernels.
#pragma once
#include "tc_sm100.cuh"

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
  int prefix_parts, own_parts;        // slots for parts
  float scale_log2;
  float *part_o;                      // [part][T * Hq][D]
  float2 *part_ml;                    // [part][T * Hq]: row maximum (base 2) and sum
  int tile_tokens, piece;             // tensor-core form: tokens of a tile, keys of one TMA box
  int cluster;                        // and key ranges of a tile that one cluster joins
  int follows_prefix;                 // the stream follows the call's tensor-core launch over the prefix
  int nseq;                           // sequences in the stream: B, or 0 without own keys
  int stream_prefix;                  // the stream of key blocks covers the prefix too
  int *prefix_runs, *own_runs;        // [T * Hq]: parts in use, or NULL: all slots are
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

// Result of a part, elements d .. d + W - 1 of one row, or the output itself when the call has one part.  l == 0 marks a
// part in which the row saw no key: its O is neither stored nor read.
template <int W>
__device__ __forceinline__ void store_row(const Params &p, int part, int t, int hd, int d, float (&f)[W], float m, float l) {
  if (p.part_o) {
    const int64_t i = (int64_t)part * p.T * p.Hq + (int64_t)t * p.Hq + hd;
    if (d == 0) p.part_ml[i] = make_float2(m, l);
    if (l != 0.f) {
      float2 *o = reinterpret_cast<float2 *>(p.part_o + i * p.D + d);
      if (W == 4) *reinterpret_cast<float4 *>(o) = make_float4(f[0], f[1], f[W - 2], f[W - 1]);
      else *o = make_float2(f[0], f[1]);
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    __half2 *o = reinterpret_cast<__half2 *>(p.out + (int64_t)t * p.so_t + (int64_t)hd * p.so_h + d);
#pragma unroll
    for (int e = 0; e < W; e += 2) o[e / 2] = __floats2half2_rn(f[e] * inv, f[e + 1] * inv);
  }
}

// Tensor maps of the two caches: boxes of 64 columns of `piece` slots of a page.
int cache_maps(const Params &p, int hkv, CUtensorMap *tm);

// Tensor-core form (paged_attention_tc.cu): seq false: rows of the batch against the prefix; true: rows of each
// sequence against the prefix and its own keys.
int tc_launch(const Params &p, int hkv, bool seq, dim3 grid, cudaStream_t st);

}  // namespace paged
}  // namespace hexb
