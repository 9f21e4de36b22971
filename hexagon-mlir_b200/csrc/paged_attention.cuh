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
  int prefix_parts;
  float scale_log2;
  // Parts: O [index][D] and (row maximum in base 2, sum) [index].  Indexes below run_base: slots of T * Hq rows (the
  // tensor-core prefix parts, or the prefix runs of whole tiles at prefix_slot, and the own runs of whole tiles at
  // own_slot; slot -1: the output).  From run_base on: two tiles of rows per CTA of the list of units, for a run
  // that begins (0) or only ends (1) inside a tile -- a CTA has one of each at most.
  float *part_o;
  float2 *part_ml;
  int64_t run_base;
  int prefix_slot, own_slot, ctas, tile_rows;
  int4 *prefix_desc, *own_desc;       // per row: runs of its tile (0: in its slot, -1: stored), CTA of the first, row in the tile
  int shared_blocks;                  // blocks of the prefix at the head of every sequence's axis
  int tile_tokens, piece;             // tensor-core form: tokens of a tile, keys of one TMA box
  int cluster;                        // and key ranges of a tile that one cluster joins
  int nseq;                           // sequences in the stream: B, or 0 without own keys
  int stream_prefix;                  // the stream of key blocks covers the prefix too
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

// Part `i` of a row, elements d .. d + W - 1, or the output itself (i < 0).  l == 0 marks a part in which the row saw no
// key: its O is neither stored nor used.
template <int W>
__device__ __forceinline__ void store_row(const Params &p, int64_t i, int t, int hd, int d, float (&f)[W], float m, float l) {
  if (i >= 0) {
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

// A place in the list of units.
struct Cursor {
  int b;                 // -1: the prefix
  int tok0, ntok, len, nb, nt;
  int h, tile, j;
};

__device__ __forceinline__ int blocks_of(const Params &p, int b, int len) {
  // a tile without keys is one unit too: its rows get an empty part
  return max((b < 0 ? 0 : p.shared_blocks) + (len + 63) / 64, 1);
}
__device__ __forceinline__ long long sequence_units(const Params &p, int rows, int b, int *tok0, int *ntok, int *len) {
  if (b < 0) {
    *tok0 = 0;
    *ntok = tokens_used(p);
    *len = p.prefix_len;
  } else {
    seq_range(p, b, *tok0, *ntok);
    *len = seq_len(p, b);
  }
  return (long long)((*ntok * p.G + rows - 1) / rows) * (p.Hq / p.G) * blocks_of(p, b, *len);
}

__device__ __forceinline__ void enter(const Params &p, int rows, Cursor &c) {
  // the next sequence from c.b on that has tokens
  for (; c.b < p.nseq; ++c.b) {
    if (sequence_units(p, rows, c.b, &c.tok0, &c.ntok, &c.len) > 0) break;
  }
  c.nb = blocks_of(p, c.b, c.len);
  c.nt = (c.ntok * p.G + rows - 1) / rows;
}

// On by `n` units, which do not pass the end of the tile.
__device__ __forceinline__ void advance(const Params &p, int rows, Cursor &c, int n = 1) {
  if ((c.j += n) < c.nb) return;
  c.j = 0;
  if (++c.tile < c.nt) return;
  c.tile = 0;
  if (++c.h < p.Hq / p.G) return;
  c.h = 0;
  ++c.b;
  enter(p, rows, c);
}

// Own keys (of the prefix: its keys) [0, end) are seen by some row of its tile.
__device__ __forceinline__ int end_of(const Params &p, int rows, const Cursor &c) {
  if (c.b < 0) return c.len;
  return min(c.len, c.len - c.ntok + min(c.ntok - 1, (c.tile * rows + rows - 1) / p.G) + 1);
}

// This CTA's stretch of the list: units [start, stop), `per` units a CTA, the cursor at start.  All NT threads call it.
template <int NT>
__device__ __forceinline__ void find_stretch(const Params &p, int rows, long long &start, long long &stop, long long &per, Cursor &c) {
  constexpr int NW = NT / 32;
  __shared__ long long s_sum[NW];
  __shared__ int s_b;
  __shared__ long long s_off;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int first_b = p.stream_prefix ? -1 : 0;
  long long total = 0;
  for (int b = first_b + tid; b < p.nseq; b += NT) {
    int t0, n, len;
    total += sequence_units(p, rows, b, &t0, &n, &len);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < NW; ++w) total += s_sum[w];
  per = max((total + gridDim.x - 1) / gridDim.x, 1ll);
  start = blockIdx.x * per;
  stop = min(start + per, total);
  if (start >= stop) return;
  long long base = 0;
  for (int b0 = first_b; b0 < p.nseq; b0 += NT) {
    int t0, n, len;
    const long long u = b0 + tid < p.nseq ? sequence_units(p, rows, b0 + tid, &t0, &n, &len) : 0;
    long long incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = incl;
    if (tid == 0) s_b = p.nseq;
    __syncthreads();
    long long excl = base + incl - u;
    for (int w = 0; w < warp; ++w) excl += s_sum[w];
    if (start >= excl && start < excl + u) {
      s_b = b0 + tid;
      s_off = start - excl;
    }
    for (int w = 0; w < NW; ++w) base += s_sum[w];
    __syncthreads();
    if (s_b < p.nseq) break;
  }
  c.b = s_b;
  enter(p, rows, c);
  const long long tiles = s_off / c.nb;     // of all key heads
  c.j = (int)(s_off - tiles * c.nb);
  c.h = (int)(tiles / c.nt);
  c.tile = (int)(tiles - (long long)c.h * c.nt);
}

// Where blocks [j0, j1) of the cursor's tile leave their result.  `tile_first`: the tile's first unit in the list.
struct RunPlace {
  int slot;         // rows in order (-1: the output); -2: at `base`
  int64_t base;
  bool last;        // the run ends the tile
  int runs, first;  // for the join
  __device__ __forceinline__ RunPlace(const Params &p, const Cursor &c, int j0, int j1, long long tile_first, long long per, int rows) {
    last = j1 == c.nb;
    base = 0;
    if (j0 == 0 && last) {
      slot = c.b < 0 ? p.prefix_slot : p.own_slot;
      runs = slot < 0 ? -1 : 0;
      first = 0;
    } else {
      slot = -2;
      base = p.run_base + ((int64_t)blockIdx.x * 2 + (j0 == 0)) * rows;
      first = (int)(tile_first / per);
      runs = (int)blockIdx.x - first + 1;
    }
  }
  __device__ __forceinline__ int64_t index(const Params &p, int t, int hd, int r) const {
    if (slot == -2) return base + r;
    return slot < 0 ? -1 : (int64_t)slot * p.T * p.Hq + (int64_t)t * p.Hq + hd;
  }
  __device__ __forceinline__ void describe(const Params &p, const Cursor &c, int t, int hd, int r) const {
    int4 *desc = c.b < 0 ? p.prefix_desc : p.own_desc;
    if (last && desc) desc[(int64_t)t * p.Hq + hd] = make_int4(runs, first, r, 0);
  }
};

// Tensor maps of the two caches: boxes of 64 columns of `piece` slots of a page.
int cache_maps(const Params &p, int hkv, CUtensorMap *tm);

// Tensor-core forms (paged_attention_tc.cu): seq false: rows of the batch against the prefix; true: tiles of the sequences
// against the prefix and their own keys, by the list of units.
int tc_launch(const Params &p, int hkv, bool seq, dim3 grid, cudaStream_t st);

}  // namespace paged
}  // namespace hexb
