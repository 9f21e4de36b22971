// Attention of a batch whose sequences share a prefix, over a paged key/value cache.
//
// Query token t of sequence b sees every key of the shared prefix and the keys j <= len[b] - nq[b] + i of its
// sequence's own pages (i = the token's index among the nq[b] new ones, whose own keys are the last nq[b] of
// the cache): out = softmax(q . K^T * scale) V over their union.  The softmax of a union is joined from
// partial results: a part holds its row maximum m (base 2, scale folded in), l = sum 2^(s - m) and
// O = sum 2^(s - m) v, and
//     out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i,
// so the prefix is read once for all queries of the batch instead of once per sequence, and a long axis is cut
// into parts that run side by side.  Query heads that share a key head (and tokens) form the rows of a tile.
//
// A row that sees no key (empty sequence, no prefix) gives zeros.  Rows behind the last sequence are not
// written.  fp32 scores, statistics and sums; P is rounded to fp16 for the second product as in the library's
// other attention kernels, and the output once.
#include "paged_attention.cuh"

namespace hexb {

namespace paged {

constexpr int THREADS = 128;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
  const int n = valid ? 16 : 0;  // 0 source bytes: the 16 are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------------ tiles of few rows
// One CTA: a tile of 16 * RW rows of one key head against a range of keys, in blocks of 64 keys staged by
// cp.async through a three-deep ring.  RW row groups times 4 / RW key groups of warps: with few rows (a decode
// step) the four warps share the rows and take 16 keys of a block each, with their own running maximum and sum,
// joined at the end; with many rows each warp owns 16 rows and all keys.
// OWN false: rows of the whole batch against the shared prefix (split blockIdx.y of it).
// OWN true: rows of sequence blockIdx.y % B against its own keys, split blockIdx.y / B.
template <int DP>
struct RowCfg {
  static constexpr int BN = 64;
  static constexpr int STAGES = 3;
  static constexpr int KV = BN * DP * 2;
  static constexpr int OFFS = STAGES * 2 * KV;           // two buffers of row offsets, K and V
  static constexpr int SMEM = OFFS + 2 * 2 * BN * 8;
};

template <int DP, int RW, bool OWN>
__global__ void __launch_bounds__(THREADS, DP == 64 ? 4 : DP == 128 ? 2 : 1)
paged_rows_kernel(const Params p) {
  using cfg = RowCfg<DP>;
  constexpr int BN = cfg::BN, KW = 4 / RW, KPW = BN / KW, ROWS = 16 * RW;
  constexpr int CH = DP / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem);
  int64_t *offs = reinterpret_cast<int64_t *>(smem + cfg::OFFS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rw = warp % RW, kw = warp / RW;
  const int h = blockIdx.z;
  // The launch over own keys does not read what the prefix launch of the same call writes until it joins them: it may
  // run beside it (the prefix launch lets it start only when all that came before is complete).
  if (!OWN || !p.follows_prefix) pdl_wait();
  if (!OWN) pdl_launch_dependents();

  int tok0 = 0, ntok, hi_all, nq = 0, part, lo, hi;
  const int *pages;
  if (OWN) {
    const int b = blockIdx.y % p.B, split = blockIdx.y / p.B;
    seq_range(p, b, tok0, ntok);
    nq = ntok;
    hi_all = seq_len(p, b);
    pages = p.table + (int64_t)b * p.table_stride;
    part = p.prefix_parts + split;
    const int chunk = ((hi_all + p.own_parts - 1) / p.own_parts + BN - 1) / BN * BN;
    lo = min(split * chunk, hi_all);
    hi = min(lo + chunk, hi_all);
  } else {
    ntok = tokens_used(p);
    hi_all = p.prefix_len;
    pages = p.prefix_pages;
    part = blockIdx.y;
    lo = min(part * p.prefix_chunk, hi_all);
    hi = min(lo + p.prefix_chunk, hi_all);
  }
  const int rows = ntok * p.G;

  for (int row0 = (int)blockIdx.x * ROWS; row0 < rows; row0 += (int)gridDim.x * ROWS) {
    // the last key any row of the tile sees
    int end = hi;
    if (OWN) end = min(end, hi_all - nq + min(ntok - 1, (row0 + ROWS - 1) / p.G) + 1);
    const int blocks = end > lo ? (end - lo + BN - 1) / BN : 0;

    // A fragments of Q: rows g and g + 8 of this warp's 16
    int tok[2], head[2];
    bool row_ok[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + rw * 16 + (lane >> 2) + 8 * i;
      row_ok[i] = r < rows;
      tok[i] = tok0 + (row_ok[i] ? r / p.G : 0);
      head[i] = h * p.G + (row_ok[i] ? r % p.G : 0);
    }
    uint32_t qa[DP / 16][4];
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = k * 16 + (i >> 1) * 8 + (lane & 3) * 2;
        qa[k][i] = 0;
        if (row_ok[i & 1] && d < p.D)
          qa[k][i] = *reinterpret_cast<const uint32_t *>(p.q + (int64_t)tok[i & 1] * p.sq_t + (int64_t)head[i & 1] * p.sq_h + d);
      }

    // row offsets of block j: thread tid < 64 looks key tid up (one block ahead of its use)
    auto lookup = [&](int j) -> int {
      const int key = lo + j * BN + tid;
      return tid < BN && key < end ? pages[key / p.page_size] : -1;
    };
    auto publish = [&](int j, int page) {
      if (tid < BN) {
        const int key = lo + j * BN + tid;
        int64_t ko = -1, vo = -1;
        if (key < end) {
          if ((unsigned)page < (unsigned)p.num_pages) {
            const int64_t in = key % p.page_size;
            ko = (int64_t)page * p.sk_p + in * p.sk_s;
            vo = (int64_t)page * p.sv_p + in * p.sv_s;
          } else {
            atomicExch(&g_paged_status, (int)HEXB_ERR_BAD_ARG);
          }
        }
        int64_t *o = offs + (j & 1) * 2 * BN;
        o[tid] = ko;
        o[BN + tid] = vo;
      }
    };
    auto fetch = [&](int j) {
      if (j < blocks) {
        const int64_t *o = offs + (j & 1) * 2 * BN;
        const uint32_t st = s0 + (uint32_t)(j % cfg::STAGES) * 2 * cfg::KV;
        const int c = tid % CH;
        const bool col = c * 8 < p.D;
#pragma unroll
        for (int i = 0; i < BN * CH / THREADS; ++i) {
          const int row = tid / CH + i * (THREADS / CH);
          const uint32_t dst = st + (uint32_t)(row * DP * 2 + ((c ^ (row & 7)) * 16));
          const int64_t ko = o[row], vo = o[BN + row];
          const bool kv = col && ko >= 0;
          cp_async16(dst, p.k + (kv ? ko + (int64_t)h * p.sk_h + c * 8 : 0), kv);
          cp_async16(dst + cfg::KV, p.v + (kv ? vo + (int64_t)h * p.sv_h + c * 8 : 0), kv);
        }
      }
      cp_async_commit();
    };

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    __syncthreads();  // the previous tile's use of the shared memory is over
    publish(0, lookup(0));
    publish(1, lookup(1));
    __syncthreads();
    fetch(0);
    fetch(1);
    int page_next = lookup(2);
    __syncthreads();
    publish(2, page_next);
    for (int j = 0; j < blocks; ++j) {
      cp_async_wait<1>();
      __syncthreads();  // block j landed for all; block j - 1's readers are done; offsets of j + 2 are visible
      fetch(j + 2);
      page_next = lookup(j + 3);
      const uint32_t sk = s0 + (uint32_t)(j % cfg::STAGES) * 2 * cfg::KV, sv = sk + cfg::KV;
      float s[KPW / 8][4];
#pragma unroll
      for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
        for (int n = 0; n < KPW / 16; ++n) {
          const int row = kw * KPW + n * 16 + (lane & 7) + ((lane >> 4) << 3);
          const int c = k * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldsm4(sk + (uint32_t)(row * DP * 2 + ((c ^ (row & 7)) * 16)), b);
          mma16816(s[2 * n], qa[k], b[0], b[1]);
          mma16816(s[2 * n + 1], qa[k], b[2], b[3]);
        }
      }
      // scores in base 2; keys past the end, and for own keys those after the row's token, drop out
      const int key0 = lo + j * BN + kw * KPW;
      int limit[2] = {end, end};
      if (OWN) {
#pragma unroll
        for (int i = 0; i < 2; ++i) limit[i] = min(end, hi_all - nq + (tok[i] - tok0) + 1);
      }
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + (lane & 3) * 2 + (e & 1);
          s[n][e] = key < limit[e >> 1] ? s[n][e] * p.scale_log2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
        }
      float base[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        base[i] = mx[i] == -INFINITY ? 0.f : mx[i];  // nothing seen yet: 2^(-inf - 0) = 0
        const float alpha = exp2f(m[i] - base[i]);
        m[i] = mx[i];
        l[i] *= alpha;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[n][2 * i] *= alpha;
          o[n][2 * i + 1] *= alpha;
        }
      }
      uint32_t pa[KPW / 16][4];
#pragma unroll
      for (int n = 0; n < KPW / 8; ++n) {
        float e4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          e4[e] = exp2f(s[n][e] - base[e >> 1]);
          l[e >> 1] += e4[e];
        }
        const __half2 lo2 = __floats2half2_rn(e4[0], e4[1]), hi2 = __floats2half2_rn(e4[2], e4[3]);
        pa[n >> 1][(n & 1) * 2] = *reinterpret_cast<const uint32_t *>(&lo2);
        pa[n >> 1][(n & 1) * 2 + 1] = *reinterpret_cast<const uint32_t *>(&hi2);
      }
#pragma unroll
      for (int k = 0; k < KPW / 16; ++k) {
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          const int row = kw * KPW + k * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
          const int c = n * 2 + (lane >> 4);
          uint32_t b[4];
          ldsm4t(sv + (uint32_t)(row * DP * 2 + ((c ^ (row & 7)) * 16)), b);
          mma16816(o[2 * n], pa[k], b[0], b[1]);
          mma16816(o[2 * n + 1], pa[k], b[2], b[3]);
        }
      }
      if (j + 3 < blocks) publish(j + 3, page_next);
    }
    cp_async_wait<0>();
    if (OWN && p.merge) pdl_wait();  // the prefix parts are complete
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }

    if (KW > 1) {
      // join the key groups of a row group: maxima and sums first, then O group by group
      __syncthreads();
      float *sm = reinterpret_cast<float *>(smem);                 // [KW][ROWS] m, then l
      float *so = sm + 2 * KW * ROWS;                              // [KW][ROWS][DP + 4]
      if ((lane & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = rw * 16 + (lane >> 2) + 8 * i;
          sm[kw * ROWS + r] = m[i];
          sm[(KW + kw) * ROWS + r] = l[i];
        }
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = rw * 16 + (lane >> 2) + 8 * i;
          *reinterpret_cast<float2 *>(so + (size_t)(kw * ROWS + r) * (DP + 4) + n * 8 + (lane & 3) * 2) =
              make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
      __syncthreads();
      for (int i = tid; i < ROWS * (DP / 4); i += THREADS) {
        const int r = i / (DP / 4), d = (i % (DP / 4)) * 4;
        if (row0 + r >= rows || d >= p.D) continue;
        float mm = -INFINITY, ll = 0.f, f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KW; ++w) mm = fmaxf(mm, sm[w * ROWS + r]);
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float lw = sm[(KW + w) * ROWS + r];
          const float a = lw == 0.f ? 0.f : exp2f(sm[w * ROWS + r] - mm);
          ll = fmaf(a, lw, ll);
          const float4 v = *reinterpret_cast<const float4 *>(so + (size_t)(w * ROWS + r) * (DP + 4) + d);
          f[0] = fmaf(a, v.x, f[0]); f[1] = fmaf(a, v.y, f[1]); f[2] = fmaf(a, v.z, f[2]); f[3] = fmaf(a, v.w, f[3]);
        }
        const int t = tok0 + (row0 + r) / p.G, hd = h * p.G + (row0 + r) % p.G;
        store_row<4>(p, part, t, hd, d, f, mm, ll);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!row_ok[i]) continue;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          const int d = n * 8 + (lane & 3) * 2;
          float f[2] = {o[n][2 * i], o[n][2 * i + 1]};
          if (d < p.D) store_row<2>(p, part, tok[i], head[i], d, f, m[i], l[i]);
        }
      }
    }
  }
  if (OWN) {
    pdl_wait();  // whoever waits for this launch waits for the prefix launch too
    pdl_launch_dependents();
  }
}

// ------------------------------------------------------------------ join of the parts
// One warp per (token, query head).
__global__ void __launch_bounds__(128) paged_join_kernel(const Params p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(row / p.Hq), hd = (int)(row - (int64_t)t * p.Hq);
  if (t >= tokens_used(p)) return;
  const int parts = p.prefix_parts + p.own_parts;
  const int64_t n = (int64_t)p.T * p.Hq;
  float mm = -INFINITY;
  for (int i = lane; i < parts; i += 32) mm = fmaxf(mm, p.part_ml[i * n + row].x);
  mm = warp_max(mm);
  for (int d = lane * 4; d < p.D; d += 128) {
    float f[4] = {0.f, 0.f, 0.f, 0.f}, ll = 0.f;
    for (int i = 0; i < parts; ++i) {
      const float2 ml = p.part_ml[i * n + row];
      if (ml.y == 0.f) continue;  // no key seen: no O either
      const float a = exp2f(ml.x - mm);
      ll = fmaf(a, ml.y, ll);
      const float4 v = *reinterpret_cast<const float4 *>(p.part_o + (i * n + row) * p.D + d);
      f[0] = fmaf(a, v.x, f[0]); f[1] = fmaf(a, v.y, f[1]); f[2] = fmaf(a, v.z, f[2]); f[3] = fmaf(a, v.w, f[3]);
    }
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;
    __half2 *o = reinterpret_cast<__half2 *>(p.out + (int64_t)t * p.so_t + (int64_t)hd * p.so_h + d);
    o[0] = __floats2half2_rn(f[0] * inv, f[1] * inv);
    o[1] = __floats2half2_rn(f[2] * inv, f[3] * inv);
  }
}

// ------------------------------------------------------------------ host
static int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is cut.  A function of the sizes alone, so that the workspace query and the launch agree.
struct Plan {
  bool seq, tc_prefix;            // tensor-core forms
  int prefix_parts, prefix_chunk, own_parts;
  int prefix_rw, own_rw;
  int tile_tokens, piece;
  int parts() const { return prefix_parts + own_parts; }
  bool merge() const { return prefix_parts > 0 && own_parts == 1; }
};

static int rw_for(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

static Plan make_plan(const hexb_paged_attention_desc *d, int sm_count) {
  Plan pl = {};
  const int64_t G = d->Hq / d->Hkv, capacity = d->table_width * d->page_size;
  const int64_t mq = d->max_q > 0 ? d->max_q : ceil_div(d->T, d->B);
  const int64_t pblocks = ceil_div(d->prefix_len, 64);
  // The tensor-core forms: what TMA can address (page pieces of at least the 8 rows of a swizzle atom, no stride of 0), a
  // positive scale, and enough rows to fill half of a 128-row tile; below that the key stream, not the products, is
  // what takes the time, and the small tiles of mma.sync read it as fast.
  pl.piece = (int)(d->page_size & -d->page_size);
  if (pl.piece > 64) pl.piece = 64;
  bool tc_ok = (d->D == 64 || d->D == 128) && pl.piece >= 8 && d->sm_scale > 0.f && G <= 128;
  const int64_t dims[10] = {d->T, d->Hq, d->num_pages, d->page_size, d->Hkv, d->num_pages, d->page_size, d->Hkv, 1, 1};
  for (int i = 0; i < 8; ++i) tc_ok = tc_ok && (dims[i] <= 1 || (d->strides[i] > 0 && d->strides[i] < ((int64_t)1 << 38)));
  tc_ok = tc_ok && (d->Hkv <= 1 || d->strides[1] * G < ((int64_t)1 << 38));
  pl.tile_tokens = tc_ok ? (int)(128 / G) : 0;
  if (tc_ok && mq * G >= 64 && capacity > 0) {
    // tiles of one sequence each, over prefix and own keys: cut the axis only when the tiles leave SMs idle
    pl.seq = true;
    const int64_t tiles = d->B * ceil_div(mq, pl.tile_tokens) * d->Hkv;
    int64_t parts = 2 * sm_count / tiles;
    const int64_t most = (pblocks + capacity / 64) / 8;
    if (parts > most) parts = most;
    if (parts > 32) parts = 32;
    pl.prefix_parts = parts > 1 ? (int)parts : 1;
    return pl;
  }
  if (d->prefix_len > 0 && tc_ok && d->T * G >= 64) {
    // One CTA an SM when own keys follow: their launch shares the SMs and streams beside the products.
    pl.tc_prefix = true;
    const int64_t tiles = (int64_t)ceil_div(d->T, pl.tile_tokens) * d->Hkv;
    int64_t parts = (capacity > 0 ? 1 : 2) * sm_count / tiles;
    if (parts < 1) parts = 1;
    if (parts > 64) parts = 64;
    if (parts > (pblocks + 1) / 2) parts = (pblocks + 1) / 2;
    const int64_t per = ceil_div(pblocks, parts);
    pl.prefix_parts = ceil_div(pblocks, per);
  } else if (d->prefix_len > 0) {
    const int per_sm = d->D <= 64 ? 4 : d->D <= 128 ? 2 : 1;
    const int64_t want = (int64_t)sm_count * per_sm * 2;
    pl.prefix_rw = rw_for(d->T * G);
    const int64_t tiles = (int64_t)ceil_div(d->T * G, 16 * pl.prefix_rw) * d->Hkv;
    int64_t parts = ceil_div(want, tiles);
    const int64_t most = ceil_div(d->prefix_len, 256);
    if (parts > most) parts = most;
    if (parts > 64) parts = 64;
    pl.prefix_chunk = ceil_div(ceil_div(d->prefix_len, parts), 64) * 64;
    pl.prefix_parts = ceil_div(d->prefix_len, pl.prefix_chunk);
  }
  if (capacity > 0) {
    pl.own_rw = rw_for(mq * G);
    const int64_t tiles = (int64_t)d->B * ceil_div(mq * G, 16 * pl.own_rw) * d->Hkv;
    int64_t parts = sm_count * 2 / tiles;   // one part (and no join launch) once the tiles fill the SMs
    const int64_t most = ceil_div(capacity, 256);
    if (parts > most) parts = most;
    if (parts > 64) parts = 64;
    pl.own_parts = parts > 1 ? (int)parts : 1;
  }
  return pl;
}

static size_t ws_need(const hexb_paged_attention_desc *d, const Plan &pl) {
  if (pl.parts() < 2) return 0;
  const size_t parts = pl.merge() ? (size_t)pl.prefix_parts : (size_t)pl.parts();
  return parts * (size_t)d->T * d->Hq * ((size_t)d->D * 4 + 8) + 256;
}

template <int DP, int RW, bool OWN>
static int launch_rows(const Params &p, dim3 grid, cudaStream_t st) {
  static PerDeviceOnce once;
  int dev = 0;
  HEXB_CUDA_OK(cudaGetDevice(&dev));
  if (!once.is_done(dev)) {
    HEXB_CUDA_OK(cudaFuncSetAttribute(paged_rows_kernel<DP, RW, OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowCfg<DP>::SMEM));
    once.mark(dev);
  }
  HEXB_CUDA_OK(launch_pdl(paged_rows_kernel<DP, RW, OWN>, grid, dim3(THREADS), (size_t)RowCfg<DP>::SMEM, st, p));
  return check_launch("paged_rows");
}

template <bool OWN>
static int dispatch_rows(const Params &p, int rw, dim3 grid, cudaStream_t st) {
#define HEXB_ROWS(DP)                                                   \
  return rw == 1 ? launch_rows<DP, 1, OWN>(p, grid, st)                 \
                 : rw == 2 ? launch_rows<DP, 2, OWN>(p, grid, st) : launch_rows<DP, 4, OWN>(p, grid, st)
  if (p.D <= 64) HEXB_ROWS(64);
  if (p.D <= 128) HEXB_ROWS(128);
  HEXB_ROWS(256);
#undef HEXB_ROWS
}

static int check_desc(const hexb_paged_attention_desc *d) {
  if (!d) return HEXB_ERR_BAD_ARG;
  if (d->T < 0 || d->B < 0 || d->Hq < 0 || d->Hkv < 0 || d->D < 0 || d->prefix_len < 0 || d->table_width < 0 ||
      d->num_pages < 0 || d->page_size < 1 || d->max_q < 0)
    return HEXB_ERR_BAD_ARG;
  if (d->T == 0 || d->Hq == 0 || d->B == 0 || d->D == 0) return HEXB_OK;
  if (d->Hkv == 0 || d->Hq % d->Hkv || (!d->q_offsets && d->T != d->B)) return HEXB_ERR_BAD_ARG;
  if (d->D % 8 || d->D > 256 || d->Hkv > 65535 || d->T > (1 << 24) || d->T * (d->Hq / d->Hkv) > (1 << 30) ||
      d->B > (1 << 20) || d->prefix_len > (1 << 30) || d->page_size > (1 << 30) || d->num_pages > 0x7fffffff ||
      d->table_width > (1 << 30) / d->page_size)
    return HEXB_ERR_UNSUPPORTED;
  return HEXB_OK;
}

}  // namespace paged

int paged_device_status_fetch_and_clear(int *out) {
  int v = 0, zero = 0;
  HEXB_CUDA_OK(cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(int)));
  if (v) HEXB_CUDA_OK(cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int)));
  *out = v;
  return HEXB_OK;
}

}  // namespace hexb

using namespace hexb;

extern "C" size_t hexb_paged_attention_workspace_bytes(const hexb_paged_attention_desc *d) {
  if (paged::check_desc(d) != HEXB_OK || d->T == 0 || d->Hq == 0 || d->B == 0 || d->D == 0) return 0;
  DeviceInfo di;
  const int sms = current_device(&di) == HEXB_OK ? di.sm_count : kNumSMsB200;
  return paged::ws_need(d, paged::make_plan(d, sms));
}

extern "C" int hexb_paged_attention_f16(const hexb_paged_attention_desc *d, void *workspace, size_t workspace_bytes,
                                        void *stream) {
  if (int e = paged::check_desc(d)) return e;
  if (d->T == 0 || d->Hq == 0 || d->B == 0 || d->D == 0) return HEXB_OK;
  if (!d->Q || !d->Out) return HEXB_ERR_BAD_ARG;
  const bool own = d->table_width > 0, prefix = d->prefix_len > 0;
  if ((own || prefix) && (!d->K_cache || !d->V_cache)) return HEXB_ERR_BAD_ARG;
  if ((own && (!d->block_table || !d->seq_lens)) || (prefix && !d->prefix_pages)) return HEXB_ERR_BAD_ARG;
  if (!aligned16(d->Q) || !aligned16(d->Out) || !aligned16(d->K_cache) || !aligned16(d->V_cache)) return HEXB_ERR_MISALIGNED;
  for (int64_t s : d->strides)
    if (s % 8) return HEXB_ERR_MISALIGNED;
  DeviceInfo di;
  if (int e = current_device(&di)) return e;
  const paged::Plan pl = paged::make_plan(d, di.sm_count);
  const size_t need = paged::ws_need(d, pl);
  if (need && (!workspace || workspace_bytes < need)) return HEXB_ERR_WORKSPACE;
  const int64_t *s = d->strides;
  paged::Params p = {};
  p.q = (const __half *)d->Q; p.k = (const __half *)d->K_cache; p.v = (const __half *)d->V_cache; p.out = (__half *)d->Out;
  p.sq_t = s[0]; p.sq_h = s[1]; p.sk_p = s[2]; p.sk_s = s[3]; p.sk_h = s[4]; p.sv_p = s[5]; p.sv_s = s[6]; p.sv_h = s[7];
  p.so_t = s[8]; p.so_h = s[9];
  p.prefix_pages = d->prefix_pages; p.table = d->block_table; p.lens = d->seq_lens; p.offsets = d->q_offsets;
  p.table_stride = d->table_stride;
  p.T = (int)d->T; p.B = (int)d->B; p.Hq = (int)d->Hq; p.G = (int)(d->Hq / d->Hkv); p.D = (int)d->D;
  p.prefix_len = (int)d->prefix_len; p.page_size = (int)d->page_size; p.num_pages = (int)d->num_pages;
  p.own_capacity = (int)(d->table_width * d->page_size);
  p.prefix_parts = pl.prefix_parts; p.prefix_chunk = pl.prefix_chunk; p.own_parts = pl.own_parts;
  p.scale_log2 = d->sm_scale * 1.44269504f;
  p.tile_tokens = pl.tile_tokens;
  p.piece = pl.piece;
  if (need) {
    const size_t n = (size_t)(pl.merge() ? pl.prefix_parts : pl.parts()) * d->T * d->Hq;
    uint8_t *w = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
    p.part_o = reinterpret_cast<float *>(w);
    p.part_ml = reinterpret_cast<float2 *>(w + n * d->D * 4);
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t mq = d->max_q > 0 ? d->max_q : paged::ceil_div(d->T, d->B);
  auto grid_of = [&](int64_t x, int64_t y, dim3 *g) {
    if (x > 0x7fffffff || y > 65535) return false;
    *g = dim3((unsigned)x, (unsigned)y, (unsigned)d->Hkv);
    return true;
  };
  dim3 grid;
  if (pl.seq) {
    if (!grid_of(paged::ceil_div(mq, pl.tile_tokens), (int64_t)pl.prefix_parts * d->B, &grid)) return HEXB_ERR_UNSUPPORTED;
    if (int e = paged::tc_launch(p, (int)d->Hkv, true, grid, st)) return e;
  } else if (pl.tc_prefix) {
    if (!grid_of(paged::ceil_div(d->T, pl.tile_tokens), pl.prefix_parts, &grid)) return HEXB_ERR_UNSUPPORTED;
    if (int e = paged::tc_launch(p, (int)d->Hkv, false, grid, st)) return e;
  } else if (pl.prefix_parts) {
    if (!grid_of(paged::ceil_div(d->T * p.G, 16 * pl.prefix_rw), pl.prefix_parts, &grid)) return HEXB_ERR_UNSUPPORTED;
    if (int e = paged::dispatch_rows<false>(p, pl.prefix_rw, grid, st)) return e;
  }
  if (pl.own_parts) {
    if (!grid_of(paged::ceil_div(mq * p.G, 16 * pl.own_rw), (int64_t)pl.own_parts * d->B, &grid)) return HEXB_ERR_UNSUPPORTED;
    paged::Params po = p;
    po.follows_prefix = pl.prefix_parts > 0;
    po.merge = pl.merge();
    if (int e = paged::dispatch_rows<true>(po, pl.own_rw, grid, st)) return e;
    if (pl.merge()) return HEXB_OK;
  }
  if (pl.parts() != 1) {
    // also the call without any key: its rows are set to zero
    const int64_t rows = d->T * d->Hq;
    HEXB_CUDA_OK(launch_pdl(paged::paged_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p));
    return check_launch("paged_join");
  }
  return HEXB_OK;
}
