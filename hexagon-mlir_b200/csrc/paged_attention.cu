// Attention of a batch whose sequences share a prefix, over a paged key/value cache.
//
// Query token t of sequence b sees every key of the shared prefix and the keys j <= len[b] - nq[b] + i of its
// sequence's own pages (i = the token's index among the nq[b] new ones, whose own keys are the last nq[b] of
// the cache): out = softmax(q . K^T * scale) V over their union.  The softmax of a union is joined from
// partial results: a part holds its row maximum m (base 2, scale folded in), l = sum 2^(s - m) and
// O = sum 2^(s - m) v, and
//     out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i,
// so the prefix can be read for a tile of rows from many sequences instead of once per sequence, and a long axis is cut
// into parts that run side by side.  Query heads that share a key head (and tokens) form the rows of a tile.  From 64 rows
// a sequence on, a tile holds one sequence alone and reads the prefix itself (make_plan).
//
// A row that sees no key (empty sequence, no prefix) gives zeros.  Rows behind the last sequence are not
// written.  fp32 scores, statistics and sums; P is rounded to fp16 for the second product as in the library's
// other attention kernels, and the output once.
#include <type_traits>

#include "attn_common.cuh"
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

// ------------------------------------------------------------------ stream of key blocks
// Tiles of 16 * RW rows of one key head against blocks of 64 keys, four consumer warps.  RW row groups times 4 / RW key
// groups of warps: with few rows (a decode step) the four warps share the rows and take 16 keys of a block each,
// with their own running maximum and sum, joined at the end of a run; with many rows each warp owns 16 rows and all
// keys.
//
// The work of a call is one list of units -- (sequence, key head, tile, block), the shared prefix counting as a
// sequence of all tokens -- cut evenly over the CTAs that fit the GPU.  A CTA streams its stretch of the list without a
// pause at the borders between sequences: the start-up (lengths, page numbers, first keys: three dependent trips
// to memory) is paid once, and ragged lengths leave no SM idle.  A run of units of one tile ends in one part; the
// join adds the parts up.
//
// The stream is bound by memory only if a block costs its warps few instructions: with every thread copying its share
// by cp.async (page, address and predicate for each 16 bytes) a block cost 550 instructions a warp and the stream
// ran at 4.9 TB/s of 8192-key sequences.  So a producer warp fetches blocks by TMA, page piece by page
// piece, the consumer warps wait on its barriers and not on each other, and O is rescaled only when a row maximum grows by
// more than 2^8.  The cp.async form remains for pages and strides that TMA cannot address.
template <int DP>
struct RowCfg {
  static constexpr int BN = 64;
  static constexpr int STAGES = 3;
  static constexpr int KV = BN * DP * 2, KV_CHUNK = BN * 128;   // 64 columns: 64 rows of 128 bytes, 128-byte swizzle
  // Exchange between the key groups: m, l, and 16 rows of DP / 4 columns a warp.  Heads of more than 128 leave no room
  // for it beside three stages: their tiles have 64 rows, a warp owns all keys of its 16.
  static constexpr int XCH = STAGES * 2 * KV;
  static constexpr int XLD = DP == 64 ? 18 : DP / 4 + 8;   // row pitch (40: no bank conflicts; 24 would cost the fourth CTA of 64-wide heads)
  static constexpr int OFFS = XCH + (DP > 128 ? 0 : (128 + 64 * XLD) * 4);   // cp.async: row offsets, K and V, two buffers
  static constexpr int BARS = OFFS;                      // TMA: full and empty barrier of every stage, abort flag
  static constexpr int SMEM = OFFS + 2 * 2 * BN * 8;
  static constexpr int SMEM_TMA = BARS + 2 * STAGES * 8 + 16 + 1024;
  static constexpr int PER_SM = DP == 64 ? 4 : DP == 128 ? 2 : 1;
};

// The running state of one tile in the consumer warps.
template <int DP, int RW>
struct Run {
  static constexpr int KW = 4 / RW, KPW = 64 / KW, ROWS = 16 * RW;
  uint32_t qa[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];       // reference maximum (base 2, scaled) of rows g and g + 8; this lane's share of the sum
  int tok[2], head[2];
  bool row_ok[2];
  int lane, rw, kw;
  int first_j;            // block the run began with

  // fragments of Q: rows g and g + 8 of this warp's 16
  __device__ __forceinline__ void begin(const Params &p, const Cursor &c) {
    const int row0 = c.tile * ROWS, rows = c.ntok * p.G;
    first_j = c.j;
    const __half *q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + rw * 16 + (lane >> 2) + 8 * i;
      row_ok[i] = r < rows;
      tok[i] = c.tok0 + (row_ok[i] ? r / p.G : 0);
      head[i] = c.h * p.G + (row_ok[i] ? r % p.G : 0);
      q[i] = p.q + (int64_t)tok[i] * p.sq_t + (int64_t)head[i] * p.sq_h + (lane & 3) * 2;
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = k * 16 + (i >> 1) * 8;
        qa[k][i] = 0;
        if (row_ok[i & 1] && d < p.D) qa[k][i] = *reinterpret_cast<const uint32_t *>(q[i & 1] + d);
      }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  }

  // One block: keys 64 * c.j .. of the tile, K at sk and V at sv.
  __device__ __forceinline__ void step(const Params &p, const Cursor &c, int end, uint32_t sk, uint32_t sv) {
    constexpr int KV_CHUNK = RowCfg<DP>::KV_CHUNK;
    float s[KPW / 8][4];
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    const uint32_t krow = (uint32_t)(kw * KPW + (lane & 7) + ((lane >> 4) << 3)), kx = krow & 7;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint32_t ch = (uint32_t)(k * 2) + ((lane >> 3) & 1);
      const uint32_t at = sk + (ch >> 3) * KV_CHUNK + krow * 128 + (((ch & 7) ^ kx) << 4);
#pragma unroll
      for (int n = 0; n < KPW / 16; ++n) {
        uint32_t b[4];
        ldsm4(at + n * 16 * 128, b);
        mma16816(s[2 * n], qa[k], b[0], b[1]);
        mma16816(s[2 * n + 1], qa[k], b[2], b[3]);
      }
    }
    // scores in base 2; keys past the end, and own keys after the row's token, drop out
    const int key0 = c.j * 64 + kw * KPW;
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] *= p.scale_log2;
    const int sees = c.b < 0 ? end : c.len - c.ntok + 1 - c.tok0;   // + token: own keys a row sees
    if (key0 + KPW > (c.b < 0 ? end : c.len - c.ntok + 1)) {        // some row may not see some key of this warp
#pragma unroll
      for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + (lane & 3) * 2 + (e & 1);
          const int limit = min(end, c.b < 0 ? end : sees + tok[e >> 1]);
          if (key >= limit) s[n][e] = -INFINITY;
        }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
    }
    // the same reference serves P, l and O, so the result does not depend on how old it is; P stays below 2^8
    if (__any_sync(0xffffffffu, mx[0] - m[0] > 8.0f || mx[1] - m[1] > 8.0f)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float mn = fmaxf(m[i], mx[i]);
        const float alpha = mn == -INFINITY ? 1.0f : attn::ex2_approx(m[i] - mn);
        m[i] = mn;
        l[i] *= alpha;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[n][2 * i] *= alpha;
          o[n][2 * i + 1] *= alpha;
        }
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};  // nothing seen: 2^(-inf - 0) = 0
    uint32_t pa[KPW / 16][4];
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n) {
      float e4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        e4[e] = attn::ex2_approx(s[n][e] - base[e >> 1]);
        l[e >> 1] += e4[e];
      }
      pa[n >> 1][(n & 1) * 2] = attn::pack_f16x2(e4[0], e4[1]);
      pa[n >> 1][(n & 1) * 2 + 1] = attn::pack_f16x2(e4[2], e4[3]);
    }
    const uint32_t vrow = (uint32_t)(kw * KPW + (lane & 7) + (((lane >> 3) & 1) << 3)), vx = vrow & 7;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      const uint32_t ch = (uint32_t)(n * 2) + (lane >> 4);
      const uint32_t at = sv + (ch >> 3) * KV_CHUNK + vrow * 128 + (((ch & 7) ^ vx) << 4);
#pragma unroll
      for (int k = 0; k < KPW / 16; ++k) {
        uint32_t b[4];
        ldsm4t(at + k * 16 * 128, b);
        mma16816(o[2 * n], pa[k], b[0], b[1]);
        mma16816(o[2 * n + 1], pa[k], b[2], b[3]);
      }
    }
  }

  // The run is over: its part, or the output itself.  All 128 consumer threads.
  __device__ __forceinline__ void end(const Params &p, const Cursor &c, long long unit, long long per, float *xch) {
    const RunPlace place(p, c, first_j, c.j + 1, unit - c.j, per, ROWS);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if (kw == 0 && (lane & 3) == 0 && row_ok[i]) place.describe(p, c, tok[i], head[i], rw * 16 + (lane >> 2) + 8 * i);
    }
    if (KW > 1) {
      // Join the key groups of a row group.  All scale to their common maximum; then key group w collects columns
      // [w, w + 1) * DP / KW from the others, one of them a round (joining 16 columns of all groups at a time, between two
      // barriers each, took 6.7 us a run; this takes a third).
      constexpr int QC = DP / KW, PC = DP / 4;                 // columns a group keeps; of them a round
      constexpr int PN = PC / 8, LD = RowCfg<DP>::XLD;         // 8-column tiles, row pitch
      float *sm = xch, *sl = xch + 64;                         // [KW][ROWS] each
      float *so = xch + 128 + (kw * RW + rw) * 16 * LD;        // what this warp sends: its 16 rows
      const int r0 = rw * 16 + (lane >> 2);
      sync();
      if ((lane & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sm[kw * ROWS + r0 + 8 * i] = m[i];
          sl[kw * ROWS + r0 + 8 * i] = l[i];
        }
      }
      sync();
      float mm[2], ll[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mm[i] = -INFINITY;
#pragma unroll
        for (int w = 0; w < KW; ++w) mm[i] = fmaxf(mm[i], sm[w * ROWS + r0 + 8 * i]);
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float lw = sl[w * ROWS + r0 + 8 * i];
          ll[i] += lw == 0.f ? 0.f : lw * attn::ex2_approx(sm[w * ROWS + r0 + 8 * i] - mm[i]);
        }
        const float a = l[i] == 0.f ? 0.f : attn::ex2_approx(m[i] - mm[i]);
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[n][2 * i] *= a;
          o[n][2 * i + 1] *= a;
        }
      }
      // fn(first 8-column tile of group w's columns) with a constant, so that O stays in registers
      auto tile_of = [&](int w, auto &&fn) {
        if (w == 0) fn(std::integral_constant<int, 0>{});
        else if (w == 1) fn(std::integral_constant<int, (KW > 1 ? 1 : 0) * QC / 8>{});
        else if (w == 2) fn(std::integral_constant<int, (KW > 2 ? 2 : 0) * QC / 8>{});
        else fn(std::integral_constant<int, (KW > 3 ? 3 : 0) * QC / 8>{});
      };
#pragma unroll
      for (int pc = 0; pc < QC / PC; ++pc) {
        float f[PN][4];
        tile_of(kw, [&](auto t) {
#pragma unroll
          for (int n = 0; n < PN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) f[n][e] = o[decltype(t)::value + pc * PN + n][e];
        });
#pragma unroll 1
        for (int d = 1; d < KW; ++d) {
          // to group (kw + d) % KW its columns; from group (kw - d) % KW this warp's
          tile_of((kw + d) % KW, [&](auto t) {
#pragma unroll
            for (int n = 0; n < PN; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                *reinterpret_cast<float2 *>(so + ((lane >> 2) + 8 * i) * LD + n * 8 + (lane & 3) * 2) =
                    make_float2(o[decltype(t)::value + pc * PN + n][2 * i], o[decltype(t)::value + pc * PN + n][2 * i + 1]);
          });
          sync();
          const float *in = xch + 128 + (((kw + KW - d) % KW) * RW + rw) * 16 * LD;
#pragma unroll
          for (int n = 0; n < PN; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 v = *reinterpret_cast<const float2 *>(in + ((lane >> 2) + 8 * i) * LD + n * 8 + (lane & 3) * 2);
              f[n][2 * i] += v.x;
              f[n][2 * i + 1] += v.y;
            }
          sync();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!row_ok[i]) continue;
#pragma unroll
          for (int n = 0; n < PN; ++n) {
            const int d = kw * QC + pc * PC + n * 8 + (lane & 3) * 2;
            float v[2] = {f[n][2 * i], f[n][2 * i + 1]};
            if (d < p.D) store_row<2>(p, place.index(p, tok[i], head[i], r0 + 8 * i), tok[i], head[i], d, v, mm[i], ll[i]);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!row_ok[i]) continue;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          const int d = n * 8 + (lane & 3) * 2;
          float f[2] = {o[n][2 * i], o[n][2 * i + 1]};
          if (d < p.D) store_row<2>(p, place.index(p, tok[i], head[i], rw * 16 + (lane >> 2) + 8 * i), tok[i], head[i], d, f, m[i], l[i]);
        }
      }
    }
  }
  // Barrier of the consumer warps.  They leave their loop together in every case (a wait that gave up does not end it).
  static __device__ __forceinline__ void sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
};

// ---- blocks fetched by TMA: warps 0-3 consume, warp 4 produces
template <int DP, int RW>
__global__ void __launch_bounds__(160, RowCfg<DP>::PER_SM)
paged_stream_tma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params p) {
  using cfg = RowCfg<DP>;
  constexpr int BN = cfg::BN, ST = cfg::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw), s0 = (raw + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (s0 - raw);
  auto full = [&](int i) { return s0 + cfg::BARS + 8 * i; };
  auto empty = [&](int i) { return s0 + cfg::BARS + 8 * (ST + i); };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + cfg::BARS + 2 * ST * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(full(i), 1);
      tc::mbar_init(empty(i), 4);
    }
    *abort_flag = 0;
    tc::fence_barrier_init();
    tc::prefetch_tensormap(&tmK);
    tc::prefetch_tensormap(&tmV);
  }
  // Also after the call's own tensor-core launch, whose results this one does not touch: what earlier kernels of the stream
  // wrote -- queries, lengths, tables, the cache -- is certain to be visible only behind the wait.
  pdl_wait();
  long long start, stop, per;
  Cursor c;
  find_stretch<160>(p, 16 * RW, start, stop, per, c);   // its barriers also publish the ones set up above
  if (start < stop) {
    const int units = (int)(stop - start);
    if (warp == 4) {
      const int pieces = BN / p.piece;
      auto lookup = [&](int u, int &slot) {
        int page = p.num_pages;                     // no key there: reads as zeros
        slot = 0;
        if (lane < pieces && u < units) {
          const int key = c.j * BN + lane * p.piece;
          if (key < end_of(p, 16 * RW, c)) {
            const int pi = key / p.page_size;
            slot = key - pi * p.page_size;
            const int got = c.b < 0 ? p.prefix_pages[pi] : p.table[(int64_t)c.b * p.table_stride + pi];
            if ((unsigned)got < (unsigned)p.num_pages) page = got;
            else atomicExch(&g_paged_status, (int)HEXB_ERR_BAD_ARG);
          }
        }
        return page;
      };
      int slot_next, page_next = lookup(0, slot_next);
      for (int u = 0; u < units; ++u) {
        const int st = u % ST, page = page_next, slot = slot_next, h = c.h;
        if (u + 1 < units) advance(p, 16 * RW, c);
        page_next = lookup(u + 1, slot_next);
        if (!tc::mbar_wait(empty(st), (uint32_t)(u / ST + 1) & 1u, abort_flag)) break;
        if (lane == 0) tc::mbar_arrive_expect_tx(full(st), 2 * cfg::KV);
        __syncwarp();
        if (lane < pieces) {
          const uint32_t dst = s0 + (uint32_t)st * 2 * cfg::KV + (uint32_t)(lane * p.piece) * 128u;
#pragma unroll
          for (int k = 0; k < DP / 64; ++k) {
            tc::tma_load_4d(dst + k * cfg::KV_CHUNK, &tmK, k * 64, h, slot, page, full(st));
            tc::tma_load_4d(dst + cfg::KV + k * cfg::KV_CHUNK, &tmV, k * 64, h, slot, page, full(st));
          }
        }
      }
    } else {
      Run<DP, RW> r;
      r.lane = lane;
      r.rw = warp % RW;
      r.kw = warp / RW;
      float *xch = reinterpret_cast<float *>(smem + cfg::XCH);
      int end = 0;
      for (int u = 0; u < units; ++u) {
        if (u == 0 || c.j == 0) {
          r.begin(p, c);
          end = end_of(p, 16 * RW, c);
        }
        const int st = u % ST;
        const uint32_t sk = s0 + (uint32_t)st * 2 * cfg::KV, sv = sk + cfg::KV;
        // Should it give up, the loop goes on, without waiting further, over whatever the stage holds: the warps meet at
        // barriers, and the status word tells the host.
        tc::mbar_wait(full(st), (uint32_t)(u / ST) & 1u, abort_flag);
        // this warp's keys behind the last one: whatever the slots hold -- NaN, perhaps -- must not meet a weight of 0
        const int k0 = r.kw * Run<DP, RW>::KPW, k1 = k0 + Run<DP, RW>::KPW;
        const int filled = max(end - c.j * BN, 0);
        if (filled < k1) {
          const int from = max(filled, k0);
          __syncwarp();
          for (int i = lane; i < (k1 - from) * (DP / 8); i += 32) {
            const int row = from + i / (DP / 8), ch = i % (DP / 8);
            *reinterpret_cast<uint4 *>(smem + (sv - s0) + (ch >> 3) * cfg::KV_CHUNK + row * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          __syncwarp();   // (warps that share the keys write the same zeros)
        }
        r.step(p, c, end, sk, sv);
        if (filled < k1) tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(empty(st));
        if (c.j == c.nb - 1 || u == units - 1) r.end(p, c, start + u, per, xch);
        if (u + 1 < units) advance(p, 16 * RW, c);
      }
    }
    if (*abort_flag) {
      for (int i = 0; i < 200; ++i) __nanosleep(1000);  // lets copies in flight land before the CTA's memory goes
      if (threadIdx.x == 0) atomicExch(&g_paged_status, (int)HEXB_ERR_TIMEOUT);
    }
  }
  pdl_launch_dependents();
}

// ---- blocks copied by cp.async
template <int DP, int RW>
__global__ void __launch_bounds__(THREADS, RowCfg<DP>::PER_SM)
paged_stream_kernel(const Params p) {
  using cfg = RowCfg<DP>;
  constexpr int BN = cfg::BN;
  constexpr int CH = DP / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem);
  int64_t *offs = reinterpret_cast<int64_t *>(smem + cfg::OFFS);
  const int tid = threadIdx.x, warp = tid >> 5;
  pdl_wait();
  long long start, stop, per;
  Cursor cc, cl;                        // the unit being computed, the one whose pages are looked up
  find_stretch<THREADS>(p, 16 * RW, start, stop, per, cc);
  if (start < stop) {
    const int units = (int)(stop - start);
    int looked = 0, fetched = 0;
    cl = cc;
    auto lookup = [&]() -> int {        // thread tid < 64: page of key tid of unit `looked`
      int page = -1;
      if (looked < units && tid < BN) {
        const int key = cl.j * BN + tid;
        if (key < end_of(p, 16 * RW, cl)) {
          const int pi = key / p.page_size;
          page = cl.b < 0 ? p.prefix_pages[pi] : p.table[(int64_t)cl.b * p.table_stride + pi];
        }
      }
      return page;
    };
    auto publish = [&](int page) {      // row offsets of unit `looked`; then the next one's turn
      if (looked < units) {
        if (tid < BN) {
          const int key = cl.j * BN + tid;
          int64_t ko = -1, vo = -1;
          if (key < end_of(p, 16 * RW, cl)) {
            if ((unsigned)page < (unsigned)p.num_pages) {
              const int64_t in = key % p.page_size;
              ko = (int64_t)page * p.sk_p + in * p.sk_s + (int64_t)cl.h * p.sk_h;
              vo = (int64_t)page * p.sv_p + in * p.sv_s + (int64_t)cl.h * p.sv_h;
            } else {
              atomicExch(&g_paged_status, (int)HEXB_ERR_BAD_ARG);
            }
          }
          int64_t *o = offs + (looked & 1) * 2 * BN;
          o[tid] = ko;
          o[BN + tid] = vo;
        }
        advance(p, 16 * RW, cl);
      }
      ++looked;
    };
    auto fetch = [&]() {
      if (fetched < units) {
        const int64_t *o = offs + (fetched & 1) * 2 * BN;
        const int c = tid % CH;
        const uint32_t st = s0 + (uint32_t)(fetched % cfg::STAGES) * 2 * cfg::KV + (c >> 3) * cfg::KV_CHUNK;
        const bool col = c * 8 < p.D;
#pragma unroll
        for (int i = 0; i < BN * CH / THREADS; ++i) {
          const int row = tid / CH + i * (THREADS / CH);
          const uint32_t dst = st + (uint32_t)(row * 128 + (((c & 7) ^ (row & 7)) * 16));
          const int64_t ko = o[row], vo = o[BN + row];
          const bool kv = col && ko >= 0;
          cp_async16(dst, p.k + (kv ? ko + c * 8 : 0), kv);
          cp_async16(dst + cfg::KV, p.v + (kv ? vo + c * 8 : 0), kv);
        }
      }
      ++fetched;
      cp_async_commit();
    };
    int page_next;
    publish(lookup());
    publish(lookup());
    __syncthreads();
    fetch();
    fetch();
    page_next = lookup();
    __syncthreads();
    publish(page_next);

    Run<DP, RW> r;
    r.lane = tid & 31;
    r.rw = warp % RW;
    r.kw = warp / RW;
    int end = 0;
    for (int u = 0; u < units; ++u) {
      if (u == 0 || cc.j == 0) {
        r.begin(p, cc);
        end = end_of(p, 16 * RW, cc);
      }
      cp_async_wait<1>();
      __syncthreads();  // unit u landed for all; unit u - 1's readers are done; offsets of u + 2 are visible
      fetch();
      page_next = lookup();
      const uint32_t sk = s0 + (uint32_t)(u % cfg::STAGES) * 2 * cfg::KV;
      r.step(p, cc, end, sk, sk + cfg::KV);
      publish(page_next);
      if (cc.j == cc.nb - 1 || u == units - 1) r.end(p, cc, start + u, per, reinterpret_cast<float *>(smem + cfg::XCH));
      if (u + 1 < units) advance(p, 16 * RW, cc);
    }
    cp_async_wait<0>();
  }
  pdl_launch_dependents();
}

// ------------------------------------------------------------------ join of the parts
// One warp per (token, query head); LPR lanes hold the row, the 32 / LPR groups of lanes take every so many-th part.
template <int LPR>
__global__ void __launch_bounds__(128) paged_join_kernel(const Params p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane / LPR, col = lane % LPR;
  constexpr int SUBS = 32 / LPR;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(row / p.Hq), hd = (int)(row - (int64_t)t * p.Hq);
  if (t >= p.T) return;
  const int used = tokens_used(p);
  const int64_t n = (int64_t)p.T * p.Hq;
  // The parts of a row: those of the prefix, then those of its own keys; each side either in row order, or the runs of
  // its tile where their CTAs left them.
  auto side = [&](const int4 *desc, int dense, int &cta, int &r) {
    if (!desc) return dense;
    const int4 v = desc[row];    // (rows that belong to no sequence have none: whatever is there stays in bounds)
    cta = min(max(v.y, 0), p.ctas - 1);
    r = min(max(v.z, 0), p.tile_rows - 1);
    return min(max(v.x, -1), p.ctas - cta);
  };
  int pc = 0, pr = 0, oc = 0, orow = 0;
  int np = side(p.prefix_desc, p.prefix_desc ? 0 : p.prefix_parts, pc, pr), no = side(p.own_desc, 0, oc, orow);
  if (t >= used || np < 0 || no < 0) return;  // no sequence's; stored by its one run
  const bool pcut = p.prefix_desc && np > 0, ocut = no > 0;
  if (p.prefix_desc && np == 0) np = 1;
  if (p.own_desc && no == 0) no = 1;
  const int parts = np + no;
  auto slot = [&](int i) -> int64_t {
    if (i < np) return pcut ? p.run_base + ((int64_t)(pc + i) * 2 + (i == 0)) * p.tile_rows + pr : i * n + row;
    i -= np;
    return ocut ? p.run_base + ((int64_t)(oc + i) * 2 + (i == 0)) * p.tile_rows + orow : p.own_slot * n + row;
  };
  float mm = -INFINITY;
  for (int i = lane; i < parts; i += 32) {
    const float2 ml = p.part_ml[slot(i)];
    if (ml.y != 0.f) mm = fmaxf(mm, ml.x);
  }
  mm = warp_max(mm);
  for (int d0 = 0; d0 < p.D; d0 += LPR * 4) {
    const int d = d0 + col * 4;
    float f[4] = {0.f, 0.f, 0.f, 0.f}, ll = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      float2 ml = make_float2(0.f, 0.f);
      if (i0 + lane < parts) ml = p.part_ml[slot(i0 + lane)];
      const float w = ml.y == 0.f ? 0.f : exp2f(ml.x - mm);  // no key seen: no O either
      ll += warp_sum(w * ml.y);
      const int m = min(32, parts - i0);
#pragma unroll 8
      for (int i = 0; i < m; i += SUBS) {
        // every lane loads, from a slot in bounds, and then selects: loads behind a branch would not overlap
        const int k = i + sub;
        const float a = __shfl_sync(0xffffffffu, w, k & 31);
        const float4 v = __ldcs(reinterpret_cast<const float4 *>(p.part_o + slot(i0 + min(k, m - 1)) * p.D + min(d, p.D - 4)));
        const bool use = k < m && a != 0.f;
        f[0] = fmaf(use ? a : 0.f, use ? v.x : 0.f, f[0]);
        f[1] = fmaf(use ? a : 0.f, use ? v.y : 0.f, f[1]);
        f[2] = fmaf(use ? a : 0.f, use ? v.z : 0.f, f[2]);
        f[3] = fmaf(use ? a : 0.f, use ? v.w : 0.f, f[3]);
      }
    }
#pragma unroll
    for (int s = LPR; s < 32; s <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] += __shfl_xor_sync(0xffffffffu, f[e], s);
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;
    if (sub == 0 && d < p.D) {
      __half2 *o = reinterpret_cast<__half2 *>(p.out + (int64_t)t * p.so_t + (int64_t)hd * p.so_h + d);
      o[0] = __floats2half2_rn(f[0] * inv, f[1] * inv);
      o[1] = __floats2half2_rn(f[2] * inv, f[3] * inv);
    }
  }
}

// ------------------------------------------------------------------ host
static int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is cut.  A function of the sizes alone, so that the workspace query and the launch agree.
struct Plan {
  bool seq, tc_prefix;            // tensor-core forms
  bool stream, stream_prefix;     // the stream of key blocks: own keys, and the prefix unless tc_prefix
  bool tma;                       // its blocks by TMA
  bool join;                      // some row may have more than one part
  int prefix_parts;               // parts in row order that the prefix leaves
  int cluster;                    // key ranges of a prefix tile that join in a cluster
  int slots;                      // parts in row order, prefix and own
  int rw, tile_rows, tile_tokens, piece;
  int64_t ctas;                   // of the launch that walks the list of units
};

static int rw_for(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
static int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

static Plan make_plan(const hexb_paged_attention_desc *d, int sm_count) {
  Plan pl = {};
  const int64_t G = d->Hq / d->Hkv, capacity = d->table_width * d->page_size;
  const int64_t mq = d->max_q > 0 ? clamp64(d->max_q, 1, d->T) : ceil_div(d->T, d->B);
  const int64_t pblocks = ceil_div(d->prefix_len, 64), oblocks = ceil_div(capacity, 64);
  // What TMA can address: page pieces of at least the 8 rows of a swizzle atom, no stride of 0.
  // The tensor-core forms want besides: a positive scale, and enough rows to fill half of a 128-row tile.
  pl.piece = (int)(d->page_size & -d->page_size);
  if (pl.piece > 64) pl.piece = 64;
  bool tma_ok = (d->D == 64 || d->D == 128) && pl.piece >= 8;
  const int64_t dims[8] = {d->T, d->Hq, d->num_pages, d->page_size, d->Hkv, d->num_pages, d->page_size, d->Hkv};
  auto fits = [&](int i) { return dims[i] <= 1 || (d->strides[i] > 0 && d->strides[i] < ((int64_t)1 << 38)); };
  for (int i = 2; i < 8; ++i) tma_ok = tma_ok && fits(i);
  pl.tma = tma_ok;
  const bool tc_ok = tma_ok && fits(0) && fits(1) && d->sm_scale > 0.f && G <= 128 && (d->Hkv <= 1 || d->strides[1] * G < ((int64_t)1 << 38));
  pl.tile_tokens = tc_ok ? (int)(128 / G) : 0;
  // CTAs for a list of at most `tiles` tiles of at most `blocks` blocks: those that fit the GPU, fewer for a short list
  auto ctas_for = [&](double units, int64_t fit) { return clamp64(units < (double)fit ? (int64_t)units : fit, 1, fit); };
  if (tc_ok && mq * G >= 64 && capacity > 0) {
    // Tiles of one sequence each, over the prefix and its own keys, from 64 rows a sequence on.  Against the stream (behind
    // the packed prefix form, if there is a prefix), 8 key heads of 128, G = 4: 16 sequences of 2048 own keys, no prefix, 32
    // rows each 38.9 us against 43.7, 64 rows 43.9 against 67.4; 64 sequences of 512 behind 8192 shared keys 333 against 159,
    // 332 against 269, and at 96 rows 345 against 502: a long prefix, which each tile reads for itself, moves the border up.
    pl.seq = true;
    pl.tile_rows = 128;
    const double tiles = (double)(ceil_div(d->T, pl.tile_tokens) + d->B) * d->Hkv;
    pl.ctas = ctas_for(tiles * (pblocks + oblocks), 2 * sm_count);
    pl.join = pblocks + oblocks > 1;
    return pl;
  }
  if (d->prefix_len > 0 && tc_ok && d->T * G >= 64) {
    pl.tc_prefix = true;
    // The prefix by 128-row tiles, from 64 rows on.  Against the stream, 8192 keys, 8 key heads of 128, G = 4: with 512 own
    // keys a sequence 32 rows 33.3 us against 30.5 (one launch more), 64 rows 36.0 against 38.9, 256 rows 61.8 against 98.3;
    // the prefix alone 20.0 against 28.8, 20.7 against 33.1, 26.5 against 57.9.
    const int64_t tiles = (int64_t)ceil_div(d->T, pl.tile_tokens) * d->Hkv;
    // Two CTAs an SM: one does not keep the tensor pipe busy (the prefix alone: 64 sequences behind 8192 keys 29.3 us against
    // 26.3, 128 behind 16385 keys 82.6 against 50.5).
    const int64_t ranges = clamp64(2 * sm_count / tiles, 1, clamp64((pblocks + 1) / 2, 1, 64));
    for (pl.cluster = 8; pl.cluster > ranges;) pl.cluster /= 2;
    pl.prefix_parts = (int)(ranges / pl.cluster);
  }
  pl.stream_prefix = d->prefix_len > 0 && !pl.tc_prefix;
  pl.stream = pl.stream_prefix || capacity > 0;
  if (pl.stream) {
    const int per_sm = d->D <= 64 ? 4 : d->D <= 128 ? 2 : 1;
    pl.rw = rw_for(mq * G);
    if ((pl.stream_prefix && d->T * G > 128) || d->D > 128) pl.rw = 4;
    pl.tile_rows = 16 * pl.rw;
    const double ptiles = pl.stream_prefix ? (double)ceil_div(d->T * G, pl.tile_rows) * d->Hkv : 0.;
    const double otiles = capacity > 0 ? (double)(ceil_div(d->T * G, pl.tile_rows) + d->B) * d->Hkv : 0.;
    pl.ctas = ctas_for(ptiles * pblocks + otiles * (oblocks > 1 ? oblocks : 1), (int64_t)sm_count * per_sm);
  }
  const int sides = (d->prefix_len > 0) + (capacity > 0);
  pl.join = sides != 1 || (pl.tc_prefix ? pl.prefix_parts > 1 : pblocks + oblocks > 1);
  if (pl.tc_prefix) pl.slots = pl.prefix_parts > 1 || sides > 1 ? pl.prefix_parts : 0;
  else if (pl.stream_prefix && sides > 1) pl.slots = 1;
  if (sides > 1) ++pl.slots;      // own keys of tiles that were not cut
  return pl;
}

static size_t parts_of(const hexb_paged_attention_desc *d, const Plan &pl) {
  return (size_t)pl.slots * d->T * d->Hq + (pl.tile_rows ? (size_t)pl.ctas * 2 * pl.tile_rows : 0);
}
static size_t ws_need(const hexb_paged_attention_desc *d, const Plan &pl) {
  if (!pl.join || !parts_of(d, pl)) return 0;
  return parts_of(d, pl) * ((size_t)d->D * 4 + 8) + (size_t)d->T * d->Hq * 2 * sizeof(int4) + 256;
}

template <int DP, int RW>
static int launch_stream(const Params &p, const CUtensorMap *tm, dim3 grid, cudaStream_t st) {
  static PerDeviceOnce once;
  int dev = 0;
  HEXB_CUDA_OK(cudaGetDevice(&dev));
  using cfg = RowCfg<DP>;
  if (!once.is_done(dev)) {
    HEXB_CUDA_OK(cudaFuncSetAttribute(paged_stream_kernel<DP, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize, cfg::SMEM));
    if constexpr (DP <= 128)
      HEXB_CUDA_OK(cudaFuncSetAttribute(paged_stream_tma_kernel<DP, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize, cfg::SMEM_TMA));
    once.mark(dev);
  }
  if constexpr (DP <= 128) {
    if (tm) {
      HEXB_CUDA_OK(launch_pdl(paged_stream_tma_kernel<DP, RW>, grid, dim3(160), (size_t)cfg::SMEM_TMA, st, tm[0], tm[1], p));
      return check_launch("paged_stream_tma");
    }
  }
  HEXB_CUDA_OK(launch_pdl(paged_stream_kernel<DP, RW>, grid, dim3(THREADS), (size_t)cfg::SMEM, st, p));
  return check_launch("paged_stream");
}

static int dispatch_stream(const Params &p, int rw, const CUtensorMap *tm, dim3 grid, cudaStream_t st) {
#define HEXB_ROWS(DP)                                                  \
  return rw == 1 ? launch_stream<DP, 1>(p, tm, grid, st)               \
                 : rw == 2 ? launch_stream<DP, 2>(p, tm, grid, st) : launch_stream<DP, 4>(p, tm, grid, st)
  if (p.D <= 64) HEXB_ROWS(64);
  if (p.D <= 128) HEXB_ROWS(128);
  return launch_stream<256, 4>(p, tm, grid, st);
#undef HEXB_ROWS
}

static int check_desc(const hexb_paged_attention_desc *d) {
  if (!d) return HEXB_ERR_BAD_ARG;
  if (d->T < 0 || d->B < 0 || d->Hq < 0 || d->Hkv < 0 || d->D < 0 || d->prefix_len < 0 || d->table_width < 0 ||
      d->num_pages < 0 || d->page_size < 1 || d->max_q < 0)
    return HEXB_ERR_BAD_ARG;
  if (d->T == 0 || d->Hq == 0 || d->B == 0 || d->D == 0) return HEXB_OK;
  if (d->Hkv == 0 || d->Hq % d->Hkv || (!d->q_offsets && d->T != d->B)) return HEXB_ERR_BAD_ARG;
  if (d->D % 8 || d->D > 256 || d->Hkv > 65535 || d->Hq > (1 << 30) || d->T > (1 << 24) ||
      d->T * (d->Hq / d->Hkv) > (1 << 30) || d->T * d->Hq > ((int64_t)1 << 32) || d->B > (1 << 20) ||
      d->prefix_len > (1 << 30) || d->page_size > (1 << 30) || d->num_pages > 0x7fffffff ||
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
  p.prefix_parts = pl.prefix_parts;
  p.nseq = p.own_capacity ? p.B : 0;
  p.scale_log2 = d->sm_scale * 1.44269504f;
  p.tile_tokens = pl.tile_tokens;
  p.piece = pl.piece;
  p.cluster = pl.cluster;
  p.ctas = (int)pl.ctas;
  p.tile_rows = pl.tile_rows;
  const bool both = d->prefix_len > 0 && p.own_capacity > 0 && !pl.seq;
  p.prefix_slot = pl.stream_prefix && both ? 0 : -1;
  p.own_slot = both ? pl.slots - 1 : -1;
  if (need) {
    const size_t rows = (size_t)d->T * d->Hq, n = parts_of(d, pl);
    uint8_t *w = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~(uintptr_t)15);
    p.part_o = reinterpret_cast<float *>(w);
    p.part_ml = reinterpret_cast<float2 *>(w + n * d->D * 4);
    p.run_base = (int64_t)pl.slots * rows;
    int4 *desc = reinterpret_cast<int4 *>(w + (n * (d->D * 4 + 8) + 15) / 16 * 16);
    if (pl.stream_prefix) p.prefix_desc = desc;
    if (p.own_capacity) p.own_desc = desc + rows;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (pl.seq) {
    p.shared_blocks = paged::ceil_div(d->prefix_len, 64);
    if (int e = paged::tc_launch(p, (int)d->Hkv, true, dim3((unsigned)pl.ctas), st)) return e;
  } else if (pl.tc_prefix) {
    const dim3 grid((unsigned)paged::ceil_div(d->T, pl.tile_tokens), (unsigned)(pl.prefix_parts * pl.cluster), (unsigned)d->Hkv);
    if (int e = paged::tc_launch(p, (int)d->Hkv, false, grid, st)) return e;
  }
  if (pl.stream) {
    p.stream_prefix = pl.stream_prefix;
    CUtensorMap tm[2];
    if (pl.tma)
      if (int e = paged::cache_maps(p, (int)d->Hkv, tm)) return e;
    if (int e = paged::dispatch_stream(p, pl.rw, pl.tma ? tm : nullptr, dim3((unsigned)pl.ctas), st)) return e;
  }
  if (pl.join) {
    // also the call without any key: its rows are set to zero
    const dim3 grid((unsigned)((d->T * d->Hq + 3) / 4));
    if (d->D <= 64) HEXB_CUDA_OK(launch_pdl(paged::paged_join_kernel<16>, grid, dim3(128), 0, st, p));
    else HEXB_CUDA_OK(launch_pdl(paged::paged_join_kernel<32>, grid, dim3(128), 0, st, p));
    return check_launch("paged_join");
  }
  return HEXB_OK;
}
