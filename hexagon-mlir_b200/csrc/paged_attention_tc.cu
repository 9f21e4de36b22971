// Paged attention on the tensor cores (tcgen05 + TMEM + TMA) for tiles of many query rows.
//
// A tile is up to 128 rows of one key head: floor(128 / G) tokens with their G query heads, fetched by one
// TMA box per 64 columns.  Keys come in blocks of 64; a block is fetched page piece by page piece (the largest
// power of two of rows that divides the page size), each lane of the producer warp looking up and fetching its
// own piece.  Two forms:
//   SEQ false   rows of the whole batch against the shared prefix: every key is read for 128 rows at once
//   SEQ true    rows of one sequence against the prefix and then its own keys, causal among the new tokens
// The pipeline is that of the library's 64-key attention kernel (attention.cu): scores of block j + 1 are
// computed into the second buffer while the softmax warps work on block j, P is written over the scores as fp16
// and read from tensor memory, O stays there and is rescaled only when a row maximum grows by more than 2^8.
// A block range that is not the whole axis leaves (O, m, l) in fp32 for the join.
//
// 192 threads: warp 0 producer, warp 1 MMA issuer, warps 2-5 one row per thread.  Every wait is bounded.
#include "attn_common.cuh"
#include "paged_attention.cuh"

namespace hexb {
namespace paged {

using attn::ex2_approx;

template <int HD>
struct TcCfg {
  static constexpr int BN = 64;
  static constexpr int CHUNKS = HD / 64;
  static constexpr int Q_BYTES = 128 * HD * 2, Q_CHUNK = 128 * 128;
  static constexpr int KV_BYTES = BN * HD * 2, KV_CHUNK = BN * 128;
  static constexpr int NBAR = 18;
  static constexpr int NEEDED = Q_BYTES + 4 * KV_BYTES + NBAR * 8 + 16 + 1024;
  static constexpr int SMEM = NEEDED < 100 * 1024 ? 100 * 1024 : NEEDED;  // at most two CTAs an SM: 2 x 256 TMEM columns
  static constexpr int TMEM_COLS = 256, O_COL = 128;                      // S0 [0,64), S1 [64,128), O [128,128+HD)
};

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

template <int HD, bool SEQ>
__global__ void __launch_bounds__(192, 2)
paged_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const Params p) {
  using cfg = TcCfg<HD>;
  constexpr int BN = cfg::BN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_addr = tc::smem_u32(smem_raw);
  const uint32_t sQ = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem = smem_raw + (sQ - raw_addr);
  const uint32_t sK0 = sQ + cfg::Q_BYTES, sV0 = sK0 + 2 * cfg::KV_BYTES;
  const uint32_t bar0 = sV0 + 2 * cfg::KV_BYTES;
  const uint32_t q_full = bar0, q_empty = bar0 + 8, o_full = bar0 + 16, o_empty = bar0 + 24, pv_done = bar0 + 32,
                 tail = bar0 + 40;
  auto k_full = [&](uint32_t b) { return bar0 + 48 + 8 * b; };
  auto k_empty = [&](uint32_t b) { return bar0 + 64 + 8 * b; };
  auto v_full = [&](uint32_t b) { return bar0 + 80 + 8 * b; };
  auto v_empty = [&](uint32_t b) { return bar0 + 96 + 8 * b; };
  auto s_full = [&](uint32_t b) { return bar0 + 112 + 8 * b; };
  auto p_full = [&](uint32_t b) { return bar0 + 128 + 8 * b; };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + cfg::Q_BYTES + 4 * cfg::KV_BYTES + cfg::NBAR * 8);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int TB = p.tile_tokens, rows_tile = TB * p.G;

  if (threadIdx.x == 0) {
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, 1);
    tc::mbar_init(o_full, 1);
    tc::mbar_init(o_empty, 4);
    tc::mbar_init(pv_done, 1);
    tc::mbar_init(tail, 1);
    for (uint32_t b = 0; b < 2; ++b) {
      tc::mbar_init(k_full(b), 1);
      tc::mbar_init(k_empty(b), 1);
      tc::mbar_init(v_full(b), 1);
      tc::mbar_init(v_empty(b), 1);
      tc::mbar_init(s_full(b), 1);
      tc::mbar_init(p_full(b), 4);
    }
    *abort_flag = 0;
    tc::fence_barrier_init();
    tc::prefetch_tensormap(&tmQ);
    tc::prefetch_tensormap(&tmK);
    tc::prefetch_tensormap(&tmV);
  }
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(tmem_slot), cfg::TMEM_COLS);
    tc::tmem_relinquish();
  }
  // rows of the Q tile that no query fills (G does not divide 128): zeros, so that their scores are
  for (int i = threadIdx.x; i < (128 - rows_tile) * 8 * cfg::CHUNKS; i += 192) {
    const int c = i / ((128 - rows_tile) * 8), k = i - c * (128 - rows_tile) * 8;
    *reinterpret_cast<uint4 *>(smem + c * cfg::Q_CHUNK + rows_tile * 128 + k * 16) = make_uint4(0, 0, 0, 0);
  }
  tc::fence_proxy_async_smem();
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  // The next launch may take the places of CTAs that are done; it waits for this whole grid before it reads anything.
  pdl_launch_dependents();
  const uint32_t tO = tmem_base + cfg::O_COL;

  // SEQ: the CTA's stretch of the list of units, segment by segment (the blocks of one tile); else one tile and range.
  long long u = 0, stop = 1, per = 1;
  Cursor cur;
  int part = 0;
  if (SEQ) {
    find_stretch<192>(p, rows_tile, u, stop, per, cur);
  } else {
    cur.b = -1;
    cur.tok0 = 0;
    cur.ntok = tokens_used(p);
    cur.len = 0;
    cur.nb = 1;
    cur.tile = blockIdx.x;
    cur.h = blockIdx.z;
    cur.j = 0;
    part = blockIdx.y;
    if (cur.tile * TB >= cur.ntok) stop = 0;
  }
  const int prefix_blocks = (p.prefix_len + BN - 1) / BN;
  // The segment at the cursor: units [j0, j1) of its tile, of which [lo, hi) hold keys that some row sees.
  struct Segment {
    int j0, j1, lo, hi, own_end;
  };
  auto segment = [&]() {
    Segment s;
    if (SEQ) {
      s.own_end = max(0, cur.len - cur.ntok + min((cur.tile + 1) * TB, cur.ntok));
      s.j0 = cur.j;
      s.j1 = (int)min((long long)cur.nb, cur.j + (stop - u));
      s.lo = s.j0;
      s.hi = min(s.j1, prefix_blocks + (s.own_end + BN - 1) / BN);
    } else {
      const int n = (prefix_blocks + (int)gridDim.y - 1) / (int)gridDim.y;
      s.own_end = 0;
      s.j0 = 0;
      s.j1 = 1;
      s.lo = min(part * n, prefix_blocks);
      s.hi = min(s.lo + n, prefix_blocks);
    }
    return s;
  };
  auto next = [&](const Segment &s) {
    u += s.j1 - s.j0;
    if (SEQ && u < stop) advance(p, rows_tile, cur, s.j1 - s.j0);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    uint32_t it = 0, t = 0, tails = 0;
    bool ok = true;
    const int pieces = BN / p.piece;
    for (; u < stop && ok;) {
      const Segment a = segment();
      if (a.lo >= a.hi) {
        next(a);
        continue;
      }
      const int oend = a.own_end, h = cur.h;
      const int *own_pages = SEQ ? p.table + (int64_t)cur.b * p.table_stride : nullptr;
      if (t > 0 && !tc::mbar_wait(q_empty, (t - 1u) & 1u, abort_flag)) break;
      ++t;
      if (lane == 0) {
        tc::mbar_arrive_expect_tx(q_full, (uint32_t)rows_tile * HD * 2);
#pragma unroll
        for (int c = 0; c < cfg::CHUNKS; ++c)
          tc::tma_load_4d(sQ + c * cfg::Q_CHUNK, &tmQ, c * 64, 0, h, cur.tok0 + cur.tile * TB, q_full);
      }
      // page of this lane's piece of block j; a piece without keys and a page outside the cache read as zeros
      auto lookup = [&](int j, int &slot) {
        const bool pre = j < prefix_blocks;
        const int key = (pre ? j : j - prefix_blocks) * BN + lane * p.piece;
        int page = p.num_pages;
        slot = 0;
        if (lane < pieces && j < a.hi && key < (pre ? p.prefix_len : oend)) {
          const int pi = key / p.page_size;
          slot = key - pi * p.page_size;
          const int got = pre ? p.prefix_pages[pi] : own_pages[pi];
          if ((unsigned)got < (unsigned)p.num_pages) page = got;
          else atomicExch(&g_paged_status, (int)HEXB_ERR_BAD_ARG);
        }
        return page;
      };
      int slot_next, page_next = lookup(a.lo, slot_next);
      for (int j = a.lo; j < a.hi; ++j, ++it) {
        const uint32_t b = it & 1u, ph = (it >> 1) & 1u;
        const int page = page_next, slot = slot_next;
        page_next = lookup(j + 1, slot_next);
        const uint32_t at = (uint32_t)lane * (uint32_t)p.piece * 128u;
        if (!tc::mbar_wait(k_empty(b), ph ^ 1u, abort_flag)) { ok = false; break; }
        if (lane == 0) tc::mbar_arrive_expect_tx(k_full(b), cfg::KV_BYTES);
        __syncwarp();
        if (lane < pieces) {
#pragma unroll
          for (int c = 0; c < cfg::CHUNKS; ++c)
            tc::tma_load_4d(sK0 + b * cfg::KV_BYTES + c * cfg::KV_CHUNK + at, &tmK, c * 64, h, slot, page, k_full(b));
        }
        if (!tc::mbar_wait(v_empty(b), ph ^ 1u, abort_flag)) { ok = false; break; }
        const bool pre = j < prefix_blocks;
        const int filled = (pre ? p.prefix_len - j * BN : oend - (j - prefix_blocks) * BN);  // keys of the block
        const uint32_t bar = filled < BN ? tail : v_full(b);
        if (lane == 0) tc::mbar_arrive_expect_tx(bar, cfg::KV_BYTES);
        __syncwarp();
        if (lane < pieces) {
#pragma unroll
          for (int c = 0; c < cfg::CHUNKS; ++c)
            tc::tma_load_4d(sV0 + b * cfg::KV_BYTES + c * cfg::KV_CHUNK + at, &tmV, c * 64, h, slot, page, bar);
        }
        if (filled < BN) {
          // the last block of an axis: whatever lies behind the keys -- NaN, perhaps -- must not meet a weight of 0
          if (!tc::mbar_wait(tail, tails & 1u, abort_flag)) { ok = false; break; }
          ++tails;
          uint8_t *v = smem + (sV0 - sQ) + b * cfg::KV_BYTES;
          for (int i = lane; i < (BN - filled) * 8 * cfg::CHUNKS; i += 32) {
            const int c = i / ((BN - filled) * 8), k = i - c * (BN - filled) * 8;
            *reinterpret_cast<uint4 *>(v + c * cfg::KV_CHUNK + filled * 128 + k * 16) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(v_full(b));
        }
      }
      next(a);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_qk = tc::make_idesc_f16_f32(128, BN, 0, 0);
      constexpr uint32_t idesc_pv = tc::make_idesc_f16_f32(128, HD, 0, 1);
      bool ok = true;
      auto issue_qk = [&](uint32_t blk, bool last) {
        const uint32_t b = blk & 1u;
        if (!tc::mbar_wait(k_full(b), (blk >> 1) & 1u, abort_flag)) { ok = false; return; }
        tc::tc_fence_after();
        const uint32_t sK = sK0 + b * cfg::KV_BYTES;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t qoff = (uint32_t)((k >> 2) * cfg::Q_CHUNK + (k & 3) * 32);
          const uint32_t koff = (uint32_t)((k >> 2) * cfg::KV_CHUNK + (k & 3) * 32);
          tc::mma_f16_ss(tmem_base + b * BN, tc::make_smem_desc_sw128(sQ + qoff, 16, 1024),
                         tc::make_smem_desc_sw128(sK + koff, 16, 1024), idesc_qk, k != 0 ? 1u : 0u);
        }
        tc::mma_commit(s_full(b));
        tc::mma_commit(k_empty(b));
        if (last) tc::mma_commit(q_empty);
      };
      uint32_t it = 0, t = 0;
      for (; u < stop && ok;) {
        const Segment a = segment();
        next(a);
        if (a.lo >= a.hi) continue;
        if (!tc::mbar_wait(q_full, t & 1u, abort_flag)) break;
        issue_qk(it, a.lo + 1 == a.hi);
        for (int j = a.lo; j < a.hi && ok; ++j, ++it) {
          if (j + 1 < a.hi) issue_qk(it + 1, j + 2 == a.hi);  // one block ahead of the softmax
          if (!ok) break;
          const uint32_t b = it & 1u, ph = (it >> 1) & 1u;
          if (!tc::mbar_wait(p_full(b), ph, abort_flag)) { ok = false; break; }
          if (!tc::mbar_wait(v_full(b), ph, abort_flag)) { ok = false; break; }
          // the first product of a later tile overwrites O: the previous epilogue must have read it
          if (j == a.lo && t > 0 && !tc::mbar_wait(o_empty, (t - 1u) & 1u, abort_flag)) { ok = false; break; }
          tc::tc_fence_after();
          const uint32_t sV = sV0 + b * cfg::KV_BYTES;
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            tc::mma_f16_ts(tO, tmem_base + b * BN + (uint32_t)(k * 8),
                           tc::make_smem_desc_sw128(sV + (uint32_t)(k * 2048), cfg::KV_CHUNK, 1024), idesc_pv,
                           (j != a.lo || k != 0) ? 1u : 0u);
          tc::mma_commit(v_empty(b));
          tc::mma_commit(pv_done);
          if (j == a.hi - 1) tc::mma_commit(o_full);
        }
        ++t;
      }
    }
  } else {
    // ------------------------------------------------------------ softmax, rescaling, epilogue
    const int q = warp & 3;
    const int r = q * 32 + lane;                    // row of the tile == TMEM lane
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const int rt = r / p.G, rg = r - rt * p.G;      // token in the tile, query head in the group
    uint32_t it = 0, t = 0;
    bool ok = true;
    float m_last = -INFINITY, l_last = 0.f;         // of the one tile of a CTA in a cluster
    const float2 mul2 = make_float2(p.scale_log2, p.scale_log2);
    for (; u < stop && ok;) {
      const Segment a = segment();
      const int idx = cur.tile * TB + rt;           // token of the sequence (or batch)
      const bool row_ok = rt < TB && idx < cur.ntok;
      const int sees = cur.len - cur.ntok + idx + 1;   // own keys this row sees (SEQ)
      const int tok = cur.tok0 + idx, hd = cur.h * p.G + rg;
      int64_t dest = part < 0 || !p.part_o ? -1 : (int64_t)part * p.T * p.Hq + (int64_t)tok * p.Hq + hd;
      if (SEQ) {
        const RunPlace place(p, cur, a.j0, a.j1, u - a.j0, per, 128);
        dest = row_ok ? place.index(p, tok, hd, r) : -1;
        if (row_ok) place.describe(p, cur, tok, hd, r);
      }
      next(a);
      float m_ref = -INFINITY, l = 0.f;
      for (int j = a.lo; j < a.hi; ++j, ++it) {
        const uint32_t b = it & 1u, ph = (it >> 1) & 1u;
        if (!tc::mbar_wait(s_full(b), ph, abort_flag)) { ok = false; break; }
        tc::tc_fence_after();
        const uint32_t tS = tmem_base + b * BN;
        uint32_t sv[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
          tc::tmem_ld_32x32(tS + lane_off + (uint32_t)(c * 32), reinterpret_cast<uint32_t(&)[32]>(sv[c * 32]));
        tc::tmem_ld_wait();
        // keys of this block that the row sees
        const bool pre = j < prefix_blocks;
        const int kv0 = (pre ? j : j - prefix_blocks) * BN;
        const int vis = (pre ? p.prefix_len : SEQ ? min(sees, a.own_end) : 0) - kv0;
        if (__any_sync(0xffffffffu, vis < BN)) {
#pragma unroll
          for (int e = 0; e < BN; ++e)
            if (e >= vis) sv[e] = 0xff800000u;
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < BN; e += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            mx4[u] = attn::max3(mx4[u], __uint_as_float(sv[e + 2 * u]), __uint_as_float(sv[e + 2 * u + 1]));
        }
        // scale > 0: the maximum commutes with the scaling
        const float m_new = fmaxf(m_ref, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2);
        if (j == a.lo) {
          m_ref = m_new;
        } else if (__any_sync(0xffffffffu, m_new - m_ref > attn::kRescaleThreshold)) {
          // O must be quiescent: P_{it-1}.V_{it-1} is the it-th completion of pv_done
          if (!tc::mbar_wait(pv_done, (it - 1u) & 1u, abort_flag)) { ok = false; break; }
          tc::tc_fence_after();
          const float alpha = m_new == -INFINITY ? 1.0f : ex2_approx(m_ref - m_new);
          m_ref = m_new;
          l *= alpha;
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tc::tmem_ld_32x32(tO + lane_off + (uint32_t)(c * 32), o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tc::tmem_st_32x32(tO + lane_off + (uint32_t)(c * 32), o);
          }
        }
        // a row that has seen no key, or only infinite ones, keeps m_ref = -inf: its weights must come out 0, not NaN
        const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
        const float2 neg_m2 = make_float2(neg_m, neg_m);
        float2 l0 = make_float2(0.f, 0.f), l1 = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float2 xa = attn::fma2(make_float2(__uint_as_float(sv[c * 32 + e]), __uint_as_float(sv[c * 32 + e + 1])), mul2, neg_m2);
            const float2 xb = attn::fma2(make_float2(__uint_as_float(sv[c * 32 + e + 2]), __uint_as_float(sv[c * 32 + e + 3])), mul2, neg_m2);
            const float2 pa = make_float2(ex2_approx(xa.x), ex2_approx(xa.y));
            const float2 pb = make_float2(ex2_approx(xb.x), ex2_approx(xb.y));
            l0 = attn::add2(l0, pa);
            l1 = attn::add2(l1, pb);
            pk[e >> 1] = attn::pack_f16x2(pa.x, pa.y);
            pk[(e >> 1) + 1] = attn::pack_f16x2(pb.x, pb.y);
          }
          tc::tmem_st_32x16(tS + lane_off + (uint32_t)(c * 16), pk);
        }
        l += (l0.x + l0.y) + (l1.x + l1.y);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(b));
      }
      if (!ok) break;
      if (!SEQ && p.cluster > 1) {                  // joined with the other CTAs of the cluster below
        if (a.lo < a.hi) {
          ok = tc::mbar_wait(o_full, 0, abort_flag);
          tc::tc_fence_after();
          m_last = m_ref;
          l_last = ok ? l : 0.f;
        }
        break;
      }
      if (a.lo >= a.hi) {                           // no key for this tile: nothing went through the pipeline
        if (row_ok) {
          float zero[4] = {0.f, 0.f, 0.f, 0.f};
          for (int d = 0; d < HD; d += 4) store_row<4>(p, dest, tok, hd, d, zero, -INFINITY, 0.f);
        }
        continue;
      }
      if (!tc::mbar_wait(o_full, t & 1u, abort_flag)) { ok = false; break; }
      tc::tc_fence_after();
      ++t;
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      __half *orow = p.out + (int64_t)tok * p.so_t + (int64_t)hd * p.so_h;
      if (dest >= 0 && row_ok) p.part_ml[dest] = make_float2(m_ref, l);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tc::tmem_ld_32x32(tO + lane_off + (uint32_t)(c * 32), o);
        tc::tmem_ld_wait();
        if (c == HD / 32 - 1) {  // O is in registers: the next tile's first product may overwrite it
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(o_empty);
        }
        if (!row_ok) continue;
        if (dest >= 0) {
          if (l != 0.f) {
            float4 *dst = reinterpret_cast<float4 *>(p.part_o + dest * HD + c * 32);
#pragma unroll
            for (int g = 0; g < 8; ++g)
              dst[g] = make_float4(__uint_as_float(o[g * 4]), __uint_as_float(o[g * 4 + 1]), __uint_as_float(o[g * 4 + 2]),
                                   __uint_as_float(o[g * 4 + 3]));
          }
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = l == 0.f ? 0.f : __uint_as_float(o[g * 8 + e]) * inv;
            Vec16<__half> ov;
            ov.pack(f);
            *reinterpret_cast<uint4 *>(orow + c * 32 + g * 8) = ov.raw;
          }
        }
      }
    }
    if (!SEQ && p.cluster > 1) {
      // The CTAs of a cluster hold the same rows against neighbouring key ranges.  Their parts meet in distributed shared
      // memory, each CTA adding up its share of the rows: the parts that reach memory, and the join kernel, are
      // fewer by the cluster's size (16 parts of 2048 rows through memory cost the join 10 us).
      const int cl = p.cluster, rank = (int)tc::cluster_ctarank();
      float2 *ml = reinterpret_cast<float2 *>(smem);                          // over Q: the last product has read it
      const uint32_t so = sK0;                                                // over K and V: [128 rows][HD], 16-byte pieces
      float2 *fin = ml + 128;                                                 // of row r: maximum and sum over the cluster
      ml[r] = make_float2(m_last, l_last);                                    // of row r at (piece ^ r)
      tc::cluster_sync_all();
      float mm = -INFINITY, ll = 0.f;
      const uint32_t mine = tc::smem_u32(&ml[r]);
      float2 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)                                             // all trips to the peers under way at once
        v[i] = i < cl ? ld_cluster_f2(tc::map_to_rank(mine, (uint32_t)i)) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i].y != 0.f) mm = fmaxf(mm, v[i].x);
#pragma unroll
      for (int i = 0; i < 8; ++i) ll += v[i].y == 0.f ? 0.f : v[i].y * ex2_approx(v[i].x - mm);
      fin[r] = make_float2(mm, ll);
      const float alpha = l_last == 0.f ? 0.f : ex2_approx(m_last - mm);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tc::tmem_ld_32x32(tO + lane_off + (uint32_t)(c * 32), o);
        tc::tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint32_t piece = (uint32_t)(c * 8 + g) ^ (uint32_t)(r & (HD / 4 - 1));
          const bool use = l_last != 0.f;
          *reinterpret_cast<float4 *>(smem + (so - sQ) + r * HD * 4 + piece * 16) =
              make_float4(use ? alpha * __uint_as_float(o[g * 4]) : 0.f, use ? alpha * __uint_as_float(o[g * 4 + 1]) : 0.f,
                          use ? alpha * __uint_as_float(o[g * 4 + 2]) : 0.f, use ? alpha * __uint_as_float(o[g * 4 + 3]) : 0.f);
        }
      }
      tc::cluster_sync_all();
      const int share = 128 / cl, tid = threadIdx.x - 64;
      for (int i = tid; i < share * (HD / 4); i += 128) {
        const int rr = rank * share + i / (HD / 4), d = (i % (HD / 4)) * 4;
        const int idx = (int)blockIdx.x * TB + rr / p.G, hd = (int)blockIdx.z * p.G + rr % p.G;
        if (rr >= rows_tile || idx >= cur.ntok) continue;
        float f[4] = {0.f, 0.f, 0.f, 0.f};
        const float2 row = fin[rr];
        const uint32_t orow = so + (uint32_t)(rr * HD * 4) + (((uint32_t)(d / 4) ^ (uint32_t)(rr & (HD / 4 - 1))) * 16);
        float4 q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          q[k] = k < cl ? ld_cluster_f4(tc::map_to_rank(orow, (uint32_t)k)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          f[0] += q[k].x; f[1] += q[k].y; f[2] += q[k].z; f[3] += q[k].w;
        }
        const int64_t dest = p.part_o ? (int64_t)(part / cl) * p.T * p.Hq + (int64_t)idx * p.Hq + hd : -1;
        store_row<4>(p, dest, idx, hd, d, f, row.x, row.y);
      }
      tc::cluster_sync_all();                                                 // no CTA leaves while its memory is read
    }
  }

  if (!SEQ && p.cluster > 1 && warp < 2) {          // the other side of the cluster's barriers
    __syncwarp();
    for (int i = 0; i < 3; ++i) tc::cluster_sync_all();
  }
  // ------------------------------------------------------------ teardown
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // lets copies in flight land before the CTA's memory goes
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, cfg::TMEM_COLS);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_paged_status, (int)HEXB_ERR_TIMEOUT);
}

// ------------------------------------------------------------------ host
template <int HD, bool SEQ>
static int launch_tc(const Params &p, const CUtensorMap *tm, dim3 grid, cudaStream_t st) {
  static PerDeviceOnce once;
  int dev = 0;
  HEXB_CUDA_OK(cudaGetDevice(&dev));
  if (!once.is_done(dev)) {
    HEXB_CUDA_OK(cudaFuncSetAttribute(paged_tc_kernel<HD, SEQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcCfg<HD>::SMEM));
    once.mark(dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = TcCfg<HD>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (option(OPT_pdl, 1)) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (!SEQ && p.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1;
    attr[n].val.clusterDim.y = (unsigned)p.cluster;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  HEXB_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_tc_kernel<HD, SEQ>, tm[0], tm[1], tm[2], p));
  return check_launch("paged_tc");
}

// a dimension of one element may come with any stride: the map gets a legal one
static uint64_t stride_bytes(int64_t n, int64_t stride) { return n > 1 ? (uint64_t)stride * 2 : (uint64_t)16; }

int cache_maps(const Params &p, int hkv, CUtensorMap *tm) {
  const uint64_t dims[4] = {(uint64_t)p.D, (uint64_t)hkv, (uint64_t)p.page_size, (uint64_t)p.num_pages};
  const uint32_t box[4] = {64, 1, (uint32_t)p.piece, 1};
  const uint64_t sk[3] = {stride_bytes(hkv, p.sk_h), stride_bytes(p.page_size, p.sk_s), stride_bytes(p.num_pages, p.sk_p)};
  const uint64_t sv[3] = {stride_bytes(hkv, p.sv_h), stride_bytes(p.page_size, p.sv_s), stride_bytes(p.num_pages, p.sv_p)};
  if (int e = encode_tmap_f16_sw128(&tm[0], p.k, 4, dims, sk, box)) return e;
  return encode_tmap_f16_sw128(&tm[1], p.v, 4, dims, sv, box);
}

int tc_launch(const Params &p, int hkv, bool seq, dim3 grid, cudaStream_t st) {
  CUtensorMap tm[3];
  const uint64_t dims[4] = {(uint64_t)p.D, (uint64_t)p.G, (uint64_t)hkv, (uint64_t)p.T};
  const uint64_t str[3] = {stride_bytes(p.G, p.sq_h), stride_bytes(hkv, p.sq_h * p.G), stride_bytes(p.T, p.sq_t)};
  const uint32_t box[4] = {64, (uint32_t)p.G, 1, (uint32_t)p.tile_tokens};
  if (int e = encode_tmap_f16_sw128(&tm[0], p.q, 4, dims, str, box)) return e;
  if (int e = cache_maps(p, hkv, tm + 1)) return e;
  if (p.D == 64) return seq ? launch_tc<64, true>(p, tm, grid, st) : launch_tc<64, false>(p, tm, grid, st);
  return seq ? launch_tc<128, true>(p, tm, grid, st) : launch_tc<128, false>(p, tm, grid, st);
}

}  // namespace paged

int paged_tc_device_status_fetch_and_clear(int *out) {
  int v = 0, zero = 0;
  HEXB_CUDA_OK(cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(int)));
  if (v) HEXB_CUDA_OK(cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int)));
  *out = v;
  return HEXB_OK;
}

}  // namespace hexb
