// Head-row operators of a serving step: per-head RMS norm with the rotary embedding in the same pass
// (hexb_qk_norm_rope), and the store of new keys and values into a paged cache with that norm and rotation
// applied on the way (hexb_kv_cache_append).
//
// Both walk rows of D elements, one per (token, head):
//   y = R(pos) . (x * rsqrt(mean(x^2) + eps) * w)
// R(pos) turns the pair p of the first rotary_dim elements by pos * theta^(-2p / rotary_dim); a pair is
// (2p, 2p + 1) when interleaved -- the convention of rope_kernel (test/python/triton/test_rope.py:98-190) --
// and (p, p + rotary_dim / 2) otherwise.  The norm is that of rms_norm_fwd_kernel
// (test/python/triton/test_rms_norm.py:37-63) on one head.  fp32 arithmetic, one rounding at the store.
//
// Every element is read once and written once: the bound is the memory traffic, and for a decode step's few
// rows the latency of one dependent load.  A row is held by a group of lanes (16 bytes a lane), so the mean
// is a few shuffles; the sines and cosines depend on (token, pair) only and are formed once for all heads that a group
// of lanes walks (in the fallback for odd sizes: once per CTA, in shared memory).
//
// The angle of a far position: a 32-bit product of position and frequency is off by up to 2^-24 * 130000 = 0.008 rad
// at position 130000, so it is formed in 64-bit fixed point and rounded to 32 bits as a fraction of a turn.
#include <cmath>

#include "common.cuh"

namespace hexb {

static __device__ int g_heads_status = 0;

namespace heads {

constexpr int THREADS = 128;
constexpr int AHEAD = 4;         // rows a group of lanes has under way
constexpr int kPowerBits = 11;   // rotary_dim <= 4096

// One of the two tensors a call walks (queries and keys, or keys and values).
struct Segment {
  const void *src;
  void *dst;
  const void *weight;         // gains of the norm, or NULL for ones
  int64_t src_t, src_h;       // element strides
  int64_t dst_t, dst_h;       // rows addressed by token (qk_norm_rope), or by cache slot: dst_p page, dst_t slot in page
  int64_t dst_p;
  int heads;
  int norm, rotate;
};

struct Params {
  Segment seg[2];
  const int64_t *positions;
  const int64_t *slots;       // NULL: destination rows follow the tokens
  int64_t tokens, num_slots, page_size;
  int D, rot, interleaved;
  int tokens_per_cta, gpt_shift;   // groups of lanes a token has: 1 << gpt_shift
  float eps;
  uint64_t power[kPowerBits];
};

// Angles are fractions of a turn in 64-bit fixed point: 2^64 is one turn, a product with the position wraps as an angle
// does, and no chain of 64-bit floating-point operations delays the first row of a CTA.  The frequency of pair p is
// 2^64 / (2 pi) * theta^(-2p / rotary_dim): the product of the powers theta^(-2^(b+1) / rotary_dim) over the bits b of p,
// which the host forms in 64-bit floating point (2^63 is 1).  A power is off by a relative 2^-52, on a frequency of at most
// 0.16 turn a position: 11 of them 2^-51 of a turn.  Their truncation to integers and that of the products add at most 3
// units of 2^-64 of a turn each, whatever is left of the frequency: 2^-58.  So the angle at position n is good to n * 2^-50.
__device__ __forceinline__ uint64_t frequency(const Params &p, int pr) {
  uint64_t f = 2935890503282001226ull;  // 2^64 / (2 pi)
#pragma unroll
  for (int b = 0; b < kPowerBits; ++b) {
    if ((p.rot - 1) >> (b + 1) == 0) break;
    const uint64_t g = __umul64hi(f, p.power[b]) << 1;
    f = pr >> b & 1 ? g : f;
  }
  return f;
}
__host__ __device__ constexpr int ring_bytes(int nv) { return AHEAD * nv * THREADS * 16; }
__device__ __forceinline__ void copy16_async(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

// cos and sin of pos * frequency
__device__ __forceinline__ float2 turn(int64_t pos, uint64_t freq) {
  const int32_t t = (int32_t)(((uint64_t)pos * freq) >> 32);
  float sn, cs;
  sincospif((float)t * 4.656612873077393e-10f, &sn, &cs);  // 2^-31: half turns
  return make_float2(cs, sn);
}

// Destination row of (token, head), or NULL when the token has no slot.
template <typename T>
__device__ __forceinline__ T *dst_row(const Segment &s, const Params &p, int64_t token, int64_t slot, int head) {
  T *base = static_cast<T *>(s.dst) + (int64_t)head * s.dst_h;
  if (!p.slots) return base + token * s.dst_t;
  if (slot < 0) return nullptr;
  const int64_t page = (slot >> 32) == 0 ? (uint32_t)slot / (uint32_t)p.page_size : slot / p.page_size;
  return base + page * s.dst_p + (slot - page * p.page_size) * s.dst_t;
}

// A slot outside the cache stores nothing and is recorded; negative slots are padding.
__device__ __forceinline__ int64_t load_slot(const Params &p, int64_t token) {
  int64_t slot = p.slots[token];
  if (slot >= p.num_slots) {
    atomicExch(&g_heads_status, (int)HEXB_ERR_BAD_ARG);
    slot = -1;
  }
  return slot;
}

// Vector form.  LPR lanes hold one row, NV 16-byte vectors each (vector v sits in lane v % LPR, register v / LPR).
// A CTA takes tokens_per_cta tokens; a token's heads (of both tensors, in one row) are dealt to 1 << gpt_shift groups
// of lanes.  Instruction issue bounds a kernel that forms addresses and rotation anew for each row (46 M warp instructions,
// 86 us for the append below, now 14 M, where the traffic takes 21 us), so what the rows of a group share is set up
// once: the addresses advance by a constant, and the linear map of a row
//   y_e = rstd * (A_e x_e + B_e x_partner(e)),   A = w cos,  B = -+ w_partner sin
// sits in registers -- two fused operations an element besides the mean.  AHEAD rows of a group are under way, the first
// before the angles are computed.  The code is kept to one copy of each step: with few tokens the time is that of
// fetching it.  8192 tokens of 16 + 4 heads of 128 (84 MB): 19 us, 4.4 TB/s; append of 16400 tokens of 8 heads (134 MB):
// 30 us, 4.5 TB/s; one token: 4.3 us back to back.  Held in registers, one row ahead, they took 26 and 37 us: 20 KB
// under way on an SM do not cover the latency of memory.  Four CTAs an SM without spills beat five with (22 against 25 us).
template <typename T, int LPR, int NV>
__global__ void __launch_bounds__(THREADS, 4)
head_rows_kernel(const Params p) {
  constexpr int E = Vec16<T>::N;
  using Raw = decltype(Vec16<T>::raw);
  // cos, sin of pair (v, e) of vector v at [token][e][v]: the lanes of a row read consecutive words
  extern __shared__ __align__(16) uint8_t s_dyn[];
  float2 *const s_cs = reinterpret_cast<float2 *>(s_dyn + ring_bytes(NV));
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int nvec = p.D / E, half = p.rot / 2, rotv = p.rot / E, hv = half / E;
  const bool inter = p.interleaved != 0;
  const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
  const int gs = p.gpt_shift, gpt = 1 << gs;
  const int t = grp >> gs, h0 = grp & (gpt - 1), h1 = (h0 - p.seg[0].heads) & (gpt - 1);
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_cta, tok = t0 + t;
  const int nt = (int)min((int64_t)p.tokens_per_cta, p.tokens - t0);
  const int pairs_v = inter ? E / 2 : E, width = half / pairs_v, plane = pairs_v * width;
  const int n0 = t < nt && h0 < p.seg[0].heads ? (p.seg[0].heads - h0 + gpt - 1) >> gs : 0;
  const int n1 = t < nt && h1 < p.seg[1].heads ? (p.seg[1].heads - h1 + gpt - 1) >> gs : 0;
  pdl_wait();

  const T *src = static_cast<const T *>(p.seg[0].src) + tok * p.seg[0].src_t + (int64_t)h0 * p.seg[0].src_h + lane * E;
  const T *src1 = static_cast<const T *>(p.seg[1].src) + tok * p.seg[1].src_t + (int64_t)h1 * p.seg[1].src_h + lane * E;
  // Rows travel through shared memory, each lane's 16-byte pieces into places of its own: no barrier, and the rows under
  // way cost no registers.
  uint4 *const ring = reinterpret_cast<uint4 *>(s_dyn) + threadIdx.x;     // [AHEAD][NV][THREADS]
  auto request = [&](int n) {
    if (n < n0 + n1) {
      if (n == n0) src = src1;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + i * LPR < nvec) copy16_async(ring + ((n % AHEAD) * NV + i) * THREADS, src + i * LPR * E);
      src += p.seg[n >= n0].src_h << gs;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int n = 0; n < AHEAD; ++n) request(n);
  // the gains are needed after the angles: their fetch overlaps that of the positions (one token: 6.7 -> 6.2 us)
  if (threadIdx.x < 2 * LPR * NV) {
    const int g = threadIdx.x >= LPR * NV, v = threadIdx.x - g * LPR * NV;
    const Segment &s = p.seg[g];
    if (s.norm && s.weight && v < nvec)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const T *>(s.weight) + v * E));
  }
  const int64_t slot = p.slots && t < nt ? load_slot(p, tok) : 0;
  if (p.rot) {
    // a thread keeps its pair and steps over tokens while the pairs are fewer than the threads
    const int lanes = half < THREADS ? THREADS / half * half : THREADS;
    for (int pr = threadIdx.x < lanes ? threadIdx.x % half : half; pr < half; pr += THREADS) {
      const uint64_t fq = frequency(p, pr);
      for (int ti = threadIdx.x / half; ti < nt; ti += max(1, lanes / half))
        s_cs[ti * plane + pr % pairs_v * width + pr / pairs_v] = turn(p.positions[t0 + ti], fq);
    }
    __syncthreads();
  }
  const float2 *cs = s_cs + t * plane;
  const float inv_d = 1.0f / (float)p.D;

  float A[NV][E], B[NV][E];
  T *dst = nullptr;
  bool norm = false, rotate = false;
  int64_t dst_step = 0;
#pragma unroll 1
  for (int n = 0; n < n0 + n1; ++n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
    Raw raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i] = Raw{};
      if (lane + i * LPR < nvec) {
        const uint4 v = ring[((n % AHEAD) * NV + i) * THREADS];
        raw[i] = *reinterpret_cast<const Raw *>(&v);
      }
    }
    request(n + AHEAD);
    if (n == 0 || n == n0) {
      const int g = n >= n0;
      const Segment &s = p.seg[g];
      norm = s.norm;
      rotate = s.rotate;
      dst_step = s.dst_h << gs;
      dst = dst_row<T>(s, p, tok, slot, g ? h1 : h0);
      if (!dst) dst_step = 0;
      else dst += lane * E;
      const Raw *w = norm ? static_cast<const Raw *>(s.weight) : nullptr;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * LPR;
        const int pv = inter ? v : v < hv ? v + hv : v - hv;
        const bool turned = rotate && v < rotv;
        float wp[E];
#pragma unroll
        for (int e = 0; e < E; ++e) A[i][e] = wp[e] = 1.0f;
        if (w && v < nvec) {
          Vec16<T> x;
          x.raw = w[v];
          x.unpack(A[i]);
          if (turned) x.raw = w[pv];
          x.unpack(wp);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float sign = (inter ? (e & 1) == 0 : v < hv) ? -1.0f : 1.0f;
          float2 c = make_float2(1.0f, 0.0f);
          if (turned) c = cs[inter ? e / 2 * width + v : e * width + min(v, pv)];
          A[i][e] *= c.x;
          B[i][e] = sign * (inter ? wp[e ^ 1] : wp[e]) * c.y;
        }
      }
    }
    if (!norm && !rotate) {  // values: the bits as they are
      if (dst) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + i * LPR < nvec) st_stream_as<Raw>(dst + i * LPR * E, raw[i]);
      }
    } else {
      float f[NV][E], o[NV][E];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Vec16<T> x;
        x.raw = raw[i];
        x.unpack(f[i]);
      }
      if (inter) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) o[i][e] = f[i][e ^ 1];
      } else if (hv == LPR) {
        // a lane holds both vectors of its pairs (the whole of a row of LPR * NV vectors is rotated)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) o[i][e] = f[NV - 1 - i][e];
      } else {
        // the partner of vector v is v + hv (first half) or v - hv (second half)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = lane + i * LPR;
          const int pv = v < hv ? v + hv : v - hv;
          const int pl = pv & (LPR - 1), pi = pv / LPR;
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            w[q] = __shfl_sync(mask, reinterpret_cast<const uint32_t *>(&raw[0])[q], pl, LPR);
            const uint32_t w1 = __shfl_sync(mask, reinterpret_cast<const uint32_t *>(&raw[NV - 1])[q], pl, LPR);
            w[q] = pi ? w1 : w[q];
          }
          Vec16<T> x;
          x.raw = *reinterpret_cast<const Raw *>(w);
          x.unpack(o[i]);
        }
      }
      float rstd = 1.0f;
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) ss = fmaf(f[i][e], f[i][e], ss);
#pragma unroll
        for (int k = LPR / 2; k > 0; k >>= 1) ss += __shfl_xor_sync(mask, ss, k);
        rstd = rsqrtf(fmaf(ss, inv_d, p.eps));
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * LPR;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float y = f[i][e] * A[i][e];
          // elements that are not rotated have no partner
          f[i][e] = rstd * (rotate && v < rotv ? fmaf(o[i][e], B[i][e], y) : y);
        }
        if (dst && v < nvec) {
          Vec16<T> x;
          x.pack(f[i]);
          st_stream_as<Raw>(dst + i * LPR * E, x.raw);
        }
      }
    }
    dst += dst_step;
  }
  pdl_launch_dependents();
}

// Element-wise form for rows that cannot be read in 16-byte vectors (odd sizes, strides or addresses): one
// warp per row.  The mean is complete before the first store, and a pair is read and written by one lane, so
// the output may be the input here too.
template <typename T>
__global__ void __launch_bounds__(THREADS)
head_rows_scalar_kernel(const Params p) {
  const int lane = threadIdx.x & 31;
  const int heads = p.seg[0].heads + p.seg[1].heads;
  const int64_t rows = p.tokens * heads, step = (int64_t)gridDim.x * (THREADS / 32);
  const int half = p.rot / 2;
  pdl_wait();
  for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); r < rows; r += step) {
    const int64_t t = r / heads;
    int h = (int)(r - t * heads);
    const int g = h >= p.seg[0].heads;
    if (g) h -= p.seg[0].heads;
    const Segment &s = p.seg[g];
    const T *src = static_cast<const T *>(s.src) + t * s.src_t + (int64_t)h * s.src_h;
    float rstd = 1.f;
    if (s.norm) {
      float ss = 0.f;
      for (int d = lane; d < p.D; d += 32) {
        const float x = to_f32<T>(src[d]);
        ss = fmaf(x, x, ss);
      }
      rstd = rsqrtf(warp_sum(ss) / (float)p.D + p.eps);
    }
    T *dst = dst_row<T>(s, p, t, p.slots ? load_slot(p, t) : 0, h);
    if (!dst) continue;
    const T *w = s.norm ? static_cast<const T *>(s.weight) : nullptr;
    const int nrot = s.rotate ? half : 0;
    auto at = [&](int d) { return to_f32<T>(src[d]) * (w ? rstd * to_f32<T>(w[d]) : rstd); };
    for (int pr = lane; pr < nrot; pr += 32) {
      const int i = p.interleaved ? 2 * pr : pr, j = p.interleaved ? 2 * pr + 1 : pr + half;
      const float2 c = turn(p.positions[t], frequency(p, pr));
      const float a = at(i), b = at(j);
      dst[i] = from_f32<T>(a * c.x - b * c.y);
      dst[j] = from_f32<T>(a * c.y + b * c.x);
    }
    for (int d = 2 * nrot + lane; d < p.D; d += 32) dst[d] = from_f32<T>(at(d));
  }
  pdl_launch_dependents();
}

template <typename T>
static bool vector_ok(const Params &p) {
  constexpr int E = Vec16<T>::N;
  if (p.D % E || p.D > 256 || p.rot % (p.interleaved ? E : 2 * E)) return false;
  for (const Segment &s : p.seg) {
    if (!s.heads) continue;
    if (!aligned16(s.src) || !aligned16(s.dst) || (s.weight && !aligned16(s.weight))) return false;
    if (s.src_t % E || s.src_h % E || s.dst_t % E || s.dst_h % E || s.dst_p % E) return false;
  }
  return true;
}

template <typename T, int LPR, int NV>
static cudaError_t launch_vec(const Params &p, dim3 grid, size_t smem, cudaStream_t st) {
  return launch_pdl(head_rows_kernel<T, LPR, NV>, grid, dim3(THREADS), smem, st, p);
}

template <typename T>
static int launch(Params p, float theta, cudaStream_t st) {
  DeviceInfo di;
  if (int e = current_device(&di)) return e;
  for (int b = 0; b < kPowerBits && (p.rot >> (b + 1)); ++b) {
    const double v = ldexp(pow((double)theta, -ldexp(2.0, b) / p.rot), 63);
    p.power[b] = v < 9223372036854775808.0 ? (uint64_t)v : 1ull << 63;
  }
  if (!vector_ok<T>(p)) {
    const int64_t warps = p.tokens * (p.seg[0].heads + p.seg[1].heads), want = (warps + 7) / 8, cap = (int64_t)di.sm_count * 32;
    HEXB_CUDA_OK(launch_pdl(head_rows_scalar_kernel<T>, dim3((unsigned)(want < cap ? want : cap)), dim3(THREADS), 0, st, p));
    return check_launch("head_rows_scalar");
  }
  constexpr int E = Vec16<T>::N;
  const int nvec = p.D / E;
  const int lpr = nvec <= 8 ? 4 : nvec <= 16 ? 8 : nvec <= 32 ? 16 : 32;   // two vectors a lane
  const int rp = THREADS / lpr;
  // Tokens per CTA: so many that a group of lanes gets sixteen of a token's heads (the map is
  // built for them once: with four, 27 us for the 8192 tokens), but no fewer CTAs than two an SM.
  int tb = 1;
  while (tb < rp && rp / tb * 16 > p.seg[0].heads) tb *= 2;
  while (tb > 1 && (p.tokens + tb - 1) / tb < 2 * (int64_t)di.sm_count) tb /= 2;
  p.tokens_per_cta = tb;
  for (p.gpt_shift = 0; (tb << (p.gpt_shift + 1)) <= rp;) ++p.gpt_shift;
  const int64_t gx = (p.tokens + tb - 1) / tb;
  if (gx > 0x7fffffff) return HEXB_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx);
  const size_t smem = ring_bytes(2) + (size_t)tb * (p.rot / 2) * sizeof(float2);
  cudaError_t e;
  if (lpr == 4) e = launch_vec<T, 4, 2>(p, grid, smem, st);
  else if (lpr == 8) e = launch_vec<T, 8, 2>(p, grid, smem, st);
  else if (lpr == 16) e = launch_vec<T, 16, 2>(p, grid, smem, st);
  else e = launch_vec<T, 32, 2>(p, grid, smem, st);
  HEXB_CUDA_OK(e);
  return check_launch("head_rows");
}

static int dispatch(int dtype, const Params &p, float theta, void *stream) {
  if (dtype == HEXB_DT_F16) return launch<__half>(p, theta, (cudaStream_t)stream);
  return launch<float>(p, theta, (cudaStream_t)stream);
}

}  // namespace heads

int heads_device_status_fetch_and_clear(int *out) {
  int v = 0, zero = 0;
  HEXB_CUDA_OK(cudaMemcpyFromSymbol(&v, g_heads_status, sizeof(int)));
  if (v) HEXB_CUDA_OK(cudaMemcpyToSymbol(g_heads_status, &zero, sizeof(int)));
  *out = v;
  return HEXB_OK;
}

}  // namespace hexb

using namespace hexb;

extern "C" int hexb_qk_norm_rope(int dtype, const void *q, const void *k, void *q_out, void *k_out,
                                 const int64_t *positions, const void *q_weight, const void *k_weight, int64_t tokens,
                                 int64_t q_heads, int64_t kv_heads, int64_t D, const int64_t *strides, int rotary_dim,
                                 int interleaved, float theta, float eps, void *stream) {
  if (dtype != HEXB_DT_F16 && dtype != HEXB_DT_F32) return HEXB_ERR_UNSUPPORTED;
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || D < 0 || rotary_dim < 0 || rotary_dim > D || rotary_dim % 2)
    return HEXB_ERR_BAD_ARG;
  if (tokens == 0 || D == 0 || q_heads + kv_heads == 0) return HEXB_OK;
  if (!strides || (q_heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)) || (rotary_dim && !positions) ||
      !(theta >= 1.f))
    return HEXB_ERR_BAD_ARG;
  if (D > 4096 || q_heads + kv_heads > 65535) return HEXB_ERR_UNSUPPORTED;
  heads::Params p = {};
  p.seg[0] = {q, q_out, q_weight, strides[0], strides[1], strides[4], strides[5], 0, (int)q_heads, 1, rotary_dim > 0};
  p.seg[1] = {k, k_out, k_weight, strides[2], strides[3], strides[6], strides[7], 0, (int)kv_heads, 1, rotary_dim > 0};
  p.positions = positions;
  p.tokens = tokens;
  p.D = (int)D;
  p.rot = rotary_dim;
  p.interleaved = interleaved != 0;
  p.eps = eps;
  return heads::dispatch(dtype, p, theta, stream);
}

extern "C" int hexb_kv_cache_append(int dtype, const void *k, const void *v, void *k_cache, void *v_cache,
                                    const int64_t *slots, const int64_t *positions, const void *k_weight, int64_t tokens,
                                    int64_t kv_heads, int64_t D, int64_t num_pages, int64_t page_size,
                                    const int64_t *strides, int k_norm, int rotary_dim, int interleaved, float theta,
                                    float eps, void *stream) {
  if (dtype != HEXB_DT_F16 && dtype != HEXB_DT_F32) return HEXB_ERR_UNSUPPORTED;
  if (tokens < 0 || kv_heads < 0 || D < 0 || num_pages < 0 || page_size < 0 || rotary_dim < 0 || rotary_dim > D ||
      rotary_dim % 2)
    return HEXB_ERR_BAD_ARG;
  if (tokens == 0 || kv_heads == 0 || D == 0) return HEXB_OK;
  if (!strides || !k || !v || !k_cache || !v_cache || !slots || (rotary_dim && !positions) || !(theta >= 1.f) ||
      page_size == 0)
    return HEXB_ERR_BAD_ARG;
  if (D > 4096 || kv_heads > 32767 || page_size > 0x7fffffff ||
      num_pages > INT64_MAX / page_size) return HEXB_ERR_UNSUPPORTED;
  heads::Params p = {};
  p.seg[0] = {k, k_cache, k_weight, strides[0], strides[1], strides[5], strides[6], strides[4], (int)kv_heads,
              k_norm != 0, rotary_dim > 0};
  p.seg[1] = {v, v_cache, nullptr, strides[2], strides[3], strides[8], strides[9], strides[7], (int)kv_heads, 0, 0};
  p.positions = positions;
  p.slots = slots;
  p.tokens = tokens;
  p.num_slots = num_pages * page_size;
  p.page_size = page_size;
  p.D = (int)D;
  p.rot = rotary_dim;
  p.interleaved = interleaved != 0;
  p.eps = eps;
  return heads::dispatch(dtype, p, theta, stream);
}
