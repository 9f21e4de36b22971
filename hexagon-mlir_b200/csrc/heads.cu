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
// is a few shuffles; the sines and cosines depend on (token, pair) only and are computed once per CTA
// into shared memory, then used by all heads of its tokens.
//
// The angle of a far position: pos * frequency is formed in 64 bits and reduced to a fraction of a turn before
// it is rounded to 32 (at position 130000 a 32-bit product is off by up to 2^-24 * 130000 = 0.008 rad); the
// frequencies, in turns, come as 64-bit kernel parameters computed by the host.
#include <cmath>

#include "common.cuh"

namespace hexb {

static __device__ int g_heads_status = 0;

namespace heads {

constexpr int kMaxPairs = 256;  // rotary_dim <= 512: the frequency table travels as a kernel parameter
constexpr int THREADS = 256;

struct Freqs {
  double turns[kMaxPairs];  // theta^(-2p / rotary_dim) / (2 pi)
};

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
  int tokens_per_cta, rows_per_split;
  float eps;
};

// cos and sin of pos * frequency
__device__ __forceinline__ float2 turn(int64_t pos, double freq_turns) {
  double t = (double)pos * freq_turns;
  t -= rint(t);
  float sn, cs;
  sincospif(2.0f * (float)t, &sn, &cs);
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

// Vector form.  LPR lanes hold one row, NV 16-byte vectors each (vector v sits in lane v % LPR, register
// v / LPR).  grid.x: blocks of tokens_per_cta tokens; grid.y: splits of a token's rows (few tokens only).
template <typename T, int LPR, int NV>
__global__ void __launch_bounds__(THREADS)
head_rows_kernel(const Params p, const __grid_constant__ Freqs fr) {
  constexpr int E = Vec16<T>::N;
  using Raw = decltype(Vec16<T>::raw);
  constexpr int RP = THREADS / LPR;  // rows at a time
  extern __shared__ float2 s_cs[];   // [tokens_per_cta][rot / 2]
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int nvec = p.D / E, half = p.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int nt = (int)min((int64_t)p.tokens_per_cta, p.tokens - t0);
  const int heads = p.seg[0].heads + p.seg[1].heads;
  const int r_lo = (int)blockIdx.y * p.rows_per_split;
  const int r_hi = min(r_lo + p.rows_per_split, nt * heads);
  pdl_wait();
  if (p.rot) {
    for (int i = threadIdx.x; i < nt * half; i += THREADS) {
      const int t = i / half, pr = i - t * half;
      s_cs[i] = turn(p.positions[t0 + t], fr.turns[pr]);
    }
  }
  // gains of this lane's columns
  Raw w[2][NV];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * LPR;
      if (p.seg[g].norm && p.seg[g].weight && v < nvec)
        w[g][i] = *(reinterpret_cast<const Raw *>(p.seg[g].weight) + v);
    }
  __syncthreads();
  const float inv_d = 1.0f / (float)p.D;
  for (int r = r_lo + grp; r < r_hi; r += RP) {
    const int t = r / heads;
    int h = r - t * heads;
    const int g = h >= p.seg[0].heads;
    if (g) h -= p.seg[0].heads;
    const Segment &s = p.seg[g];
    const int64_t slot = p.slots ? load_slot(p, t0 + t) : 0;
    const T *src = static_cast<const T *>(s.src) + (t0 + t) * s.src_t + (int64_t)h * s.src_h;
    float f[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * LPR;
      if (v < nvec) {
        Vec16<T> x;
        x.raw = ld_stream_as<Raw>(src + v * E);
        x.unpack(f[i]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] = 0.f;
      }
    }
    // lanes of one row take the same branches: a group of LPR lanes shares (t, h)
    const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u) << ((threadIdx.x & 31) / LPR * LPR);
    if (s.norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) ss = fmaf(f[i][e], f[i][e], ss);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float rstd = rsqrtf(fmaf(ss, inv_d, p.eps));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float wf[E];
        if (s.weight) {
          Vec16<T> x;
          x.raw = g ? w[1][i] : w[0][i];
          x.unpack(wf);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) f[i][e] *= s.weight ? rstd * wf[e] : rstd;
      }
    }
    if (s.rotate) {
      const float2 *cs = s_cs + t * half;
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int p0 = (lane + i * LPR) * (E / 2);
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            if (p0 + e < half) {
              const float2 c = cs[p0 + e];
              const float a = f[i][2 * e], b = f[i][2 * e + 1];
              f[i][2 * e] = a * c.x - b * c.y;
              f[i][2 * e + 1] = a * c.y + b * c.x;
            }
          }
        }
      } else {
        // the partner of vector v is v + half / E (first half) or v - half / E (second half)
        const int hv = half / E;
        float o[NV][E];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = lane + i * LPR;
          const int pv = v < hv ? v + hv : v - hv;
          const int pl = pv & (LPR - 1), pi = pv / LPR;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            float q = __shfl_sync(mask, f[0][e], pl, LPR);
            if (NV > 1) {
              const float q1 = __shfl_sync(mask, f[NV - 1][e], pl, LPR);
              q = pi ? q1 : q;
            }
            o[i][e] = q;
          }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = lane + i * LPR;
          if (v < 2 * hv) {
            const bool first = v < hv;
            const int p0 = (first ? v : v - hv) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float2 c = cs[p0 + e];
              f[i][e] = first ? f[i][e] * c.x - o[i][e] * c.y : f[i][e] * c.x + o[i][e] * c.y;
            }
          }
        }
      }
    }
    T *dst = dst_row<T>(s, p, t0 + t, slot, h);
    if (dst) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * LPR;
        if (v < nvec) {
          Vec16<T> x;
          x.pack(f[i]);
          st_stream_as<Raw>(dst + v * E, x.raw);
        }
      }
    }
  }
  pdl_launch_dependents();
}

// Element-wise form for rows that cannot be read in 16-byte vectors (odd sizes, strides or addresses): one
// warp per row.  The mean is complete before the first store, and a pair is read and written by one lane, so
// the output may be the input here too.
template <typename T>
__global__ void __launch_bounds__(THREADS)
head_rows_scalar_kernel(const Params p, const __grid_constant__ Freqs fr) {
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
      const float2 c = turn(p.positions[t], fr.turns[pr]);
      const float a = at(i), b = at(j);
      dst[i] = from_f32<T>(a * c.x - b * c.y);
      dst[j] = from_f32<T>(a * c.y + b * c.x);
    }
    for (int d = 2 * nrot + lane; d < p.D; d += 32) dst[d] = from_f32<T>(at(d));
  }
  pdl_launch_dependents();
}

// Frequencies in turns; the table of the last (theta, rotary_dim) is kept per host thread.
static const Freqs &freqs(float theta, int rot) {
  static thread_local Freqs f;
  static thread_local float f_theta = 0.f;
  static thread_local int f_rot = -1;
  if (f_rot != rot || f_theta != theta) {
    for (int i = 0; i < kMaxPairs; ++i)
      f.turns[i] = i < rot / 2 ? pow((double)theta, -2.0 * i / rot) / 6.283185307179586476925 : 0.0;
    f_rot = rot;
    f_theta = theta;
  }
  return f;
}

template <typename T>
static bool vector_ok(const Params &p) {
  constexpr int E = Vec16<T>::N;
  if (p.D % E || p.D > 256 || (!p.interleaved && p.rot % (2 * E))) return false;
  for (const Segment &s : p.seg) {
    if (!s.heads) continue;
    if (!aligned16(s.src) || !aligned16(s.dst) || (s.weight && !aligned16(s.weight))) return false;
    if (s.src_t % E || s.src_h % E || s.dst_t % E || s.dst_h % E || s.dst_p % E) return false;
  }
  return true;
}

template <typename T, int LPR, int NV>
static cudaError_t launch_vec(const Params &p, const Freqs &fr, dim3 grid, size_t smem, cudaStream_t st) {
  return launch_pdl(head_rows_kernel<T, LPR, NV>, grid, dim3(THREADS), smem, st, p, fr);
}

template <typename T>
static int launch(Params p, float theta, cudaStream_t st) {
  DeviceInfo di;
  if (int e = current_device(&di)) return e;
  const Freqs &fr = freqs(theta, p.rot);
  const int heads = p.seg[0].heads + p.seg[1].heads;
  if (!vector_ok<T>(p)) {
    const int64_t warps = p.tokens * heads, want = (warps + 7) / 8, cap = (int64_t)di.sm_count * 32;
    HEXB_CUDA_OK(launch_pdl(head_rows_scalar_kernel<T>, dim3((unsigned)(want < cap ? want : cap)), dim3(THREADS), 0, st, p, fr));
    return check_launch("head_rows_scalar");
  }
  constexpr int E = Vec16<T>::N;
  const int nvec = p.D / E;
  const int lpr = nvec <= 8 ? 8 : nvec <= 16 ? 16 : 32;
  const int rp = THREADS / lpr;
  // Enough tokens per CTA for four rounds of rows, so that the angles are shared by many rows; a step with few
  // tokens is cut over its rows instead, one round per CTA.
  int tb = 4 * rp / heads;
  const int64_t spread = p.tokens / ((int64_t)di.sm_count * 4);
  if (tb > spread) tb = (int)spread;
  if (tb > 16) tb = 16;
  if (tb < 1) tb = 1;
  p.tokens_per_cta = tb;
  int splits = 1;
  if (tb == 1 && p.tokens < di.sm_count * 4) splits = (heads + rp - 1) / rp;
  p.rows_per_split = (tb * heads + splits - 1) / splits;
  const int64_t gx = (p.tokens + tb - 1) / tb;
  if (gx > 0x7fffffff || splits > 65535) return HEXB_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)gx, (unsigned)splits);
  const size_t smem = (size_t)tb * (p.rot / 2) * sizeof(float2);
  cudaError_t e;
  if (lpr == 8) e = launch_vec<T, 8, 1>(p, fr, grid, smem, st);
  else if (lpr == 16) e = launch_vec<T, 16, 1>(p, fr, grid, smem, st);
  else if (nvec <= 32) e = launch_vec<T, 32, 1>(p, fr, grid, smem, st);
  else e = launch_vec<T, 32, 2>(p, fr, grid, smem, st);
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
      !(theta > 0.f))
    return HEXB_ERR_BAD_ARG;
  if (D > 4096 || rotary_dim > 2 * heads::kMaxPairs || q_heads + kv_heads > 65535) return HEXB_ERR_UNSUPPORTED;
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
  if (!strides || !k || !v || !k_cache || !v_cache || !slots || (rotary_dim && !positions) || !(theta > 0.f) ||
      page_size == 0)
    return HEXB_ERR_BAD_ARG;
  if (D > 4096 || rotary_dim > 2 * heads::kMaxPairs || kv_heads > 32767 || page_size > 0x7fffffff ||
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
