// Token sampling: one token per row of logits, from a given uniform random number.
//
//   w_i = exp((x_i - max x) / T)                      T <= 0: the largest logit, lowest index
//   top-k   keeps the k largest logits
//   top-p   of those, in descending order, every one before which less than p of their mass lies
//   min-p   of those, the ones with w_i >= min_p
//   token   the first kept index, in index order, whose inclusive sum of w exceeds u times the kept sum
//
// Ties are ordered by index everywhere (the lower one first).  Drawing in index order needs no sort: each filter
// is a cut (key, index) in the descending order, found by histograms.  NaN and -inf are never chosen; a row
// with nothing else gives -1.
//
// A token is a whole number, so borders decide: weights are formed in 64 bits, and sums are 64-bit sums or exact
// integers (44 bits of the mass; two 32-bit shared-memory atomics a logit), so the result does not
// depend on the order of the atomics.
//
// One cluster of C CTAs owns a row: each CTA reads its slice once into shared memory and all passes run there;
// the CTAs exchange maxima, sums and histograms through distributed shared memory.  A slice that does not fit
// is read again from L2 by each pass.
#include "tc_sm100.cuh"

namespace hexb {
namespace sampling {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int NB = 2048;           // histogram bins
constexpr int MAXC = 8;
constexpr int VEC = 4;             // elements a lane takes at a time

struct Params {
  const void *x;
  const float *u;
  int64_t *out;
  const float *temperature, *top_p, *min_p;   // per row, or NULL: the scalar
  const int *top_k;
  float temperature0, top_p0, min_p0;
  int top_k0;
  int64_t row_stride;
  int V, slice, resident;
};

// Order-preserving integer of a float (no NaN; -0 counts as +0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// 2^y for y <= 0 in 64 bits: y = n + f, |f| <= 1/2, Taylor series of e^(f ln 2) (degree 11: the first term left
// out is below 0.3466^12 / 12! = 7e-15), exponent added as an integer.  Below 2^-1000: 0.
__device__ __forceinline__ double exp2_neg(double y) {
  if (!(y > -1000.0)) return 0.0;
  const double n = rint(y);
  const double f = (y - n) * 0.693147180559945309417;
  double r = 1.0 / 39916800.0;
  r = fma(r, f, 1.0 / 3628800.0);
  r = fma(r, f, 1.0 / 362880.0);
  r = fma(r, f, 1.0 / 40320.0);
  r = fma(r, f, 1.0 / 5040.0);
  r = fma(r, f, 1.0 / 720.0);
  r = fma(r, f, 1.0 / 120.0);
  r = fma(r, f, 1.0 / 24.0);
  r = fma(r, f, 1.0 / 6.0);
  r = fma(r, f, 0.5);
  r = fma(r, f, 1.0);
  r = fma(r, f, 1.0);
  return __longlong_as_double(__double_as_longlong(r) + ((long long)n << 52));
}

// What is kept so far: keys above `key`, and of those equal to it the indices up to `index`.
struct Cut {
  uint32_t key;
  int index;
};

struct Shared {
  uint32_t count[NB], hi[NB], lo[NB];
  double warp_sum[WARPS];
  double part[2][MAXC];             // this CTA's column of each exchange is [..][rank] of every CTA
  float fmax[MAXC], fmin[MAXC];
  int imin[MAXC];
  int found_index;
  unsigned long long scan[WARPS];
  int bin;
  unsigned long long before;
  uint32_t bin_count;
  int winner;
  double rel;
};

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T, int C>
struct Row {
  const Params &p;
  Shared &s;
  const T *data;          // the slice: shared memory, or global
  int n, rank, warp, lane;
  int w0, w1;             // this warp's contiguous part of the slice
  int first;              // row index of slice element 0
  float m;
  double inv_t;           // log2(e) / T
  int flip;

  __device__ Row(const Params &p_, Shared &s_) : p(p_), s(s_), flip(0) {}

  __device__ __forceinline__ void cluster_barrier() {
    if (C > 1) tc::cluster_sync_all();
    else __syncthreads();
  }
  __device__ __forceinline__ uint32_t peer(const void *a, int r) {
    const uint32_t l = tc::smem_u32(a);
    return C > 1 ? tc::map_to_rank(l, (uint32_t)r) : l;
  }
  __device__ __forceinline__ float at(int i) const {
    const float v = to_f32<T>(data[i]);
    return v != v ? -INFINITY : v;
  }
  __device__ __forceinline__ double weight(float v) const {
    return v == m ? 1.0 : exp2_neg(((double)v - (double)m) * inv_t);
  }
  __device__ __forceinline__ bool kept(const Cut &c, float v, int i) const {
    const uint32_t k = key_of(v);
    return v > -INFINITY && (k > c.key || (k == c.key && i <= c.index));
  }
  // f(value, row index) for every element of this warp's part
  template <typename F>
  __device__ __forceinline__ void each(F &&f) {
#pragma unroll 4
    for (int i = w0 + lane; i < w1; i += 32) f(at(i), first + i);
  }

  // Sum of one 64-bit value per thread over the cluster: lanes, warps in order, CTAs in order.  Also leaves the
  // warp sums of this CTA in s.warp_sum and the CTA sums in `cta`.
  __device__ double cluster_total(double v, double (&cta)[C]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = v;
    __syncthreads();
    if (threadIdx.x < C) {
      double t = 0.0;
      for (int w = 0; w < WARPS; ++w) t += s.warp_sum[w];
      st_cluster_f64(peer(&s.part[flip][rank], threadIdx.x), t);
    }
    cluster_barrier();
    double total = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      cta[r] = s.part[flip][r];
      total += cta[r];
    }
    flip ^= 1;  // a CTA can be one exchange ahead of its peers, not two
    return total;
  }

  // Lowest row index at which the inclusive sum of f exceeds target(total); -1 if the sum is empty.  The CTA
  // that holds it returns it, others return -1.
  template <typename F, typename G>
  __device__ int ordered_find(F &&f, G &&target) {
    double v = 0.0;
    each([&](float x, int i) { v += f(x, i); });
    double cta[C];
    const double total = cluster_total(v, cta);
    if (!(total > 0.0)) return -1;
    const double t = target(total);
    double excl = 0.0;
    int win = -1;
    double win_excl = 0.0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      if (cta[r] > 0.0 && (win < 0 || excl <= t)) {
        win = r;
        win_excl = excl;
      }
      excl += cta[r];
    }
    if (win != rank) return -1;
    if (threadIdx.x == 0) {
      double e = win_excl;
      int w_win = -1;
      double w_excl = 0.0;
      for (int w = 0; w < WARPS; ++w) {
        if (s.warp_sum[w] > 0.0 && (w_win < 0 || e <= t)) {
          w_win = w;
          w_excl = e;
        }
        e += s.warp_sum[w];
      }
      s.winner = w_win;
      s.rel = w_excl;
    }
    __syncthreads();
    if (warp != s.winner) return -1;
    double run = s.rel;
    int last = -1;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const double own = i < w1 ? f(at(i), first + i) : 0.0;
      double incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned any = __ballot_sync(0xffffffffu, own > 0.0);
      if (any) last = first + i0 + 31 - __clz(any);
      const unsigned over = __ballot_sync(0xffffffffu, own > 0.0 && run + incl > t);
      if (over) return first + i0 + __ffs(over) - 1;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    return last;  // the sums of the scan and of the lanes may round apart: the last one then
  }

  // Histogram bin in which the running total of `value` first reaches `need` (bins in descending key order).
  // count / hi / lo of the cluster are summed by every CTA alike.  Leaves bin, the total before it and its count.
  template <bool MASS>
  __device__ void find_bin(double need) {
    cluster_barrier();  // all histograms are complete
    constexpr int PER = NB / THREADS;
    unsigned long long v[PER];
    uint32_t cnt[PER];
    unsigned long long sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = threadIdx.x * PER + i;
      cnt[i] = 0;
      v[i] = 0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        cnt[i] += ld_cluster_u32(peer(&s.count[b], r));
        if (MASS) v[i] += ((unsigned long long)ld_cluster_u32(peer(&s.hi[b], r)) << 14) + ld_cluster_u32(peer(&s.lo[b], r));
      }
      if (!MASS) v[i] = cnt[i];
      sum += v[i];
    }
    unsigned long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) s.scan[warp] = incl;
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
    unsigned long long excl = incl - sum;
    for (int w = 0; w < warp; ++w) excl += s.scan[w];
    // the crossing bin; without one (rounding at the far end) the last bin that holds anything
    int last = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (cnt[i]) last = threadIdx.x * PER + i;
    unsigned long long e = excl;
    bool hit = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (cnt[i] && (double)e < need && (double)(e + v[i]) >= need) {
        s.bin = threadIdx.x * PER + i;
        s.before = e;
        s.bin_count = cnt[i];
        hit = true;
      }
      e += v[i];
    }
    const int any = __syncthreads_or(hit);
    if (!any) {
      atomicMax(&s.bin, last);
      __syncthreads();
      const int b = s.bin;
      if (b / PER == (int)threadIdx.x) {
        unsigned long long f = excl;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          if (threadIdx.x * PER + i == b) {
            s.before = f;
            s.bin_count = cnt[i];
          }
          f += v[i];
        }
      }
      __syncthreads();
    }
    cluster_barrier();  // every CTA has read the histograms
  }

  __device__ void clear() {
    for (int i = threadIdx.x; i < NB; i += THREADS) s.count[i] = s.hi[i] = s.lo[i] = 0;
    __syncthreads();
  }

  // The cut of top-k (MASS false: `need` elements) or top-p (MASS true: `need` units of mass; unit = 1 / scale):
  // first by value, linear over at most 64 below the maximum -- logits spread evenly there, so the atomics do --
  // then by key within the bin until a bin is one key.
  template <bool MASS>
  __device__ Cut descend(const Cut &in, double need, double scale, float lowest) {
    const float range = fminf(m - lowest, 64.0f);
    const float f = range > 1e-20f ? (float)NB / range : 0.0f;
    auto bin_of = [&](float v) {
      const float d = v == m ? 0.0f : m - v;
      return (int)fminf(d * f, (float)(NB - 1));
    };
    auto add = [&](int b, float v) {
      atomicAdd(&s.count[b], 1u);
      if (MASS) {
        const unsigned long long q = __double2ull_rn(weight(v) * scale);
        atomicAdd(&s.hi[b], (uint32_t)(q >> 14));
        atomicAdd(&s.lo[b], (uint32_t)(q & 16383u));
      }
    };
    clear();
    each([&](float v, int i) {
      if (kept(in, v, i)) add(bin_of(v), v);
    });
    find_bin<MASS>(need);
    unsigned long long before = s.before;
    const int b = s.bin;
    // keys of the bin: bin_of does not rise with the key
    uint32_t lo = key_of(lowest), hi = key_of(m);
    {
      uint32_t l = lo, h = hi;      // lowest key with bin <= b
      while (l < h) {
        const uint32_t mid = l + (h - l) / 2;
        if (bin_of(value_of(mid)) <= b) h = mid;
        else l = mid + 1;
      }
      const uint32_t first_key = l;
      l = first_key, h = hi;        // highest key with bin >= b
      while (l < h) {
        const uint32_t mid = l + (h - l + 1) / 2;
        if (bin_of(value_of(mid)) >= b) l = mid;
        else h = mid - 1;
      }
      lo = first_key;
      hi = l;
    }
    constexpr int KS = sizeof(T) == 2 ? 13 : 0;  // a widened fp16 value leaves the low 13 bits of its key alone
    while (true) {
      const uint32_t span = (hi >> KS) - (lo >> KS);   // keys - 1
      int sh = 0;
      while ((span >> sh) >= (uint32_t)NB) ++sh;
      __syncthreads();
      clear();
      each([&](float v, int i) {
        const uint32_t k = key_of(v);
        if (k >= lo && k <= hi && kept(in, v, i)) add((int)(((hi >> KS) - (k >> KS)) >> sh), v);
      });
      find_bin<MASS>(need - (double)before);
      const uint32_t bb = (uint32_t)s.bin;
      before += s.before;
      const uint32_t top = (hi >> KS) - (bb << sh);
      if (sh == 0) {
        const uint32_t k = KS ? (top << KS | (top & (0x80000000u >> KS) ? 0u : (1u << KS) - 1u)) : top;
        const uint32_t ties = s.bin_count;
        double t;
        if (MASS) t = ceil((need - (double)before) / (weight(value_of(k)) * scale));
        else t = need - (double)before;
        if (!(t > 1.0)) t = 1.0;
        Cut c = {k, 0x7fffffff};
        if (t < (double)ties) c.index = tie_index(in, k, t);
        return c;
      }
      const uint32_t lowk = top >= (1u << sh) - 1u ? top - ((1u << sh) - 1u) : 0u;
      if ((lowk << KS) > lo) lo = lowk << KS;
      hi = KS ? (top << KS | ((1u << KS) - 1u)) : top;
    }
  }

  // Row index of the t-th kept element with key k.
  __device__ int tie_index(const Cut &in, uint32_t k, double t) {
    const int i = ordered_find([&](float v, int j) { return key_of(v) == k && kept(in, v, j) ? 1.0 : 0.0; },
                               [&](double) { return t - 0.5; });
    if (i >= 0 && (threadIdx.x & 31) == 0)
      for (int r = 0; r < C; ++r) st_cluster_u32(peer(&s.found_index, r), (uint32_t)i);
    cluster_barrier();
    const int at_index = s.found_index;
    cluster_barrier();
    return at_index;
  }
};

template <typename T, int C>
__global__ void __launch_bounds__(THREADS)
sample_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared s;
  Row<T, C> r(p, s);
  const int row = blockIdx.x / C;
  r.rank = C > 1 ? (int)tc::cluster_ctarank() : 0;
  r.warp = threadIdx.x >> 5;
  r.lane = threadIdx.x & 31;
  r.first = r.rank * p.slice;
  r.n = max(0, min(p.slice, p.V - r.first));
  const T *src = static_cast<const T *>(p.x) + (int64_t)row * p.row_stride + r.first;
  // the peers' shared memory may be written once every CTA of the cluster has started
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();
  float T0 = p.temperature ? p.temperature[row] : p.temperature0;
  float top_p = p.top_p ? p.top_p[row] : p.top_p0;
  float min_p = p.min_p ? p.min_p[row] : p.min_p0;
  int top_k = p.top_k ? p.top_k[row] : p.top_k0;
  float u = fminf(fmaxf(p.u[row], 0.0f), 0.99999994f);

  const int per = ((p.slice + WARPS - 1) / WARPS + 31) / 32 * 32;
  r.w0 = min(r.warp * per, r.n);
  r.w1 = min(r.w0 + per, r.n);
  float mx = -INFINITY, mn = INFINITY;
  auto seen = [&](float v) {
    if (v == v) {
      mx = fmaxf(mx, v);
      if (v > -INFINITY) mn = fminf(mn, v);
    }
  };
  if (p.resident) {
    T *dst = reinterpret_cast<T *>(dyn);
    constexpr int E = 16 / sizeof(T);
    // 16-byte loads between the first and the last aligned address of the slice, single elements around them
    const int head = min(r.n, (int)(((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / sizeof(T)));
    const int vecs = (r.n - head) / E;
    dst += (E - head) % E;  // the vectors are aligned in shared memory too
    r.data = dst;
    for (int i = threadIdx.x; i < head; i += THREADS) seen(to_f32<T>(dst[i] = src[i]));
    for (int i = head + vecs * E + threadIdx.x; i < r.n; i += THREADS) seen(to_f32<T>(dst[i] = src[i]));
#pragma unroll 8
    for (int i = threadIdx.x; i < vecs; i += THREADS) {
      Vec16<T> v;
      v.raw = ld_stream_as<decltype(v.raw)>(src + head + i * E);
      *reinterpret_cast<decltype(v.raw) *>(dst + head + i * E) = v.raw;
      float f[E];
      v.unpack(f);
#pragma unroll
      for (int e = 0; e < E; ++e) seen(f[e]);
    }
  } else {
    r.data = src;
    for (int i = threadIdx.x; i < r.n; i += THREADS) seen(to_f32<T>(src[i]));
  }
  mx = warp_max(mx);
  mn = -warp_max(-mn);
  if (r.lane == 0) {
    s.scan[r.warp] = ((unsigned long long)__float_as_uint(mx) << 32) | __float_as_uint(mn);
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < C) {
    for (int w = 0; w < WARPS; ++w) {
      mx = fmaxf(w ? mx : -INFINITY, __uint_as_float((uint32_t)(s.scan[w] >> 32)));
      mn = fminf(w ? mn : INFINITY, __uint_as_float((uint32_t)s.scan[w]));
    }
    st_cluster_u32(r.peer(&s.fmax[r.rank], threadIdx.x), __float_as_uint(mx));
    st_cluster_u32(r.peer(&s.fmin[r.rank], threadIdx.x), __float_as_uint(mn));
  }
  r.cluster_barrier();
  mx = -INFINITY;
  mn = INFINITY;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    mx = fmaxf(mx, s.fmax[c]);
    mn = fminf(mn, s.fmin[c]);
  }
  r.m = mx;
  int token = -1;          // held by the CTA (and warp) that found it
  if (mx == -INFINITY) {
    if (r.rank == 0) token = -2;  // nothing to choose from
  } else if (!(T0 > 0.0f) || top_k == 1) {
    token = r.ordered_find([&](float v, int) { return v == mx ? 1.0 : 0.0; }, [](double) { return 0.5; });
  } else {
    r.inv_t = 1.4426950408889634074 / (double)T0;
    Cut cut = {0u, 0x7fffffff};
    if (top_k > 0 && top_k < p.V) cut = r.template descend<false>(cut, (double)top_k, 0.0, mn);
    if (top_p < 1.0f) {
      double part = 0.0, cta[C];
      r.each([&](float v, int i) { if (r.kept(cut, v, i)) part += r.weight(v); });
      const double total = r.cluster_total(part, cta);
      const double scale = 17592186044416.0 / total;  // 2^44 units
      cut = r.template descend<true>(cut, fmax((double)top_p * 17592186044416.0, 1.0), scale, mn);
    }
    const double floor_w = (double)fminf(fmaxf(min_p, 0.0f), 1.0f);  // the largest logit (w = 1) always stays
    token = r.ordered_find(
        [&](float v, int i) {
          if (!r.kept(cut, v, i)) return 0.0;
          const double w = r.weight(v);
          return w >= floor_w ? w : 0.0;
        },
        [&](double total) { return (double)u * total; });
  }
  if (token != -1 && r.lane == 0 && (token >= 0 || threadIdx.x == 0)) p.out[row] = token >= 0 ? token : -1;
  r.cluster_barrier();  // no CTA leaves while its shared memory may still be read
  pdl_launch_dependents();
}

template <typename T, int C>
static int launch(const Params &p, int64_t rows, size_t smem, cudaStream_t st) {
  static PerDeviceOnce once;
  int dev = 0;
  HEXB_CUDA_OK(cudaGetDevice(&dev));
  if (!once.is_done(dev)) {
    HEXB_CUDA_OK(cudaFuncSetAttribute(sample_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 196 * 1024));
    once.mark(dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option(OPT_pdl, 1) ? 2 : 1;
  HEXB_CUDA_OK(cudaLaunchKernelEx(&cfg, sample_kernel<T, C>, p));
  return check_launch("sample");
}

template <typename T>
static int dispatch(Params p, int64_t rows, cudaStream_t st) {
  DeviceInfo di;
  if (int e = current_device(&di)) return e;
  // CTAs of a row: enough that a slice is at most 16384 logits, up to the 8 of a portable cluster.
  int c = 1;
  while (c < MAXC && (p.V + c - 1) / c > 16384) c *= 2;
  p.slice = ((p.V + c - 1) / c + 7) / 8 * 8;
  const size_t bytes = (size_t)p.slice * sizeof(T) + 32;
  p.resident = bytes <= 192 * 1024;
  const size_t smem = p.resident ? bytes : 0;
  switch (c) {
    case 1: return launch<T, 1>(p, rows, smem, st);
    case 2: return launch<T, 2>(p, rows, smem, st);
    case 4: return launch<T, 4>(p, rows, smem, st);
    default: return launch<T, 8>(p, rows, smem, st);
  }
}

}  // namespace sampling
}  // namespace hexb

using namespace hexb;

extern "C" int hexb_sample_tokens(int dtype, const void *logits, const float *u, int64_t *out, int64_t rows,
                                  int64_t vocab, int64_t row_stride, const float *temperature, const int32_t *top_k,
                                  const float *top_p, const float *min_p, float temperature0, int top_k0, float top_p0,
                                  float min_p0, void *stream) {
  if (dtype != HEXB_DT_F16 && dtype != HEXB_DT_F32) return HEXB_ERR_UNSUPPORTED;
  if (rows < 0 || vocab < 0) return HEXB_ERR_BAD_ARG;
  if (rows == 0) return HEXB_OK;
  if (vocab == 0 || !logits || !u || !out || row_stride < 0) return HEXB_ERR_BAD_ARG;
  if (vocab > (1 << 28) || rows > (1 << 27)) return HEXB_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == HEXB_DT_F16 ? 2 : 4)) return HEXB_ERR_MISALIGNED;
  sampling::Params p = {};
  p.x = logits; p.u = u; p.out = out;
  p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.temperature0 = temperature0; p.top_k0 = top_k0; p.top_p0 = top_p0; p.min_p0 = min_p0;
  p.row_stride = row_stride;
  p.V = (int)vocab;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == HEXB_DT_F16 ? sampling::dispatch<__half>(p, rows, st) : sampling::dispatch<float>(p, rows, st);
}
