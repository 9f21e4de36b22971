// Token sampling: one token per row of logits, from a given uniform random number.
//
//   w_i = exp((x_i - max x) / T)                      T <= 0: the largest logit, lowest index
//   top-k   keeps the k largest logits
//   top-p   of those, in descending order, every one before which less than p of their mass lies
//   min-p   of those, the ones with w_i >= min_p
//   token   the first kept index, in index order, whose inclusive sum of w exceeds u times the kept sum
//
// Ties are ordered by index everywhere (the lower one first), so each filter keeps a prefix of one descending order, and
// a cut in it -- (key, index) -- says all.  NaN and -inf are never chosen; a row with nothing else gives -1.
//
// A token is a whole number, so borders decide: weights (relative error below 2^-37, see weight()) are formed and summed in
// 64 bits, as floating-point numbers or as integers of at least 60 bits of the mass, and in an order that does not depend on
// how the threads run.
//
// Drawing in index order needs no sorted row.  A histogram of the row's values (one shared-memory atomic a logit) gives
// the cut of top-k to a bin, and with the bins' weights a guess of the cut of top-p to a few.  Then one pass
//   - collects the logits at or above the cut, if they are few: the rest happens in that sorted list; else
//   - collects the cut's bins alone and sums, exactly, the mass above them and in all, which settles the cut and proves or
//     disproves the guess; a last pass draws among what is kept.
// Where the list would not hold the bins (thousands of equal logits) or the guess was wrong, the cut is found by
// histograms of the keys, level by level.
//
// Few rows: a cluster of CTAs owns a row, each with its slice in shared memory, and exchanges maxima, sums and
// histograms through distributed shared memory; a step costs latency only.  Many rows: one CTA a row, two an SM, the
// passes read the row from L2; instruction issue is the bound (256 rows of 128000 fp16, 65 MB, 10 us of memory: 24 us for
// the maximum alone, 79 without filters, 149 with top-p).
#include "tc_sm100.cuh"

namespace hexb {
namespace sampling {

typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int NB = 2048;           // histogram bins
constexpr int CAP = 4096;          // list entries
constexpr int SHORT = 1024;        // of a list in which all the rest may happen
constexpr int MAXC = 8;
constexpr int WIDTHS = 3;          // windows around the guess: 1, 4 and 16 bins to either side
constexpr int kLevelBits = 10, kLevels = 1 << kLevelBits;  // of the exponential's table
constexpr uint32_t kNoCut = 0x007fffffu;  // key of -inf

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
// What is kept so far: keys above `key`, and of those equal to it the indices up to `index`.
struct Cut {
  uint32_t key;
  int index;
};

struct Shared {
  uint32_t count[NB];
  alignas(16) u64 list[CAP];               // (key, ~index); the key histograms' two mass words lie here too
  double mass[CAP];                 // of the sorted list: weights, then running sums
  double table[kLevels];            // 2^(-i / kLevels)
  double warp_sum[WARPS];
  double part[2][MAXC];
  double rel;
  u64 best[MAXC];              // (key, ~index) of the largest logit of every CTA
  float fmin[MAXC];
  u64 scan[WARPS];
  float fscan[WARPS];
  unsigned long long before;
  uint32_t bin_count, n;            // list length
  int found_index, bin, winner, b_k, b_p, b_last, n_last, n_first[WIDTHS], n_guess[WIDTHS], guessed;
  uint32_t before_k;
  Cut cut;
  int cut_ok;
};
static_assert(2 * NB * 4 <= CAP * 8, "mass words fit the list");

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint4 ld_cluster_u128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t add_cluster_u32(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}

template <typename T, int C>
struct Row {
  static constexpr int E = Vec16<T>::N;
  using Raw = decltype(Vec16<T>::raw);
  const Params &p;
  Shared &s;
  const T *data;          // the slice: shared memory, or global
  int n, rank, warp, lane;
  int shift;              // elements between the 16-byte boundary below `data` and data
  int v0, v1;             // this warp's contiguous part of the slice, in 16-byte vectors from that boundary
  int first;              // row index of slice element 0
  float m, f_bin;         // maximum; bins per unit of value
  double top, scale;      // the maximum; kLevels * log2(e) / T
  float scale32, v_min;
  bool infinite;          // the maximum is: the elements come as 0 (its like), or as -inf
  int flip;

  __device__ Row(const Params &p_, Shared &s_) : p(p_), s(s_), infinite(false), flip(0) {}

  __device__ __forceinline__ void cluster_barrier() {
    if (C > 1) tc::cluster_sync_all();
    else __syncthreads();
  }
  __device__ __forceinline__ uint32_t peer(const void *a, int r) {
    const uint32_t l = tc::smem_u32(a);
    return C > 1 ? tc::map_to_rank(l, (uint32_t)r) : l;
  }
  // exp((v - m) / T) in 64 bits: y = kLevels * log2(e) * (v - m) / T = k + f, |f| <= 1/2; 2^(k / kLevels) from the table and the
  // exponent, 2^(f / kLevels) by its Taylor series (degree 2: the next term is below 0.00034^3 / 6 = 7e-12, an order
  // under what the sums need).  Below v_min the weight, 2^-1000, counts as 0.
  __device__ __forceinline__ double weight(float v) const { return v < v_min ? 0.0 : weight_above(v); }
  __device__ __forceinline__ double weight_above(float v) const {   // v >= v_min
    // the difference first: it is exact where it counts, however large the logits are
    const double d = (double)v - top;
    const double magic = 6755399441055744.0;         // 1.5 * 2^52: the sum's low word is the rounded y
    const double z = fma(d, scale, magic);
    const int k = -__double2loint(z);
    const double f = fma(d, scale, magic - z);
    constexpr double L = 0.693147180559945309417 / kLevels;
    double r = fma(L * L / 2.0, f, L);
    r = fma(r, f, 1.0);
    const double w = r * s.table[k & (kLevels - 1)];
    return __hiloint2double(__double2hiint(w) - ((k & ~(kLevels - 1)) << (20 - kLevelBits)), __double2loint(w));
  }
  // Weights of the elements of one vector that the cut keeps, 0 for the others.  Without a branch an element, so that
  // the chains of a vector's elements overlap (with one, a pass over 256 rows of 128000 took 121 us).
  __device__ __forceinline__ void weigh(const Cut &c, const float (&x)[E], int i0, double (&w)[E]) const {
    const float at = value_of(c.key), low = fmaxf(at, v_min);
    float top = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
    if (top < low) {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = 0.0;
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double v = weight_above(x[e]);
      w[e] = x[e] < low ? 0.0 : v;
    }
    if (i0 + E - 1 > c.index) {                       // the cut runs through equal logits, behind the last that stays
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] == at && i0 + e > c.index) w[e] = 0.0;
    }
  }
  // sum += their sum; and, of those above the value `upper`, above += it.
  template <bool ABOVE>
  __device__ __forceinline__ void add_weights(const Cut &c, const float (&x)[E], int i0, double &sum, float upper, double &above) const {
    const float at = value_of(c.key), low = fmaxf(at, v_min);
    float top = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
    if (top < low) return;
    // Behind the cut's index the cut's equals are out; few vectors hold one (256 rows, k = 40000 of 128000: 150 -> 146 us).
    bool tie = false;
    if (i0 + E - 1 > c.index) {
#pragma unroll
      for (int e = 0; e < E; ++e) tie = tie || x[e] == at;
    }
    if (tie) {
      double w[E];
      weigh(c, x, i0, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sum += w[e];
        if (ABOVE && x[e] > upper) above += w[e];
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double w = weight_above(x[e]);
      if (x[e] >= low) sum += w;
      if (ABOVE && x[e] >= low && x[e] > upper) above += w;
    }
  }
  // Lowest key whose weight is at least min_p: weights do not fall as keys rise.
  __device__ uint32_t min_p_key(float min_p) const {
    uint32_t lo = 0x00800000u, hi = key_of(m);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (weight(value_of(mid)) >= (double)min_p) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }
  __device__ __forceinline__ bool kept(const Cut &c, float v, int i) const {
    const float at = value_of(c.key);                // (-inf for no cut: it keeps no -inf either)
    return v > at || (v == at && i <= c.index && at > -INFINITY);
  }
  // Does not fall as v falls.  (bin_of(v) < b, for b < NB, is depth(v) < b.)
  __device__ __forceinline__ float depth(float v) const { return (m - v) * f_bin; }
  // The largest value at least `bin` deep; -inf if no finite one is.  Passes compare with it instead of forming every depth.
  // Whole warps call it: one round around the estimate, and if that misses, rounds that cut the range of keys by 33.
  __device__ float value_at(int bin) const {
    if (bin <= 0) return m;
    uint32_t lo = kNoCut, hi = key_of(m);            // lo: deep enough, or the key of -inf; hi: not
    const uint32_t near = key_of(m - (float)bin / f_bin) - 16 + lane;
    const bool in = near > lo && near < hi;
    const unsigned fits = __ballot_sync(0xffffffffu, in && depth(value_of(near)) >= (float)bin);
    if (__all_sync(0xffffffffu, in) && (fits & 1u) && !(fits >> 31)) return value_of(near - lane + __popc(fits) - 1);
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo - 1) / 33 + 1, k = lo + step * (lane + 1);
      const bool deep = k > lo && k < hi && hi - lo > step * (lane + 1) && depth(value_of(k)) >= (float)bin;
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, deep));
      lo += step * n;
      hi = min(hi - lo, step) + lo;
    }
    return value_of(lo);
  }
  __device__ __forceinline__ int bin_of(float v) const { return (int)fminf(depth(v), (float)(NB - 1)); }
  // The elements of vector v, and the row index of the first.  NaN, and places outside the slice, come as -inf.
  __device__ __forceinline__ int vector(int v, float (&x)[E]) const {
    Raw raw;
    return expand(v, fetch(v, vectors(), raw), raw, x);
  }
  __device__ __forceinline__ int vectors() const { return (n + shift + E - 1) / E; }
  // Whole vectors below `end` are requested here, so that several are under way; others are read element by element.
  __device__ __forceinline__ bool fetch(int v, int end, Raw &raw) const {
    const int i = v * E - shift;
    const bool whole = v < end && i >= 0 && i + E <= n;
    if (whole) raw = *reinterpret_cast<const Raw *>(data + i);
    return whole;
  }
  __device__ __forceinline__ int expand(int v, bool whole, const Raw &raw, float (&x)[E]) const {
    const int i = v * E - shift;
    if (whole) {
      Vec16<T> q;
      q.raw = raw;
      q.unpack(x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i + e >= 0 && i + e < n ? to_f32<T>(data[i + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = fmaxf(x[e], -INFINITY);
    if (infinite) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = x[e] == INFINITY ? m : -INFINITY;
    }
    return first + i;
  }
  // f(values, row index of the first) for every vector of this warp's part, by whole warps (lanes without a vector get -inf)
  template <typename F>
  __device__ __forceinline__ void each(F &&f) const {
    constexpr int AHEAD = 4;
    for (int vb = v0; vb < v1; vb += 32 * AHEAD) {
      Raw raw[AHEAD];
      bool whole[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) whole[j] = fetch(vb + j * 32 + lane, v1, raw[j]);
#pragma unroll 1
      for (int j = 0; j < AHEAD; ++j) {
        if (vb + j * 32 >= v1) break;
        const int v = vb + j * 32 + lane;
        float x[E];
        int at = 0;
        if (v < v1) {
          at = expand(v, whole[0], raw[0], x);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) x[e] = -INFINITY;
        }
        f(x, at);
        // the next one moves up: one copy of f's code
#pragma unroll
        for (int k = 0; k + 1 < AHEAD; ++k) {
          raw[k] = raw[k + 1];
          whole[k] = whole[k + 1];
        }
      }
    }
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

  // Lowest row index at which the inclusive sum of a weighting exceeds target(total); -1 if the sum is empty.  The warp that
  // finds it returns it, all others -1.  f(x, i, w) weighs a vector, g(x, i, sum) adds its weights up.
  template <typename F, typename S, typename G>
  __device__ int ordered_find(F &&f, S &&g, G &&target) {
    double v = 0.0;
    each([&](const float (&x)[E], int i) { g(x, i, v); });
    return place(v, f, target);
  }
  // The same from the sums of the lanes of this warp.
  template <typename F, typename G>
  __device__ int place(double v, F &&f, G &&target) {
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
    // The warp whose part holds it; then that part is dealt to all warps, until a part is one vector a lane.  (One warp
    // alone over its part of 128000 logits: 20 us.)
    int lo = 0, hi = (n + shift + E - 1) / E;
    double base = win_excl;
    while (true) {
      const int len = (hi - lo + WARPS - 1) / WARPS;
      if (threadIdx.x == 0) {
        double e = base;
        s.winner = -1;
        for (int w = 0; w < WARPS; ++w) {
          if (s.warp_sum[w] > 0.0 && (s.winner < 0 || e <= t)) {
            s.winner = w;
            s.rel = e;
          }
          e += s.warp_sum[w];
        }
      }
      __syncthreads();
      lo = min(lo + s.winner * len, hi);
      hi = min(lo + len, hi);
      base = s.rel;
      if (hi - lo <= 32) break;
      const int part = (hi - lo + WARPS - 1) / WARPS, a = min(lo + warp * part, hi), b = min(a + part, hi);
      double sum = 0.0;
      for (int vv = a + lane; vv < b; vv += 32) {
        float x[E];
        double w[E];
        const int i = vector(vv, x);
        f(x, i, w);
#pragma unroll
        for (int e = 0; e < E; ++e) sum += w[e];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncthreads();
      if (lane == 0) s.warp_sum[warp] = sum;
      __syncthreads();
    }
    if (warp) return -1;
    // a lane's vector first, then the element in it
    double own[E], sum = 0.0;
    int at = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) own[e] = 0.0;
    if (lo + lane < hi) {
      float x[E];
      at = vector(lo + lane, x);
      f(x, at, own);
#pragma unroll
      for (int e = 0; e < E; ++e) sum += own[e];
    }
    double incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned any = __ballot_sync(0xffffffffu, sum > 0.0);
    const unsigned over = __ballot_sync(0xffffffffu, sum > 0.0 && base + incl > t);
    // the lane that crosses, or (sums of scan and lanes may round apart) the last that holds anything
    const int from = over ? __ffs(over) - 1 : 31 - __clz(any);
    int mine = -1;
    if (lane == from) {
      double c = base + (incl - sum);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (own[e] > 0.0 && (mine < 0 || !(c > t))) mine = at + e;
        c += own[e];
      }
    }
    return __shfl_sync(0xffffffffu, mine, from);
  }

  __device__ void clear(bool mass) {
    for (int i = threadIdx.x; i < NB; i += THREADS) s.count[i] = 0;
    if (mass) {
      uint32_t *w = reinterpret_cast<uint32_t *>(s.list);
      for (int i = threadIdx.x; i < 2 * NB; i += THREADS) w[i] = 0;
    }
    __syncthreads();
  }
  // This thread's four bins of the cluster's histogram: counts, or the mass (the high words, then the low ones).
  __device__ __forceinline__ uint4 bins4_of(const uint32_t *h, int r) {
    return C > 1 ? ld_cluster_u128(peer(h + threadIdx.x * 4, r)) : *reinterpret_cast<const uint4 *>(h + threadIdx.x * 4);
  }
  __device__ __forceinline__ uint4 bins4() {
    uint4 c = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const uint4 v = bins4_of(s.count, r);
      c.x += v.x; c.y += v.y; c.z += v.z; c.w += v.w;
    }
    return c;
  }
  __device__ __forceinline__ void mass4(u64 (&v)[4]) {
    const uint32_t *hi = reinterpret_cast<const uint32_t *>(s.list), *lo = hi + NB;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const uint4 h = bins4_of(hi, r), l = bins4_of(lo, r);
      v[0] += (u64)h.x << 32 | l.x;
      v[1] += (u64)h.y << 32 | l.y;
      v[2] += (u64)h.z << 32 | l.z;
      v[3] += (u64)h.w << 32 | l.w;
    }
  }
  // exclusive prefix over the threads of the CTA
  template <typename U>
  __device__ __forceinline__ U exclusive(U v, U *scratch) {
    U incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const U up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    U e = incl - v;
    for (int w = 0; w < warp; ++w) e += scratch[w];
    return e;
  }

  // ------------------------------------------------------------ the plan: histogram of values
  // Counts over at most 32 below the maximum, linear in the value (logits spread evenly there, so the atomics do).
  // Leaves: b_k, before_k  bin of the k-th logit and the count before it
  //         b_p            guess of the bin where p of the mass (of what top-k leaves) is reached
  //         b_last         the last bin that the list needs, n_last logits up to it; guessed: b_p set it
  //         n_first, n_guess   logits before bin b_p - 4^i, and up to bin b_p + 4^i
  __device__ void plan(const Cut &in, int top_k, float top_p, float min_p, float lowest) {
    // (a sample that is all masked, or all the maximum, says nothing about the width)
    const float range = lowest < m ? fminf(m - lowest, 32.0f) : 32.0f;
    f_bin = range > 1e-20f ? (float)NB / range : 0.0f;
    clear(false);
    each([&](const float (&x)[E], int) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > -INFINITY) atomicAdd(&s.count[bin_of(x[e])], 1u);
    });
    if (threadIdx.x == 0) {
      s.b_k = s.b_p = NB - 1;
      s.before_k = 0;
      s.n_last = 0;
      for (int i = 0; i < WIDTHS; ++i) s.n_first[i] = s.n_guess[i] = 0;
    }
    cluster_barrier();
    const uint4 c4 = bins4();
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
    const u64 before = exclusive<u64>((u64)c[0] + c[1] + c[2] + c[3], s.scan);
    const int b0 = threadIdx.x * 4;
    if (top_k > 0) {
      u64 e = before;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (e < (u64)top_k && e + c[i] >= (u64)top_k) {
          s.b_k = b0 + i;
          s.before_k = (uint32_t)e;
        }
        e += c[i];
      }
    }
    __syncthreads();
    const int b_k = s.b_k;
    if (top_p < 1.0f) {
      float w[4], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float centre = f_bin > 0.f ? ((float)(b0 + i) + 0.5f) / f_bin : 0.f;
        w[i] = b0 + i <= b_k ? (float)c[i] * exp2f(-centre * scale32) : 0.f;
        // the maximum, which may hold most of the mass, weighs 1: half a bin off, it would move the guess by many bins
        if (b0 + i == 0) w[i] += 1.0f - w[i] / (float)c[i];
        sum += w[i];
      }
      float e = exclusive<float>(sum, s.fscan);
      float all = 0.f;
      for (int i = 0; i < WARPS; ++i) all += s.fscan[i];
      const float need = fmaxf(top_p * all, 1e-30f);
      bool hit = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!hit && c[i] && e < need && e + w[i] >= need) {
          atomicMin(&s.b_p, b0 + i);
          hit = true;
        }
        e += w[i];
      }
    }
    __syncthreads();
    int limit = b_k;                              // of what any filter but top-p keeps
    if (min_p > 0.0f) {
      // the first difference that min_p drops, to 32 bits (min_p = 1 keeps what 64 bits do not tell from 1)
      const float d = fmaxf(-log2f(min_p), 4e-16f) / scale32, reach = d * f_bin;
      // behind the range all lie in the last bin, so a reach past it is no limit (the range is a sample's: in a row masked
      // but for a few logits it may be a part of what min_p keeps)
      if (reach < (float)(NB - 4)) limit = min(limit, (int)reach + 2);
    }
    // the mass that top-p takes its share of is top-k's, if there is one: then the list has to hold that
    const int last = top_p < 1.0f ? (top_k > 0 ? b_k : min(limit, s.b_p + 1)) : limit;
    u64 e = before;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int k = 0; k < WIDTHS; ++k)
        if (b0 + i == s.b_p - (1 << 2 * k)) s.n_first[k] = (int)e;
      e += c[i];
      if (b0 + i == last) s.n_last = (int)e;
#pragma unroll
      for (int k = 0; k < WIDTHS; ++k)
        if (b0 + i == min(s.b_p + (1 << 2 * k), NB - 1)) s.n_guess[k] = (int)e;
    }
    if (threadIdx.x == 0) {
      s.b_last = last;
      s.guessed = last < limit;
    }
    cluster_barrier();  // every CTA has read the histograms
  }

  // ------------------------------------------------------------ the list
  // The value behind the last of bin `bin`: a list of bins up to that one takes what lies above.
  __device__ __forceinline__ float behind(int bin) const { return bin >= NB - 1 ? -INFINITY : value_at(bin + 1); }
  __device__ __forceinline__ void list_reset() {
    if (threadIdx.x == 0) s.n = 0;
    cluster_barrier();
  }
  // Appends the elements above `below`, up to `from`, that the cut keeps to the list of CTA 0; the whole warp calls it.
  __device__ __forceinline__ void append(const Cut &c, float from, float below, const float (&x)[E], int i0) {
    bool take[E], any = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      take[e] = x[e] <= from && x[e] > below;
      any = any || take[e];
    }
    if (!__any_sync(0xffffffffu, any)) return;       // most vectors hold none
    // One reservation for the warp's vectors: with a cluster it is a trip to CTA 0 and back.
    unsigned who[E];
    int all = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      who[e] = __ballot_sync(0xffffffffu, take[e] && kept(c, x[e], i0 + e));
      all += __popc(who[e]);
    }
    if (all == 0) return;
    uint32_t at = 0;
    if (lane == 0) at = C > 1 ? add_cluster_u32(peer(&s.n, 0), (uint32_t)all) : atomicAdd(&s.n, (uint32_t)all);
    at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t mine = at + __popc(who[e] & ((1u << lane) - 1u));
      if ((who[e] >> lane & 1u) && mine < CAP) {
        const u64 entry = (u64)key_of(x[e]) << 32 | (uint32_t)~(i0 + e);
        if (C > 1) st_cluster_u64(peer(&s.list[mine], 0), entry);
        else s.list[mine] = entry;
      }
      at += __popc(who[e]);
    }
  }
  // Sorts the list, descending (all threads of CTA 0).  Entries differ, so a short list -- one entry a thread -- is ranked by
  // counting the larger ones (300 entries: 4 thousand cycles; the bitonic network takes 12, its steps are all latency).
  // The count grows with the square: 1000 entries took longer than the network.
  __device__ void sort(u64 *a, int n) {
    if (n <= THREADS) {
      const u64 mine = threadIdx.x < n ? a[threadIdx.x] : 0;
      int larger = 0;
      if (threadIdx.x == 0 && (n & 1)) a[n] = 0;
      __syncthreads();
      if (warp * 32 < n) {                             // else no entry in this warp
#pragma unroll 4
        for (int i = 0; i < n; i += 2) {
          const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(a + i);
          larger += (q.x > mine) + (q.y > mine);
        }
      }
      __syncthreads();
      if (threadIdx.x < n) a[larger] = mine;
      __syncthreads();
      return;
    }
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += THREADS) a[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        for (int i = threadIdx.x; i < size / 2; i += THREADS) {
          const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
          const u64 x = a[lo], y = a[hi];
          if ((x < y) == ((lo & k) == 0)) {
            a[lo] = y;
            a[hi] = x;
          }
        }
        // up to j = 32 a warp's pairs lie in 64 entries that only it touches
        if (j > 32 || j == 1 && k >= 64) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
  }
  // s.mass[i] <- sum of the weights of list entries 0 .. i (CTA 0).  Fixed order: consecutive entries a thread.
  __device__ void accumulate(int n) {
    const int per = (n + THREADS - 1) / THREADS, e0 = min((int)threadIdx.x * per, n), e1 = min(e0 + per, n);
    double sum = 0.0;
    for (int e = e0; e < e1; ++e) {
      const double w = weight(value_of((uint32_t)(s.list[e] >> 32)));
      s.mass[e] = w;
      sum += w;
    }
    double run = exclusive<double>(sum, s.warp_sum);
    for (int e = e0; e < e1; ++e) {
      run += s.mass[e];
      s.mass[e] = run;
    }
    __syncthreads();
  }
  // First i < n with ok(i) false (ok holds for a prefix); all threads of CTA 0.
  template <typename F>
  __device__ int prefix_length(int n, F &&ok) {
    __syncthreads();
    if (threadIdx.x == 0) s.found_index = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < n; i += THREADS)
      if (ok(i)) mine = i + 1;
    if (mine) atomicMax(&s.found_index, mine);
    __syncthreads();
    return s.found_index;
  }
  // The cut that CTA 0 found, to all.
  __device__ bool broadcast(Cut &c) {
    if (C > 1) {
      if (rank == 0 && threadIdx.x < C) {
        st_cluster_u32(peer(&s.cut.key, threadIdx.x), s.cut.key);
        st_cluster_u32(peer(&s.cut.index, threadIdx.x), (uint32_t)s.cut.index);
        st_cluster_u32(peer(&s.cut_ok, threadIdx.x), (uint32_t)s.cut_ok);
      }
    }
    cluster_barrier();
    const bool ok = s.cut_ok != 0;
    if (ok) c = s.cut;
    cluster_barrier();
    return ok;
  }

  // ------------------------------------------------------------ everything that is needed fits the list
  // CTA 0 returns the token (thread 0), others -1; -2 in every thread: the guess of top-p was too short.
  __device__ int from_list(int top_k, float top_p, float min_p, float u) {
    const int last = s.b_last;
    list_reset();
    double sum = 0.0, cta[C];
    const bool total_needed = top_p < 1.0f && top_k <= 0;
    const Cut all = {kNoCut, 0x7fffffff};
    const float below = behind(last);
    each([&](const float (&x)[E], int i) {
      append(all, m, below, x, i);
      double none;
      if (total_needed) add_weights<false>(all, x, i, sum, 0.f, none);
    });
    double total = 0.0;
    if (total_needed) total = cluster_total(sum, cta);
    cluster_barrier();
    int token = -1;
    bool short_list = false;
    if (rank == 0) {
      const int n = (int)min(s.n, (uint32_t)CAP);
      sort(s.list, n);
      accumulate(n);
      int keep = top_k > 0 ? min(top_k, n) : n;
      if (top_p < 1.0f) {
        if (!total_needed) total = s.mass[keep - 1];
        const double need = (double)top_p * total;
        const int fits = prefix_length(keep, [&](int i) { return i == 0 || s.mass[i - 1] < need; });
        // every entry belongs to the nucleus and the guess ended the list: the next logit, which is not here, may too
        short_list = s.guessed && fits == n && s.mass[n - 1] < need;
        keep = fits;
      }
      if (min_p > 0.0f) {
        const double w_min = (double)min_p;
        keep = prefix_length(keep, [&](int i) { return weight(value_of((uint32_t)(s.list[i] >> 32))) >= w_min; });
        short_list = short_list && keep == n;
      }
      if (!short_list) {
        if (keep <= 1) {
          token = (int)~(uint32_t)s.list[0];
        } else {
          // the kept entries by index: (~index, key) descending
          for (int i = threadIdx.x; i < keep; i += THREADS) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;
          __syncthreads();
          sort(s.list, keep);
          for (int i = threadIdx.x; i < keep; i += THREADS) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;
          __syncthreads();
          accumulate(keep);
          const double t = (double)u * s.mass[keep - 1];
          const int at = prefix_length(keep, [&](int i) { return s.mass[i] <= t; });
          token = (int)~(uint32_t)s.list[min(at, keep - 1)];
        }
        if (threadIdx.x) token = -1;
      }
      if (threadIdx.x == 0) s.cut_ok = short_list;
      __syncthreads();
    }
    Cut unused;
    return broadcast(unused) ? -2 : token;
  }

  // ------------------------------------------------------------ a cut whose bins fit the list
  // k-th logit: it is in bin b_k.
  __device__ bool refine_k(Cut &cut, int top_k) {
    const int b = s.b_k;
    const int rank_in = top_k - (int)s.before_k;     // 1 ..
    list_reset();
    const Cut all = {kNoCut, 0x7fffffff};
    const float from = value_at(b), below = behind(b);
    each([&](const float (&x)[E], int i) { append(all, from, below, x, i); });
    cluster_barrier();
    if (rank == 0) {
      const int n = (int)min(s.n, (uint32_t)CAP);
      const bool ok = s.n <= CAP && rank_in <= n;
      if (ok) sort(s.list, n);
      if (threadIdx.x == 0) {
        s.cut_ok = ok;
        if (ok) s.cut = {(uint32_t)(s.list[rank_in - 1] >> 32), (int)~(uint32_t)s.list[rank_in - 1]};
      }
      __syncthreads();
    }
    return broadcast(cut);
  }
  // p of the mass: guessed to lie in bin b_p, or at most `width` bins from it.
  // With one CTA a row it also leaves what draw_above needs: `above`, this lane's sum over the bins before those.
  __device__ bool refine_p(Cut &cut, float top_p, int width, double &above) {
    const int lo = s.b_p - width, hi = s.b_p + width;
    list_reset();
    double sum = 0.0, cta[C];
    above = 0.0;
    const float from = value_at(lo), below = behind(hi);
    each([&](const float (&x)[E], int i) {
      append(cut, from, below, x, i);
      add_weights<true>(cut, x, i, sum, from, above);
    });
    const double total = cluster_total(sum, cta);
    const double over = cluster_total(above, cta);
    cluster_barrier();
    if (rank == 0) {
      const int n = (int)min(s.n, (uint32_t)CAP);
      bool ok = s.n <= CAP && n > 0;
      if (ok) {
        sort(s.list, n);
        accumulate(n);
        const double need = (double)top_p * total;
        const int fits = prefix_length(n, [&](int i) { return over + (i ? s.mass[i - 1] : 0.0) < need; });
        ok = (fits > 0 || lo <= 0) && (fits < n || over + s.mass[n - 1] >= need || hi >= NB - 1);
        const int at = max(fits, 1) - 1;
        if (threadIdx.x == 0) s.n = (uint32_t)at + 1;   // the entries that stay
        if (threadIdx.x == 0) s.cut = {(uint32_t)(s.list[at] >> 32), (int)~(uint32_t)s.list[at]};
      }
      __syncthreads();
      if (threadIdx.x == 0) s.cut_ok = ok;
      __syncthreads();
    }
    return broadcast(cut);
  }

  // The draw after refine_p, without another pass over the row: a warp's kept mass is what lies above the list's bins
  // and the list entries of its part that stay.
  __device__ int draw_above(const Cut &cut, double above, float u) {
    const int keep = (int)s.n;
    for (int i = lane; i < keep; i += 32) {
      const int v = ((int)~(uint32_t)s.list[i] - first + shift) / E;
      if (v >= v0 && v < v1) above += weight(value_of((uint32_t)(s.list[i] >> 32)));
    }
    return place(above, [&](const float (&x)[E], int i, double (&w)[E]) { weigh(cut, x, i, w); },
                 [&](double total) { return (double)u * total; });
  }

  // ------------------------------------------------------------ a cut by histograms alone
  // Bin in which the running total first reaches `need` (bins in descending key order).
  template <bool MASS>
  __device__ void find_bin(double need) {
    cluster_barrier();  // all histograms are complete
    const uint4 c4 = bins4();
    const uint32_t cnt[4] = {c4.x, c4.y, c4.z, c4.w};
    u64 v[4] = {c4.x, c4.y, c4.z, c4.w};
    if (MASS) mass4(v);
    const u64 sum = v[0] + v[1] + v[2] + v[3];
    if (threadIdx.x == 0) s.bin = -1;
    const u64 excl = exclusive<u64>(sum, s.scan);
    // the crossing bin; without one (rounding at the far end) the last bin that holds anything
    int last = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (cnt[i]) last = threadIdx.x * 4 + i;
    u64 e = excl;
    bool hit = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (cnt[i] && (double)e < need && (double)(e + v[i]) >= need) {
        s.bin = threadIdx.x * 4 + i;
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
      if (b / 4 == (int)threadIdx.x) {
        u64 g = excl;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (threadIdx.x * 4 + i == b) {
            s.before = g;
            s.bin_count = cnt[i];
          }
          g += v[i];
        }
      }
      __syncthreads();
    }
    cluster_barrier();  // every CTA has read the histograms
  }

  // The cut of top-k (MASS false: `need` elements) or top-p (MASS true: `need` units of mass; unit = 1 / units, a power of
  // two, so that equal logits of weight 1 sum exactly): bins of keys, narrowed until a bin is one key.
  template <bool MASS>
  __device__ Cut descend(const Cut &in, double need, double units) {
    constexpr int KS = sizeof(T) == 2 ? 13 : 0;  // a widened fp16 value leaves the low 13 bits of its key alone
    uint32_t *hi_words = reinterpret_cast<uint32_t *>(s.list), *lo_words = hi_words + NB;
    uint32_t lo = 0x00800000u, hi = key_of(m);       // all finite values up to the maximum
    u64 before = 0;
    while (true) {
      const uint32_t span = (hi >> KS) - (lo >> KS);   // keys - 1
      int sh = 0;
      while ((span >> sh) >= (uint32_t)NB) ++sh;
      __syncthreads();
      clear(MASS);
      each([&](const float (&x)[E], int i) {
#pragma unroll 1
        for (int e = 0; e < E; ++e) {
          const uint32_t k = key_of(x[e]);
          if (k < lo || k > hi || !kept(in, x[e], i + e)) continue;
          const uint32_t b = ((hi >> KS) - (k >> KS)) >> sh;
          atomicAdd(&s.count[b], 1u);
          if (MASS) {
            // 64-bit sums in two words, the low one's carries with the high one: whatever the order, the same integer
            const u64 q = __double2ull_rn(weight(x[e]) * units);
            const uint32_t low = (uint32_t)q;
            const uint32_t high = (uint32_t)(q >> 32) + (atomicAdd(&lo_words[b], low) + low < low);
            if (high) atomicAdd(&hi_words[b], high);
          }
        }
      });
      find_bin<MASS>(need - (double)before);
      const uint32_t b = (uint32_t)s.bin;
      before += s.before;
      const uint32_t top = (hi >> KS) - (b << sh);
      if (sh == 0) {
        const uint32_t k = KS ? (top << KS | (top & (0x80000000u >> KS) ? 0u : (1u << KS) - 1u)) : top;
        const uint32_t ties = s.bin_count;
        double t;
        if (MASS) t = ceil((need - (double)before) / (weight(value_of(k)) * units));
        else t = need - (double)before;
        if (!(t > 1.0)) t = 1.0;
        Cut c = {k, k == in.key ? in.index : 0x7fffffff};   // all that were left of the key's equals, or fewer
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
    const int i = ordered_find(
        [&](const float (&x)[E], int j, double (&w)[E]) {
#pragma unroll
          for (int e = 0; e < E; ++e) w[e] = key_of(x[e]) == k && kept(in, x[e], j + e) ? 1.0 : 0.0;
        },
        [&](const float (&x)[E], int j, double &sum) {
#pragma unroll
          for (int e = 0; e < E; ++e) sum += key_of(x[e]) == k && kept(in, x[e], j + e) ? 1.0 : 0.0;
        },
                               [&](double) { return t - 0.5; });
    if (i >= 0 && lane == 0)
      for (int r = 0; r < C; ++r) st_cluster_u32(peer(&s.found_index, r), (uint32_t)i);
    cluster_barrier();
    const int at_index = s.found_index;
    cluster_barrier();
    return at_index;
  }
};

template <typename T, int C>
__global__ void __launch_bounds__(THREADS, 2)
sample_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared &s = *reinterpret_cast<Shared *>(dyn);
  constexpr int E = Vec16<T>::N;
  Row<T, C> r(p, s);
  const int row = blockIdx.x / C;
  r.rank = C > 1 ? (int)tc::cluster_ctarank() : 0;
  r.warp = threadIdx.x >> 5;
  r.lane = threadIdx.x & 31;
  r.first = r.rank * p.slice;
  r.n = max(0, min(p.slice, p.V - r.first));
  const T *src = static_cast<const T *>(p.x) + (int64_t)row * p.row_stride + r.first;
  for (int i = threadIdx.x; i < kLevels; i += THREADS) s.table[i] = exp2(-(double)i / kLevels);
  // the peers' shared memory may be written once every CTA of the cluster has started
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();
  const float T0 = p.temperature ? p.temperature[row] : p.temperature0;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p0;
  const float min_p = fminf(fmaxf(p.min_p ? p.min_p[row] : p.min_p0, 0.0f), 1.0f);  // the largest logit (w = 1) always stays
  int top_k = p.top_k ? p.top_k[row] : p.top_k0;
  const float u = fminf(fmaxf(p.u[row], 0.0f), 0.99999994f);

  r.shift = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  const int vecs = (r.n + r.shift + E - 1) / E, per = (vecs + WARPS - 1) / WARPS;
  r.v0 = min(r.warp * per, vecs);
  r.v1 = min(r.v0 + per, vecs);
  r.data = src;
  T *copy = reinterpret_cast<T *>(dyn + (sizeof(Shared) + 15) / 16 * 16) + r.shift;  // as aligned as the source
  // maximum with its place, and the minimum of a sample (each lane's first vector) for the width of the bins
  float top = -INFINITY, mn = INFINITY;
  int top_v = 0;
  auto load = [&](int v, float (&x)[E]) {
    const int i = v * E - r.shift;
    if (i >= 0 && i + E <= r.n) {
      Vec16<T> q;
      q.raw = ld_stream_as<decltype(q.raw)>(src + i);
      if (p.resident) *reinterpret_cast<decltype(q.raw) *>(copy + i) = q.raw;
      q.unpack(x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = -INFINITY;
        if (i + e >= 0 && i + e < r.n) {
          const T one = src[i + e];
          if (p.resident) copy[i + e] = one;
          x[e] = to_f32<T>(one);
        }
      }
    }
  };
#pragma unroll 4
  for (int v = r.v0 + r.lane; v < r.v1; v += 32) {
    float x[E];
    load(v, x);
    float t = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) t = fmaxf(t, x[e]);   // NaN loses
    if (t > top) {                                    // a lane's places rise: the first of equal ones stays
      top = t;
      top_v = v;
    }
    if (v == r.v0 + r.lane) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > -INFINITY) mn = fminf(mn, x[e]);
    }
  }
  u64 best = 0;
  if (top > -INFINITY) {
    const int i = top_v * E - r.shift;
    int at = 0;
    for (int e = E - 1; e >= 0; --e)
      if (i + e >= 0 && i + e < r.n && to_f32<T>(src[i + e]) == top) at = e;
    best = (u64)key_of(top) << 32 | (uint32_t)~(r.first + i + at);
  }
  if (p.resident) r.data = copy;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  mn = -warp_max(-mn);
  if (r.lane == 0) {
    s.scan[r.warp] = best;
    s.fscan[r.warp] = mn;
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < C) {
    for (int w = 0; w < WARPS; ++w) {
      best = max(w ? best : 0ull, s.scan[w]);
      mn = fminf(w ? mn : INFINITY, s.fscan[w]);
    }
    st_cluster_u64(r.peer(&s.best[r.rank], threadIdx.x), best);
    st_cluster_u32(r.peer(&s.fmin[r.rank], threadIdx.x), __float_as_uint(mn));
  }
  r.cluster_barrier();
  best = 0;
  mn = INFINITY;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    best = max(best, s.best[c]);
    mn = fminf(mn, s.fmin[c]);
  }
  int token = -1;          // held by the thread that stores it
  const bool speaker = r.rank == 0 && threadIdx.x == 0;
  if (best == 0) {
    if (speaker) p.out[row] = -1;  // nothing to choose from
  } else if (!(T0 > 0.0f) || top_k == 1) {
    if (speaker) token = (int)~(uint32_t)best;
  } else {
    r.m = value_of((uint32_t)(best >> 32));
    const double c = 1.4426950408889634074 / (double)T0;
    r.scale = c * kLevels;
    r.top = (double)r.m;
    r.scale32 = (float)c;
    if (top_k >= p.V) top_k = 0;
    r.v_min = fmaxf((float)((double)r.m - 1000.0 / c), -3.402823466e38f);   // never -inf: what is masked weighs nothing
    if (r.m == INFINITY) {        // weight 1 for its like, 0 for any other: they come as 0, the others as -inf
      r.infinite = true;
      r.m = 0.0f;                 // a value of either type: the key's low bits are those of a widened fp16 value
      r.top = 0.0;
      r.v_min = 0.0f;
    }
    Cut cut = {kNoCut, 0x7fffffff};
    bool drawn = false;
    if (top_k > 0 || top_p < 1.0f) {
      r.plan(cut, top_k, top_p, min_p, mn);
      if (s.n_last <= SHORT) {
        token = r.from_list(top_k, top_p, min_p, u);
        drawn = token != -2;
        if (!drawn) token = -1;
      }
      if (!drawn) {
        // Logits around the guess: the widest window whose list is ranked quickly.  (256 rows of 128000, mixed filters: 178 us;
        // always one bin 219, since a row that misses takes three times as long; up to 512 logits 180, and a single row 27.7
        // instead of 25.8.)
        int width = 1, n_p = s.n_guess[0] - s.n_first[0];
        for (int k = 1; k < WIDTHS && s.n_guess[k] - s.n_first[k] <= THREADS / 2; ++k) {
          width = 1 << 2 * k;
          n_p = s.n_guess[k] - s.n_first[k];
        }
        if (top_k > 0 && !r.refine_k(cut, top_k)) cut = r.template descend<false>(cut, (double)top_k, 0.0);
        double above = 0.0;
        const bool refined = top_p < 1.0f && n_p <= CAP && r.refine_p(cut, top_p, width, above);
        if (refined && C == 1 && (min_p <= 0.0f || r.min_p_key(min_p) <= cut.key)) {
          token = r.draw_above(cut, above, u);
          if (r.lane) token = -1;
          drawn = true;
        }
        if (top_p < 1.0f && !refined) {
          double part = 0.0, cta[C];
          r.each([&](const float (&x)[E], int i) {
            double none;
            r.template add_weights<false>(cut, x, i, part, 0.f, none);
          });
          // 2^60 to 2^61 units in all (the largest weighs 1, so the total is at least that): vocab / 2 of them, at most
          // 2^-33 of the mass at 2^28 logits, bound what rounding the weights to units does
          const double total = r.cluster_total(part, cta);
          const double units = __hiloint2double((2 * 1023 + 60 - (__double2hiint(total) >> 20)) << 20, 0);
          cut = r.template descend<true>(cut, fmax((double)top_p * total * units, 1.0), units);
        }
      }
    }
    if (!drawn) {
      if (min_p > 0.0f) {
        const uint32_t k = r.min_p_key(min_p);
        if (k > cut.key) cut = {k, 0x7fffffff};
      }
      token = r.ordered_find([&](const float (&x)[E], int i, double (&w)[E]) { r.weigh(cut, x, i, w); },
                             [&](const float (&x)[E], int i, double &sum) {
                               double none;
                               r.template add_weights<false>(cut, x, i, sum, 0.f, none);
                             },
                             [&](double total) { return (double)u * total; });
      if (r.lane) token = -1;
    }
  }
  if (token >= 0) p.out[row] = token;
  r.cluster_barrier();  // no CTA leaves while its shared memory may still be read
  pdl_launch_dependents();
}

template <typename T, int C>
static int launch(const Params &p, int64_t rows, size_t smem, cudaStream_t st) {
  static PerDeviceOnce once;
  int dev = 0;
  HEXB_CUDA_OK(cudaGetDevice(&dev));
  if (!once.is_done(dev)) {
    HEXB_CUDA_OK(cudaFuncSetAttribute(sample_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
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
  // CTAs of a row: one when the rows alone fill the GPU (its row stays in L2), else enough to spread the row over idle SMs,
  // up to the 8 of a portable cluster and down to slices of 4096 logits.  Rows of 128000 fp16, top-p 0.95, 1 / 2 / 4 / 8 CTAs
  // a row: 16 rows 88 / 72 / 49 / 45 us, 32 rows 92 / 70 / 48 / 54, 64 rows 89 / 71 / 91 / 100, 100 rows 92 / 134 / 163 / 162,
  // 256 rows 145 / 280 / 369 / 391.  At 37 rows the rule's 4 take 87, 2 would take 69: the clusters fill every SM but for one,
  // and do not all find a place at once.
  int c = 1;
  while (c < MAXC && rows * c * 2 <= di.sm_count && (p.V + c - 1) / c > 4096) c *= 2;
  p.slice = ((p.V + c - 1) / c + 7) / 8 * 8;
  const size_t fixed = (sizeof(Shared) + 15) / 16 * 16, bytes = (size_t)p.slice * sizeof(T) + 32;
  p.resident = c > 1 && fixed + bytes <= 220 * 1024;
  const size_t smem = fixed + (p.resident ? bytes : 0);
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
