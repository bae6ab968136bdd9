// Sampling one token a row from logits with temperature, top-k, top-p and min-p, from given random numbers (gfx950).
//
// Candidates of a row are its logits above -inf (NaN and -inf are none), in order of falling logit, ties lowest index first.
//   w_i   = exp((z_i - z_max) / T)
//   top-k   keeps the first k;  top-p the shortest prefix whose sum reaches p * (sum of the top-k set);  min-p those with
//   w_i >= m (the largest weight is 1).  All three are prefixes of the one order, so the kept set is the shortest of them.
//   token = the first candidate whose running sum exceeds u * (sum of the kept set);  prob = its w / that sum.
//
// A long row is never sorted: every decision is "the first position where the running count or weight passes a target", and a
// radix search over the sortable bits of the logit finds it -- a histogram of count or weight over the top bits, the bin in which
// the target falls, the next bits inside that bin; at the last bits all members of a bin are equal and share one weight.
//
// Weights are 64-bit fixed point, w * 2^S rounded, with S such that V of them cannot overflow: integer sums do not depend on
// their order, so a row gives the same token however it is divided among lanes and workgroups (and by whatever order its
// atomics come in), and at 2^-41 or finer they decide as 64-bit floating point would (a 32-bit running sum over a large
// vocabulary is off by more than the distance between two neighbouring tokens' borders).
//
// Three forms, by the length of a row (sizes measured at the entry point below): one wave sorts a row of up to 256 logits by
// counting; one workgroup keeps a row of up to 32768 as keys in LDS; longer ones go through four launches in which slices of a
// row work side by side and meet in a histogram and a list of the few logits that can still decide.
#include "common.h"
#include "../../include/cube_hip.h"

namespace {

// ---- logits as sortable bits ----------------------------------------------------------------------------------------------

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float as_float(bf16_t v) { return (float)v; }

// a larger logit has a larger key; 0 for what is no candidate (the smallest candidate has key 0x00800000).  -0 and +0 are one
// value (v + 0 makes them so).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return v > -INFINITY ? k : 0u;  // false for NaN too
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

template <class T> struct Granule { static constexpr int N = 16 / sizeof(T); };  // logits in 16 bytes

// The 16-byte granules of a row, counted from the aligned address at or before its first logit: granule j holds the logits
// j*N - lead .. j*N - lead + N - 1.  Whole ones are loaded at once; the first and the last element by element, so that nothing
// outside the row is read.  out: keys, 0 for what lies outside.
template <class T> struct Row {
  const T* at; int V, lead, granules;
  __device__ Row(const T* row, int v) : at(row), V(v) {
    lead = (int)(((uintptr_t)row & 15) / sizeof(T));
    granules = (V + lead + Granule<T>::N - 1) / Granule<T>::N;
  }
  __device__ __forceinline__ void keys(int j, uint32_t (&out)[Granule<T>::N]) const {
    constexpr int N = Granule<T>::N;
    typedef T vec __attribute__((ext_vector_type(N)));
    const int i0 = j * N - lead;
    if (i0 >= 0 && i0 + N <= V) {
      const vec v = *(const vec*)(at + i0);
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = key_of(as_float(v[i]));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = i0 + i >= 0 && i0 + i < V ? key_of(as_float(at[i0 + i])) : 0u;
    }
  }
};

// ---- settings and weights -------------------------------------------------------------------------------------------------

struct Settings {
  float temp, p, m; int k; double u;
  __device__ Settings(const cube_sample_args& a, int r) {
    temp = a.temperature ? a.temperature[r] : a.temperature0;
    k = a.top_k ? a.top_k[r] : a.top_k0;
    p = a.top_p ? a.top_p[r] : a.top_p0;
    m = a.min_p ? a.min_p[r] : a.min_p0;
    const double x = a.u[r];
    u = x > 0.0 ? (x < 1.0 ? x : 1.0) : 0.0;
  }
  __device__ bool greedy() const { return !(temp > 0.0f); }
  __device__ bool limited(int V) const { return k > 0 && k < V; }
  // first position whose running sum passes this target ends the top-p set of a total
  __device__ uint64_t goal(uint64_t total) const {
    const double g = ceil((p > 0.0f ? (double)p : 0.0) * (double)total);
    return g >= 1.0 ? (uint64_t)g - 1 : 0;
  }
  __device__ uint64_t draw(uint64_t kept) const {
    const uint64_t t = (uint64_t)(u * (double)kept);
    return t < kept ? t : kept - 1;
  }
};

struct Weigher {
  double top, inv_t, floor_x;  // largest logit, 1 / T, ln(min-p)
  uint32_t top_key; int S;
  __device__ Weigher(const Settings& s, uint32_t best, int bits) : top_key(best), S(bits) {
    top = (double)value_of(best);
    inv_t = 1.0 / (double)s.temp;
    floor_x = s.m > 0.0f ? log(s.m < 1.0f ? (double)s.m : 1.0) : -INFINITY;
  }
  __device__ __forceinline__ double x(uint32_t key) const { return key == top_key ? 0.0 : ((double)value_of(key) - top) * inv_t; }
  // 2^shift * exp(x), x <= 0: 2^(n + f) with |f| <= 1/2, 2^f by the series of exp(f ln 2) to the 11th power (the 12th is below
  // 2^-47 of the value).  NaN (0 * inf: an infinite temperature beside an infinite logit) counts as -1100, nothing.
  __device__ __forceinline__ double power(double x, int shift) const {
    const double y = fmax(x, -1100.0) * 1.4426950408889634;
    const double n = rint(y);
    const double f = (y - n) * 0.6931471805599453;
    double e = 1.0 / 39916800.0;
    e = fma(e, f, 1.0 / 3628800.0);
    e = fma(e, f, 1.0 / 362880.0);
    e = fma(e, f, 1.0 / 40320.0);
    e = fma(e, f, 1.0 / 5040.0);
    e = fma(e, f, 1.0 / 720.0);
    e = fma(e, f, 1.0 / 120.0);
    e = fma(e, f, 1.0 / 24.0);
    e = fma(e, f, 1.0 / 6.0);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return ldexp(e, (int)n + shift);
  }
  // to an integer: at 2^52 a double's last place is 1, and its low bits are the sum (S <= 46)
  __device__ __forceinline__ uint64_t at(double x) const {
    return (uint64_t)__double_as_longlong(power(x, S) + 4503599627370496.0) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ uint64_t operator()(uint32_t key) const { return at(x(key)); }
  __device__ float prob(uint32_t key, uint64_t kept) const { return (float)(power(x(key), S) / (double)kept); }
};

// ---- wave and workgroup helpers -------------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)v, src, 64) | ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(v >> 32), src, 64) << 32);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const uint32_t t = (uint32_t)__shfl_xor((int)v, o, 64); v = t > v ? t : v; }
  return v;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += shfl64(v, (threadIdx.x & 63) ^ o);
  return v;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const uint64_t t = shfl64(v, lane >= o ? lane - o : lane); v += lane >= o ? t : 0; }
  return v;
}

constexpr int D1 = 11, D2 = 10;  // bits of the first two digits of a key within a workgroup; the third has the rest
constexpr int LOW_BINS = 1 << D2;

struct Scratch {  // of a workgroup, in LDS
  uint64_t high[1 << D1];   // first digit
  uint64_t low[LOW_BINS];   // second digit (64-bit sums), third digit (twice as many 32-bit counts)
  uint64_t part[16];
  uint32_t part32[16];
  uint64_t before;
  uint32_t bin;
};
static_assert(sizeof(Scratch) % 16 == 0, "keys behind it are read 16 bytes at a time");

template <int WG> __device__ uint32_t block_max(Scratch& s, uint32_t v) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) s.part32[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WG / 64; ++i) v = s.part32[i] > v ? s.part32[i] : v;
  __syncthreads();
  return v;
}
template <int WG> __device__ uint64_t block_sum(Scratch& s, uint64_t v) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < WG / 64; ++i) v += s.part[i];
  __syncthreads();
  return v;
}

// Bins from the top one down, a run of neighbours per thread: what lies before this thread's run, and in it.
struct Runs { uint64_t before, sum, total; };
template <int WG, int BINS, class G> __device__ Runs scan_bins(Scratch& s, G get) {
  static_assert(BINS % WG == 0, "whole runs");
  constexpr int C = BINS / WG;
  Runs r;
  r.sum = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) r.sum += get(BINS - 1 - (int)threadIdx.x * C - c);
  const uint64_t incl = wave_scan(r.sum);
  if ((threadIdx.x & 63) == 63) s.part[threadIdx.x >> 6] = incl;
  __syncthreads();
  r.before = incl - r.sum;
  r.total = 0;
#pragma unroll
  for (int i = 0; i < WG / 64; ++i) {
    if (i < (int)(threadIdx.x >> 6)) r.before += s.part[i];
    r.total += s.part[i];
  }
  __syncthreads();
  return r;
}
// the bin in which the running sum passes target - base (base + total > target), and base + what lies before it
struct Found { uint32_t bin; uint64_t before; };
template <int WG, int BINS, class G> __device__ Found find_bin(Scratch& s, const Runs& r, uint64_t base, uint64_t target, G get) {
  constexpr int C = BINS / WG;
  uint64_t before = base + r.before;
  if (before <= target && target < before + r.sum) {
    int b = BINS - 1 - (int)threadIdx.x * C;
    for (int c = 0; c < C; ++c, --b) {
      const uint64_t v = get(b);
      if (target < before + v) break;
      before += v;
    }
    s.bin = b;
    s.before = before;
  }
  __syncthreads();
  const Found f = {s.bin, s.before};
  __syncthreads();
  return f;
}

// Inside the bin `bin` of the first `DIG1` bits: the key at which the running count (COUNT) or weight passes `target`, the place of
// the position among the logits equal to it, and how many those are.  each(f) calls f(key) for every logit of the bin at least.
struct Place { uint32_t key, tie, ties; uint64_t before, one; __device__ uint64_t end() const { return before + (uint64_t)(tie + 1) * one; } };
template <int WG, int DIG1, bool COUNT, class E>
__device__ Place refine(Scratch& s, E each, const Weigher& w, uint32_t bin, uint64_t before, uint64_t target) {
  constexpr int D3 = 32 - DIG1 - D2;
  static_assert((4 << D3) <= (int)sizeof(s.low), "the third digit's counts fit");
  for (int b = threadIdx.x; b < LOW_BINS; b += WG) s.low[b] = 0;
  __syncthreads();
  each([&](uint32_t k) {
    if (k >> (32 - DIG1) == bin) atomicAdd((unsigned long long*)&s.low[(k >> D3) & (LOW_BINS - 1)], (unsigned long long)(COUNT ? 1 : w(k)));
  });
  __syncthreads();
  auto second = [&](int b) { return s.low[b]; };
  const Found f = find_bin<WG, LOW_BINS>(s, scan_bins<WG, LOW_BINS>(s, second), before, target, second);
  const uint32_t prefix = (bin << D2) | f.bin;
  uint32_t* cnt = (uint32_t*)s.low;
  for (int b = threadIdx.x; b < (1 << D3); b += WG) cnt[b] = 0;
  __syncthreads();
  each([&](uint32_t k) { if (k >> D3 == prefix) atomicAdd(&cnt[k & ((1 << D3) - 1)], 1u); });
  __syncthreads();
  auto third = [&](int b) { return cnt[b] ? (uint64_t)cnt[b] * (COUNT ? 1 : w((prefix << D3) | (uint32_t)b)) : 0; };
  const Found h = find_bin<WG, 1 << D3>(s, scan_bins<WG, 1 << D3>(s, third), f.before, target, third);
  Place at;
  at.key = (prefix << D3) | h.bin;
  at.one = COUNT ? 1 : w(at.key);
  at.before = h.before;
  at.tie = (uint32_t)((target - h.before) / at.one);
  at.ties = cnt[h.bin];
  __syncthreads();
  return at;
}

// A row's whole decision by one workgroup: which key, the how-manieth of the logits equal to it, and the kept sum.
struct Choice { uint32_t key, tie; uint64_t kept; };
template <int WG, class E> __device__ Choice decide(Scratch& s, E each, const Settings& st, const Weigher& w, int V) {
  auto first = [&](int b) { return s.high[b]; };
  uint32_t least = 1;      // keys below it are outside the top-k set
  uint64_t surplus = 0;    // weight of the logits equal to the last of the top-k set that are outside it
  if (st.limited(V)) {
    for (int b = threadIdx.x; b < (1 << D1); b += WG) s.high[b] = 0;
    __syncthreads();
    each([&](uint32_t k) { if (k) atomicAdd((unsigned long long*)&s.high[k >> (32 - D1)], 1ull); });
    __syncthreads();
    const Runs r = scan_bins<WG, 1 << D1>(s, first);
    if ((uint64_t)st.k < r.total) {
      const uint64_t t = (uint64_t)st.k - 1;
      const Found f = find_bin<WG, 1 << D1>(s, r, 0, t, first);
      const Place at = refine<WG, D1, true>(s, each, w, f.bin, f.before, t);
      least = at.key;
      surplus = (uint64_t)(at.ties - at.tie - 1) * w(at.key);
    }
  }
  for (int b = threadIdx.x; b < (1 << D1); b += WG) s.high[b] = 0;
  __syncthreads();
  uint64_t heavy = 0;  // weight of those that min-p keeps
  each([&](uint32_t k) {
    if (k >= least) {
      const double x = w.x(k);
      const uint64_t v = w.at(x);
      if (v) atomicAdd((unsigned long long*)&s.high[k >> (32 - D1)], (unsigned long long)v);
      if (x >= w.floor_x) heavy += v;
    }
  });
  __syncthreads();
  const Runs r = scan_bins<WG, 1 << D1>(s, first);
  const uint64_t total = r.total - surplus;
  uint64_t kept = total;
  if (st.p < 1.0f) {
    const uint64_t t = st.goal(total);
    if (t < total) {
      const Found f = find_bin<WG, 1 << D1>(s, r, 0, t, first);
      const uint64_t end = refine<WG, D1, false>(s, each, w, f.bin, f.before, t).end();
      kept = end < kept ? end : kept;
    }
  }
  if (st.m > 0.0f) {
    heavy = block_sum<WG>(s, heavy);
    kept = heavy < kept ? heavy : kept;
  }
  const uint64_t t = st.draw(kept);
  const Found f = find_bin<WG, 1 << D1>(s, r, 0, t, first);
  const Place at = refine<WG, D1, false>(s, each, w, f.bin, f.before, t);
  return {at.key, at.tie, kept};
}

// ---- up to 256 logits: one wave a row ---------------------------------------------------------------------------------------
// A logit's place in the order is the number of logits before it: every lane counts for its E logits against all of them (broadcast
// reads).  Then a lane holds E neighbouring places, and sums and searches are wave scans.
constexpr int SHORT_V = 256;
template <class T, int E>
__global__ __launch_bounds__(256) void sample_short_kernel(cube_sample_args a, int S) {
  __shared__ __attribute__((aligned(16))) uint32_t s_key[4][64 * E];
  __shared__ uint32_t s_order[4][64 * E], s_sorted[4][64 * E];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, V = a.V;
  const long long r = (long long)blockIdx.x * 4 + wave;
  if (r >= a.M) return;  // no workgroup barrier below
  const T* row = (const T*)a.logits + r * a.ld;
  const Settings st(a, (int)r);
  uint32_t key[E], best = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane + 64 * e;
    key[e] = i < V ? key_of(as_float(row[i])) : 0u;
    best = key[e] > best ? key[e] : best;
    s_key[wave][i] = key[e];
  }
  best = wave_max(best);
  if (best == 0) {
    if (lane == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (st.greedy()) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned long long hit = __ballot(key[e] == best);
      if (hit) {
        if (lane == 0) { a.token[r] = 64 * e + __ffsll(hit) - 1; if (a.prob) a.prob[r] = 1.0f; }
        return;
      }
    }
  }
  // places: before an equal key of its own 64 come those of lower lanes, of earlier 64s all, of later 64s none
  int place[E];
#pragma unroll
  for (int e = 0; e < E; ++e) place[e] = 0;
  const int n4 = (V + 3) / 4;
#pragma unroll
  for (int c = 0; c < E; ++c) {
    for (int q = 16 * c; q < (n4 < 16 * c + 16 ? n4 : 16 * c + 16); ++q) {
      const uint4 o = *(const uint4*)&s_key[wave][4 * q];
      const uint32_t other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 4 * (q - 16 * c) + i;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t mine = e > c ? key[e] : e < c ? key[e] + 1 : key[e] + (at >= lane ? 1u : 0u);
          place[e] += other[i] >= mine ? 1 : 0;
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane + 64 * e;
    s_sorted[wave][i] = 0;
    s_order[wave][i] = 0;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (key[e]) { s_sorted[wave][place[e]] = key[e]; s_order[wave][place[e]] = lane + 64 * e; }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();

  const Weigher w(st, best, S);
  const bool limited = st.limited(V);
  uint32_t q[E];
  uint64_t wt[E], run[E], sum = 0;
  double x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int pos = lane * E + e;
    q[e] = s_sorted[wave][pos];
    x[e] = w.x(q[e]);
    wt[e] = q[e] && !(limited && pos >= st.k) ? w.at(x[e]) : 0;
    sum += wt[e];
    run[e] = sum;
  }
  const uint64_t incl = wave_scan(sum), before = incl - sum;
  const uint64_t total = shfl64(incl, 63);
  uint64_t kept = total;
  const uint64_t goal = st.goal(total);
  if (st.p < 1.0f || st.m > 0.0f) {
    uint64_t mine = 0;  // running sum at the last place of this lane that stays
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t c = before + run[e];
      const bool stays = wt[e] && (!(st.p < 1.0f) || c - wt[e] <= goal) && (!(st.m > 0.0f) || x[e] >= w.floor_x);
      mine = stays ? c : mine;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const uint64_t t = shfl64(mine, lane ^ o); mine = t > mine ? t : mine; }
    kept = mine;
  }
  const uint64_t t = st.draw(kept);
  if (before <= t && t < incl) {  // one lane
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t c = before + run[e];
      if (c - wt[e] <= t && t < c) {
        a.token[r] = (int)s_order[wave][lane * E + e];
        if (a.prob) a.prob[r] = w.prob(q[e], kept);
      }
    }
  }
}

// ---- up to 32768 logits: one workgroup a row, keys in LDS -------------------------------------------------------------------
constexpr int MID_V = 32768;

// every thread four neighbouring keys at a time; n4: a multiple of four
template <int WG> struct LdsKeys {
  const uint32_t* keys; int n4;
  template <class F> __device__ __forceinline__ void operator()(F f) const {
    for (int i = 4 * (int)threadIdx.x; i < n4; i += 4 * WG) {
      const uint4 k = *(const uint4*)&keys[i];
      f(k.x); f(k.y); f(k.z); f(k.w);
    }
  }
};

template <class T, int WG>
__global__ __launch_bounds__(WG) void sample_mid_kernel(cube_sample_args a, int S) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Scratch& s = *(Scratch*)smem;
  uint32_t* keys = (uint32_t*)(smem + sizeof(Scratch));
  constexpr int N = Granule<T>::N;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const Settings st(a, r);
  uint32_t best = 0;
  for (int j = threadIdx.x; j < row.granules; j += WG) {
    uint32_t k[N];
    row.keys(j, k);
#pragma unroll
    for (int i = 0; i < N; i += 4) *(uint4*)&keys[j * N + i] = make_uint4(k[i], k[i + 1], k[i + 2], k[i + 3]);
#pragma unroll
    for (int i = 0; i < N; ++i) best = k[i] > best ? k[i] : best;
  }
  best = block_max<WG>(s, best);  // its barriers also make the keys visible
  if (best == 0) {
    if (threadIdx.x == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  const int n4 = row.granules * N;
  const LdsKeys<WG> each = {keys, n4};
  Choice c = {best, 0, 0};
  float prob = 1.0f;
  if (!st.greedy()) {
    const Weigher w(st, best, S);
    c = decide<WG>(s, each, st, w, a.V);
    prob = w.prob(c.key, c.kept);
  }
  // the c.tie-th key equal to c.key in order of index: each wave counts its span (256 keys a step), the owner walks its own
  const int steps = (n4 + 255) / 256, per = (steps + WG / 64 - 1) / (WG / 64);
  const int lo = wave * per, hi = lo + per < steps ? lo + per : steps;
  auto ties4 = [&](int step, uint32_t (&k)[4]) {  // this lane's four keys of a step: how many are equal
    const int i = step * 256 + 4 * lane;
    const uint4 v = i < n4 ? *(const uint4*)&keys[i] : make_uint4(0, 0, 0, 0);
    k[0] = v.x; k[1] = v.y; k[2] = v.z; k[3] = v.w;
    return (v.x == c.key) + (v.y == c.key) + (v.z == c.key) + (v.w == c.key);
  };
  uint32_t mine = 0, k[4];
  for (int i = lo; i < hi; ++i) mine += ties4(i, k);
  mine = (uint32_t)wave_sum(mine);
  if (lane == 0) s.part32[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < wave; ++i) before += s.part32[i];
  if (c.tie < before || c.tie >= before + mine) return;
  for (int i = lo; i < hi; ++i) {
    const uint32_t n = ties4(i, k);
    const uint32_t incl = (uint32_t)wave_scan(n), all = (uint32_t)shfl64(incl, 63);
    if (c.tie < before + all) {
      uint32_t at = before + incl - n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k[e] == c.key) {
          if (at == c.tie) { a.token[r] = i * 256 + 4 * lane + e - row.lead; if (a.prob) a.prob[r] = prob; }
          ++at;
        }
      return;
    }
    before += all;
  }
}

// ---- longer rows: slices side by side ---------------------------------------------------------------------------------------
// 1 largest key of every slice, and the row's histogram cleared;  2 histogram of the first 12 bits over the row: counts for a
// top-k row, weights for another;  3 the bins in which the targets can fall are known: their logits into the row's list;
// 4 one workgroup decides from the list and the histogram.  A list that runs over (very many equal logits) sends the fourth
// launch over the whole row instead.
constexpr int DL = 12, LONG_BINS = 1 << DL;
constexpr int LIST = 16384;
constexpr int LWG = 1024;
constexpr int ROWS_AT_ONCE = 256;  // rows of one pass of the four launches: bounds the workspace
constexpr int MAX_SLICES = 256;

struct LongRow {  // of the workspace
  uint64_t hist[LONG_BINS];
  uint64_t list[LIST];  // key << 32 | index
  uint64_t heavy;       // weight of those that min-p keeps
  uint32_t top[MAX_SLICES];
  uint32_t listed;
};

__device__ __forceinline__ uint32_t row_top(const LongRow& l, int slices, Scratch& s) {
  return block_max<LWG>(s, (int)threadIdx.x < slices ? l.top[threadIdx.x] : 0u);
}

template <class T>
__global__ __launch_bounds__(LWG) void long_top_kernel(cube_sample_args a, int r0, LongRow* rows, int per) {
  __shared__ uint32_t part[LWG / 64];
  constexpr int N = Granule<T>::N;
  const int r = r0 + blockIdx.y, slices = gridDim.x;
  LongRow& l = rows[blockIdx.y];
  for (int b = blockIdx.x * LWG + threadIdx.x; b < LONG_BINS; b += slices * LWG) l.hist[b] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) { l.heavy = 0; l.listed = 0; }
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  uint32_t best = 0;
#pragma unroll 4
  for (int j = lo + threadIdx.x; j < hi; j += LWG) {
    uint32_t k[N];
    row.keys(j, k);
#pragma unroll
    for (int i = 0; i < N; ++i) best = k[i] > best ? k[i] : best;
  }
  best = wave_max(best);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x < 64) {
    best = wave_max(threadIdx.x < LWG / 64 ? part[threadIdx.x] : 0u);
    if (threadIdx.x == 0) l.top[blockIdx.x] = best;
  }
}

template <class T>
__global__ __launch_bounds__(LWG) void long_hist_kernel(cube_sample_args a, int r0, LongRow* rows, int per, int S) {
  __shared__ uint64_t hist[LONG_BINS];
  __shared__ Scratch s;
  constexpr int N = Granule<T>::N;
  const int r = r0 + blockIdx.y;
  LongRow& l = rows[blockIdx.y];
  const Settings st(a, r);
  const uint32_t best = row_top(l, gridDim.x, s);
  if (best == 0 || st.greedy()) return;
  for (int b = threadIdx.x; b < LONG_BINS; b += LWG) hist[b] = 0;
  __syncthreads();
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  if (st.limited(a.V)) {
    for (int j = lo + threadIdx.x; j < hi; j += LWG) {
      uint32_t k[N];
      row.keys(j, k);
#pragma unroll
      for (int i = 0; i < N; ++i) if (k[i]) atomicAdd((unsigned long long*)&hist[k[i] >> (32 - DL)], 1ull);
    }
  } else {
    const Weigher w(st, best, S);
    uint64_t heavy = 0;
    for (int j = lo + threadIdx.x; j < hi; j += LWG) {
      uint32_t k[N];
      row.keys(j, k);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (k[i]) {
          const double x = w.x(k[i]);
          const uint64_t v = w.at(x);
          if (v) atomicAdd((unsigned long long*)&hist[k[i] >> (32 - DL)], (unsigned long long)v);
          if (x >= w.floor_x) heavy += v;
        }
      }
    }
    if (st.m > 0.0f) {
      heavy = wave_sum(heavy);
      if ((threadIdx.x & 63) == 0 && heavy) atomicAdd((unsigned long long*)&l.heavy, (unsigned long long)heavy);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < LONG_BINS; b += LWG)
    if (hist[b]) atomicAdd((unsigned long long*)&l.hist[b], (unsigned long long)hist[b]);
}

// What the histogram of a row without a top-k limit leaves open: the bin that ends the top-p set (if that can be the shortest
// prefix), and the bins among which the drawn position lies.
struct Open { bool ends; Found end; uint64_t goal, least, most; uint32_t from, to; };
template <class G> __device__ Open open_bins(Scratch& s, const Runs& r, const Settings& st, uint64_t heavy, G get) {
  Open o;
  o.ends = false;
  o.least = o.most = r.total;
  if (st.p < 1.0f) {
    o.goal = st.goal(r.total);
    if (o.goal < r.total) {
      o.ends = true;
      o.end = find_bin<LWG, LONG_BINS>(s, r, 0, o.goal, get);
      o.least = o.goal + 1;  // the set's sum is at least the goal and at most the end of the bin
      o.most = o.end.before + get(o.end.bin);
    }
  }
  if (st.m > 0.0f) {
    if (heavy <= o.least) o.ends = false;
    o.least = heavy < o.least ? heavy : o.least;
    o.most = heavy < o.most ? heavy : o.most;
  }
  o.from = find_bin<LWG, LONG_BINS>(s, r, 0, st.draw(o.least), get).bin;
  o.to = o.least == o.most ? o.from : find_bin<LWG, LONG_BINS>(s, r, 0, st.draw(o.most), get).bin;
  return o;
}

template <class T>
__global__ __launch_bounds__(LWG) void long_list_kernel(cube_sample_args a, int r0, LongRow* rows, int per) {
  __shared__ Scratch s;
  constexpr int N = Granule<T>::N;
  const int r = r0 + blockIdx.y, lane = threadIdx.x & 63;
  LongRow& l = rows[blockIdx.y];
  const Settings st(a, r);
  const uint32_t best = row_top(l, gridDim.x, s);
  if (best == 0) return;
  // keys in [a0, a1] or [b0, b1] are listed
  uint32_t a0 = best, a1 = best, b0 = 1, b1 = 0;
  if (!st.greedy()) {
    auto get = [&](int b) { return l.hist[b]; };
    const Runs runs = scan_bins<LWG, LONG_BINS>(s, get);
    a1 = 0xffffffffu;
    if (st.limited(a.V)) {
      a0 = 1;
      if ((uint64_t)st.k < runs.total) a0 = find_bin<LWG, LONG_BINS>(s, runs, 0, (uint64_t)st.k - 1, get).bin << (32 - DL);
    } else {
      const Open o = open_bins(s, runs, st, l.heavy, get);
      a0 = o.to << (32 - DL);
      a1 = (o.from << (32 - DL)) | ((1u << (32 - DL)) - 1);
      if (o.ends) { b0 = o.end.bin << (32 - DL); b1 = b0 | ((1u << (32 - DL)) - 1); }
    }
  }
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  for (int j0 = lo; j0 < hi; j0 += LWG) {
    const int j = j0 + threadIdx.x;
    uint32_t k[N], n = 0;
    bool in[N];
    if (j < hi) {
      row.keys(j, k);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) k[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      in[i] = (k[i] >= a0 && k[i] <= a1) || (k[i] >= b0 && k[i] <= b1);
      n += in[i];
    }
    if (__ballot(n != 0) == 0) continue;
    const uint32_t incl = (uint32_t)wave_scan(n);
    uint32_t base = 0;
    if (lane == 63) base = atomicAdd(&l.listed, incl);
    uint32_t at = (uint32_t)__shfl((int)base, 63, 64) + incl - n;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) {
        if (at < LIST) l.list[at] = ((uint64_t)k[i] << 32) | (uint32_t)(j * N + i - row.lead);
        ++at;
      }
  }
}

// the listed logits of a row, or all of them
struct ListKeys {
  const uint64_t* list; int n;
  template <class F> __device__ __forceinline__ void operator()(F f) const {
    for (int i = threadIdx.x; i < n; i += LWG) f((uint32_t)(list[i] >> 32));
  }
};
template <class T> struct RowKeys {
  const Row<T>& row;
  template <class F> __device__ __forceinline__ void operator()(F f) const {
    constexpr int N = Granule<T>::N;
    for (int j = threadIdx.x; j < row.granules; j += LWG) {
      uint32_t k[N];
      row.keys(j, k);
#pragma unroll
      for (int i = 0; i < N; ++i) f(k[i]);
    }
  }
};

template <class T>
__global__ __launch_bounds__(LWG) void long_choose_kernel(cube_sample_args a, int r0, LongRow* rows, int slices, int S) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Scratch& s = *(Scratch*)smem;
  uint64_t* list = (uint64_t*)(smem + sizeof(Scratch));
  const int r = r0 + blockIdx.x;
  LongRow& l = rows[blockIdx.x];
  const Settings st(a, r);
  const uint32_t best = row_top(l, slices, s);
  if (best == 0) {
    if (threadIdx.x == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const bool whole = l.listed > LIST;  // the list ran over: decide from the row itself
  const int n = whole ? 0 : (int)l.listed;
  for (int i = threadIdx.x; i < n; i += LWG) list[i] = l.list[i];
  __syncthreads();
  Choice c = {best, 0, 0};
  float prob = 1.0f;
  if (!st.greedy()) {
    const Weigher w(st, best, S);
    const ListKeys some = {list, n};
    if (whole) {
      c = decide<LWG>(s, RowKeys<T>{row}, st, w, a.V);
    } else if (st.limited(a.V)) {
      c = decide<LWG>(s, some, st, w, a.V);
    } else {
      auto get = [&](int b) { return l.hist[b]; };
      const Runs runs = scan_bins<LWG, LONG_BINS>(s, get);
      const Open o = open_bins(s, runs, st, l.heavy, get);
      uint64_t kept = o.most;
      if (o.ends) {
        const uint64_t end = refine<LWG, DL, false>(s, some, w, o.end.bin, o.end.before, o.goal).end();
        kept = end < kept ? end : kept;
      }
      const uint64_t t = st.draw(kept);
      const Found f = find_bin<LWG, LONG_BINS>(s, runs, 0, t, get);
      const Place at = refine<LWG, DL, false>(s, some, w, f.bin, f.before, t);
      c = {at.key, at.tie, kept};
    }
    prob = w.prob(c.key, c.kept);
  }
  // the c.tie-th smallest index among the logits equal to c.key: two digits of 11 bits of the index, from below
  uint32_t prefix = 0, left = c.tie;
#pragma unroll
  for (int shift = 11; shift >= 0; shift -= 11) {
    for (int b = threadIdx.x; b < 2048; b += LWG) s.high[b] = 0;
    __syncthreads();
    auto add = [&](uint32_t i) {
      if (shift == 11 || i >> 11 == prefix) atomicAdd((unsigned long long*)&s.high[2047 - ((i >> shift) & 2047)], 1ull);
    };
    if (whole) {
      constexpr int N = Granule<T>::N;
      for (int j = threadIdx.x; j < row.granules; j += LWG) {
        uint32_t k[N];
        row.keys(j, k);
#pragma unroll
        for (int i = 0; i < N; ++i) if (k[i] == c.key) add((uint32_t)(j * N + i - row.lead));
      }
    } else {
      for (int i = threadIdx.x; i < n; i += LWG) if ((uint32_t)(list[i] >> 32) == c.key) add((uint32_t)list[i]);
    }
    __syncthreads();
    auto get = [&](int b) { return s.high[b]; };
    const Found f = find_bin<LWG, 2048>(s, scan_bins<LWG, 2048>(s, get), 0, left, get);
    prefix = (prefix << 11) | (2047 - f.bin);
    left -= (uint32_t)f.before;
  }
  if (threadIdx.x == 0) { a.token[r] = (int)prefix; if (a.prob) a.prob[r] = prob; }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------

template <class T> int launch_short(const cube_sample_args& a, int S, hipStream_t st) {
  const dim3 grid((a.M + 3) / 4), block(256);
  if (a.V <= 64) hipLaunchKernelGGL((sample_short_kernel<T, 1>), grid, block, 0, st, a, S);
  else if (a.V <= 128) hipLaunchKernelGGL((sample_short_kernel<T, 2>), grid, block, 0, st, a, S);
  else hipLaunchKernelGGL((sample_short_kernel<T, 4>), grid, block, 0, st, a, S);
  CUBE_CHECK_LAUNCH("cube_sample_rows");
  return CUBE_OK;
}

template <class T, int WG> int launch_mid(const cube_sample_args& a, int S, hipStream_t st) {
  static CubeLdsReservation lds;
  const size_t bytes = sizeof(Scratch) + 4 * (size_t)((a.V + 2 * Granule<T>::N + 3) / 4 * 4);
  if (!lds.ensure((const void*)sample_mid_kernel<T, WG>, bytes)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_sample_rows: LDS reservation failed");
  hipLaunchKernelGGL((sample_mid_kernel<T, WG>), dim3(a.M), dim3(WG), bytes, st, a, S);
  CUBE_CHECK_LAUNCH("cube_sample_rows");
  return CUBE_OK;
}

template <class T> int launch_long(const cube_sample_args& a, int S, LongRow* ws, hipStream_t st) {
  static CubeLdsReservation lds;
  const size_t bytes = sizeof(Scratch) + 8 * LIST;
  if (!lds.ensure((const void*)long_choose_kernel<T>, bytes)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_sample_rows: LDS reservation failed");
  const int granules = (a.V + 2 * Granule<T>::N - 2) / Granule<T>::N;  // of the longest row (one that starts inside a granule)
  for (int r0 = 0; r0 < a.M; r0 += ROWS_AT_ONCE) {
    const int n = a.M - r0 < ROWS_AT_ONCE ? a.M - r0 : ROWS_AT_ONCE;
    // slices of one granule a thread at least, about two workgroups a CU over all rows
    int slices = (granules + LWG - 1) / LWG;
    const int want = (512 + n - 1) / n;
    slices = slices < want ? slices : want;
    slices = slices < MAX_SLICES ? slices : MAX_SLICES;
    const int per = (granules + slices - 1) / slices;
    const dim3 grid(slices, n);
    hipLaunchKernelGGL((long_top_kernel<T>), grid, dim3(LWG), 0, st, a, r0, ws, per);
    hipLaunchKernelGGL((long_hist_kernel<T>), grid, dim3(LWG), 0, st, a, r0, ws, per, S);
    hipLaunchKernelGGL((long_list_kernel<T>), grid, dim3(LWG), 0, st, a, r0, ws, per);
    hipLaunchKernelGGL((long_choose_kernel<T>), dim3(n), dim3(LWG), bytes, st, a, r0, ws, slices, S);
    CUBE_CHECK_LAUNCH("cube_sample_rows");
  }
  return CUBE_OK;
}

bool is_long(int M, int V) { return V > MID_V; }

template <class T> int launch(const cube_sample_args& a, int S, void* ws, hipStream_t st) {
  if (a.V <= SHORT_V) return launch_short<T>(a, S, st);
  if (is_long(a.M, a.V)) return launch_long<T>(a, S, (LongRow*)ws, st);
  // 256 threads keep several rows on a CU; above 4096 logits a row's own passes are what takes time
  return a.V <= 4096 ? launch_mid<T, 256>(a, S, st) : launch_mid<T, 1024>(a, S, st);
}

}  // namespace

extern "C" size_t cube_sample_workspace_bytes(int M, int V) {
  if (M <= 0 || V <= 0 || V > CUBE_SAMPLE_MAX_V || !is_long(M, V)) return 0;
  return sizeof(LongRow) * (size_t)(M < ROWS_AT_ONCE ? M : ROWS_AT_ONCE);
}

extern "C" int cube_sample_rows(const cube_sample_args* a, void* ws, size_t ws_bytes, void* stream) {
  CUBE_ENTRY();
  if (!a) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: null args");
  if (a->M < 0 || a->V < 1 || a->V > CUBE_SAMPLE_MAX_V) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: M=%d, V=%d outside 1..%d", a->M, a->V, CUBE_SAMPLE_MAX_V);
  if (a->M == 0) return CUBE_OK;
  if (!a->logits || !a->u || !a->token) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: null logits / u / token");
  if (a->type < CUBE_T_F32 || a->type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: type=%d", a->type);
  if (a->ld < a->V) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: ld=%lld < V=%d", a->ld, a->V);
  if ((uintptr_t)a->logits % (a->type == CUBE_T_F32 ? 4 : 2) || ((uintptr_t)a->u & 7) ||
      (((uintptr_t)a->token | (uintptr_t)a->prob | (uintptr_t)a->temperature | (uintptr_t)a->top_k | (uintptr_t)a->top_p | (uintptr_t)a->min_p) & 3))
    CUBE_FAIL(CUBE_ERR_ALIGN, "cube_sample_rows: a pointer is not aligned to its type");
  const size_t need = cube_sample_workspace_bytes(a->M, a->V);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: workspace of %zu bytes (need %zu, 16-byte aligned)", ws_bytes, need);
  int bits = 0;
  while ((1 << bits) < a->V) ++bits;
  const int S = 62 - bits < 46 ? 62 - bits : 46;  // V weights of at most 2^S stay below 2^63
  hipStream_t st = (hipStream_t)stream;
  if (a->type == CUBE_T_F32) return launch<float>(*a, S, ws, st);
  if (a->type == CUBE_T_BF16) return launch<bf16_t>(*a, S, ws, st);
  return launch<_Float16>(*a, S, ws, st);
}
