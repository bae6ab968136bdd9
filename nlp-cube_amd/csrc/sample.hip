// Sampling one token a row from logits with temperature, top-k, top-p and min-p, from given random numbers (gfx950).
//
// Candidates of a row are its logits above -inf (NaN and -inf are none), in order of falling logit, ties lowest index first.
//   w_i   = exp((z_i - z_max) / T)
//   top-k   keeps the first k;  top-p the shortest prefix whose sum reaches p * (sum of the top-k set);  min-p those with
//   w_i >= m (the largest weight is 1).  All three are prefixes of the one order, so the kept set is the shortest of them.
//   token = the first candidate whose running sum exceeds u * (sum of the kept set);  prob = its w / that sum.
//
// A long row is never sorted: every decision is "the first position where the running count or weight passes a target".  A histogram
// in the candidates' order (equal steps of the logit, or the values of a 16-bit type) has the running sums; the few logits of the bin
// in which the target falls are sorted.  Where they are not few, a radix search over the sortable bits of the logit goes on inside
// it: at the last bits all members of a bin are equal and share one weight.
//
// Weights are integers, w * 2^62 cut off, and their sums have 96 bits: sums of integers do not depend on their order, so a row gives
// the same token however it is divided among lanes and workgroups (and by whatever order its atomics come in).  V cut weights are off
// by less than V * 2^-62 of the largest, 2^-40 for the longest row (64-bit sums leave a weight 62 - log2 V bits, and put a flat tail of
// 2^22 logits off by up to 2^-19 of the mass, hundreds of tokens' shares; they take 64 x 32003 25 us where these take 28, 128 x 250002
// f32 110 where these take 120).  Up to 256 logits, w * 2^46 rounded and sums of 64 bits do: 256 * 2^-47 = 2^-39.
//
// Forms, by the length and type of a row (sizes measured at the entry point below):
//   short   up to 256 logits: one wave sorts the row by counting;
//   mid     one workgroup keeps the row as keys in LDS; a histogram over equal steps of the logit, then the members of the one bin
//           that matters are sorted;
//   half    16-bit logits have 65536 values: a workgroup counts every value of a row (or of a slice of it) in LDS, and everything
//           is decided from the counts, with one exponential for each value that occurs;
//   long    f32 and few f16 rows: slices of a row meet in a histogram and in a list of the few logits that can still decide.
#include <type_traits>

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
// outside the row is read.  What lies outside comes as -inf, no candidate.
template <class T> struct Row {
  const T* at; int V, lead, granules;
  __device__ Row(const T* row, int v) : at(row), V(v) {
    lead = (int)(((uintptr_t)row & 15) / sizeof(T));
    granules = (V + lead + Granule<T>::N - 1) / Granule<T>::N;
  }
  __device__ __forceinline__ void values(int j, float (&out)[Granule<T>::N]) const {
    constexpr int N = Granule<T>::N;
    typedef T vec __attribute__((ext_vector_type(N)));
    const int i0 = j * N - lead;
    if (i0 >= 0 && i0 + N <= V) {
      const vec v = *(const vec*)(at + i0);
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = as_float(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = i0 + i >= 0 && i0 + i < V ? as_float(at[i0 + i]) : -INFINITY;
    }
  }
};

// ---- sums of weights ------------------------------------------------------------------------------------------------------

struct Sum {  // 96 bits
  uint64_t lo; uint32_t hi;
  Sum() = default;
  __device__ __forceinline__ constexpr Sum(uint64_t l, uint32_t h = 0) : lo(l), hi(h) {}
};
// word by word with the carry: comparisons of 64 bits take more than the additions
__device__ __forceinline__ uint64_t add64(uint64_t a, uint64_t b, uint32_t& carry) {
  uint32_t c;
  const uint32_t l = __builtin_addc((uint32_t)a, (uint32_t)b, 0u, &c);
  const uint32_t h = __builtin_addc((uint32_t)(a >> 32), (uint32_t)(b >> 32), c, &carry);
  return (uint64_t)h << 32 | l;
}
__device__ __forceinline__ Sum operator+(Sum a, Sum b) {
  uint32_t c;
  const uint64_t l = add64(a.lo, b.lo, c);
  return {l, a.hi + b.hi + c};
}
__device__ __forceinline__ Sum subtract(Sum a, Sum b, uint32_t& borrow) {
  uint32_t c, d;
  const uint32_t l = __builtin_subc((uint32_t)a.lo, (uint32_t)b.lo, 0u, &c);
  const uint32_t h = __builtin_subc((uint32_t)(a.lo >> 32), (uint32_t)(b.lo >> 32), c, &d);
  const uint32_t t = __builtin_subc(a.hi, b.hi, d, &borrow);
  return {(uint64_t)h << 32 | l, t};
}
__device__ __forceinline__ Sum operator-(Sum a, Sum b) { uint32_t c; return subtract(a, b, c); }
__device__ __forceinline__ bool operator<(Sum a, Sum b) { uint32_t c; subtract(a, b, c); return c != 0; }
__device__ __forceinline__ Sum& operator+=(Sum& a, Sum b) { return a = a + b; }
__device__ __forceinline__ bool operator<=(Sum a, Sum b) { return !(b < a); }
__device__ __forceinline__ bool operator==(Sum a, Sum b) { return a.lo == b.lo && a.hi == b.hi; }
__device__ __forceinline__ uint64_t choose(bool c, uint64_t a, uint64_t b) { return c ? a : b; }
__device__ __forceinline__ Sum choose(bool c, Sum a, Sum b) { return {c ? a.lo : b.lo, c ? a.hi : b.hi}; }  // (c ? a : b of structures is one of two addresses)
template <class V> __device__ __forceinline__ V smaller(V a, V b) { return choose(b < a, b, a); }
__device__ __forceinline__ Sum times(uint32_t n, uint64_t w) {
  const uint64_t p = (uint64_t)n * (uint32_t)w, q = (uint64_t)n * (uint32_t)(w >> 32) + (p >> 32);
  return {(q << 32) | (uint32_t)p, (uint32_t)(q >> 32)};
}
__device__ __forceinline__ double to_double(uint64_t s) { return (double)s; }
__device__ __forceinline__ double to_double(Sum s) { return fma((double)s.hi, 18446744073709551616.0, (double)s.lo); }
// the whole part of 0 <= d < 2^96
template <class V> __device__ __forceinline__ V whole(double d);
template <> __device__ __forceinline__ uint64_t whole<uint64_t>(double d) { return (uint64_t)d; }
template <> __device__ __forceinline__ Sum whole<Sum>(double d) {
  const uint32_t hi = (uint32_t)(d * 5.421010862427522e-20);  // 2^-64
  return {(uint64_t)fma((double)hi, -18446744073709551616.0, d), hi};
}
// d / one, where that is a number of logits
__device__ __forceinline__ uint32_t quotient(Sum d, uint64_t one) {
  uint32_t q = (uint32_t)(to_double(d) / (double)one);
  if (d < times(q, one)) --q;
  else if (times(q + 1, one) <= d) ++q;
  return q;
}
// a sum that many threads add to: the 64 bits, and what was carried out of them
__device__ __forceinline__ void add_to(uint64_t* lo, uint32_t* hi, uint64_t w) {
  const uint64_t old = atomicAdd((unsigned long long*)lo, (unsigned long long)w);
  if (old + w < old) atomicAdd(hi, 1u);
}
__device__ __forceinline__ void add_to(uint64_t* lo, uint32_t* hi, Sum w) {
  uint32_t c;
  add64(atomicAdd((unsigned long long*)lo, (unsigned long long)w.lo), w.lo, c);
  if (w.hi + c) atomicAdd(hi, w.hi + c);
}

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
  template <class V> __device__ V goal(V total) const {
    const double g = ceil((p > 0.0f ? (double)p : 0.0) * to_double(total));
    return choose(g >= 1.0, whole<V>(g) - V(1), V(0));
  }
  template <class V> __device__ V draw(V kept) const {
    const V t = whole<V>(u * to_double(kept));
    return choose(t < kept, t, kept - V(1));
  }
};

struct Weigher {
  double top, per_t, floor_x;  // largest logit, log2(e) / T, log2(min-p)
  // An infinite logit beside an infinite largest one has weight 1 and every other none: the largest finite double in place of the
  // infinity makes their differences infinite and -1.8e308, and parts() ends the range on both sides.
  __device__ Weigher(const Settings& s, float best) {
    top = fmin((double)best, 1.7976931348623157e308);
    per_t = fmax(1.4426950408889634 / (double)s.temp, 1e-290);
    floor_x = s.m > 0.0f ? log2(s.m < 1.0f ? (double)s.m : 1.0) : -INFINITY;
  }
  __device__ __forceinline__ double x(float v) const { return ((double)v - top) * per_t; }  // log2 of the weight
  // 2^x = e * 2^n: x = n + f with |f| <= 1/2 (adding 1.5 * 2^52 rounds x to n and leaves n in the low bits), e = 2^f = 1 + f * P(f),
  // P of the 9th degree through (2^f - 1) / f at the Chebyshev nodes (2^-50 of the value).  What is no candidate (NaN, -inf) comes
  // out at 2^-960, as nothing.
  __device__ __forceinline__ double parts(double x, int& n) const {
    const double y = fmin(fmax(x, -960.0), 0.0);
    const double t = y + 6755399441055744.0;
    const double f = y - (t - 6755399441055744.0);
    double e = 7.070977866508139e-09;
    e = fma(e, f, 1.0205905413765595e-07);
    e = fma(e, f, 1.3215451633221434e-06);
    e = fma(e, f, 1.5252672924850737e-05);
    e = fma(e, f, 0.00015403530424776529);
    e = fma(e, f, 0.0013333558200794592);
    e = fma(e, f, 0.009618129107618665);
    e = fma(e, f, 0.05550410866465167);
    e = fma(e, f, 0.24022650695910075);
    e = fma(e, f, 0.6931471805599462);
    e = fma(e, f, 1.0);
    n = __double2loint(t);
    return e;
  }
  __device__ __forceinline__ double power(double x, int shift) const {  // 2^(x + shift): added to the exponent bits
    int n;
    const double e = parts(x, n);
    return __hiloint2double(__double2hiint(e) + ((n + shift) << 20), __double2loint(e));
  }
  // 2^(x + 62) cut off: the fraction of e with its leading 1 in bit 62, moved down by what is missing to the exponent 62 (rounded
  // through two additions of large powers of two the middle form took 3 % more time)
  __device__ __forceinline__ uint64_t at(double x) const {
    int n;
    const double e = parts(x, n);
    const uint32_t hi = (uint32_t)__double2hiint(e), lo = (uint32_t)__double2loint(e);
    const uint64_t f = ((uint64_t)((__builtin_amdgcn_alignbit(hi, lo, 22) & 0x3fffffffu) | 0x40000000u) << 32) | (lo << 10);
    const int down = 1023 - n - (int)(hi >> 20);
    return f >> (down < 63 ? down : 63);
  }
  __device__ __forceinline__ uint64_t of(float v) const { return at(x(v)); }
  __device__ __forceinline__ uint64_t operator()(uint32_t key) const { return of(value_of(key)); }
  // the same for sums of up to 256 weights in 64 bits, 2^(x + 46) rounded: at 2^52 a double's last place is 1, and its low bits are the sum
  __device__ __forceinline__ uint64_t few(double x) const {
    return (uint64_t)__double_as_longlong(power(x, 46) + 4503599627370496.0) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ float prob(float v, Sum kept) const { return (float)(power(x(v), 62) / to_double(kept)); }
  __device__ __forceinline__ float prob(float v, uint64_t kept) const { return (float)(power(x(v), 46) / (double)kept); }
};

// ---- wave and workgroup helpers -------------------------------------------------------------------------------------------

// Sums and maxima over a wave through DPP moves (whole waves only; a cross-lane LDS shuffle takes some ten times as long): shifts
// within rows of 16 lanes, then a row's last lane to the row behind it, then lane 31 to the upper half.  What has no source is 0.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t from_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t from_lane(uint64_t v) {
  return (uint64_t)from_lane<CTRL, ROWS>((uint32_t)v) | ((uint64_t)from_lane<CTRL, ROWS>((uint32_t)(v >> 32)) << 32);
}
template <int CTRL, int ROWS> __device__ __forceinline__ Sum from_lane(Sum v) { return {from_lane<CTRL, ROWS>(v.lo), from_lane<CTRL, ROWS>(v.hi)}; }
template <class V> __device__ __forceinline__ V wave_scan(V v) {  // inclusive
  v += from_lane<0x111, 0xf>(v);
  v += from_lane<0x112, 0xf>(v);
  v += from_lane<0x114, 0xf>(v);
  v += from_lane<0x118, 0xf>(v);
  v += from_lane<0x142, 0xa>(v);
  v += from_lane<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }  // lane: uniform
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  return (uint64_t)lane_value((uint32_t)v, lane) | ((uint64_t)lane_value((uint32_t)(v >> 32), lane) << 32);
}
__device__ __forceinline__ Sum lane_value(Sum v, int lane) { return {lane_value(v.lo, lane), lane_value(v.hi, lane)}; }
template <class V> __device__ __forceinline__ V wave_sum(V v) { return lane_value(wave_scan(v), 63); }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <class V> __device__ __forceinline__ V larger(V a, V b) { return choose(b < a, a, b); }
template <class V> __device__ __forceinline__ V wave_max(V v) {
  v = larger(v, from_lane<0x111, 0xf>(v));
  v = larger(v, from_lane<0x112, 0xf>(v));
  v = larger(v, from_lane<0x114, 0xf>(v));
  v = larger(v, from_lane<0x118, 0xf>(v));
  v = larger(v, from_lane<0x142, 0xa>(v));
  v = larger(v, from_lane<0x143, 0xc>(v));
  return lane_value(v, 63);
}

constexpr int D1 = 11, D2 = 10;  // bits of the first two digits of a key within a workgroup; the third has the rest
constexpr int LOW_BINS = 1 << D2;

struct alignas(16) Scratch {  // of a workgroup, in LDS
  uint64_t high[1 << D1];   // first digit, or steps of the logit
  uint64_t low[LOW_BINS];   // second digit (64-bit sums), third digit (twice as many 32-bit counts)
  Sum part[16];
  Sum before, in;
  uint32_t part32[16];
  uint32_t bin;
  // What sums of weights carry out of 64 bits lies in the other array: `low` is idle while `high` is filled, and a thread takes its bins
  // of `high` into registers (hold) before `low` is filled.
  __device__ uint32_t* high_carry() { return (uint32_t*)low; }
  __device__ uint32_t* low_carry() { return (uint32_t*)high; }
};
static_assert(sizeof(Scratch) % 16 == 0, "keys behind it are read 16 bytes at a time");
static_assert(sizeof(Scratch::low) >= (4 << D1) && sizeof(Scratch::high) >= 4 * LOW_BINS, "room for the carries");

template <int WG> __device__ uint32_t block_max(Scratch& s, uint32_t v) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) s.part32[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WG / 64; ++i) v = s.part32[i] > v ? s.part32[i] : v;
  __syncthreads();
  return v;
}
// the running sums (inclusive) of a workgroup's waves, lane l: waves 0 .. l
template <int WG, class V> __device__ __forceinline__ V over_waves(const V* part) {
  static_assert(WG / 64 <= 16, "one row of lanes");
  const int lane = threadIdx.x & 63;
  V v = part[lane < WG / 64 ? lane : 0];
  v = choose(lane < WG / 64, v, V(0));
  v += from_lane<0x111, 0xf>(v);
  v += from_lane<0x112, 0xf>(v);
  if constexpr (WG / 64 > 4) {
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
  }
  return v;
}
template <int WG> __device__ Sum block_sum(Scratch& s, Sum v) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = over_waves<WG>(s.part);
  __syncthreads();
  return lane_value(v, WG / 64 - 1);
}

// A histogram's bins in the candidates' order in registers, a run of neighbours per thread: what is in each, what lies before the run,
// in it, and in all.  UP: the order is from the first bin up, else from the last one down.
template <class V, int C> struct Held { V v[C]; V before, sum, total; };
template <bool UP, int BINS> __device__ __forceinline__ int bin_at(int place) { return UP ? place : BINS - 1 - place; }
template <int WG, int BINS, bool UP, class G> __device__ auto hold(Scratch& s, G get) {
  static_assert(BINS % WG == 0, "whole runs");
  constexpr int C = BINS / WG;
  typedef decltype(get(0)) V;
  Held<V, C> r;
  r.sum = V(0);
#pragma unroll
  for (int c = 0; c < C; ++c) r.sum += r.v[c] = get(bin_at<UP, BINS>((int)threadIdx.x * C + c));
  const V incl = wave_scan(r.sum);
  V* part = (V*)s.part;
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = incl;
  __syncthreads();
  const V waves = over_waves<WG>(part);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  r.before = lane_value(waves, wave) - part[wave] + (incl - r.sum);
  r.total = lane_value(waves, WG / 64 - 1);
  __syncthreads();
  return r;
}
// the bin in which the running sum passes target - base (base + total > target), base + what lies before it, and what is in it
template <class V> struct Found { uint32_t bin; V before, in; };
template <int WG, int BINS, bool UP, class V, int C> __device__ Found<V> find_bin(Scratch& s, const Held<V, C>& r, V base, V target) {
  static_assert(C == BINS / WG, "");
  V before = base + r.before;
  if (before <= target && target < before + r.sum) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (before <= target && target < before + r.v[c]) {
        s.bin = (uint32_t)bin_at<UP, BINS>((int)threadIdx.x * C + c);
        *(V*)&s.before = before;
        *(V*)&s.in = r.v[c];
      }
      before += r.v[c];
    }
  }
  __syncthreads();
  const Found<V> f = {s.bin, *(const V*)&s.before, *(const V*)&s.in};
  __syncthreads();
  return f;
}

// Inside the bin `bin` of the first `DIG1` bits: the key at which the running count (COUNT) or weight passes `target`, the place of
// the position among the logits equal to it, and how many those are.  each(f) calls f(key) for every logit of the bin at least.
struct Place { uint32_t key, tie, ties; Sum before; uint64_t one; __device__ Sum end() const { return before + times(tie + 1, one); } };
template <int WG, int DIG1, bool COUNT, class V, class E>
__device__ Place refine(Scratch& s, E each, const Weigher& w, uint32_t bin, V before, V target) {
  constexpr int D3 = 32 - DIG1 - D2;
  static_assert((4 << D3) <= (int)sizeof(s.low), "the third digit's counts fit");
  static_assert(std::is_same<V, typename std::conditional<COUNT, uint64_t, Sum>::type>::value, "");
  uint32_t* carry = s.low_carry();
  for (int b = threadIdx.x; b < LOW_BINS; b += WG) { s.low[b] = 0; if (!COUNT) carry[b] = 0; }
  __syncthreads();
  each([&](uint32_t k) {
    if (k >> (32 - DIG1) == bin) {
      const uint32_t at = (k >> D3) & (LOW_BINS - 1);
      if constexpr (COUNT) atomicAdd((unsigned long long*)&s.low[at], 1ull);
      else add_to(&s.low[at], &carry[at], w(k));
    }
  });
  __syncthreads();
  const Found<V> f = find_bin<WG, LOW_BINS, false>(s, hold<WG, LOW_BINS, false>(s, [&](int b) {
    if constexpr (COUNT) return s.low[b];
    else return Sum(s.low[b], carry[b]);
  }), before, target);
  const uint32_t prefix = (bin << D2) | f.bin;
  uint32_t* cnt = (uint32_t*)s.low;
  for (int b = threadIdx.x; b < (1 << D3); b += WG) cnt[b] = 0;
  __syncthreads();
  each([&](uint32_t k) { if (k >> D3 == prefix) atomicAdd(&cnt[k & ((1 << D3) - 1)], 1u); });
  __syncthreads();
  const Found<V> h = find_bin<WG, 1 << D3, false>(s, hold<WG, 1 << D3, false>(s, [&](int b) {
    if constexpr (COUNT) return (uint64_t)cnt[b];
    else return times(cnt[b], cnt[b] ? w((prefix << D3) | (uint32_t)b) : 0);
  }), f.before, target);
  Place at;
  at.key = (prefix << D3) | h.bin;
  at.ties = cnt[h.bin];
  if constexpr (COUNT) {
    at.one = 1;
    at.before = 0;
    at.tie = (uint32_t)(target - h.before);
  } else {
    at.one = w(at.key);
    at.before = h.before;
    at.tie = quotient(target - h.before, at.one);
  }
  __syncthreads();
  return at;
}

// A row's whole decision by one workgroup: which key, the how-manieth of the logits equal to it, and the kept sum.
struct Choice { uint32_t key, tie; Sum kept; };
template <int WG, class E> __device__ Choice decide(Scratch& s, E each, const Settings& st, const Weigher& w, int V) {
  constexpr int BINS = 1 << D1;
  uint32_t least = 1;      // keys below it are outside the top-k set
  Sum surplus = 0;         // weight of the logits equal to the last of the top-k set that are outside it
  if (st.limited(V)) {
    for (int b = threadIdx.x; b < BINS; b += WG) s.high[b] = 0;
    __syncthreads();
    each([&](uint32_t k) { if (k) atomicAdd((unsigned long long*)&s.high[k >> (32 - D1)], 1ull); });
    __syncthreads();
    const auto r = hold<WG, BINS, false>(s, [&](int b) { return s.high[b]; });
    if ((uint64_t)st.k < r.total) {
      const uint64_t t = (uint64_t)st.k - 1;
      const Found<uint64_t> f = find_bin<WG, BINS, false>(s, r, (uint64_t)0, t);
      const Place at = refine<WG, D1, true>(s, each, w, f.bin, f.before, t);
      least = at.key;
      surplus = times(at.ties - at.tie - 1, w(at.key));
    }
  }
  uint32_t* carry = s.high_carry();
  for (int b = threadIdx.x; b < BINS; b += WG) { s.high[b] = 0; carry[b] = 0; }
  __syncthreads();
  Sum heavy = 0;  // weight of those that min-p keeps
  each([&](uint32_t k) {
    if (k >= least) {
      const double x = w.x(value_of(k));
      const uint64_t v = w.at(x);
      if (v) add_to(&s.high[k >> (32 - D1)], &carry[k >> (32 - D1)], v);
      if (x >= w.floor_x) heavy += v;
    }
  });
  __syncthreads();
  const auto r = hold<WG, BINS, false>(s, [&](int b) { return Sum(s.high[b], carry[b]); });
  const Sum total = r.total - surplus;
  Sum kept = total;
  if (st.p < 1.0f) {
    const Sum t = st.goal(total);
    if (t < total) {
      const Found<Sum> f = find_bin<WG, BINS, false>(s, r, Sum(0), t);
      const Sum end = refine<WG, D1, false>(s, each, w, f.bin, f.before, t).end();
      kept = smaller(end, kept);
    }
  }
  if (st.m > 0.0f) {
    heavy = block_sum<WG>(s, heavy);
    kept = smaller(heavy, kept);
  }
  const Sum t = st.draw(kept);
  const Found<Sum> f = find_bin<WG, BINS, false>(s, r, Sum(0), t);
  const Place at = refine<WG, D1, false>(s, each, w, f.bin, f.before, t);
  return {at.key, at.tie, kept};
}

// One wave, candidates in order: lane l has the places l*E .. l*E + E - 1 (key 0 behind the last).  All that a row needs beyond its
// first V is there, or st.k bounds it.  -> the chosen place.  W: the sums' type (uint64_t where the row has no more than these logits)
template <class W, int E> __device__ int choose_sorted(const uint32_t (&q)[E], const Settings& st, const Weigher& w, int V, float& prob) {
  static_assert(E <= 4, "");
  const int lane = threadIdx.x & 63;
  const bool limited = st.limited(V);
  uint64_t wt[E];
  W run[E], sum = W(0);
  double x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = w.x(value_of(q[e]));
    wt[e] = q[e] && !(limited && lane * E + e >= st.k) ? (std::is_same<W, Sum>::value ? w.at(x[e]) : w.few(x[e])) : 0;
    sum += wt[e];
    run[e] = sum;
  }
  const W incl = wave_scan(sum), before = incl - sum;
  const W total = lane_value(incl, 63);
  W kept = total;
  const W goal = st.goal(total);
  if (st.p < 1.0f || st.m > 0.0f) {
    W mine = W(0);  // running sum at the last place of this lane that stays
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const W c = before + run[e];
      const bool stays = wt[e] && (!(st.p < 1.0f) || c - wt[e] <= goal) && (!(st.m > 0.0f) || x[e] >= w.floor_x);
      mine = choose(stays, c, mine);
    }
    kept = wave_max(mine);
  }
  const W t = st.draw(kept);
  int at = 0;
  float pr = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const W c = before + run[e];
    if (c - wt[e] <= t && t < c) { at = lane * E + e; pr = w.prob(value_of(q[e]), kept); }
  }
  const int owner = __ffsll(__ballot(before <= t && t < incl)) - 1;
  prob = __uint_as_float(lane_value(__float_as_uint(pr), owner));
  return (int)lane_value((uint32_t)at, owner);
}

// ---- up to 256 logits: one wave a row ---------------------------------------------------------------------------------------
// A logit's place in the order is the number of logits before it: every lane counts for its E logits against all of them (broadcast
// reads).  Then a lane holds E neighbouring places, and sums and searches are wave scans.
constexpr int SHORT_V = 256;
template <class T, int E>
__global__ __launch_bounds__(256) void sample_short_kernel(cube_sample_args a) {
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
  }
  best = wave_max(best);
  if (best == 0) {
    if (lane == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
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
  // places: before an equal key of its own 64 come those of lower lanes, of earlier 64s all, of later 64s none.  A key of 16 bits has
  // room for its lane below them, so that none are equal.  Others are counted as if none were, and put right where two then have one
  // place (8192 x 102 f32: 12.6 us, 15.9 with the lanes compared in every step; 22 where all logits are equal).
  int place[E];
  uint32_t plain[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    place[e] = 0;
    plain[e] = key[e];
    if (sizeof(T) == 2 && key[e]) key[e] = (key[e] & ~255u) | (255u - (lane + 64 * e));
    s_key[wave][lane + 64 * e] = key[e];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int n4 = (V + 3) / 4;
#pragma unroll
  for (int c = 0; c < E; ++c) {
    for (int q = 16 * c; q < (n4 < 16 * c + 16 ? n4 : 16 * c + 16); ++q) {
      const uint4 o = *(const uint4*)&s_key[wave][4 * q];
      const uint32_t other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) place[e] += other[i] >= key[e] + (e > c ? 0u : 1u) ? 1 : 0;
    }
  }
  if constexpr (sizeof(T) == 4) {
    bool twice = false;
#pragma unroll
    for (int e = 0; e < E; ++e) if (key[e]) s_order[wave][place[e]] = lane + 64 * e;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < E; ++e) twice |= key[e] && s_order[wave][place[e]] != (uint32_t)(lane + 64 * e);
    if (__ballot(twice)) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
#pragma unroll 4
        for (int i = 0; i < 64; ++i) place[e] += i < lane && s_key[wave][64 * e + i] == key[e] ? 1 : 0;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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
    if (key[e]) { s_sorted[wave][place[e]] = plain[e]; s_order[wave][place[e]] = lane + 64 * e; }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();

  uint32_t q[E];
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = s_sorted[wave][lane * E + e];
  const Weigher w(st, value_of(best));
  float prob;
  const int at = choose_sorted<uint64_t>(q, st, w, V, prob);
  if (lane == 0) { a.token[r] = (int)s_order[wave][at]; if (a.prob) a.prob[r] = prob; }
}

// ---- lists of a few candidates ----------------------------------------------------------------------------------------------
// Entries are key << 32 | ~index: larger is earlier in the order.
constexpr int FEW = 256;
struct alignas(16) Few {  // in LDS
  uint64_t entry[FEW], sorted[FEW];
  uint32_t place[FEW];
  uint32_t n;
  uint32_t key, index;
  float prob;
  Sum end;
};
static_assert(sizeof(Few) % 16 == 0, "keys behind it are read 16 bytes at a time");
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t index) { return ((uint64_t)key << 32) | (uint32_t)~index; }
__device__ __forceinline__ void append(Few& f, uint64_t entry) {
  const uint32_t at = atomicAdd(&f.n, 1u);
  if (at < FEW) f.entry[at] = entry;
}
// sorts f.entry[0 .. n), n <= FEW, into f.sorted (0 behind): an entry's place is the number of larger ones; the workgroup's
// threads share the counting
template <int WG> __device__ void sort_few(Few& f) {
  const int n = (int)f.n;
  for (int i = threadIdx.x; i < FEW; i += WG) { f.sorted[i] = 0; f.place[i] = 0; }
  __syncthreads();
  constexpr int PARTS = WG / FEW;
  const int e = threadIdx.x % FEW, part = threadIdx.x / FEW;
  if (e < n) {
    const uint64_t mine = f.entry[e];
    uint32_t before = 0;
    for (int i = part; i < n; i += PARTS) before += f.entry[i] > mine ? 1 : 0;
    atomicAdd(&f.place[e], before);
  }
  __syncthreads();
  if ((int)threadIdx.x < n) f.sorted[f.place[threadIdx.x]] = f.entry[threadIdx.x];
  __syncthreads();
}
// One wave: in the sorted entries, with `before` in front of them, the first place whose running weight exceeds target (there is
// one) -> f.key, f.index, f.end (the running weight up to and with it)
__device__ void place_few(Few& f, const Weigher& w, Sum before, Sum target) {
  constexpr int E = FEW / 64;
  const int lane = threadIdx.x & 63;
  uint64_t q[E], wt[E];
  Sum sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = f.sorted[lane * E + e];
    wt[e] = q[e] ? w((uint32_t)(q[e] >> 32)) : 0;
    sum += wt[e];
  }
  Sum c = before + (wave_scan(sum) - sum);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (c <= target && target < c + wt[e]) {
      f.key = (uint32_t)(q[e] >> 32);
      f.index = ~(uint32_t)q[e];
      f.end = c + wt[e];
    }
    c += wt[e];
  }
}

// Equal steps of the logit below the largest one, 32 wide in all (32 T for temperatures above 1): in the region that matters a bin
// then holds few logits whatever their scale.  Falls monotonically with the key, so bins are in the candidates' order.
struct Steps {
  float top, scale; uint32_t last;
  __device__ Steps(float best, float temp, int bins) : top(best), last((uint32_t)bins - 1) { scale = (float)(bins / 32) / (temp > 1.0f ? temp : 1.0f); }
  __device__ __forceinline__ int operator()(float v) const {
    uint32_t b;  // the conversion ends at 2^32 - 1 and takes NaN (an infinite logit beside an infinite largest one)
                 // to 0: as an instruction, since in C++ both are undefined
    asm("v_cvt_u32_f32 %0, %1" : "=v"(b) : "v"((top - v) * scale));
    return (int)(b < last ? b : last);
  }
  __device__ __forceinline__ int operator()(uint32_t key) const { return (*this)(value_of(key)); }
};
// A span of bins as a span of logits, a little wider (2^-20 of the numbers it is computed from, where their roundings take 2^-22): two
// comparisons tell nearly all logits outside it, and the bins of the others are computed.
struct Span {
  float lo, hi; int from, to;
  __device__ Span(const Steps& step, int from_, int to_) : from(from_), to(to_) {
    const float slack = fabsf(step.top) * 9.6e-7f, least = step.top - (float)(to + 1) / step.scale * 1.000001f - slack;
    const float most = step.top - (float)from / step.scale * 0.999999f + slack;
    lo = to == (int)step.last || !(least >= -INFINITY) ? -INFINITY : least;  // (infinities: the span may come out empty-handed as NaN)
    hi = from == 0 || !(most >= -INFINITY) ? INFINITY : most;
  }
  __device__ __forceinline__ bool near(float v) const { return v >= lo && v <= hi; }  // false for NaN
  __device__ __forceinline__ bool has(const Steps& step, float v) const {
    const int b = step(v);
    return v > -INFINITY && b >= from && b <= to;
  }
};

// ---- mid: one workgroup a row, keys in LDS ----------------------------------------------------------------------------------
constexpr int MID_V = 32768;

// every thread four neighbouring logits at a time; n4: a multiple of four
template <int WG> struct LdsValues {
  const float* at; int n4;
  template <class F> __device__ __forceinline__ void fours(F f) const {
    for (int i = 4 * (int)threadIdx.x; i < n4; i += 4 * WG) {
      const f32x4 v = *(const f32x4*)&at[i];
      f({v[0], v[1], v[2], v[3]});
    }
  }
  template <class F> __device__ __forceinline__ void values(F f) const {
    fours([&](const float (&v)[4]) { f(v[0]); f(v[1]); f(v[2]); f(v[3]); });
  }
  template <class F> __device__ __forceinline__ void operator()(F f) const {
    values([&](float v) { f(key_of(v)); });
  }
  // f(value, index) for those in the span
  template <class F> __device__ __forceinline__ void inside(const Steps& step, const Span& span, F f) const {
    for (int i = 4 * (int)threadIdx.x; i < n4; i += 4 * WG) {
      const f32x4 v = *(const f32x4*)&at[i];
      if (span.near(v[0]) || span.near(v[1]) || span.near(v[2]) || span.near(v[3])) {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (span.has(step, v[e])) f(v[e], i + e);
      }
    }
  }
};
// The weights of many logits into a histogram over steps; MIN_P: and the sum of those that min-p keeps.  N at a time: an addition that
// says what was there before (for the carry) takes the LDS some hundred cycles, and these are on their way together.
template <bool MIN_P> struct Gather {
  const Weigher& w; const Steps& step; uint64_t* hist; uint32_t* carry; Sum& heavy;
  template <int N> __device__ __forceinline__ void operator()(const float (&v)[N]) const {
    uint64_t one[N], old[N];
    int b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double x = w.x(v[i]);
      one[i] = w.at(x);
      b[i] = step(v[i]);
      if (MIN_P && x >= w.floor_x) heavy += one[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      old[i] = 0;
      if (one[i]) old[i] = atomicAdd((unsigned long long*)&hist[b[i]], (unsigned long long)one[i]);  // (none for what is no candidate)
    }
    bool some = false;
#pragma unroll
    for (int i = 0; i < N; ++i) some |= old[i] + one[i] < old[i];
    if (some) {
#pragma unroll
      for (int i = 0; i < N; ++i) if (old[i] + one[i] < old[i]) atomicAdd(&carry[b[i]], 1u);
    }
  }
};

// The row's decision through the histogram over steps; false where more than FEW logits share the bin that matters (many equal
// ones, a very flat row, a top-k set of hundreds): nothing is decided then.
template <int WG, int BINS, class K>
__device__ bool decide_few(Scratch& s, Few& f, const K& keys, int lead, const Settings& st, const Weigher& w, uint32_t best, int V) {
  static_assert(BINS <= (1 << D1) && BINS % WG == 0, "the histogram lies in Scratch::high");
  const Steps step(value_of(best), st.temp, BINS);
  uint32_t* carry = s.high_carry();
  auto clear = [&] {
    for (int b = threadIdx.x; b < BINS; b += WG) { s.high[b] = 0; carry[b] = 0; }
    if (threadIdx.x == 0) f.n = 0;
    __syncthreads();
  };
  if (st.limited(V)) {
    clear();
    keys.values([&](float v) { if (v > -INFINITY) atomicAdd((unsigned long long*)&s.high[step(v)], 1ull); });
    __syncthreads();
    const auto r = hold<WG, BINS, true>(s, [&](int b) { return s.high[b]; });
    if ((uint64_t)st.k < r.total || r.total <= FEW) {
      uint32_t bin = BINS - 1;
      if ((uint64_t)st.k < r.total) {
        const Found<uint64_t> at = find_bin<WG, BINS, true>(s, r, (uint64_t)0, (uint64_t)st.k - 1);
        if (at.before + at.in > FEW) return false;
        bin = at.bin;
      }
      keys.inside(step, Span(step, 0, (int)bin), [&](float v, int i) { append(f, entry_of(key_of(v), (uint32_t)(i - lead))); });
      __syncthreads();
      sort_few<WG>(f);
      if (threadIdx.x < 64) {
        uint32_t q[FEW / 64];
#pragma unroll
        for (int e = 0; e < FEW / 64; ++e) q[e] = (uint32_t)(f.sorted[threadIdx.x * (FEW / 64) + e] >> 32);
        float prob;
        const int at = choose_sorted<Sum>(q, st, w, V, prob);
        if (threadIdx.x == 0) { f.index = ~(uint32_t)f.sorted[at]; f.prob = prob; }
      }
      __syncthreads();
      return true;
    }
    // no more candidates than k: not limited
  }
  clear();
  Sum heavy = 0;  // weight of those that min-p keeps
  if (st.m > 0.0f) keys.fours(Gather<true>{w, step, s.high, carry, heavy});
  else keys.fours(Gather<false>{w, step, s.high, carry, heavy});
  __syncthreads();
  const auto r = hold<WG, BINS, true>(s, [&](int b) { return Sum(s.high[b], carry[b]); });
  // the place in which the running weight passes a target: the members of its bin, sorted
  auto place = [&](Sum target) {
    const Found<Sum> at = find_bin<WG, BINS, true>(s, r, Sum(0), target);
    keys.inside(step, Span(step, (int)at.bin, (int)at.bin), [&](float v, int i) { append(f, entry_of(key_of(v), (uint32_t)(i - lead))); });
    __syncthreads();
    if (f.n > FEW) return false;
    sort_few<WG>(f);
    if (threadIdx.x < 64) place_few(f, w, at.before, target);
    __syncthreads();
    return true;
  };
  Sum kept = r.total;
  if (st.p < 1.0f) {
    const Sum t = st.goal(r.total);
    if (t < r.total) {
      if (!place(t)) return false;
      kept = f.end;
      __syncthreads();
      if (threadIdx.x == 0) f.n = 0;
      __syncthreads();
    }
  }
  if (st.m > 0.0f) {
    heavy = block_sum<WG>(s, heavy);
    kept = smaller(heavy, kept);
  }
  if (!place(st.draw(kept))) return false;
  if (threadIdx.x == 0) f.prob = w.prob(value_of(f.key), kept);
  __syncthreads();
  return true;
}

template <class T, int WG>
__global__ __launch_bounds__(WG) void sample_mid_kernel(cube_sample_args a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Scratch& s = *(Scratch*)smem;
  Few& few = *(Few*)(smem + sizeof(Scratch));
  float* keys = (float*)(smem + sizeof(Scratch) + sizeof(Few));
  constexpr int N = Granule<T>::N;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const Settings st(a, r);
  float largest = -INFINITY;
  for (int j = threadIdx.x; j < row.granules; j += WG) {
    float v[N];
    row.values(j, v);
#pragma unroll
    for (int i = 0; i < N; i += 4) *(f32x4*)&keys[j * N + i] = (f32x4){v[i], v[i + 1], v[i + 2], v[i + 3]};
#pragma unroll
    for (int i = 0; i < N; ++i) largest = fmaxf(largest, v[i]);  // (NaN is passed over)
  }
  const uint32_t best = block_max<WG>(s, key_of(largest));  // its barriers also make the logits visible
  if (best == 0) {
    if (threadIdx.x == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  const int n4 = row.granules * N;
  const LdsValues<WG> each = {keys, n4};
  Choice c = {best, 0, 0};
  float prob = 1.0f;
  if (!st.greedy()) {
    const Weigher w(st, value_of(best));
    if (decide_few<WG, WG == 256 ? 1024 : 2048>(s, few, each, row.lead, st, w, best, a.V)) {
      if (threadIdx.x == 0) { a.token[r] = (int)few.index; if (a.prob) a.prob[r] = few.prob; }
      return;
    }
    __syncthreads();
    c = decide<WG>(s, each, st, w, a.V);
    prob = w.prob(value_of(c.key), c.kept);
  }
  // the c.tie-th logit equal to that of c.key in order of index: each wave counts its span (256 a step), the owner walks its own
  const float chosen = value_of(c.key);
  const int steps = (n4 + 255) / 256, per = (steps + WG / 64 - 1) / (WG / 64);
  const int lo = wave * per, hi = lo + per < steps ? lo + per : steps;
  auto ties4 = [&](int step, float (&k)[4]) {  // this lane's four of a step: how many are equal
    const int i = step * 256 + 4 * lane;
    const f32x4 v = i < n4 ? *(const f32x4*)&keys[i] : (f32x4){-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    k[0] = v[0]; k[1] = v[1]; k[2] = v[2]; k[3] = v[3];
    return (v[0] == chosen) + (v[1] == chosen) + (v[2] == chosen) + (v[3] == chosen);
  };
  uint32_t mine = 0;
  float k[4];
  for (int i = lo; i < hi; ++i) mine += ties4(i, k);
  mine = wave_sum(mine);
  if (lane == 0) s.part32[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < wave; ++i) before += s.part32[i];
  if (c.tie < before || c.tie >= before + mine) return;
  for (int i = lo; i < hi; ++i) {
    const uint32_t n = ties4(i, k);
    const uint32_t incl = wave_scan(n), all = lane_value(incl, 63);
    if (c.tie < before + all) {
      uint32_t at = before + incl - n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k[e] == chosen) {
          if (at == c.tie) { a.token[r] = i * 256 + 4 * lane + e - row.lead; if (a.prob) a.prob[r] = prob; }
          ++at;
        }
      return;
    }
    before += all;
  }
}

// ---- half: 16-bit logits by the counts of their values ----------------------------------------------------------------------
// A slice's counts: one 32-bit word per magnitude (the 15 bits without the sign), the number of its logits in the low half and
// of its negative ones in the high half; a slice has at most 65528 logits, so neither runs over.  Groups of 64 * E magnitudes, E
// to a lane: an octave of bf16, half an octave of f16 (quarters of that, 128 x 250002: 88 us, these 61:
// a row then has 130 groups).
// In the candidates' order group g comes GROUPS - 1 - g-th for positive values, falling inside, and GROUPS + g-th for negative
// ones, rising.
constexpr int HWG = 1024;
constexpr int MAGS = 32768;
constexpr int MAX_GROUPS = 256;
constexpr int HALF_GRANULES = 8191;  // of 8 logits, per slice

template <class T> struct Half;
template <> struct Half<bf16_t> { static constexpr uint32_t INF = 0x7f80; static constexpr int E = 2; };
template <> struct Half<_Float16> { static constexpr uint32_t INF = 0x7c00; static constexpr int E = 8; };
template <class T> constexpr int half_groups() { return MAGS / (64 * Half<T>::E); }
template <class T> __device__ __forceinline__ float half_value(uint32_t raw) { return as_float(__builtin_bit_cast(T, (uint16_t)raw)); }

struct HalfSlice {  // of the workspace: the counts of the groups that `has` marks
  uint32_t count[MAGS];
  uint64_t has[MAX_GROUPS / 64];
};

// E neighbouring words
template <int E> struct Words { uint32_t v[E]; };
__device__ __forceinline__ Words<2> load_words(const uint32_t* p, Words<2>) {
  const uint2 c = *(const uint2*)p;
  return {{c.x, c.y}};
}
__device__ __forceinline__ Words<8> load_words(const uint32_t* p, Words<8>) {
  const uint4 a = *(const uint4*)p, b = *(const uint4*)(p + 4);
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}

// The granules lo .. hi - 1 of a row: f(word) for the two logits of each 32-bit word of the whole ones, g(raw) for the logits of the
// row's first and last granule where those are not whole.  Four loads of a thread are on their way together (with each followed by
// its use 128 x 250002 took 3 us more in all).
template <class T, class F, class G> __device__ __forceinline__ void half_words(const Row<T>& row, int lo, int hi, F f, G g) {
  const uint16_t* at = (const uint16_t*)row.at - row.lead;
  const int whole = (row.V + row.lead) / 8;
  const int from = lo == 0 && row.lead ? 1 : lo, to = hi < whole ? hi : whole;
  for (int j = from + (int)threadIdx.x; j < to; j += 4 * HWG) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *(const uint4*)(at + 8 * (j + u * HWG < to ? j + u * HWG : j));
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (j + u * HWG < to) { f(v[u].x); f(v[u].y); f(v[u].z); f(v[u].w); }
  }
  const int i = threadIdx.x;  // a logit each
  if (from != lo && i >= row.lead && i < 8 && i < row.lead + row.V) g(at[i]);
  if (hi > whole && whole >= from && i < row.V + row.lead - 8 * whole) g(at[8 * whole + i]);
}
// counts of granules lo .. hi - 1 into `count` (LDS)
template <class T> __device__ void count_half(uint32_t* count, const Row<T>& row, int lo, int hi) {
  for (int i = threadIdx.x; i < MAGS / 4; i += HWG) ((uint4*)count)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  auto one = [&](uint32_t raw) { atomicAdd(&count[raw & 0x7fffu], 1u + ((raw & 0x8000u) << 1)); };
  half_words(row, lo, hi, [&](uint32_t w) { one(w & 0xffffu); one(w >> 16); }, one);
  __syncthreads();
}
// marks of the groups that have a logit, a wave its own run of groups: into part (LDS), then has[0 .. GROUPS / 64); f(group, words) for
// each marked one
template <class T, class F> __device__ void mark_half(const uint32_t* count, uint32_t* part, uint64_t* has, F f) {
  constexpr int E = Half<T>::E, G = half_groups<T>() / (HWG / 64), WAVES = 64 / G;  // groups of a wave, waves of a word of `has`
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t mask = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int group = wave * G + g;
    const Words<E> c = load_words(count + (group * 64 + lane) * E, Words<E>{});
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) any |= c.v[i];
    if (__ballot(any != 0)) {
      mask |= 1u << g;
      f(group, c);
    }
  }
  if (lane == 0) part[wave] = mask;
  __syncthreads();
  if (threadIdx.x < half_groups<T>() / 64) {
    uint64_t h = 0;
    for (int i = 0; i < WAVES; ++i) h |= (uint64_t)part[WAVES * threadIdx.x + i] << (G * i);
    has[threadIdx.x] = h;
  }
}

template <class T>
__global__ __launch_bounds__(HWG) void half_count_kernel(cube_sample_args a, int r0, HalfSlice* ws, int per) {
  extern __shared__ __attribute__((aligned(16))) uint32_t count[];
  __shared__ uint32_t part[HWG / 64];
  constexpr int E = Half<T>::E;
  const int r = r0 + blockIdx.y, lane = threadIdx.x & 63;
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  HalfSlice& out = ws[(size_t)blockIdx.y * gridDim.x + blockIdx.x];
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  count_half(count, row, lo, hi);
  mark_half<T>(count, part, out.has, [&](int group, const Words<E>& c) {
    uint32_t* to = out.count + (group * 64 + lane) * E;
    if constexpr (E == 2) {
      *(uint2*)to = make_uint2(c.v[0], c.v[1]);
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 4) *(uint4*)(to + i) = make_uint4(c.v[i], c.v[i + 1], c.v[i + 2], c.v[i + 3]);
    }
  });
}

struct HalfScratch {  // in LDS
  Sum weight[2 * MAX_GROUPS];  // by order; after prefix_half: running sums
  uint32_t count[2 * MAX_GROUPS];
  uint64_t has[MAX_GROUPS / 64];
  uint64_t heavy;
  uint32_t heavy_carry;
  uint32_t raw, tie, ties, slice;
  float prob;
  uint32_t part[HWG / 64];
};

// Counts of a lane's E neighbouring magnitudes of a group: all and negative.  From LDS, or summed over the slices of the workspace
// (and kept in LDS for the groups of the first SLOTS marks: a search comes back to a group).
template <int E> struct Counts { uint32_t all[E], neg[E]; };
template <class T> struct LdsCounts {
  static constexpr int E = Half<T>::E;
  const uint32_t* count;
  __device__ __forceinline__ Counts<E> load(int g) const {
    const Words<E> c = load_words(count + (g * 64 + (threadIdx.x & 63)) * E, Words<E>{});
    Counts<E> r;
#pragma unroll
    for (int i = 0; i < E; ++i) { r.all[i] = c.v[i] & 0xffffu; r.neg[i] = c.v[i] >> 16; }
    return r;
  }
  __device__ __forceinline__ Counts<E> again(const HalfScratch&, int g) const { return load(g); }
  __device__ __forceinline__ void keep(const HalfScratch&, int, const Counts<E>&) const {}
};
constexpr int HALF_SLICES = 96;  // of a row, at most: 65 cover 2^22 logits
constexpr int KEPT_BYTES = 128 * 1024;
template <class T> struct SliceCounts {
  static constexpr int E = Half<T>::E, SLOTS = KEPT_BYTES / (64 * E * 8), BATCH = 32 / E;
  const HalfSlice* slice; int n;
  const uint64_t (*has)[MAX_GROUPS / 64];  // of every slice, in LDS
  uint32_t* kept;                          // [SLOTS][2 * E][64], in LDS
  __device__ __forceinline__ int slot(const HalfScratch& s, int g) const {  // marked groups before g
    int r = 0;
    for (int i = 0; i < (g >> 6); ++i) r += __popcll(s.has[i]);
    return r + __popcll(s.has[g >> 6] & ((1ull << (g & 63)) - 1));
  }
  __device__ __forceinline__ Counts<E> load(int g) const {
    const int lane = threadIdx.x & 63, at = (g * 64 + lane) * E;
    Counts<E> r;
#pragma unroll
    for (int i = 0; i < E; ++i) r.all[i] = r.neg[i] = 0;
    for (int i0 = 0; i0 < n; i0 += 64) {
      uint64_t left = __ballot(i0 + lane < n && ((has[i0 + lane < n ? i0 + lane : i0][g >> 6] >> (g & 63)) & 1));
      while (left) {  // several slices' loads at a time
        Words<E> c[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          c[u] = {};
          if (left) {
            c[u] = load_words(slice[i0 + __ffsll((long long)left) - 1].count + at, Words<E>{});
            left &= left - 1;
          }
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
#pragma unroll
          for (int i = 0; i < E; ++i) { r.all[i] += c[u].v[i] & 0xffffu; r.neg[i] += c[u].v[i] >> 16; }
      }
    }
    return r;
  }
  __device__ __forceinline__ void keep(const HalfScratch& s, int g, const Counts<E>& c) const {
    const int at = slot(s, g);
    if (at >= SLOTS) return;
    uint32_t* to = kept + at * 2 * E * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < E; ++i) { to[2 * i * 64] = c.all[i]; to[(2 * i + 1) * 64] = c.neg[i]; }
  }
  __device__ __forceinline__ Counts<E> again(const HalfScratch& s, int g) const {
    const int at = slot(s, g);
    if (at >= SLOTS) return load(g);
    const uint32_t* from = kept + at * 2 * E * 64 + (threadIdx.x & 63);
    Counts<E> r;
#pragma unroll
    for (int i = 0; i < E; ++i) { r.all[i] = from[2 * i * 64]; r.neg[i] = from[(2 * i + 1) * 64]; }
    return r;
  }
};
template <class T> __device__ __forceinline__ uint32_t half_raw(int g, bool neg, int i) {
  return (uint32_t)((g * 64 + ((int)threadIdx.x & 63)) * Half<T>::E + i) | (neg ? 0x8000u : 0u);
}
// the candidates among them: negative counts for `neg` (below the infinity), positive ones else (up to it; zero takes both signs)
template <class T> __device__ __forceinline__ void valid(int g, bool neg, const Counts<Half<T>::E>& p, uint32_t (&c)[Half<T>::E]) {
#pragma unroll
  for (int i = 0; i < Half<T>::E; ++i) {
    const uint32_t mag = half_raw<T>(g, false, i);
    if (neg) c[i] = mag != 0 && mag < Half<T>::INF ? p.neg[i] : 0;
    else c[i] = mag == 0 ? p.all[i] : mag <= Half<T>::INF ? p.all[i] - p.neg[i] : 0;
  }
}
template <int E> __device__ __forceinline__ uint32_t sum_of(const uint32_t (&c)[E]) {
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) s += c[i];
  return s;
}
template <class T> __device__ __forceinline__ int group_of(int order) {
  return order < half_groups<T>() ? half_groups<T>() - 1 - order : order - half_groups<T>();
}

// One wave: counts and weights by order become running sums
template <class T> __device__ __forceinline__ void prefix_half(HalfScratch& s) {
  constexpr int R = 2 * half_groups<T>() / 64;
  const int lane = threadIdx.x & 63;
  uint32_t c[R], cs = 0;
  Sum w[R], ws = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    cs += s.count[lane * R + i];
    ws += s.weight[lane * R + i];
    c[i] = cs;
    w[i] = ws;
  }
  cs = wave_scan(cs) - cs;
  ws = wave_scan(ws) - ws;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    s.count[lane * R + i] = cs + c[i];
    s.weight[lane * R + i] = ws + w[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct Spot { uint32_t raw, tie, ties; Sum before; uint64_t one; __device__ Sum end() const { return before + times(tie + 1, one); } };
// One wave: the value at which the running count (BY_COUNT) or weight passes target (the total does); before, one: weights
template <class T, bool BY_COUNT, class C> __device__ Spot spot_half(const HalfScratch& s, const C& counts, const Weigher& w, Sum target) {
  const int lane = threadIdx.x & 63;
  constexpr int E = Half<T>::E, R = 2 * half_groups<T>() / 64;
  // 64 running sums, R apart, then the R between them
  auto sum = [&](int i) { return BY_COUNT ? Sum(s.count[i]) : s.weight[i]; };
  int order = R * (__ffsll(__ballot(target < sum(lane * R + R - 1))) - 1);
  order += __ffsll(__ballot(lane < R && target < sum(order + (lane < R ? lane : 0)))) - 1;
  Sum bc(order > 0 ? s.count[order - 1] : 0), bw = choose(order > 0, s.weight[order > 0 ? order - 1 : 0], Sum(0));
  const bool neg = order >= half_groups<T>();
  const int g = group_of<T>(order);
  uint32_t c[E];
  valid<T>(g, neg, counts.again(s, g), c);
  Sum v[E], sw = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    v[i] = times(c[i], c[i] ? w.of(half_value<T>(half_raw<T>(g, neg, i))) : 0);
    sw += v[i];
  }
  // in falling order: negative values as they lie, positive ones from the other end
  const uint32_t sc = sum_of(c), ic = wave_scan(sc);
  const Sum iw = wave_scan(sw);
  bc += neg ? ic - sc : lane_value(ic, 63) - ic;
  bw += choose(neg, iw - sw, lane_value(iw, 63) - iw);
  Spot out = {0, 0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const uint32_t ci = neg ? c[j] : c[E - 1 - j];
    const Sum vi = choose(neg, v[j], v[E - 1 - j]);
    const Sum here = choose(BY_COUNT, bc, bw), mine = choose(BY_COUNT, Sum(ci), vi);
    if (here <= target && target < here + mine) {
      out.raw = half_raw<T>(g, neg, neg ? j : E - 1 - j);
      out.ties = ci;
      out.before = bw;
      out.tie = BY_COUNT ? (uint32_t)(target - here).lo : 0;
    }
    bc += ci;
    bw += vi;
  }
  const int owner = __ffsll(__ballot(out.ties != 0)) - 1;
  out.raw = lane_value(out.raw, owner);
  out.tie = lane_value(out.tie, owner);
  out.ties = lane_value(out.ties, owner);
  out.before = lane_value(out.before, owner);
  out.one = w.of(half_value<T>(out.raw));
  if (!BY_COUNT) out.tie = quotient(target - out.before, out.one);
  return out;
}

// The workgroup's decision for a row from its counts (s.has filled): s.raw, s.tie, s.ties, s.prob; false for an empty row.
template <class T, class C> __device__ bool decide_half(HalfScratch& s, const C& counts, const Settings& st, int V) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int E = Half<T>::E, GROUPS = half_groups<T>(), R = 2 * GROUPS / 64;
  for (int i = threadIdx.x; i < 2 * GROUPS; i += HWG) { s.weight[i] = 0; s.count[i] = 0; }
  if (threadIdx.x == 0) { s.heavy = 0; s.heavy_carry = 0; }
  __syncthreads();
  // the marked groups, the waves in turn: candidates of both signs
  auto groups = [&](auto f) {
    int turn = 0;
    for (int word = 0; word < GROUPS / 64; ++word)
      for (uint64_t left = s.has[word]; left; left &= left - 1)
        if (turn++ % (HWG / 64) == wave) f(64 * word + __ffsll((long long)left) - 1);
  };
  groups([&](int g) {
    const Counts<E> p = counts.load(g);
    counts.keep(s, g, p);
    uint32_t pos[E], neg[E];
    valid<T>(g, false, p, pos);
    valid<T>(g, true, p, neg);
    const uint32_t np = wave_sum(sum_of(pos)), nn = wave_sum(sum_of(neg));
    if (lane == 0) { s.count[GROUPS - 1 - g] = np; s.count[GROUPS + g] = nn; }
  });
  __syncthreads();
  // the largest candidate, in the first order that has one (every wave finds it)
  uint32_t first = 2 * GROUPS;
#pragma unroll
  for (int i = R - 1; i >= 0; --i) first = s.count[lane * R + i] ? lane * R + i : first;
  const unsigned long long some = __ballot(first < 2 * GROUPS);
  if (!some) return false;
  const int order = (int)lane_value(first, __ffsll(some) - 1);
  const bool below = order >= GROUPS;
  uint32_t c[E], mine = 0;
  valid<T>(group_of<T>(order), below, counts.again(s, group_of<T>(order)), c);
#pragma unroll
  for (int j = 0; j < E; ++j) {  // of a lane's own the largest: the first of the negative ones, the last of the others
    const int i = below ? E - 1 - j : j;
    mine = (below ? c[E - 1 - j] : c[j]) ? half_raw<T>(group_of<T>(order), below, i) : mine;
  }
  const unsigned long long hit = __ballot(sum_of(c) != 0);
  const int at = below ? __ffsll(hit) - 1 : 63 - __clzll((long long)hit);
  const Weigher w(st, half_value<T>(lane_value(mine, at)));
  const bool greedy = st.greedy();
  if (!greedy) {
    groups([&](int g) {
      const Counts<E> p = counts.again(s, g);
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        uint32_t c[E];
        valid<T>(g, side != 0, p, c);
        if (!__ballot(sum_of(c) != 0)) continue;
        Sum sum = 0, heavy = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (!__ballot(c[i] != 0)) continue;
          const double x = w.x(half_value<T>(half_raw<T>(g, side != 0, i)));
          const Sum v = times(c[i], w.at(x));
          sum += v;
          if (x >= w.floor_x) heavy += v;
        }
        sum = wave_sum(sum);
        if (lane == 0) s.weight[side ? GROUPS + g : GROUPS - 1 - g] = sum;
        if (st.m > 0.0f) {
          heavy = wave_sum(heavy);
          if (lane == 0) add_to(&s.heavy, &s.heavy_carry, heavy);
        }
      }
    });
  }
  __syncthreads();  // of a greedy row too: every wave has read the counts that become running sums now
  if (wave == 0) {
    prefix_half<T>(s);
    Spot at;
    float prob = 1.0f;
    if (greedy) {
      at = spot_half<T, true>(s, counts, w, Sum(0));
    } else {
      Sum total = s.weight[2 * GROUPS - 1];
      if (st.limited(V) && (uint32_t)st.k < s.count[2 * GROUPS - 1]) total = spot_half<T, true>(s, counts, w, Sum((uint64_t)st.k - 1)).end();
      Sum kept = total;
      if (st.p < 1.0f) {
        const Sum t = st.goal(total);
        if (t < total) {
          const Sum end = spot_half<T, false>(s, counts, w, t).end();
          kept = smaller(end, kept);
        }
      }
      if (st.m > 0.0f) {
        const Sum heavy(s.heavy, s.heavy_carry);
        kept = smaller(heavy, kept);
      }
      at = spot_half<T, false>(s, counts, w, st.draw(kept));
      prob = w.prob(half_value<T>(at.raw), kept);
    }
    if (lane == 0) { s.raw = at.raw; s.tie = at.tie; s.ties = at.ties; s.prob = prob; }
  }
  __syncthreads();
  return true;
}

// The tie-th logit of value `raw` (0: of either sign) among granules lo .. hi - 1, in order of index; one of `ties` there.  Every wave
// has a run of at most 512 granules, every lane 8 of them as bits.
template <class T> __device__ void find_half(HalfScratch& s, const Row<T>& row, int lo, int hi, uint32_t raw, uint32_t tie, uint32_t ties, int32_t* token) {
  static_assert(HALF_GRANULES <= 8 * HWG, "a lane's granules as bytes of 64 bits");
  const uint16_t* at = (const uint16_t*)row.at - row.lead;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t mask = raw == 0 ? 0x7fffu : 0xffffu;
  const int whole = (row.V + row.lead) / 8, from = lo == 0 && row.lead ? 1 : lo, to = hi < whole ? hi : whole;  // whole granules: from .. to - 1
  const int span = ((hi - lo + HWG / 64 - 1) / (HWG / 64) + 63) / 64 * 64;  // a wave's granules
  const int w0 = lo + wave * span, w1 = w0 + span < hi ? w0 + span : hi;
  uint64_t bits = 0;
#pragma unroll
  for (int b = 0; b < 8; b += 4) {
    if (64 * b < span && from < to) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = w0 + 64 * (b + u) + lane;
        v[u] = *(const uint4*)(at + 8 * (j < from ? from : j < to ? j : to - 1));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = w0 + 64 * (b + u) + lane;
        const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m |= (w[i] & mask) == raw ? 1u << (2 * i) : 0;
          m |= ((w[i] >> 16) & mask) == raw ? 2u << (2 * i) : 0;
        }
        if (j >= from && j < to && j < w1) bits |= (uint64_t)m << (8 * (b + u));
      }
    }
  }
  auto edge = [&](int j) {  // a granule that is not whole, where it is this lane's
    if (j < w0 || j >= w1 || (j - w0) % 64 != lane) return;
    for (int i = 0; i < 8; ++i) {
      const int e = 8 * j + i - row.lead;
      if (e >= 0 && e < row.V && (at[8 * j + i] & mask) == raw) bits |= 1ull << (8 * ((j - w0) / 64) + i);
    }
  };
  if (from != lo) edge(0);
  if (hi > whole) edge(whole);
  if (ties == 1) {  // the only one: no order to keep
    if (bits) {
      const int i = __ffsll((long long)bits) - 1;
      *token = (w0 + 64 * (i / 8) + lane) * 8 + i % 8 - row.lead;
    }
    return;
  }
  const uint32_t mine = wave_sum((uint32_t)__popcll(bits));
  if (lane == 0) s.part[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < wave; ++i) before += s.part[i];
  if (tie < before || tie >= before + mine) return;
  for (int b = 0; b < 8; ++b) {
    uint32_t m = (uint32_t)(bits >> (8 * b)) & 255u;
    const uint32_t n = __popc(m), incl = wave_scan(n), all = lane_value(incl, 63);
    if (tie < before + all) {
      const uint32_t first = before + incl - n;
      if (tie >= first && tie < first + n) {
        for (uint32_t i = first; i < tie; ++i) m &= m - 1;
        *token = (w0 + 64 * b + lane) * 8 + __ffs(m) - 1 - row.lead;
      }
      return;
    }
    before += all;
  }
}

// the counts of a row's slices -> its token
template <class T>
__global__ __launch_bounds__(HWG) void half_choose_kernel(cube_sample_args a, int r0, const HalfSlice* ws, int slices, int per) {
  extern __shared__ __attribute__((aligned(16))) uint32_t kept[];
  __shared__ HalfScratch s;
  __shared__ uint64_t has[HALF_SLICES][MAX_GROUPS / 64];
  constexpr int WORDS = half_groups<T>() / 64, GROUP = 64 * Half<T>::E;
  const int r = r0 + blockIdx.x, lane = threadIdx.x & 63;
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const Settings st(a, r);
  const SliceCounts<T> counts = {ws + (size_t)blockIdx.x * slices, slices, has, kept};
  if ((int)threadIdx.x < slices * WORDS) has[threadIdx.x / WORDS][threadIdx.x % WORDS] = counts.slice[threadIdx.x / WORDS].has[threadIdx.x % WORDS];
  __syncthreads();
  if (threadIdx.x < WORDS) {
    uint64_t h = 0;
    for (int i = 0; i < slices; ++i) h |= has[i][threadIdx.x];
    s.has[threadIdx.x] = h;
  }
  if (!decide_half<T>(s, counts, st, a.V)) {
    if (threadIdx.x == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  if (threadIdx.x < 64) {  // which slice has the tie-th of them
    const uint32_t mag = s.raw & 0x7fffu, g = mag / GROUP;
    uint32_t before = 0;
    for (int i0 = 0; i0 < slices; i0 += 64) {
      const int i = i0 + lane;
      uint32_t n = 0;
      if (i < slices && ((has[i][g >> 6] >> (g & 63)) & 1)) {
        const uint32_t c = counts.slice[i].count[mag];
        n = mag == 0 ? c & 0xffffu : s.raw & 0x8000u ? c >> 16 : (c & 0xffffu) - (c >> 16);
      }
      const uint32_t incl = wave_scan(n), all = lane_value(incl, 63);
      const uint32_t first = before + incl - n;
      const bool here = s.tie >= first && s.tie < first + n;
      if (__ballot(here)) {
        const uint32_t tie = s.tie;
        if (here) { s.slice = i; s.tie = tie - first; s.ties = n; }
        break;
      }
      before += all;
    }
  }
  __syncthreads();
  const int lo = (int)s.slice * per, hi = lo + per < row.granules ? lo + per : row.granules;
  if (threadIdx.x == 0 && a.prob) a.prob[r] = s.prob;
  find_half(s, row, lo, hi, s.raw, s.tie, s.ties, &a.token[r]);
}

// a row of one slice in one launch: the counts stay in LDS
template <class T>
__global__ __launch_bounds__(HWG) void half_row_kernel(cube_sample_args a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t count[];
  HalfScratch& s = *(HalfScratch*)(count + MAGS);
  const int r = blockIdx.x;
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const Settings st(a, r);
  count_half(count, row, 0, row.granules);
  mark_half<T>(count, s.part, s.has, [](int, const Words<Half<T>::E>&) {});
  if (!decide_half<T>(s, LdsCounts<T>{count}, st, a.V)) {
    if (threadIdx.x == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  if (threadIdx.x == 0 && a.prob) a.prob[r] = s.prob;
  find_half(s, row, 0, row.granules, s.raw, s.tie, s.ties, &a.token[r]);
}

// ---- long: f32 rows (and few f16 ones) in slices side by side ------------------------------------------------------------------
// 1 largest key of every slice, and the row's histogram cleared;  2 histogram over steps of the logit: counts for a top-k row,
// weights for another;  3 the bins in which the targets can fall are known: their logits into the row's list;  4 one workgroup
// decides from the list and the histogram.  A list that runs over (very many equal logits) sends the fourth launch over the
// whole row instead.
constexpr int LONG_BINS = 4096;
constexpr int LIST = 16384;
constexpr int LWG = 1024;
constexpr int ROWS_AT_ONCE = 256;  // rows of one pass of the four launches: bounds the workspace
constexpr int MAX_SLICES = 256;

struct LongRow {  // of the workspace
  uint64_t hist[LONG_BINS];
  uint64_t list[LIST];  // entries
  uint32_t carry[LONG_BINS];  // out of hist
  uint64_t heavy;       // weight of those that min-p keeps
  uint32_t heavy_carry;
  uint32_t listed;
  uint32_t top[MAX_SLICES];
  __device__ Sum weight(int b) const { return {hist[b], carry[b]}; }
};

__device__ __forceinline__ uint32_t row_top(const LongRow& l, int slices, Scratch& s) {
  return block_max<LWG>(s, (int)threadIdx.x < slices ? l.top[threadIdx.x] : 0u);
}

template <class T> __global__ __launch_bounds__(LWG) void long_top_kernel(cube_sample_args a, int r0, LongRow* rows, int per) {
  __shared__ uint32_t part[LWG / 64];
  constexpr int N = Granule<T>::N;
  const int r = r0 + blockIdx.y, slices = gridDim.x;
  LongRow& l = rows[blockIdx.y];
  for (int b = blockIdx.x * LWG + threadIdx.x; b < LONG_BINS; b += slices * LWG) { l.hist[b] = 0; l.carry[b] = 0; }
  if (blockIdx.x == 0 && threadIdx.x == 0) { l.heavy = 0; l.heavy_carry = 0; l.listed = 0; }
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  float largest = -INFINITY;
#pragma unroll 4
  for (int j = lo + threadIdx.x; j < hi; j += LWG) {
    float v[N];
    row.values(j, v);
#pragma unroll
    for (int i = 0; i < N; ++i) largest = fmaxf(largest, v[i]);
  }
  uint32_t best = wave_max(key_of(largest));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x < 64) {
    best = wave_max(threadIdx.x < LWG / 64 ? part[threadIdx.x] : 0u);
    if (threadIdx.x == 0) l.top[blockIdx.x] = best;
  }
}

template <class T> __global__ __launch_bounds__(LWG, 8) void long_hist_kernel(cube_sample_args a, int r0, LongRow* rows, int per) {
  __shared__ uint64_t hist[LONG_BINS];
  __shared__ Scratch s;
  constexpr int N = Granule<T>::N;
  const int r = r0 + blockIdx.y;
  LongRow& l = rows[blockIdx.y];
  const Settings st(a, r);
  const uint32_t best = row_top(l, gridDim.x, s);
  if (best == 0 || st.greedy()) return;
  uint32_t* carry = (uint32_t*)s.high;  // (row_top is done with it)
  static_assert(sizeof(s.high) >= 4 * LONG_BINS, "room for the carries");
  for (int b = threadIdx.x; b < LONG_BINS; b += LWG) { hist[b] = 0; carry[b] = 0; }
  __syncthreads();
  const Steps step(value_of(best), st.temp, LONG_BINS);
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  auto all = [&](auto f) {
#pragma unroll 2
    for (int j = lo + threadIdx.x; j < hi; j += LWG) {
      float v[N];
      row.values(j, v);
#pragma unroll
      for (int i = 0; i < N; i += 2) f({v[i], v[i + 1]});
    }
  };
  if (st.limited(a.V)) {
    all([&](const float (&v)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) if (v[i] > -INFINITY) atomicAdd((unsigned long long*)&hist[step(v[i])], 1ull);
    });
  } else {
    const Weigher w(st, value_of(best));
    Sum heavy = 0;
    if (st.m > 0.0f) {
      all(Gather<true>{w, step, hist, carry, heavy});
      heavy = wave_sum(heavy);
      if ((threadIdx.x & 63) == 0) add_to(&l.heavy, &l.heavy_carry, heavy);
    } else {
      all(Gather<false>{w, step, hist, carry, heavy});
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < LONG_BINS; b += LWG)
    if (hist[b] | carry[b]) add_to(&l.hist[b], &l.carry[b], Sum(hist[b], carry[b]));
}

// What the histogram of a row without a top-k limit leaves open: the bin that ends the top-p set (if that can be the shortest
// prefix), and the bins among which the drawn position lies.
struct Open { bool ends; Found<Sum> end; Sum goal, least, most; uint32_t from, to; };
typedef Held<Sum, LONG_BINS / LWG> LongHeld;
__device__ Open open_bins(Scratch& s, const LongHeld& r, const Settings& st, Sum heavy) {
  Open o;
  o.ends = false;
  o.least = o.most = r.total;
  if (st.p < 1.0f) {
    o.goal = st.goal(r.total);
    if (o.goal < r.total) {
      o.ends = true;
      o.end = find_bin<LWG, LONG_BINS, true>(s, r, Sum(0), o.goal);
      o.least = o.goal + Sum(1);  // the set's sum is at least the goal and at most the end of the bin
      o.most = o.end.before + o.end.in;
    }
  }
  if (st.m > 0.0f) {
    if (heavy <= o.least) o.ends = false;
    o.least = smaller(heavy, o.least);
    o.most = smaller(heavy, o.most);
  }
  o.from = find_bin<LWG, LONG_BINS, true>(s, r, Sum(0), st.draw(o.least)).bin;
  o.to = o.least == o.most ? o.from : find_bin<LWG, LONG_BINS, true>(s, r, Sum(0), st.draw(o.most)).bin;
  return o;
}

template <class T> __global__ __launch_bounds__(LWG, 8) void long_list_kernel(cube_sample_args a, int r0, LongRow* rows, int per) {
  __shared__ Scratch s;
  constexpr int N = Granule<T>::N;
  const int r = r0 + blockIdx.y, lane = threadIdx.x & 63;
  LongRow& l = rows[blockIdx.y];
  const Settings st(a, r);
  const uint32_t best = row_top(l, gridDim.x, s);
  if (best == 0) return;
  const Steps step(value_of(best), st.greedy() ? 1.0f : st.temp, LONG_BINS);
  // candidates in the bins from .. to and in the bin `end` are listed; of a greedy row those equal to the largest
  int from = 0, to = 0, end = -1;
  if (!st.greedy()) {
    if (st.limited(a.V)) {
      const auto counts = hold<LWG, LONG_BINS, true>(s, [&](int b) { return l.hist[b]; });
      to = LONG_BINS - 1;
      if ((uint64_t)st.k < counts.total) to = (int)find_bin<LWG, LONG_BINS, true>(s, counts, (uint64_t)0, (uint64_t)st.k - 1).bin;
    } else {
      const Open o = open_bins(s, hold<LWG, LONG_BINS, true>(s, [&](int b) { return l.weight(b); }), st, Sum(l.heavy, l.heavy_carry));
      from = (int)o.from;
      to = (int)o.to;
      if (o.ends) end = (int)o.end.bin;
    }
  }
  const Row<T> row((const T*)a.logits + (size_t)r * a.ld, a.V);
  const int lo = blockIdx.x * per, hi = lo + per < row.granules ? lo + per : row.granules;
  const float largest = value_of(best);
  const Span span(step, from, to), last(step, end < 0 ? from : end, end < 0 ? to : end);
#pragma unroll 2
  for (int j0 = lo; j0 < hi; j0 += LWG) {
    const int j = j0 + threadIdx.x;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = -INFINITY;
    if (j < hi) row.values(j, v);
    bool some = false;
#pragma unroll
    for (int i = 0; i < N; ++i) some |= span.near(v[i]) | last.near(v[i]);
    if (__ballot(some) == 0) continue;
    uint32_t n = 0;
    bool in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      in[i] = (span.has(step, v[i]) || last.has(step, v[i])) && (!st.greedy() || v[i] == largest);
      n += in[i];
    }
    if (__ballot(n != 0) == 0) continue;
    const uint32_t incl = wave_scan(n);
    uint32_t base = 0;
    if (lane == 63) base = atomicAdd(&l.listed, incl);
    uint32_t at = lane_value(base, 63) + incl - n;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) {
        if (at < LIST) l.list[at] = entry_of(key_of(v[i]), (uint32_t)(j * N + i - row.lead));
        ++at;
      }
  }
}

// the listed logits of a row, or all of a row's
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
      float v[N];
      row.values(j, v);
#pragma unroll
      for (int i = 0; i < N; ++i) f(key_of(v[i]));
    }
  }
};
// the key at which the running weight passes target among the keys that each() gives, `before` in front of them
template <class E> __device__ Place search(Scratch& s, E each, const Weigher& w, Sum before, Sum target) {
  uint32_t* carry = s.high_carry();
  for (int b = threadIdx.x; b < (1 << D1); b += LWG) { s.high[b] = 0; carry[b] = 0; }
  __syncthreads();
  each([&](uint32_t k) { add_to(&s.high[k >> (32 - D1)], &carry[k >> (32 - D1)], w(k)); });
  __syncthreads();
  const Found<Sum> f = find_bin<LWG, 1 << D1, false>(s, hold<LWG, 1 << D1, false>(s, [&](int b) { return Sum(s.high[b], carry[b]); }), before, target);
  return refine<LWG, D1, false>(s, each, w, f.bin, f.before, target);
}

template <class T> __global__ __launch_bounds__(LWG) void long_choose_kernel(cube_sample_args a, int r0, LongRow* rows, int slices) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  Scratch& s = *(Scratch*)smem;
  Few& few = *(Few*)(smem + sizeof(Scratch));
  uint64_t* list = (uint64_t*)(smem + sizeof(Scratch) + sizeof(Few));
  constexpr int N = Granule<T>::N;
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
  if (threadIdx.x == 0) few.n = 0;
  __syncthreads();
  Choice c = {best, 0, 0};
  float prob = 1.0f;
  if (!st.greedy()) {
    const Weigher w(st, value_of(best));
    if (whole) {
      c = decide<LWG>(s, RowKeys<T>{row}, st, w, a.V);
    } else if (st.limited(a.V)) {
      if (n <= FEW) {
        for (int i = threadIdx.x; i < n; i += LWG) few.entry[i] = list[i];
        if (threadIdx.x == 0) few.n = n;
        __syncthreads();
        sort_few<LWG>(few);
        if (threadIdx.x < 64) {
          uint32_t q[FEW / 64];
#pragma unroll
          for (int e = 0; e < FEW / 64; ++e) q[e] = (uint32_t)(few.sorted[threadIdx.x * (FEW / 64) + e] >> 32);
          const int at = choose_sorted<Sum>(q, st, w, a.V, prob);
          if (threadIdx.x == 0) { a.token[r] = (int)~(uint32_t)few.sorted[at]; if (a.prob) a.prob[r] = prob; }
        }
        return;
      }
      c = decide<LWG>(s, ListKeys{list, n}, st, w, a.V);
    } else {
      const Steps step(value_of(best), st.temp, LONG_BINS);
      const LongHeld runs = hold<LWG, LONG_BINS, true>(s, [&](int b) { return l.weight(b); });
      const Open o = open_bins(s, runs, st, Sum(l.heavy, l.heavy_carry));
      // where the running weight passes a target, inside a bin of the list: a few members are sorted, more are searched
      auto place = [&](const Found<Sum>& at, Sum target, Place& out) {
        for (int i = threadIdx.x; i < n; i += LWG) if (step((uint32_t)(list[i] >> 32)) == (int)at.bin) append(few, list[i]);
        __syncthreads();
        if (few.n <= FEW) {
          sort_few<LWG>(few);
          if (threadIdx.x < 64) place_few(few, w, at.before, target);
          __syncthreads();
          return true;
        }
        out = search(s, [&](auto f) {
          for (int i = threadIdx.x; i < n; i += LWG) { const uint32_t k = (uint32_t)(list[i] >> 32); if (step(k) == (int)at.bin) f(k); }
        }, w, at.before, target);
        return false;
      };
      Sum kept = o.most;
      Place at;
      if (o.ends) {
        const Sum end = place(o.end, o.goal, at) ? few.end : at.end();
        kept = smaller(end, kept);
        __syncthreads();
        if (threadIdx.x == 0) few.n = 0;
        __syncthreads();
      }
      const Sum t = st.draw(kept);
      if (place(find_bin<LWG, LONG_BINS, true>(s, runs, Sum(0), t), t, at)) {
        if (threadIdx.x == 0) { a.token[r] = (int)few.index; if (a.prob) a.prob[r] = w.prob(value_of(few.key), kept); }
        return;
      }
      c = {at.key, at.tie, kept};
    }
    prob = w.prob(value_of(c.key), c.kept);
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
      for (int j = threadIdx.x; j < row.granules; j += LWG) {
        float v[N];
        row.values(j, v);
#pragma unroll
        for (int i = 0; i < N; ++i) if (key_of(v[i]) == c.key) add((uint32_t)(j * N + i - row.lead));
      }
    } else {
      for (int i = threadIdx.x; i < n; i += LWG) if ((uint32_t)(list[i] >> 32) == c.key) add(~(uint32_t)list[i]);
    }
    __syncthreads();
    const auto f = find_bin<LWG, 2048, false>(s, hold<LWG, 2048, false>(s, [&](int b) { return s.high[b]; }), (uint64_t)0, (uint64_t)left);
    prefix = (prefix << 11) | (2047 - f.bin);
    left -= (uint32_t)f.before;
  }
  if (threadIdx.x == 0) { a.token[r] = (int)prefix; if (a.prob) a.prob[r] = prob; }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------

// A launch has fewer than 2^32 threads: where every row has a wave or a workgroup, rows go in parts of 2^21.
template <class T, class F> int in_parts(const cube_sample_args& all, F f) {
  constexpr int PART = 1 << 21;
  for (long long r0 = 0; r0 < all.M; r0 += PART) {
    cube_sample_args a = all;
    a.M = (int)(all.M - r0 < PART ? all.M - r0 : PART);
    a.logits = (const T*)all.logits + r0 * all.ld;
    a.u += r0;
    a.token += r0;
    if (a.prob) a.prob += r0;
    if (a.temperature) a.temperature += r0;
    if (a.top_k) a.top_k += r0;
    if (a.top_p) a.top_p += r0;
    if (a.min_p) a.min_p += r0;
    f(a);
    CUBE_CHECK_LAUNCH("cube_sample_rows");
  }
  return CUBE_OK;
}

template <class T> int launch_short(const cube_sample_args& all, hipStream_t st) {
  return in_parts<T>(all, [&](const cube_sample_args& a) {
    const dim3 grid((a.M + 3) / 4), block(256);
    if (a.V <= 64) hipLaunchKernelGGL((sample_short_kernel<T, 1>), grid, block, 0, st, a);
    else if (a.V <= 128) hipLaunchKernelGGL((sample_short_kernel<T, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((sample_short_kernel<T, 4>), grid, block, 0, st, a);
  });
}

template <class T, int WG> int launch_mid(const cube_sample_args& all, hipStream_t st) {
  static CubeLdsReservation lds;
  const size_t bytes = sizeof(Scratch) + sizeof(Few) + 4 * (size_t)((all.V + 2 * Granule<T>::N + 3) / 4 * 4);
  if (!lds.ensure((const void*)sample_mid_kernel<T, WG>, bytes)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_sample_rows: LDS reservation failed");
  return in_parts<T>(all, [&](const cube_sample_args& a) { hipLaunchKernelGGL((sample_mid_kernel<T, WG>), dim3(a.M), dim3(WG), bytes, st, a); });
}

template <class T> int launch_long(const cube_sample_args& a, LongRow* ws, hipStream_t st) {
  static CubeLdsReservation lds;
  const size_t bytes = sizeof(Scratch) + sizeof(Few) + 8 * LIST;
  if (!lds.ensure((const void*)long_choose_kernel<T>, bytes)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_sample_rows: LDS reservation failed");
  const int granules = (a.V + 2 * Granule<T>::N - 2) / Granule<T>::N;  // of a row that starts inside a granule
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
    hipLaunchKernelGGL((long_hist_kernel<T>), grid, dim3(LWG), 0, st, a, r0, ws, per);
    hipLaunchKernelGGL((long_list_kernel<T>), grid, dim3(LWG), 0, st, a, r0, ws, per);
    hipLaunchKernelGGL((long_choose_kernel<T>), dim3(n), dim3(LWG), bytes, st, a, r0, ws, slices);
    CUBE_CHECK_LAUNCH("cube_sample_rows");
  }
  return CUBE_OK;
}

// slices of a 16-bit row, and rows of one pass of the two launches
constexpr int HALF_AT_ONCE = 1024;  // slices
struct HalfPlan { int slices, per, rows; };
HalfPlan half_plan(int M, int V) {
  const int granules = (V + 2 * 8 - 2) / 8;
  HalfPlan p;
  p.slices = (granules + HALF_GRANULES - 1) / HALF_GRANULES;
  p.rows = HALF_AT_ONCE / p.slices < M ? HALF_AT_ONCE / p.slices : M;  // V <= 2^22: at most 65 slices
  if (p.slices > 1 || M < 64) {
    // few rows: more and shorter slices, up to one workgroup a CU, but eight of four granules a thread at most: the second launch
    // has one workgroup to add the slices' counts (1 x 250002: 31 slices took 64 us where 8 took 23)
    const int most = (granules + 4 * HWG - 1) / (4 * HWG), want = 256 / p.rows < 8 ? 256 / p.rows : 8;
    const int more = most < want ? most : want;
    p.slices = more > p.slices ? more : p.slices;
    p.slices = p.slices < HALF_SLICES ? p.slices : HALF_SLICES;
  }
  p.per = (granules + p.slices - 1) / p.slices;
  return p;
}
template <class T> int launch_half(const cube_sample_args& a, HalfSlice* ws, hipStream_t st) {
  constexpr size_t bytes = 4 * MAGS;
  const HalfPlan p = half_plan(a.M, a.V);
  if (p.slices == 1) {
    static CubeLdsReservation lds;
    constexpr size_t all = bytes + sizeof(HalfScratch);
    if (!lds.ensure((const void*)half_row_kernel<T>, all)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_sample_rows: LDS reservation failed");
    return in_parts<T>(a, [&](const cube_sample_args& part) { hipLaunchKernelGGL((half_row_kernel<T>), dim3(part.M), dim3(HWG), all, st, part); });
  }
  static CubeLdsReservation lds, lds2;
  constexpr size_t kept = KEPT_BYTES;
  if (!lds.ensure((const void*)half_count_kernel<T>, bytes) || !lds2.ensure((const void*)half_choose_kernel<T>, kept))
    CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_sample_rows: LDS reservation failed");
  for (int r0 = 0; r0 < a.M; r0 += p.rows) {
    const int n = a.M - r0 < p.rows ? a.M - r0 : p.rows;
    hipLaunchKernelGGL((half_count_kernel<T>), dim3(p.slices, n), dim3(HWG), bytes, st, a, r0, ws, p.per);
    hipLaunchKernelGGL((half_choose_kernel<T>), dim3(n), dim3(HWG), kept, st, a, r0, ws, p.slices, p.per);
    CUBE_CHECK_LAUNCH("cube_sample_rows");
  }
  return CUBE_OK;
}

// 16-bit rows longer than this are counted by value (us, top-p: bf16 64 x 16000 17 against 18; 256 x 32000 20 against 30).  f16
// has eight times as many values to an octave: 256 x 32000 33 against 29, top-k 35 against 16, and 1 x 20000 28 against 17.
template <class T> constexpr int half_v() { return std::is_same<T, bf16_t>::value ? 16000 : MID_V; }

// Rows that go through slices, histogram and list: f32 beyond what a workgroup holds; of f16 up to 32 rows of 2^23 logits in all, while
// counting by value costs more (us, plain, top-p, top-k: 1 x 250002 22 and 30 against 40 and 45;  32 x 40000 27 and 33 against 36 and 39;
// 8 x 500000 40, 54, 33 against 48, 52, 55;  24 x 250002 52, 60, 40 against 48, 52, 56;  64 x 40000 35 and 41 against 30 and 33).  bf16
// has too many equal values for the list (1 x 250002, top-p 33 against 24).
bool sliced(int type, int M, int V) {
  return V > MID_V && (type == CUBE_T_F32 || (type == CUBE_T_F16 && M <= 32 && (long long)M * V <= 1 << 23));
}

template <class T> int launch(const cube_sample_args& a, void* ws, hipStream_t st) {
  if (a.V <= SHORT_V) return launch_short<T>(a, st);
  if constexpr (!std::is_same<T, bf16_t>::value) {
    if (sliced(a.type, a.M, a.V)) return launch_long<T>(a, (LongRow*)ws, st);
  }
  if constexpr (sizeof(T) == 2) {
    if (a.V > half_v<T>()) return launch_half<T>(a, (HalfSlice*)ws, st);
  }
  // 256 threads keep several rows on a CU; above 4096 logits a row's own passes are what takes time
  return a.V <= 4096 ? launch_mid<T, 256>(a, st) : launch_mid<T, 1024>(a, st);
}

}  // namespace

extern "C" size_t cube_sample_workspace_bytes(int type, int M, int V) {
  if (M <= 0 || V <= 0 || V > CUBE_SAMPLE_MAX_V) return 0;
  if (type == CUBE_T_F32 || sliced(type, M, V)) return V > MID_V ? sizeof(LongRow) * (size_t)(M < ROWS_AT_ONCE ? M : ROWS_AT_ONCE) : 0;
  if (V <= (type == CUBE_T_BF16 ? half_v<bf16_t>() : half_v<_Float16>())) return 0;
  const HalfPlan p = half_plan(M, V);
  return p.slices > 1 ? sizeof(HalfSlice) * (size_t)p.slices * p.rows : 0;
}

extern "C" int cube_sample_rows(const cube_sample_args* a, void* ws, size_t ws_bytes, void* stream) {
  CUBE_ENTRY();
  if (!a) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: null args");
  if (a->M < 0 || a->V < 1 || a->V > CUBE_SAMPLE_MAX_V) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: M=%d, V=%d outside 1..%d", a->M, a->V, CUBE_SAMPLE_MAX_V);
  if (a->M == 0) return CUBE_OK;
  if (!a->logits || !a->u || !a->token) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: null logits / u / token");
  if (a->type < CUBE_T_F32 || a->type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: type=%d", a->type);
  if (a->ld < a->V || a->ld > 1LL << 40) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: ld=%lld outside V=%d..2^40", a->ld, a->V);
  if ((uintptr_t)a->logits % (a->type == CUBE_T_F32 ? 4 : 2) || ((uintptr_t)a->u & 7) ||
      (((uintptr_t)a->token | (uintptr_t)a->prob | (uintptr_t)a->temperature | (uintptr_t)a->top_k | (uintptr_t)a->top_p | (uintptr_t)a->min_p) & 3))
    CUBE_FAIL(CUBE_ERR_ALIGN, "cube_sample_rows: a pointer is not aligned to its type");
  const size_t need = cube_sample_workspace_bytes(a->type, a->M, a->V);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: workspace of %zu bytes (need %zu, 16-byte aligned)", ws_bytes, need);
  const long long es = a->type == CUBE_T_F32 ? 4 : 2, M4 = 4LL * a->M;
  const CubeArea in[] = {{a->logits, a->ld * es, a->V * es, a->M}, {a->u, 2 * M4}, {a->temperature, M4}, {a->top_k, M4}, {a->top_p, M4}, {a->min_p, M4}};
  const CubeArea out[] = {{a->token, M4}, {a->prob, M4}, {need ? ws : nullptr, (long long)need}};
  for (const CubeArea& o : out)
    for (const CubeArea& i : in)
      if (cube_overlap(i, o)) CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: an input overlaps token, prob or the workspace");
  if (cube_overlap(out[0], out[1]) || cube_overlap(out[0], out[2]) || cube_overlap(out[1], out[2]))
    CUBE_FAIL(CUBE_ERR_ARG, "cube_sample_rows: token, prob and the workspace overlap");
  hipStream_t st = (hipStream_t)stream;
  if (a->type == CUBE_T_F32) return launch<float>(*a, ws, st);
  if (a->type == CUBE_T_BF16) return launch<bf16_t>(*a, ws, st);
  return launch<_Float16>(*a, ws, st);
}
