// Sampling one token a row from logits with temperature, top-k, top-p and min-p, from given random numbers (gfx950).
//
// Candidates of a row are its logits above -inf (NaN and -inf are none), in order of falling logit, ties lowest index first.
//   w_i   = exp((z_i - z_max) / T)
//   top-k   keeps the first k;  top-p the shortest prefix whose sum reaches p * (sum of the top-k set);  min-p those with
//   w_i >= m (the largest weight is 1).  All three are prefixes of the one order, so the kept set is the shortest of them.
//   token = the first candidate whose running sum exceeds u * (sum of the kept set);  prob = its w / that sum.
//
// The order is never sorted out: every decision is "the first position where the running count or weight passes a target", and
// a radix search over the sortable bits of the logit finds it -- a histogram of count and weight over the top bits, the bin in
// which the target falls, the next bits inside that bin.
//
// Weights are 64-bit fixed point, w * 2^S rounded, with S such that V of them cannot overflow: integer sums do not depend on
// their order, so a row gives the same token however it is divided among lanes and workgroups, and at 2^-45 relative they
// decide as 64-bit floating point would (a 32-bit running sum over a large vocabulary is off by more than the distance
// between two neighbouring tokens' borders).
#include "common.h"
#include "../../include/cube_hip.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float as_float(bf16_t v) { return (float)v; }

// sortable bits: a larger logit has a larger key; 0 for what is no candidate.  -0 and +0 are one value (v + 0 makes them so).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return v > -INFINITY ? k : 0u;  // false for NaN too
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

struct Weigher {
  double top, inv_t, one;  // largest logit, 1 / T, 2^S
  uint32_t top_key;
  __device__ double exact(uint32_t key) const {  // w; the largest is 1 even where it is +inf
    if (key == top_key) return 1.0;
    const double x = ((double)value_of(key) - top) * inv_t;
    return x > -700.0 ? exp(x) : 0.0;  // (0 too where an infinite temperature meets an infinite logit: 0 * inf)
  }
  __device__ uint64_t operator()(uint32_t key) const { return (uint64_t)(exact(key) * one + 0.5); }
};

struct Shared {
  uint64_t wgt[BINS];
  uint32_t cnt[BINS];
  uint32_t part_c[WAVES];
  uint32_t bin;
  uint64_t before, before_w;
};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)v, src, 64) | ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(v >> 32), src, 64) << 32);
}

template <class T, class F> __device__ __forceinline__ void each(const T* row, int V, F f) {
  for (int i = threadIdx.x; i < V; i += THREADS) f(i, as_float(row[i]));
}

// where a target falls: the key of the position and the position's place among equal logits
struct Place { uint32_t key; uint32_t tie; uint64_t before_w; };

// First position, in falling order, at which the running count (BY_COUNT) or weight exceeds `target`.  The caller guarantees
// that the sum over all candidates does.
template <bool BY_COUNT, class T>
__device__ Place find(Shared& s, const T* row, int V, const Weigher& weigh, uint64_t target) {
  uint32_t prefix = 0;
  int shift = 32;
  uint64_t before = 0, before_w = 0;
  while (shift > 0) {
    const int bits = shift >= DIGIT ? DIGIT : shift;
    const int next = shift - bits;
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += THREADS) { s.wgt[b] = 0; s.cnt[b] = 0; }
    __syncthreads();
    each(row, V, [&](int, float v) {
      const uint32_t k = key_of(v);
      if (k && (shift == 32 || (k >> shift) == prefix)) {
        const int b = (k >> next) & (bins - 1);
        atomicAdd(&s.cnt[b], 1u);
        atomicAdd((unsigned long long*)&s.wgt[b], (unsigned long long)weigh(k));
      }
    });
    __syncthreads();
    if (threadIdx.x < 64) {  // one wave walks the bins from the top, 64 at a time
      const int lane = threadIdx.x;
      uint64_t acc = before, acc_w = before_w;
      for (int top = bins - 1; top >= 0; top -= 64) {
        const int b = top - lane;
        const uint64_t w = b >= 0 ? s.wgt[b] : 0;
        const uint64_t c = BY_COUNT ? (b >= 0 ? s.cnt[b] : 0) : w;
        uint64_t run = c, run_w = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint64_t t = shfl64(run, lane - o), tw = shfl64(run_w, lane - o);
          if (lane >= o) { run += t; run_w += tw; }
        }
        const unsigned long long hit = __ballot(acc + run > target);
        if (hit) {
          const int at = __ffsll(hit) - 1;
          if (lane == at) { s.bin = b; s.before_w = acc_w + run_w - w; s.before = acc + run - c; }
          break;
        }
        acc += shfl64(run, 63);
        acc_w += shfl64(run_w, 63);
      }
    }
    __syncthreads();
    prefix = (shift == 32 ? 0 : prefix << bits) | s.bin;
    before = s.before;
    before_w = s.before_w;
    shift = next;
    __syncthreads();
  }
  const uint64_t each_one = BY_COUNT ? 1 : weigh(prefix);
  return {prefix, (uint32_t)((target - before) / each_one), before_w};
}

template <class T>
__global__ __launch_bounds__(THREADS) void sample_kernel(cube_sample_args a, int S) {
  __shared__ Shared s;
  const int r = blockIdx.x, V = a.V, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* row = (const T*)a.logits + (size_t)r * a.ld;
  const float temp = a.temperature ? a.temperature[r] : a.temperature0;
  const int k = a.top_k ? a.top_k[r] : a.top_k0;
  const float p = a.top_p ? a.top_p[r] : a.top_p0;
  const float m = a.min_p ? a.min_p[r] : a.min_p0;

  uint32_t best = 0;
  each(row, V, [&](int, float v) { const uint32_t q = key_of(v); best = q > best ? q : best; });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const uint32_t t = (uint32_t)__shfl_xor((int)best, o, 64); best = t > best ? t : best; }
  if (lane == 0) s.part_c[wave] = best;
  __syncthreads();
  for (int i = 0; i < WAVES; ++i) best = s.part_c[i] > best ? s.part_c[i] : best;
  if (best == 0) {  // nothing is left of the row
    if (threadIdx.x == 0) { a.token[r] = -1; if (a.prob) a.prob[r] = 0.0f; }
    return;
  }
  __syncthreads();

  uint32_t key = best, tie = 0;
  double prob = 1.0;
  if (temp > 0.0f) {
    Weigher weigh;
    weigh.top = (double)value_of(best); weigh.inv_t = 1.0 / (double)temp; weigh.one = (double)(1ull << S); weigh.top_key = best;
    uint64_t total = 0, kept_m = 0;
    uint32_t n = 0;
    const double floor_x = m > 0.0f ? log(m < 1.0f ? (double)m : 1.0) : -INFINITY;
    each(row, V, [&](int, float v) {
      const uint32_t q = key_of(v);
      if (q) {
        const uint64_t w = weigh(q);
        total += w;
        ++n;
        if (q == best || ((double)value_of(q) - weigh.top) * weigh.inv_t >= floor_x) kept_m += w;
      }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { total += shfl64(total, lane ^ o); kept_m += shfl64(kept_m, lane ^ o); n += __shfl_xor((int)n, o, 64); }
    if (lane == 0) { s.wgt[wave] = total; s.wgt[WAVES + wave] = kept_m; s.cnt[wave] = n; }
    __syncthreads();
    total = kept_m = 0; n = 0;
    for (int i = 0; i < WAVES; ++i) { total += s.wgt[i]; kept_m += s.wgt[WAVES + i]; n += s.cnt[i]; }
    __syncthreads();
    if (k > 0 && (uint32_t)k < n) {
      const Place at = find<true>(s, row, V, weigh, (uint64_t)k - 1);
      total = at.before_w + (uint64_t)(at.tie + 1) * weigh(at.key);
    }
    uint64_t kept = total;
    if (p < 1.0f) {
      const double goal = ceil((p > 0.0f ? (double)p : 0.0) * (double)total);
      const uint64_t t = goal >= 1.0 ? (uint64_t)goal - 1 : 0;
      if (t < total) {
        const Place at = find<false>(s, row, V, weigh, t);
        const uint64_t end = at.before_w + (uint64_t)(at.tie + 1) * weigh(at.key);
        kept = end < kept ? end : kept;
      }
    }
    kept = kept_m < kept ? kept_m : kept;
    const double u = a.u[r];
    const double goal = (u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0) * (double)kept;
    uint64_t t = (uint64_t)goal;
    t = t < kept ? t : kept - 1;
    const Place at = find<false>(s, row, V, weigh, t);
    key = at.key;
    tie = at.tie;
    prob = weigh.exact(key) * weigh.one / (double)kept;
  }

  // the tie-th logit equal to `key` in order of index: each wave counts its span, the owner walks its own
  const int span = ((V + WAVES - 1) / WAVES + 63) / 64 * 64;
  const int lo = wave * span < V ? wave * span : V, hi = lo + span < V ? lo + span : V;
  uint32_t mine = 0;
  for (int i = lo; i < hi; i += 64) mine += __popcll(__ballot(i + lane < hi && key_of(as_float(row[i + lane < hi ? i + lane : lo])) == key));
  if (lane == 0) s.part_c[wave] = mine;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < wave; ++i) before += s.part_c[i];
  if (tie >= before && tie < before + mine) {
    for (int i = lo; i < hi; i += 64) {
      const unsigned long long hit = __ballot(i + lane < hi && key_of(as_float(row[i + lane < hi ? i + lane : lo])) == key);
      const uint32_t c = __popcll(hit);
      if (tie < before + c) {
        const bool me = ((hit >> lane) & 1) && before + __popcll(hit & ((1ull << lane) - 1)) == tie;
        if (me) { a.token[r] = i + lane; if (a.prob) a.prob[r] = (float)prob; }
        break;
      }
      before += c;
    }
  }
}

}  // namespace

extern "C" int cube_sample_rows(const cube_sample_args* a, void* stream) {
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
  int bits = 0;
  while ((1 << bits) < a->V) ++bits;
  const int S = 62 - bits < 46 ? 62 - bits : 46;  // V weights of at most 2^S stay below 2^63
  hipStream_t st = (hipStream_t)stream;
  if (a->type == CUBE_T_F32) hipLaunchKernelGGL(sample_kernel<float>, dim3(a->M), dim3(THREADS), 0, st, *a, S);
  else if (a->type == CUBE_T_BF16) hipLaunchKernelGGL(sample_kernel<bf16_t>, dim3(a->M), dim3(THREADS), 0, st, *a, S);
  else hipLaunchKernelGGL(sample_kernel<_Float16>, dim3(a->M), dim3(THREADS), 0, st, *a, S);
  CUBE_CHECK_LAUNCH("cube_sample_rows");
  return CUBE_OK;
}
