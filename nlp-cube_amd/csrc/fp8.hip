// 8-bit floating-point Linear layers with one power-of-two scale for each block of 128 columns (gfx950).
//
//   quantise   e = the smallest integer >= -127 with max|x| <= 448 * 2^e over the block's finite values,
//              q = e4m3(x * 2^-e) (nearest, ties to even), scale byte e + 127 (E8M0)
//   product    out[m, n] = act(bias[n] + sum over blocks of 2^(ea[m,b] + ew[n,b]) * sum over the block of qa[m,k] * qw[n,k])
//
// A power of two and not max/448: x * 2^-e is exact, so a value is rounded once, and the scaled matrix instruction
// (v_mfma_scale_f32_16x16x128_f8f6f4) takes E8M0 bytes itself -- the block scales cost no vector arithmetic and the sum over
// all blocks stays in the instruction's fp32 accumulators.  The rounding error of an e4m3 value does not depend on which
// power of two its block carries, so nothing is lost against a full fp32 scale but up to one bit at the subnormal end.
//
// Layout of quantised rows (the same for activations and weights): bytes [rows, ld], ld >= 128 * ceil(K/128), zeros behind
// column K; scales as 32-bit words [ceil(KB/4), ld_s], KB = ceil(K/128), byte j of word [i, row] = block 4i + j: one 4-byte
// load per row feeds four matrix instructions, and the 16 rows of a fragment are neighbours in memory.
#include <type_traits>

#include "common.h"
#include "../../include/cube_hip.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int BLK = 128;       // columns per scale
constexpr int MAX_K = 1 << 24;  // column indices stay far inside 32 bits,
constexpr int MAX_MN = 1 << 30;  // and rounded-up row and output counts inside them;
constexpr long long MAX_LD = 1LL << 40;  // distances of rows in bytes inside 64

__device__ __forceinline__ float load_val(const float* p) { return *p; }
__device__ __forceinline__ float load_val(const _Float16* p) { return (float)*p; }
__device__ __forceinline__ float load_val(const bf16_t* p) { return (float)*p; }

// eight consecutive values from a 16-byte aligned address
__device__ __forceinline__ void load8(const float* p, float* v) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void load8(const bf16_t* p, float* v) {
  const bf16x8 a = *(const bf16x8*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}
__device__ __forceinline__ void load8(const _Float16* p, float* v) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  const f16x8 a = *(const f16x8*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}

// eight consecutive values from any address: the aligned 16-byte vectors around them, put in place (lo, hi: the bounds of the
// matrix; where a vector would pass them, value by value).  13769x3418 f32 in rows of 8-byte alignment: 87 us value by value.
__device__ __forceinline__ void load8_any(const float* p, const float* lo, const float* hi, float* v) {
  const int mis = (int)(((uintptr_t)p & 15) >> 2);
  const float* a = p - mis;
  if (a >= lo && a + 12 <= hi) {
    const f32x4 w0 = *(const f32x4*)a, w1 = *(const f32x4*)(a + 4), w2 = *(const f32x4*)(a + 8);
    const float w[12] = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3], w2[0], w2[1], w2[2], w2[3]};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mis == 0 ? w[i] : mis == 1 ? w[i + 1] : mis == 2 ? w[i + 2] : w[i + 3];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
  }
}
template <class T> __device__ __forceinline__ void load8_any(const T* p, const T* lo, const T* hi, float* v) {
  static_assert(sizeof(T) == 2, "");
  const int mis = (int)(((uintptr_t)p & 15) >> 1), d = mis >> 1;
  const T* a = p - mis;
  if (a >= lo && a + 16 <= hi) {
    const uint4 w0 = *(const uint4*)a, w1 = *(const uint4*)(a + 8);
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint32_t q[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) q[i] = d == 0 ? w[i] : d == 1 ? w[i + 1] : d == 2 ? w[i + 2] : w[i + 3];
    if (mis & 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = __builtin_amdgcn_alignbit(q[i + 1], q[i], 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)__builtin_bit_cast(T, (uint16_t)(q[i / 2] >> (16 * (i & 1))));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_val(p + i);
  }
}

// columns c .. c+7 of a row of K columns; zeros behind the last one.  VEC: every row starts on 16 bytes
template <class T, bool VEC> __device__ __forceinline__ void load_cols(const T* row, int c, int K, const T* lo, const T* hi, float* v) {
  if (c + 8 <= K) {
    if constexpr (VEC) load8(row + c, v);
    else load8_any(row + c, lo, hi, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? load_val(row + c + i) : 0.0f;
  }
}

// bits of max |x| over the finite values among v[0..8)
__device__ __forceinline__ uint32_t amax_bits(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    const uint32_t f = b < 0x7f800000u ? b : 0u;
    m = f > m ? f : m;
  }
  return m;
}
// maximum over the 16 lanes that share a block: rotations within a DPP row
template <int CTRL> __device__ __forceinline__ uint32_t max_rot(uint32_t m) {
  const uint32_t t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xf, 0xf, false);
  return t > m ? t : m;
}
__device__ __forceinline__ uint32_t max16(uint32_t m) {
  return max_rot<0x128>(max_rot<0x124>(max_rot<0x122>(max_rot<0x121>(m))));
}
// E8M0 byte of a block whose largest finite magnitude has these bits.  448 = 1.75 * 2^8: with max = f * 2^E the exponent is
// E - 8 for f <= 1.75 and E - 7 above; what would fall under 2^-127 (magnitudes below 2^-119, zero among them) stays there
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23) - ((amax & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return e < 0 ? 0 : e;
}
__device__ __forceinline__ uint2 quant8(const float* v, int byte) {
  const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);  // 2^-e, normal for every byte 0 .. 247
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // an infinity becomes NaN, as a NaN does: 8 bits have no infinity, and a saturated one would pass for a number
    s[i] = fabsf(v[i]) < INFINITY ? v[i] * inv : __uint_as_float(0x7fc00000u);
  }
  uint2 r;
  r.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  r.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], (int)r.x, true);
  r.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[4], s[5], 0, false);
  r.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[6], s[7], (int)r.y, true);
  return r;
}

// ---- rows -> quantised rows: one wave per (row, 4 blocks): 8 columns a lane, 16 lanes a block ---------------------------
constexpr int Q_ROWS = 16;  // rows of a workgroup: its scale words are neighbours
template <class T, bool VEC>
__global__ __launch_bounds__(256) void quant_kernel(const T* __restrict__ x, long long ld_x, int M, int K, uint8_t* __restrict__ q,
                                                    long long ld_q, uint32_t* __restrict__ scale, int ld_s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kp = (K + BLK - 1) / BLK * BLK, quads = (kp / BLK + 3) / 4;
  const int quad = blockIdx.x % quads;
  const int c = quad * 4 * BLK + lane * 8;
  const long long r0 = (long long)(blockIdx.x / quads) * Q_ROWS + wave * (Q_ROWS / 4);
  float v[Q_ROWS / 4][8];
#pragma unroll
  for (int i = 0; i < Q_ROWS / 4; ++i) {
    if (r0 + i < M) {
      load_cols<T, VEC>(x + (r0 + i) * ld_x, c, K, x, x + (M - 1) * ld_x + K, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < Q_ROWS / 4; ++i) {
    const long long r = r0 + i;
    const int byte = scale_byte(max16(amax_bits(v[i])));
    const uint2 b = quant8(v[i], byte);
    if (r < M && c < kp) *(uint2*)(q + r * ld_q + c) = b;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) word |= (uint32_t)__builtin_amdgcn_readlane(byte, 16 * j) << (8 * j);
    if (r < M && lane == 0) scale[(long long)quad * ld_s + r] = word;
  }
}

// ---- product ------------------------------------------------------------------------------------------------------------
struct Fp8Params {
  const uint8_t* A; const uint32_t* A_scale; long long lda; int lds_a; int M;
  const uint8_t* W; const uint32_t* W_scale; long long ldw; int lds_w; int N;
  int K, KB; const float* bias; int act; void* out; int out_type; long long ldo; int out_align;  // 16, 4 or a value's size: what every row starts on
  int m_tiles; int n_tiles;
};

// tanh to 2^-22 of itself, as the fp32 sums are (1 - 2 / (e^2v + 1) alone keeps 3e-7 of 1: 1 % of a value of 1e-5).  Up to 0.875 the odd
// polynomial v + v^3 P(v^2), P of the 6th degree through (tanh(v) / v - 1) / v^2 at the Chebyshev nodes: 0.7 * 2^-23 in fp32;
// beyond, the quotient with the instructions' exponential and reciprocal (1 ulp each): at most 1.7 * 2^-23, at 0.875.
__device__ __forceinline__ float tanh_rel(float v) {
  const float a = fabsf(v), t = v * v;
  float q = -5.4758578696049e-04f;
  q = fmaf(q, t, 2.818473154724279e-03f);
  q = fmaf(q, t, -8.499057582911165e-03f);
  q = fmaf(q, t, 2.1777295537199697e-02f);
  q = fmaf(q, t, -5.395686152012646e-02f);
  q = fmaf(q, t, 1.3333279689711994e-01f);
  q = fmaf(q, t, -3.3333332915565317e-01f);
  const float near = fmaf(v * t, q, v);
  const float far = fmaf(-2.0f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(a * 2.8853900817779268f) + 1.0f), 1.0f);
  return a < 0.875f ? near : copysignf(far, v);  // (NaN is not below 0.875, and stays)
}

__device__ __forceinline__ float activate(float v, int act) {
  if (act == CUBE_FP8_TANH) return tanh_rel(v);
  if (act == CUBE_FP8_RELU) return v > 0.0f ? v : (v != v ? v : 0.0f);
  return v;
}

// bias of the columns n .. n+3, read once at a kernel's start: behind the first store the compiler must assume it changed
__device__ __forceinline__ f32x4 bias4(const Fp8Params& p, int n) {
  f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = p.bias[n + i < p.N ? n + i : p.N - 1];
  }
  return b;
}

// four columns n .. n+3 of row m: activation, one rounding to the output type
__device__ __forceinline__ void store4(const Fp8Params& p, int m, int n, f32x4 c) {
  if (m >= p.M || n >= p.N) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = activate(c[i], p.act);
  const bool whole = p.out_align == 16 && n + 4 <= p.N;
  const long long at = (long long)m * p.ldo + n;
  if (p.out_type == CUBE_T_F32) {
    float* o = (float*)p.out + at;
    if (whole) *(f32x4*)o = c;
    else for (int i = 0; i < 4; ++i) if (n + i < p.N) o[i] = c[i];
  } else {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = p.out_type == CUBE_T_BF16 ? f32_to_bf16(c[i]) : __builtin_bit_cast(uint16_t, (_Float16)c[i]);
    uint16_t* o = (uint16_t*)p.out + at;
    if (whole) *(uint2*)o = make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
    else for (int i = 0; i < 4; ++i) if (n + i < p.N) o[i] = h[i];
  }
}

// 32 codes times their block's scale (the low byte of `e`) as bf16: exact, a code has 4 significant bits
struct Frag16 { bf16x8 v[4]; };
__device__ __forceinline__ Frag16 widen(i32x8 q, uint32_t e) {
  const float scale = __uint_as_float((e & 255u) << 23);
  Frag16 f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * h], scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * h], scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * h + 1], scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * h + 1], scale, true);
    f.v[h] = (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  return f;
}

// One block of 128 columns: a fragment is 32 codes and, in the low byte of e, its scale.
// EXACT.  The 8-bit matrix instructions align the products of 8 neighbouring columns to their largest and keep 13 bits below
// it before they reach the fp32 accumulator (measured, the scaled and the unscaled form alike: 1.5e-5 of the result's 2-norm on
// normal data, whatever K): a hundredth of a bf16 step, but too coarse for an fp32 result.  For fp32 outputs the codes are
// widened to bf16 on their way from LDS, the conversion applying the block's scale, and multiplied at half the rate: exactly for
// values from 2^-133 to below 2^128 (what is smaller rounds to a multiple of 2^-133, and 2^128 is infinite, as it is in fp32).
template <bool EXACT> struct Operand;
template <> struct Operand<false> {
  i32x8 q; uint32_t e;
  __device__ __forceinline__ Operand(i32x8 q_, uint32_t e_) : q(q_), e(e_) {}
  __device__ __forceinline__ Operand() {}
};
template <> struct Operand<true> {
  Frag16 f;
  __device__ __forceinline__ Operand(i32x8 q, uint32_t e) : f(widen(q, e)) {}
  __device__ __forceinline__ Operand() {}
};
// c + w . a: the weights are the instruction's first operand, so a lane ends up with four neighbouring output columns of one row
__device__ __forceinline__ f32x4 mma(const Operand<false>& w, const Operand<false>& a, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.q, a.q, c, 0, 0, 0, (int)w.e, 0, (int)a.e);
}
__device__ __forceinline__ f32x4 mma(const Operand<true>& w, const Operand<true>& a, f32x4 c) {
#pragma unroll
  for (int h = 0; h < 4; ++h) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.f.v[h], a.f.v[h], c, 0, 0, 0);
  return c;
}

// LDS-DMA: 64 lanes x 16 (4) bytes to l + lane * 16 (4), l wave-uniform
__device__ __forceinline__ void dma16(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
__device__ __forceinline__ void dma4(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 4, 0, 0);
}
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Tiles of BM rows x BN columns, WM x WN waves; one block of 128 columns of K a step.  A stage in LDS: BM + BN rows of 128 bytes
// whose 16-byte chunks are XOR-swizzled by (row >> 1) & 7 (the swizzle rides on the DMA source address; the 16 rows of a fragment
// read then cover all 64 banks: by row & 7 they met in pairs), and the scale word of every row.  ST stages: step k computes while k + 1 .. k + ST - 1 are on their way; the
// wait for step k counts the later stages' loads instead of draining them.
// Which 32 of the 128 columns a lane group holds does not matter as long as both operands agree, since a step shares its scales.
// KS > 1: as many groups of WM x WN waves share K (each a stretch of its own through stages of its own) and meet in LDS at the end,
// in group order: for few tiles with a long K.
template <int BM, int BN, int WM, int WN, int ST, int KS, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN * KS) void gemm_fp8_kernel(const Fp8Params p) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;      // 1-KiB DMA pieces (8 rows) a wave issues per step
  constexpr int SP = (BM + BN) / 64, PS = (SP + NW - 1) / NW;  // pieces of 64 scale words (waves without one load the last again)
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM % 64 == 0 && BN % 64 == 0, "every wave issues whole pieces");
  constexpr int ROWS = (BM + BN) * BLK, STAGE = ROWS + (BM + BN) * 4;
  constexpr int LOADS = PA + PB + PS;                    // a wave's loads per stage
  // EARLY: a step's barrier and first fragment reads come under the last products of the step before it.  With 8 row tiles a wave, where
  // a workgroup has the CU for itself, that takes up to 1 % off (8192x8192x8192 427 -> 424 us, 8192x4096x4096 109 either way); with fewer,
  // where another workgroup covers them, nothing (2048x2048x2048 13.7 -> 13.8 us, 8192x500x768 f32 13.3 -> 13.4).
  constexpr bool EARLY = TM >= 8;
  constexpr int SLOTS = EARLY ? TM / 2 + 1 : TM;         // row tiles whose products loads go out with
  constexpr int PER = (LOADS + SLOTS - 1) / SLOTS;
  static_assert(!EARLY || KS == 1, "the barriers of wave groups along K are counted for the other form");
  extern __shared__ __attribute__((aligned(16))) unsigned char all_smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / NW, wid = wave % NW;
  unsigned char* smem = all_smem + kg * ST * STAGE;
  const int wm = wid / WN, wn = wid % WN;
  // Workgroups go round-robin over the 8 XCDs, each with an L2 of its own.  The tiles are counted in groups of four row tiles, column
  // by column, and an XCD gets an eighth of that count: the 32 workgroups it runs at once then cover 4 x 8 tiles and share 12 operand
  // tiles (2 x 16 of a row-major order share 18: 3 % more time at 8192x4096x4096), and no XCD has more than one tile over another.
  const int tiles = p.m_tiles * p.n_tiles, eighth = (tiles + 7) / 8;
  const int tile = (blockIdx.x & 7) * eighth + (blockIdx.x >> 3);
  if (tile >= tiles) return;  // whole workgroup, before any barrier
  const int group = tile / (4 * p.n_tiles), in = tile - group * 4 * p.n_tiles;
  const int high = p.m_tiles - 4 * group < 4 ? p.m_tiles - 4 * group : 4;  // row tiles of the group
  const int nt = in / high, mt = 4 * group + in - nt * high;
  const int m0 = mt * BM, n0 = nt * BN;

  // a load's address: the tile's first row (uniform) and 32 bits of offset inside the tile (255 rows of at most 2^24 bytes)
  const uint8_t* a_base = p.A + (long long)m0 * p.lda;
  const uint8_t* b_base = p.W + (long long)n0 * p.ldw;
  uint32_t off[PA + PB], s_off[PS];
  const int pr = lane >> 3, chunk = (lane & 7) ^ ((4 * (wid & 1) + (pr >> 1)) & 7);  // (row >> 1) & 7: a wave's pieces are NW apart
  static_assert(NW % 2 == 0, "so that their rows agree in bit 3");
#pragma unroll
  for (int i = 0; i < PA; ++i) {  // rows behind the last one read the last one; their results are not stored
    const int r = 8 * (wid + NW * i) + pr;
    off[i] = (uint32_t)(r < p.M - m0 ? r : p.M - 1 - m0) * (uint32_t)p.lda + chunk * 16;
  }
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int r = 8 * (wid + NW * i) + pr;
    off[PA + i] = (uint32_t)(r < p.N - n0 ? r : p.N - 1 - n0) * (uint32_t)p.ldw + chunk * 16;
  }
#pragma unroll
  for (int i = 0; i < PS; ++i) {
    const int piece = wid + NW * i < SP ? wid + NW * i : SP - 1;
    const int t = 64 * piece + lane;  // row of the stage: activations, then weights (64 | BM: a piece is of one kind)
    const bool of_a = 64 * piece < BM;
    const int r = of_a ? t : t - BM, last = (of_a ? p.M - m0 : p.N - n0) - 1;
    s_off[i] = 4 * (uint32_t)(r < last ? r : last);
  }
  // this group's steps
  const int per = (p.KB + KS - 1) / KS, first = kg * per;
  const int steps = KS == 1 ? p.KB : p.KB - first < per ? (p.KB > first ? p.KB - first : 0) : per;
  // load `i` of this group's step k: activations, weights, scale words
  auto load = [&](int k, int i) {
    unsigned char* buf = smem + (k % ST) * STAGE;
    if (i < PA) {
      dma16(a_base + (size_t)(first + k) * BLK + off[i], buf + 8 * (wid + NW * i) * BLK);
    } else if (i < PA + PB) {
      dma16(b_base + (size_t)(first + k) * BLK + off[i], buf + (BM + 8 * (wid + NW * (i - PA))) * BLK);
    } else {
      const int of = wid + NW * (i - PA - PB), t = of < SP ? of : SP - 1;
      const uint32_t* s = 64 * t < BM ? p.A_scale + (long long)((first + k) >> 2) * p.lds_a + m0 : p.W_scale + (long long)((first + k) >> 2) * p.lds_w + n0;
      dma4((const uint8_t*)s + s_off[i - PA - PB], buf + ROWS + 64 * t * 4);
    }
  };
  auto fill = [&](int k) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(k, i);
  };
  const int l15 = lane & 15, g = lane >> 4;
  f32x4 bias[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) bias[j] = bias4(p, n0 + (wn * TN + j) * 16 + 4 * g);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = KS == 1 || kg == 0 ? bias[j] : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  // this lane's two chunks of a row of a fragment
  const int o0 = l15 * BLK + ((g ^ (l15 >> 1)) << 4), o1 = l15 * BLK + (((g + 4) ^ (l15 >> 1)) << 4);
  auto meet = [&] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // fragment and scale word of one of a stage's tiles of 16 rows
  auto frag = [&](const unsigned char* cur, int tile) {
    return __builtin_shufflevector(*(const i32x4*)(cur + tile * 16 * BLK + o0), *(const i32x4*)(cur + tile * 16 * BLK + o1), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto scale = [&](const unsigned char* cur, int k, int tile) { return *(const uint32_t*)(cur + ROWS + (tile * 16 + l15) * 4) >> (8 * ((first + k) & 3)); };
  // One step.  CONT: loads of stage k + ST - 1 between the products (all at once in front of them they held up the fragment reads).
  // EARLY: the step's first fragments are in registers already; when its last row tile's fragment has been read, the wait and the
  // barrier of the next step come -- all waves are then done with this step's stage -- and the last products cover the reads of the
  // next fragments.  START: the first loads of stage k + ST behind that barrier; NEXT: there is a next step.
  i32x8 wq[TN], next;
  uint32_t we[TN], ea[TM];
  auto begin = [&](int k) {
    const unsigned char* cur = smem + (k % ST) * STAGE;
#pragma unroll
    for (int i = 0; i < TM; ++i) ea[i] = scale(cur, k, wm * TM + i);
    next = frag(cur, wm * TM);
  };
  auto weight = [&](int k, int j) {
    const unsigned char* cur = smem + (k % ST) * STAGE;
    wq[j] = frag(cur, BM / 16 + wn * TN + j);
    we[j] = scale(cur, k, BM / 16 + wn * TN + j);
  };
  auto step = [&](int k, auto CONT, auto START, auto NEXT) {
    const unsigned char* cur = smem + (k % ST) * STAGE;
    if constexpr (!EARLY) {
      meet();
      begin(k);
#pragma unroll
      for (int j = 0; j < TN; ++j) weight(k, j);
    }
    Operand<EXACT> w[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) w[j] = Operand<EXACT>(wq[j], we[j]);
#pragma unroll
    for (int i = 0; i < TM; ++i) {  // a row tile's fragment is read while the one before it is multiplied
      const Operand<EXACT> a(next, ea[i]);
      if (i + 1 < TM) next = frag(cur, wm * TM + i + 1);
      if constexpr (decltype(CONT)::value) {
#pragma unroll
        for (int u = (i + EARLY) * PER; u < (i + EARLY + 1) * PER && u < LOADS; ++u) load(k + ST - 1, u);
      }
      if (EARLY && i == TM - 1) {
        if constexpr (decltype(NEXT)::value) {
          // step k + 1 has landed once no more loads are open than the later stages'; the barrier says so for every wave's pieces
          if constexpr (decltype(CONT)::value) wait_vm<(ST - 2) * LOADS>();
          else wait_vm<0>();
          meet();
          begin(k + 1);
        }
        if constexpr (decltype(START)::value) {
#pragma unroll
          for (int u = 0; u < PER && u < LOADS; ++u) load(k + ST, u);
        }
      }
      if constexpr (!EXACT) __builtin_amdgcn_sched_barrier(0);  // the compiler would put the read right in front of its use
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[i][j] = mma(w[j], a, acc[i][j]);
        if constexpr (decltype(NEXT)::value) {
          if (i == TM - 1) weight(k + 1, j);
        }
      }
      if constexpr (!EXACT) __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int k = 0; k < ST - 1; ++k)
    if (k < steps) fill(k);
  int k = 0;
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  if constexpr (EARLY) {
    if (steps >= ST) {
#pragma unroll
      for (int u = 0; u < PER && u < LOADS; ++u) load(ST - 1, u);
      wait_vm<(ST - 2) * LOADS + (PER < LOADS ? PER : LOADS)>();
    } else {
      wait_vm<0>();
    }
    meet();
    begin(0);
#pragma unroll
    for (int j = 0; j < TN; ++j) weight(0, j);
    for (; k + ST < steps; ++k) step(k, yes, yes, yes);
    if (k + ST == steps) step(k++, yes, no, yes);
    for (; k + 1 < steps; ++k) step(k, no, no, yes);
    step(k, no, no, no);
  } else {
    // step k has landed once no more loads are open than the later stages'; the barrier in the step says so for every wave's pieces,
    // and that all waves are done with the stage that is filled next
    for (; k < steps - (ST - 1); ++k) {
      wait_vm<(ST - 2) * LOADS>();
      step(k, yes, no, no);
    }
    for (; k < steps; ++k) {
      wait_vm<0>();
      step(k, no, no, no);
    }
  }
  if constexpr (KS > 1) {
    for (; k < per; ++k) meet();  // a group with fewer steps comes to as many barriers
    meet();
    f32x4* part = (f32x4*)all_smem;  // [KS - 1][waves][TM][TN][64]
    static_assert((KS - 1) * NW * TM * TN * 1024 <= KS * ST * STAGE, "the partial sums fit in the stages' LDS");
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) part[((((kg - 1) * NW + wid) * TM + i) * TN + j) * 64 + lane] = acc[i][j];
    }
    meet();
    if (kg > 0) return;
#pragma unroll
    for (int q = 0; q < KS - 1; ++q)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const f32x4 o = part[(((q * NW + wid) * TM + i) * TN + j) * 64 + lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] += o[r];
        }
  }

  // ---- results: activation and rounding in registers, then through LDS (a wave its own part), so that whole rows of the wave's
  // columns go out 16 bytes a lane; 16-byte chunks XOR-swizzled by the row
  if (p.act == CUBE_FP8_TANH) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = activate(acc[i][j][r], CUBE_FP8_TANH);
  } else if (p.act == CUBE_FP8_RELU) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = activate(acc[i][j][r], CUBE_FP8_RELU);
  }
  constexpr int ES = EXACT ? 4 : 2, RB = 16 * TN * ES, SWZ = RB >= 128 ? 7 : RB / 16 - 1;  // bytes of a value, of a row
  static_assert((RB & (RB - 1)) == 0 && RB >= 32, "the swizzle stays inside the row");
  static_assert(NW * 16 * TM * RB <= KS * ST * STAGE, "the results fit in the stages' LDS");
  meet();  // all waves are done with the last stage (and with the partial sums)
  unsigned char* mine = smem + wid * 16 * TM * RB;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const f32x4 c = acc[i][j];
      unsigned char* row = mine + (16 * i + l15) * RB;
      const int byte = (16 * j + 4 * g) * ES;
      unsigned char* at = row + ((((byte >> 4) ^ (l15 & SWZ)) << 4) | (byte & 15));
      if constexpr (EXACT) {
        *(f32x4*)at = c;
      } else {
        uint16_t h[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          h[r] = p.out_type == CUBE_T_BF16 ? f32_to_bf16(c[r]) : __builtin_bit_cast(uint16_t, (_Float16)c[r]);
        *(uint2*)at = make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
      }
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int mw = m0 + wm * TM * 16, nw = n0 + wn * TN * 16;  // the wave's part of the output
  unsigned char* out = (unsigned char*)p.out;
  // units of U bytes, as wide as the output's rows are aligned; a unit that would pass the last column makes it single values
  auto copy = [&](auto unit) {
    using U = decltype(unit);
    constexpr int UNITS = RB / (int)sizeof(U), PER_UNIT = (int)sizeof(U) / ES, WIDE = UNITS < 64 ? UNITS : 64, R = 64 / WIDE;
#pragma unroll 4
    for (int row0 = 0; row0 < 16 * TM; row0 += R) {
      const int row = row0 + lane / WIDE;
      if (mw + row < p.M) {
#pragma unroll
        for (int u = lane % WIDE; u < UNITS; u += WIDE) {
          const int byte = u * (int)sizeof(U);
          const U v = *(const U*)(mine + row * RB + ((((byte >> 4) ^ (row & SWZ)) << 4) | (byte & 15)));
          if (nw + u * PER_UNIT < p.N) *(U*)(out + ((long long)(mw + row) * p.ldo + nw) * ES + byte) = v;
        }
      }
    }
  };
  const int align = nw + 16 * TN <= p.N ? p.out_align : ES;
  if (align == 16) copy(uint4{});
  else if (align == 4 || ES == 4) copy(uint32_t{});
  else copy(uint16_t{});
}

// Few rows: the weights are read once, straight into registers, in tiles of 16 columns.  KW = 8: a workgroup has a tile and its 8
// waves share K (wave v takes the blocks v, v + 8, ...); their sums meet in LDS, in wave order.  KW = 1: every wave has a tile of its
// own and all of K (no barrier), where there are tiles enough for all waves.  T: the type of the activations.  Plain rows are quantised into LDS
// by every workgroup for itself (the first weight loads are already on their way); e4m3 rows are read where they are.
constexpr int FEW_ROWS = 32, FUSED_ROWS = 48, FEW_WAVES = 8, FEW_LDS = 38 * 1024, FEW_AHEAD = 4, FEW_GRID = 1024;
__host__ __device__ inline int few_stride(int KB) { return KB * BLK + 16; }  // bytes of a row in LDS: 16 rows then cover all banks
__host__ __device__ inline long long few_rows_bytes(int rows, int KB) { return ((long long)rows * (few_stride(KB) + KB) + 15) / 16 * 16; }  // with scales
template <class T, bool VEC, int MT, int KW, bool EXACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_fp8_kernel(const Fp8Params p) {
  constexpr bool PLAIN = !std::is_same<T, uint8_t>::value;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l15 = lane & 15, g = lane >> 4;
  const int kw = KW == 1 ? 0 : wave;  // this wave's first block of K
  int n0 = (KW == 1 ? blockIdx.x * FEW_WAVES + wave : blockIdx.x) * 16;
  const int n_step = (KW == 1 ? gridDim.x * FEW_WAVES : gridDim.x) * 16;
  const int rows = p.M;  // at most 16 * MT
  const uint8_t* wrow;
  const uint32_t* ws;
  auto columns = [&](int n) {
    const int nr = n + l15 < p.N ? n + l15 : p.N - 1;
    wrow = p.W + (long long)nr * p.ldw + g * 32;
    ws = p.W_scale + nr;
  };
  columns(n0);
  i32x4 wq[FEW_AHEAD][2];
  uint32_t we[FEW_AHEAD];
  auto load_w = [&](int u, int kb) {
    if (kb < p.KB) {
      wq[u][0] = *(const i32x4*)(wrow + (size_t)kb * BLK);
      wq[u][1] = *(const i32x4*)(wrow + (size_t)kb * BLK + 16);
      we[u] = ws[(long long)(kb >> 2) * p.lds_w];
    }
  };
#pragma unroll
  for (int u = 0; u < FEW_AHEAD; ++u) load_w(u, kw + KW * u);

  const int stride = few_stride(p.KB);
  unsigned char* a_scale = smem + (size_t)rows * stride;  // [rows][KB] scale bytes
  if constexpr (PLAIN) {
    const T* x = (const T*)p.A;
    const int per = p.KB * (BLK / 8), total = rows * per;  // pieces of 8 columns; 16 lanes a block, so blocks never straddle waves
    constexpr int BATCH = 4;  // pieces of a thread whose loads are on their way together
    for (int i0 = threadIdx.x; i0 < (total + 63) / 64 * 64; i0 += 64 * FEW_WAVES * BATCH) {
      float v[BATCH][8];
      int r[BATCH], c[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + 64 * FEW_WAVES * u;
        if (i - lane >= total) break;  // whole waves
        r[u] = i < total ? i / per : 0;
        c[u] = i < total ? (i - r[u] * per) * 8 : 0;
        load_cols<T, VEC>(x + (long long)r[u] * p.lda, c[u], i < total ? p.K : 0, x, x + (long long)(p.M - 1) * p.lda + p.K, v[u]);
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        if (i0 + 64 * FEW_WAVES * u - lane >= total) break;
        const int byte = scale_byte(max16(amax_bits(v[u])));
        const uint2 q = quant8(v[u], byte);
        if (i0 + 64 * FEW_WAVES * u < total) {
          *(uint2*)(smem + (size_t)r[u] * stride + c[u]) = q;
          if ((lane & 15) == 0) a_scale[r[u] * p.KB + c[u] / BLK] = (unsigned char)byte;
        }
      }
    }
    __syncthreads();
  }
  int ar[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) ar[t] = 16 * t + l15 < rows ? 16 * t + l15 : rows - 1;
  f32x4* part = (f32x4*)(smem + (PLAIN ? few_rows_bytes(rows, p.KB) : 0));
  // column tiles in turn: the activations in LDS serve them all (KW = 8: a workgroup's waves come to the end together)
  while (KW != 1 || n0 < p.N) {
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const f32x4 bias = bias4(p, n0 + 4 * g);
    const int n_next = n0 + n_step;
    for (int kb0 = kw; kb0 < p.KB; kb0 += KW * FEW_AHEAD) {
#pragma unroll
      for (int u = 0; u < FEW_AHEAD; ++u) {
        const int kb = kb0 + KW * u;
        if (kb < p.KB) {  // wave-uniform
          const Operand<EXACT> w((i32x8){wq[u][0][0], wq[u][0][1], wq[u][0][2], wq[u][0][3], wq[u][1][0], wq[u][1][1], wq[u][1][2], wq[u][1][3]},
                                 we[u] >> (8 * (kb & 3)));
          load_w(u, kb + KW * FEW_AHEAD);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            i32x4 lo, hi;
            uint32_t e;
            if constexpr (PLAIN) {
              const unsigned char* b = smem + (size_t)ar[t] * stride + kb * BLK + g * 32;
              lo = *(const i32x4*)b;
              hi = *(const i32x4*)(b + 16);
              e = a_scale[ar[t] * p.KB + kb];
            } else {
              const uint8_t* b = p.A + (long long)ar[t] * p.lda + (size_t)kb * BLK + g * 32;
              lo = *(const i32x4*)b;
              hi = *(const i32x4*)(b + 16);
              e = p.A_scale[(long long)(kb >> 2) * p.lds_a + ar[t]] >> (8 * (kb & 3));
            }
            const Operand<EXACT> a((i32x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, e);
            acc[t] = mma(w, a, acc[t]);
          }
        }
      }
    }
    if (n_next < p.N) {  // the next tile's first weights, under the sums
      columns(n_next);
#pragma unroll
      for (int u = 0; u < FEW_AHEAD; ++u) load_w(u, kw + KW * u);
    }
    if constexpr (KW == 1) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4 c = acc[t];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += bias[i];
        store4(p, 16 * t + l15, n0 + 4 * g, c);
      }
      n0 = n_next;
      continue;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) part[(wave * MT + t) * 64 + lane] = acc[t];
    __syncthreads();
    if (wave < MT) {
      f32x4 c = bias;
#pragma unroll
      for (int v = 0; v < FEW_WAVES; ++v) {
        const f32x4 o = part[(v * MT + wave) * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += o[i];
      }
      store4(p, 16 * wave + l15, n0 + 4 * g, c);
    }
    if (n_next >= p.N) break;
    n0 = n_next;
    __syncthreads();  // the sums in LDS have been read
  }
}

inline int type_size(int t) { return t == CUBE_T_F32 ? 4 : 2; }
inline int kblocks(int K) { return (K - 1) / BLK + 1; }

template <class T> int launch_quant(const void* x, long long ld_x, int M, int K, void* q, long long ld_q, uint32_t* scale, int ld_s,
                                    hipStream_t st) {
  const int quads = (kblocks(K) + 3) / 4;
  // 16-byte loads where every row starts on a 16-byte boundary
  const bool vec = ((uintptr_t)x & 15) == 0 && (ld_x * (long long)sizeof(T)) % 16 == 0;
  const int part = (1 << 23) / quads * Q_ROWS;  // rows of a launch: fewer than 2^32 threads (K <= 2^24: at most 2^15 quads)
  for (long long r0 = 0; r0 < M; r0 += part) {
    const int n = (int)(M - r0 < part ? M - r0 : part);
    const dim3 grid((unsigned)quads * ((n + Q_ROWS - 1) / Q_ROWS));
    const T* from = (const T*)x + r0 * ld_x;
    uint8_t* to = (uint8_t*)q + r0 * ld_q;
    if (vec) hipLaunchKernelGGL((quant_kernel<T, true>), grid, dim3(256), 0, st, from, ld_x, n, K, to, ld_q, scale + r0, ld_s);
    else hipLaunchKernelGGL((quant_kernel<T, false>), grid, dim3(256), 0, st, from, ld_x, n, K, to, ld_q, scale + r0, ld_s);
    CUBE_CHECK_LAUNCH("cube_quant_fp8");
  }
  return CUBE_OK;
}
int quant_any(const void* x, int type, long long ld_x, int M, int K, void* q, long long ld_q, uint32_t* scale, int ld_s, hipStream_t st) {
  if (type == CUBE_T_F32) return launch_quant<float>(x, ld_x, M, K, q, ld_q, scale, ld_s, st);
  if (type == CUBE_T_BF16) return launch_quant<bf16_t>(x, ld_x, M, K, q, ld_q, scale, ld_s, st);
  return launch_quant<_Float16>(x, ld_x, M, K, q, ld_q, scale, ld_s, st);
}

template <int BM, int BN, int WM, int WN, int ST, int KS, bool EXACT> int launch_tiles(Fp8Params& p, hipStream_t st) {
  constexpr int LDS = KS * ST * (BM + BN) * (BLK + 4);
  static CubeLdsReservation lds;
  p.m_tiles = (p.M + BM - 1) / BM;
  p.n_tiles = (p.N + BN - 1) / BN;
  const long long blocks = ((long long)p.m_tiles * p.n_tiles + 7) / 8 * 8;
  if (blocks > 0x7ffffff0LL) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: %d x %d outputs are too many", p.M, p.N);
  if (!lds.ensure((const void*)gemm_fp8_kernel<BM, BN, WM, WN, ST, KS, EXACT>, LDS)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_gemm_fp8: LDS reservation failed");
  hipLaunchKernelGGL((gemm_fp8_kernel<BM, BN, WM, WN, ST, KS, EXACT>), dim3((unsigned)blocks), dim3(64 * WM * WN * KS), LDS, st, p);
  CUBE_CHECK_LAUNCH("cube_gemm_fp8");
  return CUBE_OK;
}

template <class T, bool VEC, int MT, int KW, bool EXACT> int launch_few(const Fp8Params& p, hipStream_t st) {
  static CubeLdsReservation lds;
  const int rows = p.M;
  const size_t bytes = (size_t)FEW_WAVES * MT * 64 * 16 + (std::is_same<T, uint8_t>::value ? 0 : few_rows_bytes(rows, p.KB));
  if (!lds.ensure((const void*)few_fp8_kernel<T, VEC, MT, KW, EXACT>, bytes)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_gemm_fp8: LDS reservation failed");
  const int tiles = KW == 1 ? (p.N + 16 * FEW_WAVES - 1) / (16 * FEW_WAVES) : (p.N + 15) / 16;
  const dim3 grid(tiles < FEW_GRID ? tiles : FEW_GRID);
  hipLaunchKernelGGL((few_fp8_kernel<T, VEC, MT, KW, EXACT>), grid, dim3(64 * FEW_WAVES), bytes, st, p);
  CUBE_CHECK_LAUNCH("cube_gemm_fp8");
  return CUBE_OK;
}
template <class T, bool VEC, int MT> int launch_few(const Fp8Params& p, hipStream_t st) {
  const bool exact = p.out_type == CUBE_T_F32;
  // a tile for every wave of four workgroups a CU (1 row, 768 columns, 250002 outputs: 38 us, the weights' bytes at the rate of a
  // copy; shared tiles 71)
  if (p.N >= 16 * FEW_WAVES * FEW_GRID) return exact ? launch_few<T, VEC, MT, 1, true>(p, st) : launch_few<T, VEC, MT, 1, false>(p, st);
  return exact ? launch_few<T, VEC, MT, FEW_WAVES, true>(p, st) : launch_few<T, VEC, MT, FEW_WAVES, false>(p, st);
}
template <class T, bool VEC> int launch_few(const Fp8Params& p, hipStream_t st) {
  if (p.M <= 16) return launch_few<T, VEC, 1>(p, st);
  if (p.M <= 32) return launch_few<T, VEC, 2>(p, st);
  return launch_few<T, VEC, 3>(p, st);
}

// The few-row kernel reads the weights once for up to 32 rows (4096x4096: 16 rows 6.5 us, tiles 9.8; 40 rows 13, tiles 10).  It also
// saves the launch that quantises, while every workgroup quantising all rows costs less: up to 48 rows of some 36000 values in all
// (768x768: 33 rows 6.9 us, two launches 8.8; 64 rows 10.4, two launches 8.8;  4096x4096: 4 rows 8.6 us, 16 rows 16, two launches 11).
bool fused(int M, int K) { return M <= FUSED_ROWS && few_rows_bytes(M, kblocks(K)) <= FEW_LDS; }

int launch_gemm(Fp8Params& p, hipStream_t st) {
  const bool exact = p.out_type == CUBE_T_F32;
  if (p.M <= 16) return launch_few<uint8_t, true, 1>(p, st);
  if (p.M <= FEW_ROWS) return launch_few<uint8_t, true, 2>(p, st);
  // The largest tile that still gives every CU work, by the number of tiles (launches one behind the other from a graph, 16-bit
  // output and no activation unless said):
  //   256x256: 8192x4096x4096 111 us (128x128: 139 us), where their last round fills 4 of 5 CUs:  5000x4000x2000, 320 of them,
  //     60 us (54 us), 8192x3000x1024, 384, 43 us (39 us).  A narrow output fills no such tile, and the count does not see it:
  //     65536x16x768 23 us (128x64 13)
  //   128x128 (two workgroups a CU): 8192x768x768 10.8 us (128x64 12.8, 64x64 14.8), 8000x520x8000 53 us (67, 68);
  //     256 of them, one a CU, lose: 2048x2048x2048 16.2 us (128x64 14.4)
  //   128x64: 4096x1024x1024 9.3 us (64x64 11.4), 8192x500x768 f32 13.4 us (15.7)
  //   64x64 with four stages: 512x768x768 4.6 us (128x64 5.7), 1001x500x300 f32 5.1 us (6.5)
  //   the same with four wave groups along K: 65x4096x4096 9.8 us (one group 12.2), 65x64x8000 f32 20.5 us (28.4); with a K of
  //     1024 and less it loses: 65x4096x1024 5.6 us (5.1)
  auto tiles = [&](int bm, int bn) { return (long long)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  const long long big = tiles(256, 256), rounds = (big + 255) / 256;
  if (!exact && 5 * big >= 4 * 256 * rounds) return launch_tiles<256, 256, 2, 4, 2, 1, false>(p, st);
  if (tiles(128, 128) > 256) return exact ? launch_tiles<128, 128, 2, 2, 2, 1, true>(p, st) : launch_tiles<128, 128, 2, 2, 2, 1, false>(p, st);
  if (tiles(64, 64) > 512) return exact ? launch_tiles<128, 64, 4, 1, 3, 1, true>(p, st) : launch_tiles<128, 64, 4, 1, 3, 1, false>(p, st);
  if (tiles(64, 64) <= 256 && p.KB >= 16) return exact ? launch_tiles<64, 64, 2, 2, 2, 4, true>(p, st) : launch_tiles<64, 64, 2, 2, 2, 4, false>(p, st);
  return exact ? launch_tiles<64, 64, 2, 2, 4, 1, true>(p, st) : launch_tiles<64, 64, 2, 2, 4, 1, false>(p, st);
}

size_t quant_bytes(int M, int K) {
  const size_t q = (size_t)M * kblocks(K) * BLK;
  return q + (size_t)((kblocks(K) + 3) / 4) * M * 4;
}

CubeArea code_area(const void* q, long long ld, int rows, int K) { return {q, ld, (long long)kblocks(K) * BLK, rows}; }
CubeArea scale_area(const uint32_t* s, int ld, int rows, int K) { return {s, 4LL * ld, 4LL * rows, (kblocks(K) + 3) / 4}; }
CubeArea plain_area(const void* x, int type, long long ld, int rows, int columns) {
  return {x, ld * type_size(type), (long long)columns * type_size(type), rows};
}
// what neither the output nor the workspace may touch; A_scale: NULL where A is plain
const char* touches(const CubeArea& to, const cube_fp8_args* a, const uint32_t* A_scale, const CubeArea& A) {
  if (cube_overlap(A, to)) return "A";
  if (A_scale && cube_overlap(scale_area(A_scale, a->lds_a, a->M, a->K), to)) return "A_scale";
  if (cube_overlap(code_area(a->W, a->ldw, a->N, a->K), to)) return "W";
  if (cube_overlap(scale_area(a->W_scale, a->lds_w, a->N, a->K), to)) return "W_scale";
  if (cube_overlap({a->bias, 4LL * a->N}, to)) return "bias";
  return nullptr;
}

// what cube_gemm_fp8 and cube_linear_fp8 check alike
int check_args(const cube_fp8_args* a, const char* who) {
  if (a->M < 0 || a->N < 0 || a->M > MAX_MN || a->N > MAX_MN || a->K < 1 || a->K > MAX_K) CUBE_FAIL(CUBE_ERR_ARG, "%s: M=%d N=%d K=%d", who, a->M, a->N, a->K);
  if (a->M == 0 || a->N == 0) return CUBE_OK;
  if (!a->A || !a->W || !a->W_scale || !a->out) CUBE_FAIL(CUBE_ERR_ARG, "%s: null A / W / W_scale / out", who);
  if (a->out_type < CUBE_T_F32 || a->out_type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "%s: out_type=%d", who, a->out_type);
  if (a->act < CUBE_FP8_NONE || a->act > CUBE_FP8_RELU) CUBE_FAIL(CUBE_ERR_ARG, "%s: act=%d", who, a->act);
  if (a->ldw < (long long)kblocks(a->K) * BLK || a->lds_w < a->N || a->ldo < a->N || a->ldo > MAX_LD)
    CUBE_FAIL(CUBE_ERR_ARG, "%s: ldw=%lld (>= %lld), lds_w=%d (>= N=%d), ldo=%lld (>= N)", who, a->ldw, (long long)kblocks(a->K) * BLK,
              a->lds_w, a->N, a->ldo);
  if (a->ldw > MAX_K) CUBE_FAIL(CUBE_ERR_ARG, "%s: ldw=%lld is over %d", who, a->ldw, MAX_K);
  if (((uintptr_t)a->W & 15) || a->ldw % 16) CUBE_FAIL(CUBE_ERR_ALIGN, "%s: rows of W are not 16-byte aligned", who);
  if (((uintptr_t)a->W_scale | (uintptr_t)a->bias) & 3) CUBE_FAIL(CUBE_ERR_ALIGN, "%s: W_scale / bias are not 4-byte aligned", who);
  if ((uintptr_t)a->out % type_size(a->out_type)) CUBE_FAIL(CUBE_ERR_ALIGN, "%s: out is not aligned to its type", who);
  return CUBE_OK;
}

Fp8Params params(const cube_fp8_args* a) {
  Fp8Params p;
  p.A = (const uint8_t*)a->A; p.A_scale = a->A_scale; p.lda = a->lda; p.lds_a = a->lds_a; p.M = a->M;
  p.W = (const uint8_t*)a->W; p.W_scale = a->W_scale; p.ldw = a->ldw; p.lds_w = a->lds_w; p.N = a->N;
  p.K = a->K; p.KB = kblocks(a->K); p.bias = a->bias; p.act = a->act; p.out = a->out; p.out_type = a->out_type; p.ldo = a->ldo;
  const int es = type_size(a->out_type);
  const uintptr_t at = (uintptr_t)a->out | (uintptr_t)(a->ldo * es);
  p.out_align = at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : es;
  return p;
}

}  // namespace

extern "C" int cube_quant_fp8(const void* x, int x_type, long long ld_x, int M, int K, void* q, long long ld_q, uint32_t* scale,
                              int ld_s, void* stream) {
  CUBE_ENTRY();
  if (M < 0 || M > MAX_MN || K < 1 || K > MAX_K) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: M=%d K=%d", M, K);
  if (M == 0) return CUBE_OK;
  if (!x || !q || !scale) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: null x / q / scale");
  if (x_type < CUBE_T_F32 || x_type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: x_type=%d", x_type);
  if (ld_x < K || ld_x > MAX_LD || ld_q > MAX_LD || ld_q < (long long)kblocks(K) * BLK || ld_s < M)
    CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: ld_x=%lld (>= K=%d), ld_q=%lld (>= %lld), ld_s=%d (>= M=%d)", ld_x, K, ld_q,
              (long long)kblocks(K) * BLK, ld_s, M);
  if (((uintptr_t)q & 15) || ld_q % 16) CUBE_FAIL(CUBE_ERR_ALIGN, "cube_quant_fp8: rows of q are not 16-byte aligned");
  if ((uintptr_t)x % type_size(x_type) || ((uintptr_t)scale & 3)) CUBE_FAIL(CUBE_ERR_ALIGN, "cube_quant_fp8: x / scale not aligned to their types");
  const CubeArea from = plain_area(x, x_type, ld_x, M, K), codes = code_area(q, ld_q, M, K), words = scale_area(scale, ld_s, M, K);
  if (cube_overlap(from, codes) || cube_overlap(from, words) || cube_overlap(codes, words))
    CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: x, q and scale overlap");
  return quant_any(x, x_type, ld_x, M, K, q, ld_q, scale, ld_s, (hipStream_t)stream);
}

extern "C" int cube_gemm_fp8(const cube_fp8_args* a, void* stream) {
  CUBE_ENTRY();
  if (!a) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: null args");
  if (a->a_type != CUBE_T_E4M3) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: a_type=%d, want CUBE_T_E4M3 (cube_linear_fp8 takes plain rows)", a->a_type);
  const int rc = check_args(a, "cube_gemm_fp8");
  if (rc) return rc;
  if (a->M == 0 || a->N == 0) return CUBE_OK;
  if (!a->A_scale || a->lda < (long long)kblocks(a->K) * BLK || a->lds_a < a->M || a->lda > MAX_K)
    CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: null A_scale, lda=%lld (>= %lld, <= 2^24) or lds_a=%d (>= M=%d)", a->lda, (long long)kblocks(a->K) * BLK,
              a->lds_a, a->M);
  if (((uintptr_t)a->A & 15) || a->lda % 16 || ((uintptr_t)a->A_scale & 3))
    CUBE_FAIL(CUBE_ERR_ALIGN, "cube_gemm_fp8: rows of A are not 16-byte aligned, or A_scale not 4-byte aligned");
  const char* met = touches(plain_area(a->out, a->out_type, a->ldo, a->M, a->N), a, a->A_scale, code_area(a->A, a->lda, a->M, a->K));
  if (met) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: out overlaps %s", met);
  Fp8Params p = params(a);
  return launch_gemm(p, (hipStream_t)stream);
}

extern "C" size_t cube_linear_fp8_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || M > MAX_MN || N <= 0 || K <= 0 || K > MAX_K || fused(M, K)) return 0;
  return quant_bytes(M, K);
}

extern "C" int cube_linear_fp8(const cube_fp8_args* a, void* ws, size_t ws_bytes, void* stream) {
  CUBE_ENTRY();
  if (!a) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: null args");
  if (a->a_type < CUBE_T_F32 || a->a_type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: a_type=%d, want f32, bf16 or f16 rows", a->a_type);
  const int rc = check_args(a, "cube_linear_fp8");
  if (rc) return rc;
  if (a->M == 0 || a->N == 0) return CUBE_OK;
  if (a->lda < a->K || a->lda > MAX_LD) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: lda=%lld (>= K=%d)", a->lda, a->K);
  if ((uintptr_t)a->A % type_size(a->a_type)) CUBE_FAIL(CUBE_ERR_ALIGN, "cube_linear_fp8: A is not aligned to its type");
  const size_t need = cube_linear_fp8_workspace_bytes(a->M, a->N, a->K);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: workspace of %zu bytes (need %zu, 16-byte aligned)", ws_bytes, need);
  const CubeArea from = plain_area(a->A, a->a_type, a->lda, a->M, a->K), out = plain_area(a->out, a->out_type, a->ldo, a->M, a->N);
  const char* met = touches(out, a, nullptr, from);
  if (met) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: out overlaps %s", met);
  if (need) {
    const CubeArea work = {ws, (long long)need};
    met = cube_overlap(out, work) ? "out" : touches(work, a, nullptr, from);
    if (met) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: the workspace overlaps %s", met);
  }
  Fp8Params p = params(a);
  hipStream_t st = (hipStream_t)stream;
  if (!need) {
    const bool vec = ((uintptr_t)a->A & 15) == 0 && (a->lda * type_size(a->a_type)) % 16 == 0;
    if (a->a_type == CUBE_T_F32) return vec ? launch_few<float, true>(p, st) : launch_few<float, false>(p, st);
    if (a->a_type == CUBE_T_BF16) return vec ? launch_few<bf16_t, true>(p, st) : launch_few<bf16_t, false>(p, st);
    return vec ? launch_few<_Float16, true>(p, st) : launch_few<_Float16, false>(p, st);
  }
  const long long kp = (long long)kblocks(a->K) * BLK;
  uint32_t* scale = (uint32_t*)((uint8_t*)ws + (size_t)a->M * kp);
  const int qc = quant_any(a->A, a->a_type, a->lda, a->M, a->K, ws, kp, scale, a->M, st);
  if (qc) return qc;
  p.A = (const uint8_t*)ws; p.A_scale = scale; p.lda = kp; p.lds_a = a->M;
  return launch_gemm(p, st);
}
