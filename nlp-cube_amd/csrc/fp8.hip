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
constexpr int MAX_K = 1 << 24;  // column indices stay far inside 32 bits

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

// columns c .. c+7 of a row of K columns; zeros behind the last one
template <class T, bool VEC> __device__ __forceinline__ void load_cols(const T* row, int c, int K, float* v) {
  if (VEC && c + 8 <= K) {
    load8(row + c, v);
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
// maximum over the 16 lanes that share a block
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_xor((int)m, o, 64);
    m = t > m ? t : m;
  }
  return m;
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
      load_cols<T, VEC>(x + (r0 + i) * ld_x, c, K, v[i]);
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
  int K, KB; const float* bias; int act; void* out; int out_type; long long ldo; int vec_out;
  int m_tiles; int n_tiles;
};

__device__ __forceinline__ float activate(float v, int act) {
  if (act == CUBE_FP8_TANH) return tanhf_(v);
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
  const bool whole = p.vec_out && n + 4 <= p.N;
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
// widened to bf16 on their way from LDS, the conversion applying the block's scale, and multiplied at half the rate.
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
// whose 16-byte chunks are XOR-swizzled by row & 7 (the swizzle rides on the DMA source address; fragment reads of 8 lanes then
// cover all banks), and the scale word of every row.  ST stages: step k computes while k + 1 .. k + ST - 1 are on their way; the
// wait for step k counts the later stages' loads instead of draining them.
// Which 32 of the 128 columns a lane group holds does not matter as long as both operands agree, since a step shares its scales.
template <int BM, int BN, int WM, int WN, int ST, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void gemm_fp8_kernel(const Fp8Params p) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;      // 1-KiB DMA pieces (8 rows) a wave issues per step
  constexpr int PS = (BM + BN) / 64 / NW;                // pieces of 64 scale words
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && (BM + BN) % (64 * NW) == 0, "every wave issues whole pieces");
  constexpr int ROWS = (BM + BN) * BLK, STAGE = ROWS + (BM + BN) * 4;
  constexpr int LOADS = PA + PB + PS;                    // a wave's loads per stage
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid / WN, wn = wid % WN;
  // workgroups go round-robin over the 8 XCDs: the column tiles of a row tile get consecutive slots of one XCD, whose L2 then
  // holds that row tile's activations once
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const int mt = (slot / p.n_tiles) * 8 + xcd, nt = slot % p.n_tiles;
  if (mt >= p.m_tiles) return;  // whole workgroup, before any barrier
  const int m0 = mt * BM, n0 = nt * BN;

  const uint8_t* src[PA + PB];
  const uint32_t* s_src[PS];
  const int pr = lane >> 3, chunk = (lane & 7) ^ (pr & 7);
#pragma unroll
  for (int i = 0; i < PA; ++i) {  // rows behind the last one read the last one; their results are not stored
    const int r = m0 + 8 * (wid + NW * i) + pr;
    src[i] = p.A + (long long)(r < p.M ? r : p.M - 1) * p.lda + chunk * 16;
  }
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int r = n0 + 8 * (wid + NW * i) + pr;
    src[PA + i] = p.W + (long long)(r < p.N ? r : p.N - 1) * p.ldw + chunk * 16;
  }
  long long s_step[PS];
#pragma unroll
  for (int i = 0; i < PS; ++i) {
    const int t = 64 * (wid + NW * i) + lane;  // row of the stage: activations, then weights (64 | BM: a piece is of one kind)
    const bool of_a = 64 * (wid + NW * i) < BM;
    const int r = of_a ? m0 + t : n0 + t - BM, last = (of_a ? p.M : p.N) - 1;
    s_src[i] = (of_a ? p.A_scale : p.W_scale) + (r < last ? r : last);
    s_step[i] = of_a ? p.lds_a : p.lds_w;
  }
  auto fill = [&](int k) {
    unsigned char* buf = smem + (k % ST) * STAGE;
#pragma unroll
    for (int i = 0; i < PA; ++i) dma16(src[i] + (size_t)k * BLK, buf + 8 * (wid + NW * i) * BLK);
#pragma unroll
    for (int i = 0; i < PB; ++i) dma16(src[PA + i] + (size_t)k * BLK, buf + (BM + 8 * (wid + NW * i)) * BLK);
#pragma unroll
    for (int i = 0; i < PS; ++i) dma4(s_src[i] + (long long)(k >> 2) * s_step[i], buf + ROWS + 64 * (wid + NW * i) * 4);
  };
  const int l15 = lane & 15, g = lane >> 4;
  f32x4 bias[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) bias[j] = bias4(p, n0 + (wn * TN + j) * 16 + 4 * g);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = bias[j];

#pragma unroll
  for (int k = 0; k < ST - 1; ++k)
    if (k < p.KB) fill(k);
  const int c0 = ((2 * g) ^ (l15 & 7)) << 4, c1 = ((2 * g + 1) ^ (l15 & 7)) << 4;  // this lane's two chunks of a row
  for (int k = 0; k < p.KB; ++k) {
    const unsigned char* cur = smem + (k % ST) * STAGE;
    // step k has landed once no more loads are open than the later stages'; the barrier says so for every wave's pieces, and
    // that all waves are done with the stage that is filled next
    if (k + ST - 2 < p.KB) wait_vm<(ST - 2) * LOADS>(); else wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (k + ST - 1 < p.KB) fill(k + ST - 1);
    const int shift = 8 * (k & 3);
    auto frag = [&](int row) {
      const unsigned char* b = cur + row * BLK;
      const i32x4 lo = *(const i32x4*)(b + c0), hi = *(const i32x4*)(b + c1);
      return Operand<EXACT>((i32x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]},
                            *(const uint32_t*)(cur + ROWS + row * 4) >> shift);
    };
    Operand<EXACT> w[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) w[j] = frag(BM + (wn * TN + j) * 16 + l15);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const Operand<EXACT> a = frag((wm * TM + i) * 16 + l15);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mma(w[j], a, acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
      store4(p, m0 + (wm * TM + i) * 16 + l15, n0 + (wn * TN + j) * 16 + 4 * g, acc[i][j]);
}

// Few rows: the weights are read once, straight into registers, 16 columns a workgroup, and its 8 waves share K (wave v takes the
// blocks v, v + 8, ...); their sums meet in LDS, in wave order.  T: the type of the activations.  Plain rows are quantised into LDS
// by every workgroup for itself (the first weight loads are already on their way); e4m3 rows are read where they are.
constexpr int FEW_ROWS = 64, FEW_WAVES = 8, FEW_LDS = 64 * 1024, FEW_AHEAD = 4;
__host__ __device__ inline int few_stride(int KB) { return KB * BLK + 16; }  // bytes of a row in LDS: 16 rows then cover all banks
template <class T, bool VEC, int MT, bool EXACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_fp8_kernel(const Fp8Params p) {
  constexpr bool PLAIN = !std::is_same<T, uint8_t>::value;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l15 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MT);
  const int rows = p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT;
  const int nr = n0 + l15 < p.N ? n0 + l15 : p.N - 1;
  const uint8_t* wrow = p.W + (long long)nr * p.ldw + g * 32;
  const uint32_t* ws = p.W_scale + nr;
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
  for (int u = 0; u < FEW_AHEAD; ++u) load_w(u, wave + FEW_WAVES * u);
  const f32x4 bias = bias4(p, n0 + 4 * g);

  const int stride = few_stride(p.KB);
  unsigned char* a_scale = smem + (size_t)rows * stride;  // [rows][KB] scale bytes
  if constexpr (PLAIN) {
    const T* x = (const T*)p.A + (long long)m0 * p.lda;
    const int per = p.KB * (BLK / 8), total = rows * per;  // pieces of 8 columns; 16 lanes a block, so blocks never straddle waves
    for (int i = threadIdx.x; i < (total + 63) / 64 * 64; i += 64 * FEW_WAVES) {
      const bool on = i < total;
      const int r = on ? i / per : 0, c = on ? (i - r * per) * 8 : 0;
      float v[8];
      load_cols<T, VEC>(x + (long long)r * p.lda, c, on ? p.K : 0, v);
      const int byte = scale_byte(max16(amax_bits(v)));
      const uint2 q = quant8(v, byte);
      if (on) {
        *(uint2*)(smem + (size_t)r * stride + c) = q;
        if ((lane & 15) == 0) a_scale[r * p.KB + c / BLK] = (unsigned char)byte;
      }
    }
    __syncthreads();
  }
  int ar[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) ar[t] = 16 * t + l15 < rows ? 16 * t + l15 : rows - 1;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb0 = wave; kb0 < p.KB; kb0 += FEW_WAVES * FEW_AHEAD) {
#pragma unroll
    for (int u = 0; u < FEW_AHEAD; ++u) {
      const int kb = kb0 + FEW_WAVES * u;
      if (kb < p.KB) {  // wave-uniform
        const Operand<EXACT> w((i32x8){wq[u][0][0], wq[u][0][1], wq[u][0][2], wq[u][0][3], wq[u][1][0], wq[u][1][1], wq[u][1][2], wq[u][1][3]},
                               we[u] >> (8 * (kb & 3)));
        load_w(u, kb + FEW_WAVES * FEW_AHEAD);
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
            const uint8_t* b = p.A + (long long)(m0 + ar[t]) * p.lda + (size_t)kb * BLK + g * 32;
            lo = *(const i32x4*)b;
            hi = *(const i32x4*)(b + 16);
            e = p.A_scale[(long long)(kb >> 2) * p.lds_a + m0 + ar[t]] >> (8 * (kb & 3));
          }
          const Operand<EXACT> a((i32x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, e);
          acc[t] = mma(w, a, acc[t]);
        }
      }
    }
  }
  __syncthreads();  // the activations in LDS are done with
  f32x4* part = (f32x4*)smem;
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
    store4(p, m0 + 16 * wave + l15, n0 + 4 * g, c);
  }
}

inline int type_size(int t) { return t == CUBE_T_F32 ? 4 : 2; }
inline int kblocks(int K) { return (K - 1) / BLK + 1; }

template <class T> int launch_quant(const void* x, long long ld_x, int M, int K, void* q, long long ld_q, uint32_t* scale, int ld_s,
                                    hipStream_t st) {
  const long long blocks = (long long)((kblocks(K) + 3) / 4) * ((M + Q_ROWS - 1) / Q_ROWS);
  if (blocks > 0x7fffffffLL) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: %d x %d values are too many for one launch", M, K);
  const dim3 grid((unsigned)blocks);
  // 16-byte loads where every row starts on a 16-byte boundary
  const bool vec = ((uintptr_t)x & 15) == 0 && (ld_x * (long long)sizeof(T)) % 16 == 0;
  if (vec) hipLaunchKernelGGL((quant_kernel<T, true>), grid, dim3(256), 0, st, (const T*)x, ld_x, M, K, (uint8_t*)q, ld_q, scale, ld_s);
  else hipLaunchKernelGGL((quant_kernel<T, false>), grid, dim3(256), 0, st, (const T*)x, ld_x, M, K, (uint8_t*)q, ld_q, scale, ld_s);
  CUBE_CHECK_LAUNCH("cube_quant_fp8");
  return CUBE_OK;
}
int quant_any(const void* x, int type, long long ld_x, int M, int K, void* q, long long ld_q, uint32_t* scale, int ld_s, hipStream_t st) {
  if (type == CUBE_T_F32) return launch_quant<float>(x, ld_x, M, K, q, ld_q, scale, ld_s, st);
  if (type == CUBE_T_BF16) return launch_quant<bf16_t>(x, ld_x, M, K, q, ld_q, scale, ld_s, st);
  return launch_quant<_Float16>(x, ld_x, M, K, q, ld_q, scale, ld_s, st);
}

template <int BM, int BN, int WM, int WN, int ST, bool EXACT> int launch_tiles(Fp8Params& p, hipStream_t st) {
  constexpr int LDS = ST * (BM + BN) * (BLK + 4);
  static CubeLdsReservation lds;
  p.m_tiles = (p.M + BM - 1) / BM;
  p.n_tiles = (p.N + BN - 1) / BN;
  const long long blocks = (long long)((p.m_tiles + 7) / 8 * 8) * p.n_tiles;
  if (blocks > 0x7fffffffLL) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: %d x %d outputs are too many", p.M, p.N);
  if (!lds.ensure((const void*)gemm_fp8_kernel<BM, BN, WM, WN, ST, EXACT>, LDS)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_gemm_fp8: LDS reservation failed");
  hipLaunchKernelGGL((gemm_fp8_kernel<BM, BN, WM, WN, ST, EXACT>), dim3((unsigned)blocks), dim3(64 * WM * WN), LDS, st, p);
  CUBE_CHECK_LAUNCH("cube_gemm_fp8");
  return CUBE_OK;
}

template <class T, bool VEC, int MT, bool EXACT> int launch_few(const Fp8Params& p, hipStream_t st) {
  static CubeLdsReservation lds;
  const int rows = p.M < 16 * MT ? p.M : 16 * MT;
  const size_t sums = (size_t)FEW_WAVES * MT * 64 * 16;
  const size_t act = std::is_same<T, uint8_t>::value ? 0 : (size_t)rows * (few_stride(p.KB) + p.KB);
  const size_t bytes = act > sums ? act : sums;
  if (!lds.ensure((const void*)few_fp8_kernel<T, VEC, MT, EXACT>, bytes)) CUBE_FAIL(CUBE_ERR_LAUNCH, "cube_gemm_fp8: LDS reservation failed");
  const dim3 grid((p.N + 15) / 16, (p.M + 16 * MT - 1) / (16 * MT));
  if (grid.y > 65535u) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: %d rows are too many", p.M);
  hipLaunchKernelGGL((few_fp8_kernel<T, VEC, MT, EXACT>), grid, dim3(64 * FEW_WAVES), bytes, st, p);
  CUBE_CHECK_LAUNCH("cube_gemm_fp8");
  return CUBE_OK;
}
template <class T, bool VEC> int launch_few(const Fp8Params& p, hipStream_t st) {
  const bool exact = p.out_type == CUBE_T_F32;
  if (p.M <= 16) return exact ? launch_few<T, VEC, 1, true>(p, st) : launch_few<T, VEC, 1, false>(p, st);
  if (p.M <= 32) return exact ? launch_few<T, VEC, 2, true>(p, st) : launch_few<T, VEC, 2, false>(p, st);
  return exact ? launch_few<T, VEC, 4, true>(p, st) : launch_few<T, VEC, 4, false>(p, st);
}

// plain rows that the few-row kernel quantises by itself: few, and short enough to lie in LDS beside each other
bool fused(int M, int K) { return M <= FEW_ROWS && (long long)M * few_stride(kblocks(K)) <= FEW_LDS; }

int launch_gemm(Fp8Params& p, hipStream_t st) {
  const bool exact = p.out_type == CUBE_T_F32;
  if (p.M <= FEW_ROWS) return launch_few<uint8_t, true>(p, st);
  const long long big = (long long)((p.M + 255) / 256) * ((p.N + 255) / 256);
  if (!exact && big >= 256) return launch_tiles<256, 256, 2, 4, 2, false>(p, st);
  const long long mid = (long long)((p.M + 127) / 128) * ((p.N + 127) / 128);
  if (mid >= 128) return exact ? launch_tiles<128, 128, 2, 2, 2, true>(p, st) : launch_tiles<128, 128, 2, 2, 2, false>(p, st);
  return exact ? launch_tiles<64, 64, 2, 1, 4, true>(p, st) : launch_tiles<64, 64, 2, 1, 4, false>(p, st);
}

size_t quant_bytes(int M, int K) {
  const size_t q = (size_t)M * kblocks(K) * BLK;
  return q + (size_t)((kblocks(K) + 3) / 4) * M * 4;
}

// what cube_gemm_fp8 and cube_linear_fp8 check alike
int check_args(const cube_fp8_args* a, const char* who) {
  if (a->M < 0 || a->N < 0 || a->K < 1 || a->K > MAX_K) CUBE_FAIL(CUBE_ERR_ARG, "%s: M=%d N=%d K=%d", who, a->M, a->N, a->K);
  if (a->M == 0 || a->N == 0) return CUBE_OK;
  if (!a->A || !a->W || !a->W_scale || !a->out) CUBE_FAIL(CUBE_ERR_ARG, "%s: null A / W / W_scale / out", who);
  if (a->out_type < CUBE_T_F32 || a->out_type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "%s: out_type=%d", who, a->out_type);
  if (a->act < CUBE_FP8_NONE || a->act > CUBE_FP8_RELU) CUBE_FAIL(CUBE_ERR_ARG, "%s: act=%d", who, a->act);
  if (a->ldw < (long long)kblocks(a->K) * BLK || a->lds_w < a->N || a->ldo < a->N)
    CUBE_FAIL(CUBE_ERR_ARG, "%s: ldw=%lld (>= %lld), lds_w=%d (>= N=%d), ldo=%lld (>= N)", who, a->ldw, (long long)kblocks(a->K) * BLK,
              a->lds_w, a->N, a->ldo);
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
  p.vec_out = (uintptr_t)a->out % (4 * es) == 0 && a->ldo % 4 == 0;
  return p;
}

}  // namespace

extern "C" int cube_quant_fp8(const void* x, int x_type, long long ld_x, int M, int K, void* q, long long ld_q, uint32_t* scale,
                              int ld_s, void* stream) {
  CUBE_ENTRY();
  if (M < 0 || K < 1 || K > MAX_K) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: M=%d K=%d", M, K);
  if (M == 0) return CUBE_OK;
  if (!x || !q || !scale) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: null x / q / scale");
  if (x_type < CUBE_T_F32 || x_type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: x_type=%d", x_type);
  if (ld_x < K || ld_q < (long long)kblocks(K) * BLK || ld_s < M)
    CUBE_FAIL(CUBE_ERR_ARG, "cube_quant_fp8: ld_x=%lld (>= K=%d), ld_q=%lld (>= %lld), ld_s=%d (>= M=%d)", ld_x, K, ld_q,
              (long long)kblocks(K) * BLK, ld_s, M);
  if (((uintptr_t)q & 15) || ld_q % 16) CUBE_FAIL(CUBE_ERR_ALIGN, "cube_quant_fp8: rows of q are not 16-byte aligned");
  if ((uintptr_t)x % type_size(x_type) || ((uintptr_t)scale & 3)) CUBE_FAIL(CUBE_ERR_ALIGN, "cube_quant_fp8: x / scale not aligned to their types");
  return quant_any(x, x_type, ld_x, M, K, q, ld_q, scale, ld_s, (hipStream_t)stream);
}

extern "C" int cube_gemm_fp8(const cube_fp8_args* a, void* stream) {
  CUBE_ENTRY();
  if (!a) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: null args");
  if (a->a_type != CUBE_T_E4M3) CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: a_type=%d, want CUBE_T_E4M3 (cube_linear_fp8 takes plain rows)", a->a_type);
  const int rc = check_args(a, "cube_gemm_fp8");
  if (rc) return rc;
  if (a->M == 0 || a->N == 0) return CUBE_OK;
  if (!a->A_scale || a->lda < (long long)kblocks(a->K) * BLK || a->lds_a < a->M)
    CUBE_FAIL(CUBE_ERR_ARG, "cube_gemm_fp8: null A_scale, lda=%lld (>= %lld) or lds_a=%d (>= M=%d)", a->lda, (long long)kblocks(a->K) * BLK,
              a->lds_a, a->M);
  if (((uintptr_t)a->A & 15) || a->lda % 16 || ((uintptr_t)a->A_scale & 3))
    CUBE_FAIL(CUBE_ERR_ALIGN, "cube_gemm_fp8: rows of A are not 16-byte aligned, or A_scale not 4-byte aligned");
  Fp8Params p = params(a);
  return launch_gemm(p, (hipStream_t)stream);
}

extern "C" size_t cube_linear_fp8_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > MAX_K || fused(M, K)) return 0;
  return quant_bytes(M, K);
}

extern "C" int cube_linear_fp8(const cube_fp8_args* a, void* ws, size_t ws_bytes, void* stream) {
  CUBE_ENTRY();
  if (!a) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: null args");
  if (a->a_type < CUBE_T_F32 || a->a_type > CUBE_T_F16) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: a_type=%d, want f32, bf16 or f16 rows", a->a_type);
  const int rc = check_args(a, "cube_linear_fp8");
  if (rc) return rc;
  if (a->M == 0 || a->N == 0) return CUBE_OK;
  if (a->lda < a->K) CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: lda=%lld < K=%d", a->lda, a->K);
  if ((uintptr_t)a->A % type_size(a->a_type)) CUBE_FAIL(CUBE_ERR_ALIGN, "cube_linear_fp8: A is not aligned to its type");
  const size_t need = cube_linear_fp8_workspace_bytes(a->M, a->N, a->K);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    CUBE_FAIL(CUBE_ERR_ARG, "cube_linear_fp8: workspace of %zu bytes (need %zu, 16-byte aligned)", ws_bytes, need);
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
