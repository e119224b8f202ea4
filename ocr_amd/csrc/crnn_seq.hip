// Kernels of the sequence operators (include/crnn_hip.h: crnn_linear, crnn_rms_norm, crnn_cross_attention), gfx950.
// Compiled without packed fp32 (crnn_kernels_nopk.hip says why).
#include "crnn_seq.h"
#include "crnn_kernels.h"

#include <cmath>
#include <type_traits>

namespace crnn {

typedef int i32x2b __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned char e4m3;   // the byte of an e4m3 value

// Workgroups of a launch: a grid of 2^24 workgroups of 256 would pass the 2^32 threads a launch may have, so the kernels
// below take their tiles or rows in strides of the grid.
static dim3 grid_for(int64_t tiles) { return dim3((unsigned)(tiles < (1 << 22) ? tiles : 1 << 22)); }

template <int TYPE> struct TypeOf;
template <> struct TypeOf<CRNN_FP32> { typedef float t; };
template <> struct TypeOf<CRNN_BF16> { typedef __bf16 t; };
template <> struct TypeOf<CRNN_E4M3> { typedef e4m3 t; };

// C/D map of the 32x32 MFMAs: lane l, register r hold column l & 31 and row (r & 3) + 8 (r >> 2) + 4 (l >> 5), rows being the
// FIRST operand's index
__device__ __forceinline__ int acc_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// Lane exchanges without LDS: x of lane ^ F for F 1, 2, 8 (F 4: of the other four of eight lanes, where each four agree), and for 16
// and 32 both halves' values, in the same order in both.
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
struct Two {
  float a, b;
};
template <int F> __device__ __forceinline__ Two two(float x) {
  if constexpr (F == 1) return Two{x, dpp<0xB1>(x)};        // quad_perm 1 0 3 2
  else if constexpr (F == 2) return Two{x, dpp<0x4E>(x)};   // quad_perm 2 3 0 1
  else if constexpr (F == 8) return Two{x, dpp<0x128>(x)};  // row_ror 8
  else if constexpr (F == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return Two{__uint_as_float(r[0]), __uint_as_float(r[1])};
  } else if constexpr (F == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return Two{__uint_as_float(r[0]), __uint_as_float(r[1])};
  } else {
    return Two{x, __shfl_xor(x, F)};
  }
}
// Sum over N neighbouring lanes.
template <int N> __device__ __forceinline__ float group_sum(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  if constexpr (N > 4) x += dpp<0x141>(x);   // row_half_mirror
  if constexpr (N > 8) x += dpp<0x140>(x);   // row_mirror
  if constexpr (N > 16) {
    const Two t = two<16>(x);
    x = t.a + t.b;
  }
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
  const Two t = two<32>(group_sum<32>(x));
  return t.a + t.b;
}

// x Phi(x) = max(x, 0) - |x| Phi(-|x|), and Phi(-y) = erfc(y / sqrt 2) / 2 by Abramowitz & Stegun 7.1.26: (a1 t + ... + a5 t^5)
// exp(-y^2 / 2) / 2, t = 1 / (1 + p y / sqrt 2), off by at most 0.75e-7; with what 32 bits lose on the way x Phi(x) is off by at
// most 11.4 2^-24 |x| (largest seen 4.8 2^-24 |x|, near 0), also where the result is far smaller, as 1 + erf in 32 bits is.  (With
// erff and expf 18176 x 512 x 2048 took 32 us more than without activation.)  Infinities give their limits, inf and 0,
// because in one product 0 times infinity is 0 (v_mul_legacy_f32; a cap on |x| costs an instruction more, 4 us there).
// (A vector instruction that reads v_rcp_f32's result waits for one state, which the compiler does not see to in assembly.)
__device__ __forceinline__ float mul_legacy(float a, float b) {
  float r;
  asm("s_nop 0\n\tv_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float gelu(float v) {
  const float y = fabsf(v), t = __builtin_amdgcn_rcpf(fmaf(0.23164190f, y, 1.f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5307027145f, -0.7265760135f), 0.7107068705f), -0.142248368f), 0.127414796f);
  const float e = __builtin_amdgcn_exp2f(v * v * -0.72134752044448170f);
  float yp;
  asm("v_mul_legacy_f32 %0, |%1|, %2" : "=v"(yp) : "v"(v), "v"(p));   // (p is a product: nothing to wait for)
  return fmaf(-yp, e, v > 0.f ? v : 0.f);
}
__device__ __forceinline__ float silu(float v) { return mul_legacy(v, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f))); }
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case CRNN_ACT_RELU: return v < 0.f ? 0.f : v;   // (a NaN stays one)
    case CRNN_ACT_LEAKY: return v < 0.f ? 0.2f * v : v;
    case CRNN_ACT_GELU: return gelu(v);
    case CRNN_ACT_SILU: return silu(v);
    default: return v;
  }
}

// Eight neighbouring values of a row, at the alignment of one.
template <typename T> struct Eight { typedef T t __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const typename Eight<T>::t a = *(const typename Eight<T>::t*)p;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  typename Eight<T>::t a;
#pragma unroll
  for (int i = 0; i < 8; i++) a[i] = (T)v[i];
  *(typename Eight<T>::t*)p = a;
}
__device__ __forceinline__ void store8(e4m3* p, const float (&v)[8]) {
  i32x2b a;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
    a[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], u, true);
  }
  *(i32x2b*)p = a;
}

__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }
__device__ __forceinline__ void store1(e4m3* p, float v) { *p = (e4m3)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xFF); }
// Of a row of n values those at i .. i + 7 that exist.
template <typename T>
__device__ __forceinline__ void part8(const T* row, int i, int n, float (&v)[8]) {
  if (i + 8 <= n) load8(row + i, v);
  else if (i < n) {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (i + e < n) v[e] = (float)row[i + e];
  }
}
template <typename T>
__device__ __forceinline__ void put8(T* row, int i, int n, const float (&v)[8]) {
  if (i + 8 <= n) store8(row + i, v);
  else if (i < n) {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (i + e < n) store1(row + i + e, v[e]);
  }
}

// Direct loads from memory into LDS: lane l's 16 bytes at `voff` + `soff` land at `lds` + 16 l; offsets past the resource give zeros.
// The compiler does not count them: every use of the data is behind a wait of its own.
__device__ __forceinline__ void dma16(i32x4 rsrc, unsigned lds, unsigned voff, unsigned soff = 0) {
  unsigned m0_saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(m0_saved) : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}
constexpr unsigned OUTSIDE = 0x80000000u;   // past every resource below
__device__ __forceinline__ i32x4 resource(const void* p) {
  const unsigned long long u = (unsigned long long)p;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((unsigned)u), (int)(__builtin_amdgcn_readfirstlane((unsigned)(u >> 32)) & 0xFFFF), 0x7FFFFFFF, 0x00020000};
}

template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
  if (act == CRNN_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = gelu(v[e]);
  } else if (act == CRNN_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = silu(v[e]);
  } else if (act != CRNN_ACT_NONE) {
    const float slope = act == CRNN_ACT_LEAKY ? 0.2f : 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = v[e] < 0.f ? (act == CRNN_ACT_RELU ? 0.f : slope * v[e]) : v[e];
  }
}

// ---------------------------------------------------------------------------
// linear, rows of whole 16-byte chunks (8 bits: with bf16 results): a tile of 64 MT rows x 32 NT WN columns of y per workgroup,
// 2 x WN waves of 32 MT x 32 NT each.  A step is 128 bytes of k of every row, straight from memory into one of NST LDS stages.
// 16-byte chunk c of row r sits at c ^ ((r >> 1) & 7): the 16 rows that ds_read_b128 reads at once then lie in
// different parts of the 256 bytes that LDS serves in a cycle, and SQ_LDS_BANK_CONFLICT stays 0.  w is the first operand,
// so that a lane holds four neighbouring columns of one row of y (v_mfma_f32_32x32x16_bf16, four slices a step; 8 bits:
// v_mfma_f32_32x32x64_f8f6f4, two).  Each slice's operands are read during the slice before.  One barrier a step, in its last
// slice: by then everybody has read this step's stage, and the loads for NST steps on go into it.  Steps past the end load zeros,
// which keeps the count of loads in flight the same to the last step.  KG groups of waves take steps in turn and add up at the
// end where tiles are few.
// Where k is long matrix instructions are busy 65 % of the time, at the 1.6 to 1.9 GHz that power leaves the chip then: bf16 8192 x
// 8192 x 8192 828 to 844 us, 1300 to 1330 TF/s (the library's product in turn with it: 680 to 760); 8 bits 18176 x 2048 x 2048 81
// to 85 us, 1830 TF/s.  Where k is short, by the way in and out, which
// nothing hides: 18176 x k x 2048 takes 24 us and 30 more for each 512 of k, 14 of the 24 being the rows that leave.  (One workgroup a CU
// that loads its next tile before it writes the last: 59 us for k = 512, this 56.)
// ---------------------------------------------------------------------------
template <int IN> struct Slice;
template <> struct Slice<CRNN_BF16> {
  static constexpr int KB = 32;   // bytes of k of a slice
  typedef i32x4 frag;
  static __device__ __forceinline__ frag read(const unsigned char* row, int ks, int half, int swz) { return *(const i32x4*)(row + (((2 * ks + half) ^ swz) << 4)); }
  static __device__ __forceinline__ f32x16 mfma(frag w, frag x, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
  }
};
template <> struct Slice<CRNN_E4M3> {
  static constexpr int KB = 64;
  typedef i32x8 frag;
  static __device__ __forceinline__ frag read(const unsigned char* row, int ks, int half, int swz) {
    const int c = 4 * ks + 2 * half;
    const i32x4 a = *(const i32x4*)(row + ((c ^ swz) << 4)), b = *(const i32x4*)(row + (((c + 1) ^ swz) << 4));
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  static __device__ __forceinline__ f32x16 mfma(frag w, frag x, f32x16 c) { return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 0, 0, 0, 0, 0, 0); }
};

template <> struct Slice<CRNN_FP32> {   // one 16-byte chunk a lane: four v_mfma_f32_32x32x2_f32, each with one value of both halves
  static constexpr int KB = 32;
  typedef f32x4 frag;
  static __device__ __forceinline__ frag read(const unsigned char* row, int ks, int half, int swz) { return *(const f32x4*)(row + (((2 * ks + half) ^ swz) << 4)); }
  static __device__ __forceinline__ f32x16 mfma(frag w, frag x, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(w[i], x[i], c, 0, 0, 0);
    return c;
  }
};

// fp32 in three bfloat16 parts: x = h + m + l, each what is left rounded to 8 bits, so that l holds the rest exactly and the parts have
// either sign (bits of them below 2^-126 may be lost, what a product with subnormal operands taken as 0 loses of a whole
// operand).  m is at most 2^-8 of x and l 2^-17.  Of the nine products the six largest are multiplied (v_mfma_f32_32x32x16_bf16 at 16
// times the rate of the f32 instructions); the others come to at most 2^-24 of the product, of either sign.  (Parts that are cut off
// have x's sign and are twice as large: up to 7.8 2^-24 of a product are missing then, which sums do not average out.  They took
// 719 us where these take 779; with v_cvt_pk_bf16_f32 4544 x 512 x 512 34 and 33.)  An infinity makes h infinite and m NaN, a NaN l, and
// values near the largest may overflow on the way: results that are not finite are computed again (finite_sums).  4096 x 4096 x
// 4096 722 to 779 us by box, 176 to 190 TF/s; on the f32 instructions 1057 us, 130 TF/s.
struct Parts {
  bf16x8 p[3];
};
__device__ __forceinline__ Parts split3(i32x8 raw) {
  Parts s;
#pragma unroll
  for (int part = 0; part < 3; part++) {
    i32x4 packed;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      unsigned up[2];   // (half a step added; l has no bits to round)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const unsigned r = (unsigned)raw[2 * i + e];
        up[e] = r + (part < 2 ? 0x8000u : 0u);
        if (part < 2) raw[2 * i + e] = (int)__float_as_uint(__uint_as_float(r) - __uint_as_float(up[e] & 0xFFFF0000u));
      }
      packed[i] = __builtin_amdgcn_perm(up[1], up[0], 0x07060302);   // the upper halves of both
    }
    s.p[part] = __builtin_bit_cast(bf16x8, packed);
  }
  return s;
}
__device__ __forceinline__ f32x16 mfma3(const Parts& w, const Parts& x, f32x16 c) {   // the small products first
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.p[2], x.p[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.p[0], x.p[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.p[1], x.p[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.p[1], x.p[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.p[0], x.p[1], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.p[0], x.p[0], c, 0, 0, 0);
}

// Results of the three-part products that are not finite, again on the f32 instructions: sums of a wave's 32 MT x 32 NT part of y
// whose first row and column are m0, n0.
template <int MT, int NT>
__device__ __forceinline__ void finite_sums(const crnn_linear_args& a, f32x16 (&acc)[NT][MT], int64_t m0, int64_t n0, int lane) {
  bool fine = true;
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) fine = fine && fabsf(acc[i][j][r]) < INFINITY;
  if (__all(fine)) return;
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int j = 0; j < MT; j++) {
      const int64_t n = n0 + i * 32 + (lane & 31), m = m0 + j * 32 + (lane & 31);
      f32x16 t;
#pragma unroll
      for (int r = 0; r < 16; r++) t[r] = 0.f;
#pragma unroll 4
      for (int64_t k = lane >> 5; k < ((a.k + 1) & ~(int64_t)1); k += 2) {   // (every lane to the same end)
        const float w = n < a.n && k < a.k ? ((const float*)a.w)[n * a.ldw + k] : 0.f;
        const float x = m < a.m && k < a.k ? ((const float*)a.x)[m * a.ldx + k] : 0.f;
        t = __builtin_amdgcn_mfma_f32_32x32x2f32(w, x, t, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = fabsf(acc[i][j][r]) < INFINITY ? acc[i][j][r] : t[r];
    }
}

// Up to eight values of a row of y, one by one: residual, rounding, store.
template <typename TO>
__device__ __forceinline__ void put(const crnn_linear_args& a, int64_t m, int64_t n, int count, const float (&v)[8]) {
  TO* y = (TO*)a.y + m * a.ldy + n;
  const TO* r = a.residual ? (const TO*)a.residual + m * a.ldr + n : nullptr;
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < count) y[i] = (TO)(r ? v[i] + (float)r[i] : v[i]);
}

// The sums of a wave's 32 MT x 32 NT part of y become y: 32 rows at a time go through LDS (4096 NT bytes of the wave's own at
// `ex`; 16-byte chunk c of row r at c ^ swizzle(r)), after which a lane holds eight neighbours of a row: bias, activation and
// residual happen there, and rows leave as whole lines, 16 bytes a lane at whatever alignment the rows have.  m0, n0: the
// part's first row and column.
template <int IN, int OUT, int MT, int NT>
__device__ __forceinline__ void linear_out(const crnn_linear_args& a, f32x16 (&acc)[NT][MT], unsigned char* ex, int64_t m0, int64_t n0, int lane) {
  typedef typename TypeOf<OUT>::t TO;
  typedef typename Eight<TO>::t E8;
  constexpr int LPR = 4 * NT, RPI = 64 / LPR, RI = 32 / RPI;   // lanes a row, rows at a time, times
  auto swizzle = [](int r) { return NT == 1 ? (r >> 1) & 7 : r & 15; };
  const int half = lane >> 5, c = lane % LPR;
  const int64_t n = n0 + c * 8, left = a.n - n, mw = m0 + lane / LPR;   // this lane's rows: mw + 32 j + RPI i
  float bias[8], wsc[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    bias[e] = a.bias && e < left ? a.bias[n + e] : 0.f;
    wsc[e] = IN == CRNN_E4M3 && a.w_scale && e < left ? a.w_scale[n + e] : 1.f;
  }
  // the residual of the next 32 rows (fp32: of these, registers are short) is on its way while these are worked on
  constexpr int AHEAD = sizeof(TO) == 2;
  E8 res[1 + AHEAD][RI];
  auto fetch = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RI; i++) {
      const int64_t m = mw + 32 * j + RPI * i;
      if (a.residual && left >= 8 && m < a.m) res[j & AHEAD][i] = *(const E8*)((const TO*)a.residual + m * a.ldr + n);
    }
  };
  if (AHEAD) fetch(0);
#pragma unroll
  for (int j = 0; j < MT; j++) {
    const int r = lane & 31;
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        *(f32x4*)(ex + r * 128 * NT + (((8 * i + 2 * g + half) ^ swizzle(r)) << 4)) = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
    if (j + AHEAD < MT) fetch(j + AHEAD);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    float v[8 * RI];
#pragma unroll
    for (int i = 0; i < RI; i++) {
      const int r = lane / LPR + RPI * i;
      const f32x4 lo = *(const f32x4*)(ex + r * 128 * NT + (((2 * c) ^ swizzle(r)) << 4)), hi = *(const f32x4*)(ex + r * 128 * NT + (((2 * c + 1) ^ swizzle(r)) << 4));
      float sx = 1.f;
      if (IN == CRNN_E4M3 && a.x_scale && mw + 32 * j + RPI * i < a.m) sx = a.x_scale[mw + 32 * j + RPI * i];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float u = e < 4 ? lo[e & 3] : hi[e & 3];
        v[8 * i + e] = IN == CRNN_E4M3 ? u * sx * wsc[e] + bias[e] : u + bias[e];
      }
    }
    activate_all(v, a.act);
#pragma unroll
    for (int i = 0; i < RI; i++) {
      const int64_t m = mw + 32 * j + RPI * i;
      float u[8];
#pragma unroll
      for (int e = 0; e < 8; e++) u[e] = v[8 * i + e];
      if (m >= a.m || left <= 0) continue;
      if (left < 8) {
        put<TO>(a, m, n, (int)left, u);
        continue;
      }
      E8 y;
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = (TO)(a.residual ? u[e] + (float)res[j & AHEAD][i][e] : u[e]);
      *(E8*)((TO*)a.y + m * a.ldy + n) = y;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

// EPC neighbours of a row of k values from k0 on, at the alignment of one value; zeros past the end.  A chunk that the end cuts is
// read from where it ends with the row, and moved down.
template <typename T, int EPC> struct Chunk {
  typedef int raw __attribute__((ext_vector_type(EPC * sizeof(T) / 4)));
  typedef int raw_at __attribute__((ext_vector_type(EPC * sizeof(T) / 4), aligned(sizeof(T))));
  static __device__ __forceinline__ raw whole(const T* p) { return *(const raw_at*)p; }
  typedef typename std::conditional<sizeof(raw) == 16, unsigned __int128, unsigned long long>::type bits;
  typedef typename std::conditional<sizeof(T) == 4, unsigned, typename std::conditional<sizeof(T) == 2, unsigned short, unsigned char>::type>::type word;
  static __device__ __forceinline__ raw cut(const T* row, int64_t k0, int64_t k) {   // (k0 below k)
    const int64_t at = k0 + EPC <= k ? k0 : k - EPC;
    if (k >= EPC) return __builtin_bit_cast(raw, __builtin_bit_cast(bits, whole(row + at)) >> (int)((k0 - at) * sizeof(T) * 8));
    bits b = 0;   // (a row shorter than a chunk)
#pragma unroll 1
    for (int e = (int)k - 1; e >= 0; e--) b = (b << (sizeof(T) * 8)) | ((const word*)row)[e];
    return __builtin_bit_cast(raw, b);
  }
  // `row` exists or the chunk is zeros; `inside`: it ends before k, for every lane
  static __device__ __forceinline__ raw get(const T* row, int64_t k0, int64_t k, bool exists, bool inside) {
    raw v = {};
    if (exists && (inside || k0 < k)) v = inside ? whole(row + k0) : cut(row, k0, k);
    return v;
  }
};

// ---------------------------------------------------------------------------
// linear, any strides, alignments and sizes: tiles as linear_tile_kernel's, but operands go to LDS through registers, because
// loads straight to LDS want whole 16-byte chunks: a step's loads are on their way while the step before is multiplied.  Bound
// by what a CU's cache delivers of rows that cross its lines: bf16 18176 x 2047 x 2048 215 us (2048: 145), 18176 x 511 x 2048
// 68 us (512: 54).  8-bit values become bfloat16 on the way, which holds them exactly: the 8-bit matrix instructions keep
// only 13 bits below the largest of each few products that they add first (measured: 2^8 + 2^-5 in one group is exact,
// 2^8 + 2^-6 is 2^8; between groups and with the accumulator all 24 bits are kept), too few for results in 32 bits.
// ---------------------------------------------------------------------------
template <int IN, int OUT, int MT, int NT, int WN, int KG>
__global__ __launch_bounds__(128 * WN * KG, 2) void linear_loose_kernel(const crnn_linear_args a) {
  typedef typename TypeOf<IN>::t T;
  constexpr bool F32 = IN == CRNN_FP32;
  typedef Slice<F32 ? CRNN_E4M3 : CRNN_BF16> S;   // (fp32: 32 bytes a lane)
  constexpr int RB = 128, NKS = RB / S::KB, KE = F32 ? 32 : 64, EPC = KE / 8;   // bytes of a row of a step in LDS, slices, values, of a chunk
  constexpr int NW = 2 * WN, TH = 64 * NW, BM = 64 * MT, BN = 32 * WN * NT, STAGE = (BM + BN) * RB;
  constexpr int RPC = TH / 8, LX = BM / RPC, CH = (BM + BN) / RPC;   // rows of all threads' chunks, chunks of a thread and step (of x, all)
  constexpr int JOIN = (KG - 1) * NW * MT * NT * 4096;   // bytes of the other groups' sums
  __shared__ __attribute__((aligned(1024))) unsigned char smem_all[KG * 2 * STAGE];
  static_assert(BM % RPC == 0, "a thread's chunk is of x or of w");
  static_assert(sizeof(smem_all) >= JOIN + NW * 4096 * NT, "the epilogue's exchange fits");
  typedef Chunk<T, EPC> C;
  const int tid = threadIdx.x % TH, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x / TH), wm = wave / WN, wn = wave % WN;
  unsigned char* smem = smem_all + kg * 2 * STAGE;
  auto swizzle = [](int r) { return (r >> 1) & 7; };
  const int64_t ntm = (a.m + BM - 1) / BM, ntn = (a.n + BN - 1) / BN, total = ntm * ntn, per = (total + 7) / 8;
  const int64_t nk = (a.k + KE * KG - 1) / (KE * KG);   // steps of a group: KG t + kg
  for (int64_t at = blockIdx.x >> 3; at < per; at += gridDim.x >> 3) {   // (the order of linear_tile_kernel)
    const int64_t t0 = (blockIdx.x & 7) * per + at;
    if (t0 >= total) break;
    const int64_t grp = t0 / (8 * ntn), in = t0 - grp * 8 * ntn, gm = min((int64_t)8, ntm - grp * 8);
    const int64_t m0 = (grp * 8 + in % gm) * BM, n0 = in / gm * BN;
    // chunk i of this thread: tid & 7 of row tid / 8 + RPC i, of x below LX
    const T* px = (const T*)a.x + (m0 + (tid >> 3)) * a.ldx;
    const T* pw = (const T*)a.w + (n0 + (tid >> 3)) * a.ldw;
    const int left_x = (int)min(a.m - m0 - (tid >> 3), (int64_t)BM), left_w = (int)min(a.n - n0 - (tid >> 3), (int64_t)BN);
    typename C::raw st[CH];
    auto fetch = [&](int64_t step) __attribute__((always_inline)) {
      const int64_t ks = (step * KG + kg) * KE, k0 = ks + (tid & 7) * EPC;
      const bool inside = ks + KE <= a.k;   // (the same for all)
      int64_t hx = RPC * a.ldx, hw = RPC * a.ldw;
      asm volatile("" : "+s"(hx), "+s"(hw));   // (else every chunk's address is kept in registers over the loop)
#pragma unroll
      for (int i = 0; i < CH; i++)
        st[i] = i < LX ? C::get(px + i * hx, k0, a.k, RPC * i < left_x, inside) : C::get(pw + (i - LX) * hw, k0, a.k, RPC * (i - LX) < left_w, inside);
    };
    auto put_stage = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < CH; i++) {
        const int r = (tid >> 3) + RPC * i;
        i32x4 v;
        if constexpr (IN == CRNN_E4M3) {
          bf16x8 b;
#pragma unroll
          for (int e = 0; e < 2; e++)
            b[4 * e] = (__bf16)__builtin_amdgcn_cvt_f32_fp8(st[i][e], 0), b[4 * e + 1] = (__bf16)__builtin_amdgcn_cvt_f32_fp8(st[i][e], 1),
            b[4 * e + 2] = (__bf16)__builtin_amdgcn_cvt_f32_fp8(st[i][e], 2), b[4 * e + 3] = (__bf16)__builtin_amdgcn_cvt_f32_fp8(st[i][e], 3);
          v = __builtin_bit_cast(i32x4, b);
        } else {
          v = st[i];
        }
        *(i32x4*)(smem + stage * STAGE + r * RB + (((tid & 7) ^ swizzle(r)) << 4)) = v;
      }
    };
    auto meet = []() __attribute__((always_inline)) {   // LDS writes and reads done, of everybody; loads stay on their way
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    f32x16 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int j = 0; j < MT; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
    fetch(0);
    put_stage(0);
    fetch(1);
    meet();
    const int swz = swizzle(lane & 31);
    const unsigned char* xrow = smem + (wm * 32 * MT + (lane & 31)) * RB;
    const unsigned char* wrow = smem + BM * RB + (wn * 32 * NT + (lane & 31)) * RB;
#pragma unroll 1
    for (int64_t t = 0; t < nk; t++) {
      const int stage = (int)(t & 1);
#pragma unroll
      for (int ks = 0; ks < NKS; ks++) {
        typename S::frag fx[MT], fw[NT];
#pragma unroll
        for (int i = 0; i < NT; i++) fw[i] = S::read(wrow + stage * STAGE + i * 32 * RB, ks, half, swz);
#pragma unroll
        for (int j = 0; j < MT; j++) fx[j] = S::read(xrow + stage * STAGE + j * 32 * RB, ks, half, swz);
        if constexpr (F32) {
          Parts px[MT], pw[NT];
#pragma unroll
          for (int i = 0; i < NT; i++) pw[i] = split3(fw[i]);
#pragma unroll
          for (int j = 0; j < MT; j++) px[j] = split3(fx[j]);
#pragma unroll
          for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[i][j] = mfma3(pw[i], px[j], acc[i][j]);
        } else {
#pragma unroll
          for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[i][j] = S::mfma(fw[i], fx[j], acc[i][j]);
        }
      }
      if (t + 1 < nk) {
        put_stage(stage ^ 1);
        if (t + 2 < nk) fetch(t + 2);
      }
      meet();
    }
    if constexpr (KG > 1) {   // the groups' sums, added in their order
      float* part = (float*)smem_all + (wave * MT * NT * 16) * 64 + lane;
      if (kg > 0) {
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
          for (int j = 0; j < MT; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) part[((kg - 1) * NW * MT * NT * 16 + (i * MT + j) * 16 + r) * 64] = acc[i][j][r];
      }
      meet();
      if (kg == 0) {
#pragma unroll
        for (int k = 0; k < KG - 1; k++)
#pragma unroll
          for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < MT; j++)
#pragma unroll
              for (int r = 0; r < 16; r++) acc[i][j][r] += part[(k * NW * MT * NT * 16 + (i * MT + j) * 16 + r) * 64];
      }
    }
    if (kg == 0) {
      if constexpr (F32) finite_sums<MT, NT>(a, acc, m0 + wm * 32 * MT, n0 + wn * 32 * NT, lane);
      int l = lane;
      asm volatile("" : "+v"(l));   // (else what only the way out needs is kept in registers over the loop)
      linear_out<IN, OUT, MT, NT>(a, acc, smem_all + JOIN + wave * 4096 * NT, m0 + wm * 32 * MT, n0 + wn * 32 * NT, l);
    }
    meet();   // (the next tile's operands)
  }
}

template <int N> __device__ __forceinline__ void wait_loads() {   // all but the last N loads have landed; LDS reads done
  static_assert(N < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

template <int IN, int OUT, int MT, int NT, int WN, int NST, int KG>
__global__ __launch_bounds__(128 * WN * KG, 2) void linear_tile_kernel(const crnn_linear_args a) {
  constexpr bool F32 = IN == CRNN_FP32;
  typedef Slice<F32 ? CRNN_E4M3 : IN> S;   // (fp32: 32 bytes a lane, as 8 bits)
  typedef typename TypeOf<OUT>::t TO;
  constexpr int RB = 128, ES = IN == CRNN_FP32 ? 4 : IN == CRNN_BF16 ? 2 : 1, NKS = RB / S::KB, RPL = 1024 / RB;   // slices of a step, rows of a load
  constexpr int NW = 2 * WN, BM = 64 * MT, BN = 32 * WN * NT, STAGE = (BM + BN) * RB;
  constexpr int LX = BM / (RPL * NW), LT = (BM + BN) / (RPL * NW);   // dma16 instructions of a wave and step: of x, all
  constexpr int JOIN = (KG - 1) * NW * MT * NT * 4096;   // bytes of the other groups' sums
  __shared__ __attribute__((aligned(1024))) unsigned char smem_all[KG * NST * STAGE];
  static_assert(sizeof(smem_all) >= JOIN + NW * 4096 * NT, "the epilogue's exchange fits");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NW, half = lane >> 5;
  const int kg = __builtin_amdgcn_readfirstlane(tid >> 6) / NW;
  unsigned char* smem = smem_all + kg * NST * STAGE;
  const int wm = wave / WN, wn = wave % WN;
  // Tiles in groups of eight rows of tiles, column by column; a run of consecutive tiles per XCD, so that the 32 tiles it works
  // on at a time are 8 x 4 and share their operands in its L2
  const int ntm = (int)((a.m + BM - 1) / BM), ntn = (int)((a.n + BN - 1) / BN), total = ntm * ntn;
  const int per = (total + 7) / 8, t0 = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (t0 >= total || (int)(blockIdx.x >> 3) >= per) return;
  const int grp = t0 / (8 * ntn), in = t0 - grp * 8 * ntn, gm = min(8, ntm - grp * 8);
  const int64_t m0 = (int64_t)(grp * 8 + in % gm) * BM, n0 = (int64_t)(in / gm) * BN;

  const unsigned kbytes = (unsigned)a.k * ES;
  const int nk = (int)((kbytes + RB * KG - 1) / (RB * KG));   // steps of a group: KG t + kg
  const i32x4 rx = resource((const char*)a.x + m0 * a.ldx * ES), rw = resource((const char*)a.w + n0 * a.ldw * ES);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem;
  // lane l of load i of this wave: row r = (wave + NW i) RPL + l / (RB / 16), chunk (l mod RB / 16) ^ swizzle(r), the same for all i
  auto swizzle = [](int r) { return (r >> 1) & 7; };
  const int lr = lane / (RB / 16);
  const unsigned cb = (unsigned)(((lane & (RB / 16 - 1)) ^ swizzle(wave * RPL + lr)) * 16);
  static_assert(NW * RPL % 16 == 0, "a load's rows start at the same place of the swizzle");
  unsigned off[LT];
#pragma unroll
  for (int i = 0; i < LT; i++) {
    const int r = (wave + NW * (i < LX ? i : i - LX)) * RPL + lr;
    if (i < LX) off[i] = m0 + r < a.m ? (unsigned)(r * (int)a.ldx * ES) + cb : OUTSIDE;
    else off[i] = n0 + r < a.n ? (unsigned)(r * (int)a.ldw * ES) + cb : OUTSIDE;
  }
  // load i of LT of `step` into `stage` (x before w); past the end of a row, zeros
  auto load = [&](int step, int stage, int i) __attribute__((always_inline)) {
    const unsigned kb = (unsigned)(step * KG + kg) * RB, to = lds0 + stage * STAGE + (i < LX ? (wave + NW * i) * 1024 : BM * RB + (wave + NW * (i - LX)) * 1024);
    dma16(i < LX ? rx : rw, to, kb + cb < kbytes ? off[i] : OUTSIDE, kb);
  };
  f32x16 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;
  typename S::frag fx[F32 ? 1 : 2][MT], fw[F32 ? 1 : 2][NT];
  const int swz = swizzle(lane & 31);
  const unsigned char* xrow = smem + (wm * 32 * MT + (lane & 31)) * RB;
  const unsigned char* wrow = smem + BM * RB + (wn * 32 * NT + (lane & 31)) * RB;
  auto read = [&](int set, int stage, int ks, int f) __attribute__((always_inline)) {   // operand f: w 0, x 0 .. MT - 1, w 1 ..
    if (f == 0) fw[set][0] = S::read(wrow + stage * STAGE, ks, half, swz);
    else if (f <= MT) fx[set][f - 1] = S::read(xrow + stage * STAGE + (f - 1) * 32 * RB, ks, half, swz);
    else fw[set][f - MT] = S::read(wrow + stage * STAGE + (f - MT) * 32 * RB, ks, half, swz);
  };
#pragma unroll
  for (int t = 0; t < NST; t++)
#pragma unroll
    for (int i = 0; i < (t == NST - 1 ? LT / 2 : LT); i++) load(t, t, i);
  wait_loads<(NST - 1) * LT - (LT - LT / 2)>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int f = 0; f < MT + NT; f++) read(0, 0, 0, f);
  int st = 0;
#pragma unroll 1
  for (int t = 0; t < nk; t++) {
#pragma unroll
    for (int u = 0; u < NKS; u++) {
      const int set = F32 ? 0 : u & 1, last = u == NKS - 1;
      const int nxt = last ? (st + 1 == NST ? 0 : st + 1) : st;
      Parts px[F32 ? MT : 1], pw[F32 ? NT : 1];
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < NT; i++) pw[i] = split3(fw[0][i]);
#pragma unroll
        for (int j = 0; j < MT; j++) px[j] = split3(fx[0][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      // a matrix instruction takes 32 cycles (8 bits: 64), so what goes out between two of them costs nothing
#pragma unroll
      for (int q = 0; q < MT * NT; q++) {
        const int i = q / MT, j = q % MT;
        if constexpr (F32) acc[i][j] = mfma3(pw[i], px[j], acc[i][j]);
        else acc[i][j] = S::mfma(fw[set][i], fx[set][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
        if (last && q == 0) {
          wait_loads<(NST - 2) * LT>();
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        // operands of the next slice
        constexpr int RPQ = (MT + NT + MT * NT - 1) / (MT * NT);
#pragma unroll
        for (int f = q * RPQ; f < (q + 1) * RPQ && f < MT + NT; f++) read(F32 ? 0 : set ^ 1, nxt, last ? 0 : u + 1, f);
        // loads for NST steps on into the stage that the last barrier freed, evenly over the two slices behind it: a burst of
        // them holds the wave up (each takes the address unit, which four waves share, 16 cycles)
        constexpr int SLOTS = 2 * MT * NT;
        const int p = last ? q : MT * NT + q;
        if (last || u == 0) {
#pragma unroll
          for (int l = p * LT / SLOTS; l < (p + 1) * LT / SLOTS; l++) load((last ? t : t - 1) + NST, last ? st : st == 0 ? NST - 1 : st - 1, l);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      st = nxt;
    }
  }
  wait_loads<0>();   // (zeros for steps past the end may still be on their way)
  // Epilogue: the sums of 32 rows at a time go through LDS (each wave has its own part), after which a lane holds eight
  // neighbours of a row: bias, activation and residual happen there, and rows leave as whole lines.
  __syncthreads();   // (nobody reads the stages any more)
  if constexpr (KG > 1) {   // the groups' sums, added in their order
    float* part = (float*)smem_all + (wave * MT * NT * 16) * 64 + lane;
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
          for (int r = 0; r < 16; r++) part[((kg - 1) * NW * MT * NT * 16 + (i * MT + j) * 16 + r) * 64] = acc[i][j][r];
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int k = 0; k < KG - 1; k++)
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
          for (int r = 0; r < 16; r++) acc[i][j][r] += part[(k * NW * MT * NT * 16 + (i * MT + j) * 16 + r) * 64];
  }
  if constexpr (F32) {
    finite_sums<MT, NT>(a, acc, m0 + wm * 32 * MT, n0 + wn * 32 * NT, lane);
  }
  linear_out<IN, OUT, MT, NT>(a, acc, smem_all + JOIN + wave * 4096 * NT, m0 + wm * 32 * MT, n0 + wn * 32 * NT, lane);
}

// ---------------------------------------------------------------------------
// linear, five to sixteen rows of whole 16-byte chunks: 32 columns of y per workgroup, whose KW waves take 128 bytes of k of every
// row of w in turn and add up through LDS in a fixed order.  No LDS on the way in, every lane loads its operands as they lie
// (the products may be added in any order, so a lane's half of a block is 64 neighbouring bytes), the next block's while this
// one is multiplied.  x is the first operand: lanes hold neighbouring columns.  Bound by reading w, and where n gives few
// workgroups by what one CU reads: bf16 16 x 512 x 5530 4.6 us, 16 x 8192 x 8192 40 us (3.4 TB/s), 12 x 8192 x 512 25 us.
// ---------------------------------------------------------------------------
template <int IN, int OUT, int KW>
__global__ __launch_bounds__(64 * KW, 2) void linear_rows_kernel(const crnn_linear_args a) {
  typedef typename TypeOf<OUT>::t TO;
  typedef Slice<IN> S;
  constexpr int ES = IN == CRNN_FP32 ? 4 : IN == CRNN_BF16 ? 2 : 1;
  __shared__ float part[KW][16][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  const unsigned kbytes = (unsigned)a.k * ES;
  const int nb = (int)((kbytes + 127) / 128);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)a.x, 0, 0x7FFFFFFF, 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.w + n0 * a.ldw * ES), 0, 0x7FFFFFFF, 0x00020000);
  const unsigned ow = n0 + (lane & 31) < a.n ? (unsigned)((lane & 31) * (int)a.ldw * ES) + half * 64u : OUTSIDE;
  const unsigned ox = (lane & 31) < a.m ? (unsigned)((lane & 31) * (int)a.ldx * ES) + half * 64u : OUTSIDE;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; r++) acc[r] = 0.f;
  i32x4 w[2][4], x[2][4];
  auto load = [&](int set, int blk) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const unsigned kb = (unsigned)blk * 128 + c * 16;
      const bool in = kb + half * 64u < kbytes;   // (a block past the end: zeros)
      w[set][c] = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? ow + kb : OUTSIDE, 0, 0);
      x[set][c] = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? ox + kb : OUTSIDE, 0, 0);
    }
  };
  auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 4; c += IN == CRNN_E4M3 ? 2 : 1) {
      if constexpr (IN == CRNN_E4M3) {
        const i32x4 x0 = x[set][c], x1 = x[set][c + 1], w0 = w[set][c], w1 = w[set][c + 1];
        acc = S::mfma(i32x8{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]}, i32x8{w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]}, acc);
      } else {
        acc = S::mfma(__builtin_bit_cast(typename S::frag, x[set][c]), __builtin_bit_cast(typename S::frag, w[set][c]), acc);
      }
    }
  };
  load(0, wave);
  for (int blk = wave; blk < nb; blk += 2 * KW) {
    load(1, blk + KW);
    multiply(0);
    load(0, blk + 2 * KW);
    multiply(1);
  }
#pragma unroll
  for (int r = 0; r < 16; r++) part[wave][r][lane] = acc[r];
  __syncthreads();
  const int64_t n = n0 + (lane & 31);
  if (n >= a.n) return;
  const float bias = a.bias ? a.bias[n] : 0.f, wsc = IN == CRNN_E4M3 && a.w_scale ? a.w_scale[n] : 1.f;
  for (int i = wave; i < 16; i += KW) {
    const int m = acc_row(i, lane);
    if (m >= a.m) continue;
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < KW; s++) v += part[s][i][lane];
    if (IN == CRNN_E4M3) v = v * (a.x_scale ? a.x_scale[m] : 1.f) * wsc;
    v = activate(v + bias, a.act);
    if (a.residual) v += (float)((const TO*)a.residual)[m * a.ldr + n];
    ((TO*)a.y)[m * a.ldy + n] = (TO)v;
  }
}

// One to four rows: a wave per NC columns of y, its lanes side by side along k, 16 bytes of every column and row each; fp32 FMAs
// (also for 8-bit values with results in 32 bits, since nothing is lost).  Bound by the way of the first bytes, then by reading
// w: four loads of each column are on their way at a time.  bf16 1 x 512 x 512 3.2 us, 1 x 8192 x 8192
// 27 us (4.9 TB/s); rows at odd places (CHUNKS false): 1 x 511 x 512 3.8 us, 3 x 8191 x 8192 39 us.
template <int IN, int OUT, int M, int NC, bool CHUNKS>
__global__ __launch_bounds__(256, 2) void linear_vector_kernel(const crnn_linear_args a) {
  typedef typename TypeOf<IN>::t T;
  typedef typename TypeOf<OUT>::t TO;
  constexpr int ES = sizeof(T), EPC = 16 / ES, U = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * NC;
  if (n0 >= a.n) return;
  const unsigned kbytes = (unsigned)a.k * ES;
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)a.x, 0, 0x7FFFFFFF, 0x00020000);
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.w + n0 * a.ldw * ES), 0, 0x7FFFFFFF, 0x00020000);
  auto widen = [](i32x4 u, float (&v)[EPC]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (ES == 4) v[i] = __uint_as_float((unsigned)u[i]);
      else if constexpr (ES == 2) v[2 * i] = __uint_as_float((unsigned)u[i] << 16), v[2 * i + 1] = __uint_as_float((unsigned)u[i] & 0xFFFF0000u);
      else v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(u[i], 0), v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(u[i], 1), v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(u[i], 2), v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(u[i], 3);
    }
  };
  float acc[M][NC];
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int c = 0; c < NC; c++) acc[m][c] = 0.f;
  for (unsigned k0 = lane * 16; k0 < kbytes; k0 += U * 1024) {
    i32x4 w[U][NC], x[U][M];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const unsigned kb = k0 + u * 1024;
      const bool in = kb < kbytes;
      if constexpr (CHUNKS) {
#pragma unroll
        for (int c = 0; c < NC; c++) w[u][c] = __builtin_amdgcn_raw_buffer_load_b128(rw, in && n0 + c < a.n ? (unsigned)(c * (int)a.ldw * ES) + kb : OUTSIDE, 0, 0);
#pragma unroll
        for (int m = 0; m < M; m++) x[u][m] = __builtin_amdgcn_raw_buffer_load_b128(rx, in && m < a.m ? (unsigned)(m * (int)a.ldx * ES) + kb : OUTSIDE, 0, 0);
      } else {
#pragma unroll
        for (int c = 0; c < NC; c++) w[u][c] = Chunk<T, EPC>::get((const T*)a.w + (n0 + c) * a.ldw, kb / ES, a.k, n0 + c < a.n, kb - lane * 16 + 1024 <= kbytes);
#pragma unroll
        for (int m = 0; m < M; m++) x[u][m] = Chunk<T, EPC>::get((const T*)a.x + m * a.ldx, kb / ES, a.k, m < a.m, kb - lane * 16 + 1024 <= kbytes);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float wv[NC][EPC], xv[M][EPC];
#pragma unroll
      for (int c = 0; c < NC; c++) widen(w[u][c], wv[c]);
#pragma unroll
      for (int m = 0; m < M; m++) widen(x[u][m], xv[m]);
#pragma unroll
      for (int m = 0; m < M; m++)
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
          for (int i = 0; i < EPC; i++) acc[m][c] = fmaf(xv[m][i], wv[c][i], acc[m][c]);
    }
  }
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int c = 0; c < NC; c++) acc[m][c] = wave_sum(acc[m][c]);
  // lane m NC + c has the value of row m, column c
  float v = 0.f;
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int c = 0; c < NC; c++)
      if (lane == m * NC + c) v = acc[m][c];
  const int m = lane / NC;
  const int64_t n = n0 + lane % NC;
  if (m >= M || m >= a.m || n >= a.n) return;
  if (IN == CRNN_E4M3) v = v * (a.x_scale ? a.x_scale[m] : 1.f) * (a.w_scale ? a.w_scale[n] : 1.f);
  v = activate(v + (a.bias ? a.bias[n] : 0.f), a.act);
  if (a.residual) v += (float)((const TO*)a.residual)[m * a.ldr + n];
  ((TO*)a.y)[m * a.ldy + n] = (TO)v;
}

// Rows of whole 16-byte chunks, and offsets within a tile below 2^31 bytes.
static bool linear_chunks(const crnn_linear_args& a) {
  const int64_t es = a.in_type == CRNN_FP32 ? 4 : a.in_type == CRNN_BF16 ? 2 : 1, c = 16 / es;
  return a.k % c == 0 && a.ldx % c == 0 && a.ldw % c == 0 && (((uintptr_t)a.x | (uintptr_t)a.w) & 15) == 0 &&
         (256 * (a.ldx > a.ldw ? a.ldx : a.ldw) + a.k) * es < 0x7FFFF000;
}

template <int IN, int OUT, int MT, int NT, int WN, int NST, int KG = 1>
static void linear_tile(const crnn_linear_args& a, hipStream_t s) {
  const int64_t total = ((a.m + 64 * MT - 1) / (64 * MT)) * ((a.n + 32 * WN * NT - 1) / (32 * WN * NT));
  hipLaunchKernelGGL((linear_tile_kernel<IN, OUT, MT, NT, WN, NST, KG>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(128 * WN * KG), 0, s, a);
}
static double tile_rounds(const crnn_linear_args& a, int bm, int bn, int at_once) {
  return (double)(((a.m + bm - 1) / bm * ((a.n + bn - 1) / bn) + at_once - 1) / at_once);
}
template <int IN, int OUT>
static bool linear_tiles(const crnn_linear_args& a, hipStream_t s) {
  if ((a.m + 63) / 64 * ((a.n + 63) / 64) >= 1 << 22) return false;   // (a launch has fewer than 2^32 threads)
  // Tiles come in rounds of what the 256 CUs hold; a round takes its tile's size (256 x 256: 4), 128 x 128 ones two a CU with
  // less use of what is loaded.  18176 x 512 x 2048: 256 rows 54 us, 192 rows 50, 128 x 128 59; 16384 x 4096 x 4096: 455, 488, 556.
  const double c4 = 4.0 * tile_rounds(a, 256, 256, 256), c3 = 3.0 * tile_rounds(a, 192, 256, 256), c2 = 2.4 * tile_rounds(a, 128, 128, 512);
  const int64_t small = ((a.m + 127) / 128) * ((a.n + 127) / 128), tiny = ((a.m + 63) / 64) * ((a.n + 31) / 32);
  if constexpr (IN != CRNN_FP32) {
    if (c4 <= c3 && c4 <= c2) return linear_tile<IN, OUT, 4, 2, 4, 2>(a, s), true;
    if (c3 <= c2) return linear_tile<IN, OUT, 3, 2, 4, 2>(a, s), true;
  }
  if (small >= 256) linear_tile<IN, OUT, 2, 2, 2, 2>(a, s);
  // (fp32: a larger tile halves the work of splitting; two groups of waves over k where it leaves CUs with one workgroup.  It pays from
  // where 64 x 64 ones come to more than two a CU, and where k is long enough to share: 8000 x 512 x 512, 252 tiles, 36 us, in 64 x 64
  // ones 46; 4544 x 512 x 512, 144, 28 and 30; 4096 x 512 x 512, 128, 28 and 24; 4544 x 64 x 512 11.1 and 8.9)
  else if (IN == CRNN_FP32 && small >= (a.k < 512 ? 192 : 129)) linear_tile<IN, OUT, 2, 2, 2, 2, 2>(a, s);
  // (few small tiles: four groups of waves share k.  64 x 2048 x 2048 9.2 us, without 12.5; 300 x 512 x 5530 20 us, without 11)
  else if (tiny <= 256) linear_tile<IN, OUT, 1, 1, 1, 3, 4>(a, s);
  else linear_tile<IN, OUT, 1, 1, 2, 3>(a, s);
  return true;
}

template <int IN, int OUT>
static void linear_rows(const crnn_linear_args& a, hipStream_t s) {
  constexpr int ES = IN == CRNN_FP32 ? 4 : IN == CRNN_BF16 ? 2 : 1;
  const dim3 g((unsigned)((a.n + 31) / 32));
  // waves over k: 8 x 512 x 2048 4.1 us with four, 4.8 with sixteen; 8 x 8192 x 2048 26 and 24
  if (a.k * ES <= 1024) hipLaunchKernelGGL((linear_rows_kernel<IN, OUT, 4>), g, dim3(256), 0, s, a);
  else if (a.k * ES <= 4096) hipLaunchKernelGGL((linear_rows_kernel<IN, OUT, 8>), g, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((linear_rows_kernel<IN, OUT, 16>), g, dim3(1024), 0, s, a);
}
template <int IN, int OUT, int M, bool CHUNKS>
static void linear_vector(const crnn_linear_args& a, hipStream_t s) {
  // A wave takes one column; of many columns for several rows it takes four, which read the rows of x once: 4 x 8192 x 8192
  // 33 us, by one column 41; 4 x 512 x 5530 7.0 and 6.8; 1 x 8192 x 8192 30 and 27.
  if constexpr (M > 1) {
    if (a.n >= 8192) {
      hipLaunchKernelGGL((linear_vector_kernel<IN, OUT, M, 4, CHUNKS>), dim3((unsigned)((a.n + 15) / 16)), dim3(256), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((linear_vector_kernel<IN, OUT, M, 1, CHUNKS>), dim3((unsigned)((a.n + 3) / 4)), dim3(256), 0, s, a);
}
template <int IN, int OUT, bool CHUNKS>
static void linear_vector(const crnn_linear_args& a, hipStream_t s) {
  if (a.m == 1) linear_vector<IN, OUT, 1, CHUNKS>(a, s);
  else if (a.m == 2) linear_vector<IN, OUT, 2, CHUNKS>(a, s);
  else linear_vector<IN, OUT, 4, CHUNKS>(a, s);
}
template <int IN, int OUT, int MT, int NT, int WN, int KG>
static void linear_loose(const crnn_linear_args& a, hipStream_t s) {
  const int64_t total = ((a.m + 64 * MT - 1) / (64 * MT)) * ((a.n + 32 * WN * NT - 1) / (32 * WN * NT));
  hipLaunchKernelGGL((linear_loose_kernel<IN, OUT, MT, NT, WN, KG>), dim3((unsigned)(total < (1 << 20) ? (total + 7) / 8 * 8 : 1 << 20)), dim3(128 * WN * KG), 0, s, a);
}

template <int IN, int OUT>
static void linear_of(const crnn_linear_args& a, hipStream_t s) {
  const bool chunks = linear_chunks(a);
  // (a launch has fewer than 2^32 threads, of which one row takes 64 a column; places in a row are 32-bit)
  const bool few = a.n <= (1 << 26) - 4 && a.k < 1 << 28;
  if (a.m <= 4 && few) return chunks ? linear_vector<IN, OUT, true>(a, s) : linear_vector<IN, OUT, false>(a, s);
  if constexpr (IN != CRNN_E4M3 || OUT == CRNN_BF16) {
    if (chunks && a.m <= 16 && few) return linear_rows<IN, OUT>(a, s);
    if (chunks && linear_tiles<IN, OUT>(a, s)) return;
  }
  const int64_t small = ((a.m + 127) / 128) * ((a.n + 127) / 128), tiny = ((a.m + 63) / 64) * ((a.n + 63) / 64);
  // (as in linear_tiles; 9000 x 1023 x 1023: 192 x 256 in one round 43 us, 128 x 128 in two 54)
  if constexpr (IN != CRNN_FP32) {
    if (3.0 * tile_rounds(a, 192, 256, 256) <= 1.9 * tile_rounds(a, 128, 128, 512)) return linear_loose<IN, OUT, 3, 2, 4, 1>(a, s);
  }
  // (few small tiles: two groups of waves share k, as in linear_tiles)
  if (small >= 256) linear_loose<IN, OUT, 2, 2, 2, 1>(a, s);
  else if (tiny <= 256) linear_loose<IN, OUT, 1, 1, 2, 2>(a, s);
  else linear_loose<IN, OUT, 1, 1, 2, 1>(a, s);
}

void launch_linear(const crnn_linear_args& a, hipStream_t s) {
  if (a.in_type == CRNN_FP32) a.out_type == CRNN_FP32 ? linear_of<CRNN_FP32, CRNN_FP32>(a, s) : linear_of<CRNN_FP32, CRNN_BF16>(a, s);
  else if (a.in_type == CRNN_BF16) a.out_type == CRNN_FP32 ? linear_of<CRNN_BF16, CRNN_FP32>(a, s) : linear_of<CRNN_BF16, CRNN_BF16>(a, s);
  else a.out_type == CRNN_FP32 ? linear_of<CRNN_E4M3, CRNN_FP32>(a, s) : linear_of<CRNN_E4M3, CRNN_BF16>(a, s);
}

// ---------------------------------------------------------------------------
// rms_norm.  y = t r g with r = (sum t^2 / n + eps)^-1/2.  Where the sum of squares leaves the range in which a 32-bit one is
// exact (rows around 1e-20 or above 1e18) it is taken again in 64 bits, and r is applied as a power of two near 1 / |t| and
// the rest, so that no product on the way leaves the normal numbers.
// ---------------------------------------------------------------------------
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
  return v;
}
__device__ __forceinline__ bool squares_ok(float ss) { return ss > 0x1p-90f && ss < 0x1p126f; }
// r = r1 r2 from a sum of squares in 64 bits
__device__ __forceinline__ void row_factors(double ss, double n, float eps, float* r1, float* r2) {
  const double ms = ss / n, r = 1.0 / sqrt(ms + (double)eps);
  int e = 0;
  if (ms > 0.0 && ms < INFINITY) e = -(ilogb(ms) >> 1);
  e = e > 126 ? 126 : e < -126 ? -126 : e;
  *r1 = ldexpf(1.f, e);
  *r2 = (float)ldexp(r, -e);
}
// |y| as an unsigned integer: the order of the bits is the order of the values with NaN above infinity, so a NaN is kept
__device__ __forceinline__ unsigned abs_bits(float y) { return __float_as_uint(y) & 0x7FFFFFFFu; }
__device__ __forceinline__ float row_scale(unsigned top) {
  const float t = __uint_as_float(top), low = 448.f * 0x1p-126f;   // (a row of zeros: a scale that divides)
  return (t < low ? low : t) / 448.f;
}
// y / c, from 1 / c: the product, and what it leaves of y divided likewise, which a fused multiply-add gives exactly.  (The product
// alone lies up to 1.5 steps off and takes quotients in the middle between two e4m3 values to the wrong one; v_div_* for each value
// would be ten instructions for these three.)  An infinite c gives 0, or NaN for an infinite y, as the division does.
struct RowQuotient {
  float c, ic;
  __device__ __forceinline__ explicit RowQuotient(float scale) : c(scale < INFINITY ? scale : 0.f), ic(1.f / scale) {}
  __device__ __forceinline__ float of(float y) const {
    const float q = y * ic;
    return copysignf(fmaf(fmaf(-q, c, y), ic, q), y);   // (-0 stays)
  }
};

// Sum over the 64 or 256 threads of a row (256: through LDS, between barriers).
template <int TPR, typename V> __device__ __forceinline__ V row_sum(V v, V* part) {
  v = wave_sum(v);
  if (TPR == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}
template <int TPR> __device__ __forceinline__ unsigned row_max(unsigned v, unsigned* part) {
  v = wave_max(v);
  if (TPR == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return max(max(part[0], part[1]), max(part[2], part[3]));
}

// Rows longer than 8192: one workgroup per row, the row read again for each of the passes (sum of squares, with 8-bit outputs
// the largest |y|, the outputs); bound by those readings, element by element: 18176 x 2049 took 180 us here, below 97.  The
// outputs are written in the last pass by the thread that reads the same element, so they may be the inputs themselves.  Squares are
// added in 64 bits: in 32 a thread's n / 256 of them lose 2.5e-5 of the sum at n = 2^20 and 6.5e-4 at 2^24.
template <int IN, int OUT>
__global__ __launch_bounds__(256) void rms_norm_any_kernel(const crnn_rms_norm_args a) {
  typedef typename TypeOf<IN>::t T;
  typedef typename TypeOf<OUT>::t TO;
  __shared__ double partd[4];
  __shared__ unsigned partu[4];
  const int tid = threadIdx.x;
  for (int64_t m = blockIdx.x; m < a.m; m += gridDim.x) {
    const T* x = (const T*)a.x + m * a.ldx;
    const T* r = a.residual ? (const T*)a.residual + m * a.ldr : nullptr;
    auto value = [&](int64_t i) { return r ? (float)x[i] + (float)r[i] : (float)x[i]; };
    double sd = 0.0;
    for (int64_t i = tid; i < a.n; i += 256) {
      const double t = value(i);
      sd += t * t;
    }
    sd = row_sum<256>(sd, partd);
    const float ss = (float)sd;
    float r1 = 1.f, r2;
    if (squares_ok(ss)) r2 = 1.f / sqrtf(ss / (float)a.n + a.eps);
    else row_factors(sd, (double)a.n, a.eps, &r1, &r2);
    float c = 1.f;
    if (OUT == CRNN_E4M3) {
      unsigned top = 0;
      for (int64_t i = tid; i < a.n; i += 256) top = max(top, abs_bits(value(i) * r1 * r2 * a.gain[i]));
      c = row_scale(row_max<256>(top, partu));
    }
    const RowQuotient by(c);
    for (int64_t i = tid; i < a.n; i += 256) {
      const float t = value(i), y = t * r1 * r2 * a.gain[i];
      if (a.sum) ((T*)a.sum)[m * a.lds + i] = (T)t;
      store1((TO*)a.y + m * a.ldy + i, OUT == CRNN_E4M3 ? by.of(y) : y);
    }
    if (OUT == CRNN_E4M3 && tid == 0) a.y_scale[m] = c;
    __syncthreads();   // (partd, partu)
  }
}

// Rows that fit the registers of one wave (TPR 64: four rows a workgroup) or one workgroup (TPR 256): x and the residual are
// read once, everything else happens in registers.  A thread holds C groups of eight values, which it loads and stores whole at
// whatever alignment rows have, one by one where the row ends; the gain stays in registers over the rows that a workgroup takes.
// Bound by HBM: 18176 x 2048 bf16 with residual and sum to 8 bits 56 to 61 us (4.5 TB/s and more), 18176 x 8192 to bf16 219 us
// (5.4 TB/s); 18176 x 2047 to 8 bits 75 us, rows crossing cache lines.
template <int IN, int OUT, int TPR, int C>
__global__ __launch_bounds__(256) void rms_norm_kernel(const crnn_rms_norm_args a) {
  typedef typename TypeOf<IN>::t T;
  typedef typename TypeOf<OUT>::t TO;
  __shared__ float part[4];
  __shared__ double partd[4];
  __shared__ unsigned partu[4];
  constexpr int RPB = 256 / TPR;
  const int at = threadIdx.x & (TPR - 1), n = (int)a.n;
  float g[C][8], t[C][8];
#pragma unroll
  for (int c = 0; c < C; c++) {
    const int i = (c * TPR + at) * 8;
#pragma unroll
    for (int e = 0; e < 8; e++) g[c][e] = 0.f;
    part8(a.gain, i, n, g[c]);
  }
  // (TPR 256: every thread of the workgroup has the same row, so the barriers in row_sum are met by all)
  for (int64_t m = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; m < a.m; m += (int64_t)gridDim.x * RPB) {
    const T* x = (const T*)a.x + m * a.ldx;
    const T* res = (const T*)a.residual + m * a.ldr;
    float ss = 0.f, r1 = 1.f, r2;
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int i = (c * TPR + at) * 8;
#pragma unroll
      for (int e = 0; e < 8; e++) t[c][e] = 0.f;
      part8(x, i, n, t[c]);
      if (a.residual) {
        float r[8] = {};
        part8(res, i, n, r);
#pragma unroll
        for (int e = 0; e < 8; e++) t[c][e] += r[e];
      }
    }
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) ss += t[c][e] * t[c][e];
    ss = row_sum<TPR>(ss, part);
    if (squares_ok(ss)) {
      r2 = 1.f / sqrtf(ss / (float)n + a.eps);
    } else {
      double sd = 0.0;
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) sd += (double)t[c][e] * (double)t[c][e];
      row_factors(row_sum<TPR>(sd, partd), (double)n, a.eps, &r1, &r2);
    }
    if (a.sum) {
#pragma unroll
      for (int c = 0; c < C; c++) put8((T*)a.sum + m * a.lds, (c * TPR + at) * 8, n, t[c]);
    }
    unsigned top = 0;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        t[c][e] = t[c][e] * r1 * r2 * g[c][e];
        // (past the end of the row t is 0, but 0 times an infinite factor would be NaN)
        if (OUT == CRNN_E4M3) top = max(top, (c * TPR + at) * 8 + e < n ? abs_bits(t[c][e]) : 0u);
      }
    float sc = 1.f;
    if (OUT == CRNN_E4M3) {
      sc = row_scale(row_max<TPR>(top, partu));
      if (at == 0) a.y_scale[m] = sc;
    }
    const RowQuotient by(sc);
#pragma unroll
    for (int c = 0; c < C; c++) {
      if (OUT == CRNN_E4M3) {
#pragma unroll
        for (int e = 0; e < 8; e++) t[c][e] = by.of(t[c][e]);
      }
      put8((TO*)a.y + m * a.ldy, (c * TPR + at) * 8, n, t[c]);
    }
  }
}

template <int IN, int OUT>
static void rms_norm_of(const crnn_rms_norm_args& a, hipStream_t s) {
  // at most 8 workgroups a CU at a time: more rows are taken in turn, with the gain at hand
  auto grid = [&](int rows) { return dim3((unsigned)((a.m + rows - 1) / rows < 2048 ? (a.m + rows - 1) / rows : 2048)); };
  if (a.n > 8192) hipLaunchKernelGGL((rms_norm_any_kernel<IN, OUT>), grid_for(a.m), dim3(256), 0, s, a);
  else if (a.n <= 512) hipLaunchKernelGGL((rms_norm_kernel<IN, OUT, 64, 1>), grid(4), dim3(256), 0, s, a);
  else if (a.n <= 1024) hipLaunchKernelGGL((rms_norm_kernel<IN, OUT, 64, 2>), grid(4), dim3(256), 0, s, a);
  else if (a.n <= 2048) hipLaunchKernelGGL((rms_norm_kernel<IN, OUT, 64, 4>), grid(4), dim3(256), 0, s, a);
  else if (a.n <= 4096) hipLaunchKernelGGL((rms_norm_kernel<IN, OUT, 256, 2>), grid(1), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rms_norm_kernel<IN, OUT, 256, 4>), grid(1), dim3(256), 0, s, a);
}

void launch_rms_norm(const crnn_rms_norm_args& a, hipStream_t s) {
  if (a.in_type == CRNN_FP32) {
    if (a.out_type == CRNN_FP32) rms_norm_of<CRNN_FP32, CRNN_FP32>(a, s);
    else rms_norm_of<CRNN_FP32, CRNN_E4M3>(a, s);
  } else {
    if (a.out_type == CRNN_BF16) rms_norm_of<CRNN_BF16, CRNN_BF16>(a, s);
    else rms_norm_of<CRNN_BF16, CRNN_E4M3>(a, s);
  }
}

// ---------------------------------------------------------------------------
// cross_attention.  A "row" is a pair (t, query head) that reads one key head: row r of (b, g) is t = r / G and head
// g G + r % G, G = heads / kv_heads, so the heads that share keys read them once.  Running maximum M and sum L of a row over
// tiles of keys: M' = max(M, max s), L' = L e^(M - M') + sum e^(s - M'), O' likewise; keys that are left out have s = -inf and
// v = 0.  While M is -inf nothing has been added (M' - M' is taken as 0).
//
// Any strides, sizes and types: 16 rows per workgroup, tiles of 32 keys in LDS as fp32, scores and sums by fp32 FMAs.  For rows
// that are not whole 16-byte chunks.  Bound by its LDS reads, two a FMA: bf16 64 lines x 48 queries over 71 states, head_dim 63
// 73 us, 64 by attention_tile_kernel 9.3.
// ---------------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(256, 2) void attention_any_kernel(const crnn_cross_attention_args a) {
  typedef typename TypeOf<TYPE>::t T;
  constexpr int R = 16, KT = 32, LD = 129;
  __shared__ float qs[R * LD], ks[KT * LD], vs[KT * LD], ps[R * (KT + 1)];
  __shared__ int ok[KT];
  const int tid = threadIdx.x, G = a.heads / a.kv_heads, D = a.head_dim;
  const int64_t rows = a.q_len * G, nrb = (rows + R - 1) / R, blocks = a.batch * a.kv_heads * nrb;
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t rb = blk % nrb, bg = blk / nrb, b = bg / a.kv_heads, g = bg % a.kv_heads;
    const int64_t len = a.lengths ? max((int64_t)0, min((int64_t)a.lengths[b], a.kv_len)) : a.kv_len;
    const T* q = (const T*)a.q + b * a.q_stride[0];
    const T* k = (const T*)a.k + b * a.k_stride[0] + g * a.k_stride[2];
    const T* v = (const T*)a.v + b * a.v_stride[0] + g * a.v_stride[2];
    __syncthreads();
    for (int i = tid; i < R * D; i += 256) {
      const int64_t r = rb * R + i / D;
      qs[i / D * LD + i % D] = r < rows ? (float)q[r / G * a.q_stride[1] + (g * G + r % G) * a.q_stride[2] + i % D] : 0.f;
    }
    const int row = tid >> 4, c = tid & 15;
    const float sc = a.scale * 1.4426950408889634f;   // exp(x) = 2^(x log2 e)
    float M = -INFINITY, L = 0.f, o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = 0.f;
    for (int64_t j0 = 0; j0 < len; j0 += KT) {
      __syncthreads();
      if (tid < KT) ok[tid] = j0 + tid < len && (!a.mask || a.mask[b * a.mask_stride + j0 + tid]);
      __syncthreads();
      for (int i = tid; i < KT * D; i += 256) {
        const int j = i / D, d = i % D;
        ks[j * LD + d] = ok[j] ? (float)k[(j0 + j) * a.k_stride[1] + d] : 0.f;
        vs[j * LD + d] = ok[j] ? (float)v[(j0 + j) * a.v_stride[1] + d] : 0.f;
      }
      __syncthreads();
      float s0 = 0.f, s1 = 0.f;
      for (int d = 0; d < D; d++) {
        s0 += qs[row * LD + d] * ks[c * LD + d];
        s1 += qs[row * LD + d] * ks[(c + 16) * LD + d];
      }
      s0 = ok[c] ? s0 * sc : -INFINITY;
      s1 = ok[c + 16] ? s1 * sc : -INFINITY;
      // fmaxf drops a NaN: it still reaches L and O through its own exponential below
      float mt = fmaxf(s0, s1);
#pragma unroll
      for (int f = 1; f < 16; f <<= 1) mt = fmaxf(mt, __shfl_xor(mt, f));
      const float Mn = fmaxf(M, mt), Ms = Mn == -INFINITY ? 0.f : Mn;
      const float p0 = exp2f(s0 - Ms), p1 = exp2f(s1 - Ms), al = exp2f(M - Ms);
      float pl = p0 + p1;
#pragma unroll
      for (int f = 1; f < 16; f <<= 1) pl += __shfl_xor(pl, f);
      L = L * al + pl;
      M = Mn;
      ps[row * (KT + 1) + c] = p0;          // (a row's sixteen threads are lanes of one wave; its p are read by them only)
      ps[row * (KT + 1) + c + 16] = p1;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int d = c + 16 * i;
        float t = o[i] * al;
        if (d < D)
#pragma unroll 4
          for (int j = 0; j < KT; j++) t += ps[row * (KT + 1) + j] * vs[j * LD + d];
        o[i] = t;
      }
    }
    const int64_t r = rb * R + row;
    if (r >= rows) continue;
    T* out = (T*)a.out + b * a.out_stride[0] + r / G * a.out_stride[1] + (g * G + r % G) * a.out_stride[2];
    const float il = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int d = c + 16 * i;
      if (d < D) out[d] = (T)(o[i] * il);
    }
  }
}

// The blocks of one key head (its row blocks and splits, `each` of them) belong on one XCD, whose L2 then holds their keys.  Key
// heads go round the XCDs one by one, because neighbours share their length; with too few of them to fill all XCDs evenly
// runs of blocks are dealt instead.  -1: no block.
__host__ __device__ __forceinline__ bool attention_deal(int64_t key_heads) { return key_heads >= 64 || key_heads % 8 == 0; }
static int64_t attention_grid(int64_t key_heads, int64_t each) { return attention_deal(key_heads) ? (key_heads + 7) / 8 * 8 * each : (key_heads * each + 7) / 8 * 8; }
__device__ __forceinline__ int64_t attention_block(unsigned id, int64_t key_heads, int64_t each) {
  const int64_t xcd = id & 7, at = id >> 3;
  if (attention_deal(key_heads)) {
    const int64_t head = at / each * 8 + xcd;
    return head < key_heads ? head * each + at % each : -1;
  }
  const int64_t total = key_heads * each, per = (total + 7) / 8, blk = xcd * per + at;
  return blk < total && at < per ? blk : -1;
}

// Where split s of nsplit leaves row r of all rows (batch, key head, row): D unnormalised values, then (M, L) behind all of them.
constexpr int MAX_SPLIT = 64, JOIN_ROWS = 1024;
struct SplitRow {
  float *o, *ml;
  __device__ __forceinline__ SplitRow(const crnn_cross_attention_args& a, int nsplit, int s, int64_t r) {
    const int64_t all = a.batch * a.heads * a.q_len;
    o = (float*)a.workspace + (s * all + r) * a.head_dim;
    ml = (float*)a.workspace + nsplit * all * a.head_dim + (s * all + r) * 2;
  }
};

// head_dim and strides in whole 16-byte chunks.  RW waves side by side over 32 rows each, KW times as many over different tiles
// of KT keys; head_dim padded to DP.  Both products run transposed, S^T = K Q^T and O^T = V^T P^T
// (v_mfma_f32_32x32x16_bf16): a lane then holds one query row in both results, so maximum, sum and rescaling are per lane, and
// the exponentials are the second product's operand as they stand, because its sum may run over the keys in any order: register
// r of S^T is key (r & 3) + 8 (r >> 2) + 4 (lane >> 5), and ds_read_tr16_b64 takes V's columns for four such keys at a time.
// K and V tiles go straight to LDS, two stages; 16-byte chunk c of row j sits at chunk c ^ swizzle(j), which spreads what is
// read at once -- 16 rows of K, 64 bytes of four rows of V -- over the 256 bytes that LDS serves in a cycle.  fp32 runs the same
// way on v_mfma_f32_32x32x2_f32: a 16-byte chunk feeds four of them, register r of S^T is one's second operand, and V is read
// value by value (its rows r and r + 4 half a row apart).  Keys that are left out are never loaded: their
// offset lies outside the resource, LDS gets zeros, and their score is -inf.  bf16: p is rounded to bf16 for the second product, while
// L adds it in 32 bits -- its matrix instructions take no wider operand beside bf16 values, and p in two parts would be half as
// many products again.  Each p is off by at most 2^-8; the case below is 2.06e-3 of its result from 64 bits, 1.66e-3 being the
// results' own rounding.
// With nsplit > 1 workgroups share the keys of one row block and leave (O, M, L) for attention_join_kernel.
// Bound by both products and the exponentials between them, which the two waves of a SIMD hardly ever do side by side (matrix
// instructions are busy 38 % of the time, vector ones 46): bf16 8 x 1024 queries of 16 heads over 4096 keys of 4, head_dim 128,
// 300 us, 915 TF/s (two groups of waves in turn 286, but 188 for 174 at head_dim 64 and 88 for 69 in small batches; 64 rows a wave
// 313 to 387); head_dim 64 171 us.  fp32 by the rate of its instructions: 2 x 1024 queries, head_dim 128 594 us, 116 of 153 TF/s.
template <int TYPE, int DP, int RW, int KW, int KT>
__global__ __launch_bounds__(64 * RW * KW, 2) void attention_tile_kernel(const crnn_cross_attention_args a, int nsplit) {
  typedef typename TypeOf<TYPE>::t T;
  constexpr int ES = sizeof(T), EPC = 16 / ES, ROWB = DP * ES, NCH = ROWB / 16, TILE = KT * ROWB;   // values of a chunk, bytes and chunks of a row
  constexpr int LOADS = TILE / 1024;                                          // dma16 instructions a tile, shared by RW waves
  __shared__ __attribute__((aligned(1024))) unsigned char smem[KW * 4 * TILE];   // [KW][2 stages][K, V]
  static_assert(KW == 1 || sizeof(smem) >= (RW * DP * 32 + RW * 64) * 4, "the join's exchange fits the tiles");
  // (LDS leaves a SIMD one wave: the compiler then uses AccVGPRs)
  if constexpr (sizeof(smem) > 80 * 1024 || (ES == 4 && 163840 / sizeof(smem) * RW * KW < 8)) CRNN_WHOLE_REGISTER_FILE();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int kw = wave / RW, rw = wave % RW;
  const int G = a.heads / a.kv_heads, D = a.head_dim;
  const int64_t rows = a.q_len * G, nrb = (rows + 32 * RW - 1) / (32 * RW);
  const int64_t blk = attention_block(blockIdx.x, a.batch * a.kv_heads, nrb * nsplit);
  if (blk < 0) return;
  const int sp = (int)(blk % nsplit);
  const int64_t rb = blk / nsplit % nrb, bg = blk / nsplit / nrb, b = bg / a.kv_heads, g = bg % a.kv_heads;
  const int len = a.lengths ? max(0, (int)min((int64_t)a.lengths[b], a.kv_len)) : (int)a.kv_len;
  // this workgroup's keys: whole steps of KW tiles
  const int steps_all = (len + KT * KW - 1) / (KT * KW), steps_per = (steps_all + nsplit - 1) / nsplit;
  const int step0 = min(sp * steps_per, steps_all), steps = min(steps_per, steps_all - step0);
  const T* kp = (const T*)a.k + b * a.k_stride[0] + g * a.k_stride[2];
  const T* vp = (const T*)a.v + b * a.v_stride[0] + g * a.v_stride[2];
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;

  // query rows, as the second operand: lane & 31 the row, its chunks 2 kk + half.  A negative scale turns their sign
  const float sc = fmaxf(fabsf(a.scale), 1e-38f) * 1.4426950408889634f;
  const int64_t row = rb * 32 * RW + rw * 32 + (lane & 31);
  const bool live = row < rows;
  i32x4 q[NCH / 2];
  {
    const T* qp = (const T*)a.q + b * a.q_stride[0] + (live ? row / G : 0) * a.q_stride[1] + (g * G + (live ? row % G : 0)) * a.q_stride[2];
    const unsigned flip = a.scale < 0.f ? (ES == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
    for (int kk = 0; kk < NCH / 2; kk++) {
      const int d = (2 * kk + half) * EPC;
      q[kk] = i32x4{0, 0, 0, 0};
      if (live && d < D) q[kk] = *(const i32x4*)(qp + d);
#pragma unroll
      for (int i = 0; i < 4; i++) q[kk][i] ^= flip;
    }
  }
  auto swz_k = [](int r) { return NCH % 16 == 0 ? r & 15 : NCH % 8 == 0 ? (r >> 1) & 7 : (r >> 2) & 3; };
  auto swz_v = [](int r) {
    if (ES == 4) return NCH % 16 == 0 ? 2 * (r & 4) : 0;
    return NCH == 16 ? 4 * (r & 3) : NCH == 8 ? 2 * (r & 2) : 0;
  };
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem + kw * 4 * TILE;
  const unsigned char* base = smem + kw * 4 * TILE;

  // keys that count in tile `t` of this key wave, one bit each
  auto bits_of = [&](int step, int mbyte) __attribute__((always_inline)) -> unsigned long long {
    const int j0 = (step * KW + kw) * KT;
    unsigned long long w = len - j0 >= 64 ? ~0ull : len - j0 <= 0 ? 0ull : (1ull << (len - j0)) - 1;
    if (KT < 64) w &= (1ull << (KT & 63)) - 1;
    if (mask) w &= __ballot(mbyte != 0);
    return w;
  };
  auto mask_byte = [&](int step) __attribute__((always_inline)) -> int {
    const int j = (step * KW + kw) * KT + lane;
    return mask && (KT == 64 || lane < KT) && j < len ? mask[j] : 0;
  };
  auto load = [&](int step, int stage, unsigned long long w) __attribute__((always_inline)) {
    if (w == 0) return;
    const int64_t j0 = (int64_t)(step * KW + kw) * KT;
    const i32x4 rk = resource(kp + j0 * a.k_stride[1]), rv = resource(vp + j0 * a.v_stride[1]);
#pragma unroll
    for (int i = 0; i < (LOADS + RW - 1) / RW; i++) {
      const int n = i * RW + rw;
      if (LOADS % RW != 0 && n >= LOADS) break;
      const int pos = n * 64 + lane, r = pos / NCH, c = pos % NCH;
      const bool key = (w >> r) & 1;
      const int ck = c ^ swz_k(r), cv = c ^ swz_v(r);
      dma16(rk, lds0 + stage * 2 * TILE + n * 1024, key && ck * EPC < D ? (unsigned)(r * (int)a.k_stride[1] + ck * EPC) * ES : OUTSIDE);
      dma16(rv, lds0 + stage * 2 * TILE + TILE + n * 1024, key && cv * EPC < D ? (unsigned)(r * (int)a.v_stride[1] + cv * EPC) * ES : OUTSIDE);
    }
  };

  f32x16 o[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[i][r] = 0.f;
  float M = -INFINITY, L = 0.f;   // M in units of the raw score; L of this half-wave's keys only, joined at the end

  unsigned long long w0 = 0, w1 = 0;
  if (steps > 0) {
    w0 = bits_of(step0, mask_byte(step0));
    load(step0, 0, w0);
    if (steps > 1) w1 = bits_of(step0 + 1, mask_byte(step0 + 1));
  }
  for (int it = 0; it < steps; it++) {
    const int st = it & 1;
    int mb = 0;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // this step's tiles are in LDS, the last one's reads done
    if (RW > 1) __syncthreads();                       // ... of all waves, and the other stage is no longer read
    if (it + 1 < steps) load(step0 + it + 1, st ^ 1, w1);
    if (it + 2 < steps) mb = mask_byte(step0 + it + 2);
    const unsigned long long w = w0;
    if (w != 0) {
      const unsigned char* kt = base + st * 2 * TILE;
      const unsigned char* vt = kt + TILE;
      f32x16 s[KT / 32];
#pragma unroll
      for (int kb = 0; kb < KT / 32; kb++) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[kb][r] = 0.f;
        const int r = kb * 32 + (lane & 31);
#pragma unroll
        for (int kk = 0; kk < NCH / 2; kk++) {
          const i32x4 f = *(const i32x4*)(kt + r * ROWB + (((2 * kk + half) ^ swz_k(r)) << 4));
          s[kb] = Slice<TYPE>::mfma(__builtin_bit_cast(typename Slice<TYPE>::frag, f), __builtin_bit_cast(typename Slice<TYPE>::frag, q[kk]), s[kb]);
        }
      }
      const unsigned long long full = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
      if (w != full) {
        const unsigned long long wl = w >> (4 * half);
#pragma unroll
        for (int kb = 0; kb < KT / 32; kb++)
#pragma unroll
          for (int r = 0; r < 16; r++)
            if (!((wl >> (kb * 32 + (r & 3) + 8 * (r >> 2))) & 1)) s[kb][r] = -INFINITY;
      }
      float mt = s[0][0];
#pragma unroll
      for (int kb = 0; kb < KT / 32; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++) mt = fmaxf(mt, s[kb][r]);
      const Two both = two<32>(mt);
      const float Mn = fmaxf(M, fmaxf(both.a, both.b)), Mz = Mn == -INFINITY ? 0.f : Mn, Ms = Mz * sc;
      if (__any(Mn > M)) {   // (wave-uniform: most tiles after the first few raise no row's maximum)
        const float al = __builtin_amdgcn_exp2f((M - Mz) * sc);
        L *= al;
#pragma unroll
        for (int i = 0; i < DP / 32; i++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[i][r] *= al;
        M = Mn;
      }
#pragma unroll
      for (int kb = 0; kb < KT / 32; kb++) {
#pragma unroll
        for (int r = 0; r < 16; r++) {
          // (fp32: the difference first, so that the largest is exactly 1; one instruction more, which bf16 has no use for)
          s[kb][r] = __builtin_amdgcn_exp2f(TYPE == CRNN_FP32 ? (s[kb][r] - Mz) * sc : fmaf(s[kb][r], sc, -Ms));
          L += s[kb][r];
        }
        if constexpr (TYPE == CRNN_BF16) {
#pragma unroll
          for (int j = 0; j < 2; j++) {
            bf16x8 pj;
#pragma unroll
            for (int i = 0; i < 8; i++) pj[i] = (__bf16)s[kb][8 * j + i];
#pragma unroll
            for (int db = 0; db < DP / 32; db++) {
              s16x4 f[2];
#pragma unroll
              for (int i = 0; i < 2; i++) {
                const int r = kb * 32 + 16 * j + 8 * i + 4 * half + ((lane & 15) >> 2), c = db * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
                f[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + r * ROWB + ((c ^ swz_v(r)) << 4) + (lane & 1) * 8));
              }
              const s16x8 v8 = __builtin_shufflevector(f[0], f[1], 0, 1, 2, 3, 4, 5, 6, 7);
              o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v8), pj, o[db], 0, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int j = kb * 32 + acc_row(r, lane);
#pragma unroll
            for (int db = 0; db < DP / 32; db++) {
              const int d = db * 32 + (lane & 31);
              o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(*(const float*)(vt + j * ROWB + (((d >> 2) ^ swz_v(j)) << 4) + (d & 3) * 4), s[kb][r], o[db], 0, 0, 0);
            }
          }
        }
      }
    }
    w0 = w1;
    if (it + 2 < steps) w1 = bits_of(step0 + it + 2, mb);
  }
  L += __shfl_xor(L, 32);
  // M in exponent units from here on
  float Me = M * sc;
  if constexpr (KW > 1) {   // join the key waves of a row block: through LDS, one wave after the other
    float* xo = (float*)smem;                       // [RW][DP][32]
    float* xm = xo + RW * DP * 32;                  // [RW][2][32]
    for (int w = 1; w < KW; w++) {
      __syncthreads();
      if (kw == w) {
#pragma unroll
        for (int i = 0; i < DP / 32; i++)
#pragma unroll
          for (int r = 0; r < 16; r++) xo[(rw * DP + i * 32 + acc_row(r, lane)) * 32 + (lane & 31)] = o[i][r];
        if (half == 0) xm[(rw * 2) * 32 + lane] = Me, xm[(rw * 2 + 1) * 32 + lane] = L;
      }
      __syncthreads();
      if (kw == 0) {
        const float m2 = xm[(rw * 2) * 32 + (lane & 31)], l2 = xm[(rw * 2 + 1) * 32 + (lane & 31)];
        const float mn = fmaxf(Me, m2), ms = mn == -INFINITY ? 0.f : mn;
        const float a1 = __builtin_amdgcn_exp2f(Me - ms), a2 = __builtin_amdgcn_exp2f(m2 - ms);
#pragma unroll
        for (int i = 0; i < DP / 32; i++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[i][r] = o[i][r] * a1 + xo[(rw * DP + i * 32 + acc_row(r, lane)) * 32 + (lane & 31)] * a2;
        L = L * a1 + l2 * a2;
        Me = mn;
      }
    }
    if (kw != 0) return;
  }
  if (!live) return;
  if (nsplit > 1) {
    const SplitRow w(a, nsplit, sp, bg * rows + row);
#pragma unroll
    for (int i = 0; i < DP / 32; i++)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = i * 32 + acc_row(r, lane);   // four neighbours; head_dim is a multiple of 4
        if (d < D) *(f32x4*)(w.o + d) = f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
      }
    if (half == 0) w.ml[0] = Me, w.ml[1] = L;
    return;
  }
  T* out = (T*)a.out + b * a.out_stride[0] + row / G * a.out_stride[1] + (g * G + row % G) * a.out_stride[2];
  const float il = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int i = 0; i < DP / 32; i++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
      const int d = i * 32 + acc_row(r, lane);   // four neighbours; head_dim is a multiple of 4
      if (d < D) *(T4*)(out + d) = T4{(T)(o[i][r] * il), (T)(o[i][r + 1] * il), (T)(o[i][r + 2] * il), (T)(o[i][r + 3] * il)};
    }
}

// Two groups of lanes' maximum, sum and result become one.
template <int F, int EPC> __device__ __forceinline__ void join_lanes(float& M, float& L, float (&o)[EPC]) {
  const Two m = two<F>(M), l = two<F>(L);
  M = fmaxf(m.a, m.b);
  const float ms = M == -INFINITY ? 0.f : M, a1 = __builtin_amdgcn_exp2f(m.a - ms), a2 = __builtin_amdgcn_exp2f(m.b - ms);
  L = l.a * a1 + l.b * a2;
#pragma unroll
  for (int i = 0; i < EPC; i++) {
    const Two t = two<F>(o[i]);
    o[i] = t.a * a1 + t.b * a2;
  }
}

// A few rows (at most four) per key head: no matrix instructions, no LDS on the way in.  LPK lanes share a key (16 bytes of it
// each), so an instruction loads 64 / LPK keys; a wave takes chunks of U such groups, the next chunk's loads on their way while
// this one is worked on.  Every group of lanes keeps a maximum, a sum and a result over its own keys; they are joined at the
// end, lanes by exchange, the KW waves through LDS, nsplit workgroups by attention_join_kernel.  Keys that are left out are not
// loaded.  Bound by reading the keys: bf16 256 lines over ragged 71 states of 8 x 64 10.0 us (37 MB if they were full), two over
// 18176 20.7 us (74 MB).  (Sums over a key's lanes by LDS exchanges: 10.4.)
template <int TYPE, int LPK, int U, int R, int KW>
__global__ __launch_bounds__(64 * KW, 2) void attention_few_kernel(const crnn_cross_attention_args a, int nsplit) {
  typedef typename TypeOf<TYPE>::t T;
  constexpr int ES = sizeof(T), EPC = 16 / ES, KPI = 64 / LPK, KEYS = U * KPI;
  __shared__ float part[KW][R][LPK * EPC + 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane % LPK, grp = lane / LPK;
  const int G = a.heads / a.kv_heads, D = a.head_dim, rows = (int)a.q_len * G;
  const int64_t blk = attention_block(blockIdx.x, a.batch * a.kv_heads, nsplit);
  if (blk < 0) return;
  const int sp = (int)(blk % nsplit);
  const int64_t bg = blk / nsplit, b = bg / a.kv_heads, g = bg % a.kv_heads;
  const int len = a.lengths ? max(0, (int)min((int64_t)a.lengths[b], a.kv_len)) : (int)a.kv_len;
  const int steps_all = (len + KEYS * KW - 1) / (KEYS * KW), steps_per = (steps_all + nsplit - 1) / nsplit;
  const int step0 = min(sp * steps_per, steps_all), steps = min(steps_per, steps_all - step0);
  const T* kp = (const T*)a.k + b * a.k_stride[0] + g * a.k_stride[2];
  const T* vp = (const T*)a.v + b * a.v_stride[0] + g * a.v_stride[2];
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
  const bool din = c * EPC < D;
  // keys of a chunk that count, one bit each
  auto mask_byte = [&](int step) __attribute__((always_inline)) -> int {
    const int j = (step * KW + wave) * KEYS + lane;
    return mask && lane < KEYS && j < len ? mask[j] : 0;
  };
  auto bits_of = [&](int step, int mb) __attribute__((always_inline)) -> unsigned long long {
    const int left = len - (step * KW + wave) * KEYS;
    unsigned long long w = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
    if (KEYS < 64) w &= (1ull << (KEYS & 63)) - 1;
    return mask ? w & __ballot(mb != 0) : w;
  };
  i32x4 kr[2][U], vr[2][U];
  auto load = [&](int set, int step, unsigned long long w) __attribute__((always_inline)) {
    const int64_t j0 = (int64_t)(step * KW + wave) * KEYS;
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + j0 * a.k_stride[1]), 0, 0x7FFFFFFF, 0x00020000);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(vp + j0 * a.v_stride[1]), 0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int r = u * KPI + grp;
      const bool in = din && ((w >> r) & 1);
      kr[set][u] = __builtin_amdgcn_raw_buffer_load_b128(rk, in ? (unsigned)(r * (int)a.k_stride[1] * ES) + c * 16u : OUTSIDE, 0, 0);
      vr[set][u] = __builtin_amdgcn_raw_buffer_load_b128(rv, in ? (unsigned)(r * (int)a.v_stride[1] * ES) + c * 16u : OUTSIDE, 0, 0);
    }
  };
  auto widen = [](i32x4 x, float (&v)[EPC]) __attribute__((always_inline)) {
    if constexpr (ES == 4) {
      const f32x4 f = __builtin_bit_cast(f32x4, x);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = f[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float((unsigned)x[i] << 16), v[2 * i + 1] = __uint_as_float((unsigned)x[i] & 0xFFFF0000u);
    }
  };
  unsigned long long w = 0, wn = 0;
  if (steps > 0) {
    const int mb1 = steps > 1 ? mask_byte(step0 + 1) : 0;
    w = bits_of(step0, mask_byte(step0));
    load(0, step0, w);
    if (steps > 1) wn = bits_of(step0 + 1, mb1);
  }
  // the queries, with scale and log2 e in them (exp(x) = 2^(x log2 e))
  float q[R][EPC];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const bool in = r < rows && din;
    i32x4 x = {0, 0, 0, 0};
    if (in) x = *(const i32x4*)((const T*)a.q + b * a.q_stride[0] + r / G * a.q_stride[1] + (g * G + r % G) * a.q_stride[2] + c * EPC);
    widen(x, q[r]);
#pragma unroll
    for (int i = 0; i < EPC; i++) q[r][i] *= a.scale * 1.4426950408889634f;
  }
  float M[R], L[R], o[R][EPC];
#pragma unroll
  for (int r = 0; r < R; r++) {
    M[r] = -INFINITY, L[r] = 0.f;
#pragma unroll
    for (int i = 0; i < EPC; i++) o[r][i] = 0.f;
  }
  auto work = [&](int set, unsigned long long bits) __attribute__((always_inline)) {
    if (bits == 0) return;
    float s[R][U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      float k[EPC];
      widen(kr[set][u], k);
      const bool in = (bits >> (u * KPI + grp)) & 1;
#pragma unroll
      for (int r = 0; r < R; r++) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < EPC; i++) t = fmaf(q[r][i], k[i], t);
        s[r][u] = in ? group_sum<LPK>(t) : -INFINITY;
      }
    }
    float al[R], Ms[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      float m = M[r];
#pragma unroll
      for (int u = 0; u < U; u++) m = fmaxf(m, s[r][u]);
      Ms[r] = m == -INFINITY ? 0.f : m;
      al[r] = __builtin_amdgcn_exp2f(M[r] - Ms[r]);
      M[r] = m;
      L[r] *= al[r];
#pragma unroll
      for (int i = 0; i < EPC; i++) o[r][i] *= al[r];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float v[EPC];
      widen(vr[set][u], v);
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float p = __builtin_amdgcn_exp2f(s[r][u] - Ms[r]);
        L[r] += p;
#pragma unroll
        for (int i = 0; i < EPC; i++) o[r][i] = fmaf(p, v[i], o[r][i]);
      }
    }
  };
  auto turn = [&](int set, int it) __attribute__((always_inline)) {
    if (it >= steps) return;
    int mb = 0;
    if (it + 2 < steps) mb = mask_byte(step0 + it + 2);
    if (it + 1 < steps) load(set ^ 1, step0 + it + 1, wn);
    work(set, w);
    w = wn;
    if (it + 2 < steps) wn = bits_of(step0 + it + 2, mb);
  };
  for (int it = 0; it < steps; it += 2) {
    turn(0, it);
    turn(1, it + 1);
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    if constexpr (LPK <= 4) join_lanes<4>(M[r], L[r], o[r]);
    if constexpr (LPK <= 8) join_lanes<8>(M[r], L[r], o[r]);
    if constexpr (LPK <= 16) join_lanes<16>(M[r], L[r], o[r]);
    join_lanes<32>(M[r], L[r], o[r]);
  }
  if constexpr (KW > 1) {
    if (grp == 0) {
#pragma unroll
      for (int r = 0; r < R; r++) {
#pragma unroll
        for (int i = 0; i < EPC; i++) part[wave][r][c * EPC + i] = o[r][i];
        if (c == 0) part[wave][r][LPK * EPC] = M[r], part[wave][r][LPK * EPC + 1] = L[r];
      }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int k = 1; k < KW; k++) {
        const float m2 = part[k][r][LPK * EPC], l2 = part[k][r][LPK * EPC + 1], m = fmaxf(M[r], m2), ms = m == -INFINITY ? 0.f : m;
        const float a1 = __builtin_amdgcn_exp2f(M[r] - ms), a2 = __builtin_amdgcn_exp2f(m2 - ms);
        L[r] = L[r] * a1 + l2 * a2;
#pragma unroll
        for (int i = 0; i < EPC; i++) o[r][i] = o[r][i] * a1 + part[k][r][c * EPC + i] * a2;
        M[r] = m;
      }
  }
  if (grp != 0 || !din) return;
#pragma unroll
  for (int r = 0; r < R; r++) {
    if (r >= rows) break;
    if (nsplit > 1) {
      const SplitRow w(a, nsplit, sp, bg * rows + r);
#pragma unroll
      for (int i = 0; i < EPC; i += 4) *(f32x4*)(w.o + c * EPC + i) = f32x4{o[r][i], o[r][i + 1], o[r][i + 2], o[r][i + 3]};
      if (c == 0) w.ml[0] = M[r], w.ml[1] = L[r];
    } else {
      T* out = (T*)a.out + b * a.out_stride[0] + r / G * a.out_stride[1] + (g * G + r % G) * a.out_stride[2] + c * EPC;
      const float il = L[r] == 0.f ? 0.f : 1.f / L[r];
#pragma unroll
      for (int i = 0; i < EPC; i++) out[i] = (T)(o[r][i] * il);
    }
  }
}

// out = sum_s O_s 2^(M_s - M) / sum_s L_s 2^(M_s - M): a workgroup per row, LP lanes with four values each per split, 256 / LP
// splits side by side, so that everything is asked for at once; the groups meet in LDS.  Bound by the way of the bytes, twice:
// 3.9 us for 16 rows of 64 splits (one row a thread, split by split: 17).
template <int TYPE, int LP>
__global__ __launch_bounds__(256) void attention_join_kernel(const crnn_cross_attention_args a, int nsplit) {
  typedef typename TypeOf<TYPE>::t T;
  constexpr int GR = 256 / LP, PER = MAX_SPLIT / GR;
  __shared__ float po[GR][LP * 4], pm[GR][2];
  const int G = a.heads / a.kv_heads, D = a.head_dim, tid = threadIdx.x, c = tid % LP, grp = tid / LP;
  const int64_t rows = a.q_len * G, all = a.batch * a.kv_heads * rows;
  for (int64_t r = blockIdx.x; r < all; r += gridDim.x) {
    f32x4 o[PER];
    float m[PER], l[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int s = grp + i * GR;
      const SplitRow w(a, nsplit, s, r);
      o[i] = f32x4{0.f, 0.f, 0.f, 0.f}, m[i] = -INFINITY, l[i] = 0.f;
      if (s < nsplit) {
        m[i] = w.ml[0], l[i] = w.ml[1];
        if (4 * c < D) o[i] = *(const f32x4*)(w.o + 4 * c);
      }
    }
    float M = m[0];
#pragma unroll
    for (int i = 1; i < PER; i++) M = fmaxf(M, m[i]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const float e = __builtin_amdgcn_exp2f(m[i] - Ms);
      L = fmaf(l[i], e, L);
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = fmaf(o[i][k], e, v[k]);
    }
    *(f32x4*)&po[grp][4 * c] = v;
    if (c == 0) pm[grp][0] = M, pm[grp][1] = L;
    __syncthreads();
    if (tid < D) {
      M = pm[0][0];
#pragma unroll
      for (int i = 1; i < GR; i++) M = fmaxf(M, pm[i][0]);
      const float Mz = M == -INFINITY ? 0.f : M;
      float x = 0.f;
      L = 0.f;
#pragma unroll
      for (int i = 0; i < GR; i++) {
        const float e = __builtin_amdgcn_exp2f(pm[i][0] - Mz);
        L = fmaf(pm[i][1], e, L);
        x = fmaf(po[i][tid], e, x);
      }
      const int64_t bg = r / rows, row = r - bg * rows;
      T* out = (T*)a.out + bg / a.kv_heads * a.out_stride[0] + row / G * a.out_stride[1] + (bg % a.kv_heads * G + row % G) * a.out_stride[2];
      out[tid] = (T)(L == 0.f ? 0.f : x / L);
    }
    __syncthreads();
  }
}

// The same for many rows: LP lanes a row, four values each, 256 / LP rows a workgroup, the splits one after the other.
template <int TYPE, int LP>
__global__ __launch_bounds__(256) void attention_join_rows_kernel(const crnn_cross_attention_args a, int nsplit) {
  typedef typename TypeOf<TYPE>::t T;
  typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  constexpr int RPB = 256 / LP;
  const int G = a.heads / a.kv_heads, D = a.head_dim, c = threadIdx.x % LP;
  const int64_t rows = a.q_len * G, all = a.batch * a.kv_heads * rows;
  if (4 * c >= D) return;
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / LP; r < all; r += (int64_t)gridDim.x * RPB) {
    float M = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < nsplit; s++) M = fmaxf(M, SplitRow(a, nsplit, s, r).ml[0]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < nsplit; s++) {
      const SplitRow w(a, nsplit, s, r);
      const float e = __builtin_amdgcn_exp2f(w.ml[0] - Ms);
      const f32x4 o = *(const f32x4*)(w.o + 4 * c);
      L = fmaf(w.ml[1], e, L);
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = fmaf(o[k], e, v[k]);
    }
    const float d = L == 0.f ? 1.f : L;   // (divided, not multiplied: where one key counts its value comes out as it is)
    const int64_t bg = r / rows, row = r - bg * rows;
    T* out = (T*)a.out + bg / a.kv_heads * a.out_stride[0] + row / G * a.out_stride[1] + (bg % a.kv_heads * G + row % G) * a.out_stride[2];
    *(T4*)(out + 4 * c) = T4{(T)(v[0] / d), (T)(v[1] / d), (T)(v[2] / d), (T)(v[3] / d)};
  }
}

static bool attention_chunks(const crnn_cross_attention_args& a) {   // (sizes, type and strides only)
  const int c = a.type == CRNN_BF16 ? 8 : 4;
  if (a.head_dim % c != 0 || a.kv_len == 0 || a.kv_len > 0x7FF00000) return false;   // (key numbers a few steps past the end are ints)
  const int64_t qn[3] = {a.batch, a.q_len, a.heads}, kn[3] = {a.batch, a.kv_len, a.kv_heads};
  for (int i = 0; i < 3; i++)   // (a stride that no step is made by may be anything)
    if ((qn[i] > 1 && a.q_stride[i] % c != 0) || (kn[i] > 1 && (a.k_stride[i] % c != 0 || a.v_stride[i] % c != 0))) return false;
  return a.kv_len == 1 || (a.k_stride[1] < (1 << 22) && a.v_stride[1] < (1 << 22));   // offsets within 64 keys stay below 2^31 bytes
}
static bool attention_aligned(const crnn_cross_attention_args& a) { return (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0; }

// How the work is cut: `rw` waves side by side over 32 rows each, or 0 for attention_few_kernel; `kw` waves over the keys;
// nsplit workgroups over the keys where there are too few row blocks to fill the chip.
struct AttnPlan {
  int rw, kw, nsplit;
};
static AttnPlan attention_plan(const crnn_cross_attention_args& a) {
  const int64_t rows = a.q_len * (a.heads / a.kv_heads), bg = a.batch * a.kv_heads;
  AttnPlan p;
  int64_t blocks, keys;   // row blocks; keys of a workgroup's step
  // Few rows without matrix instructions: bf16 one (1 over 300 keys of 100 lines 16.0 us, by tiles 20.4; 3 over 256 lines of 71
  // 17.4 and 11.6), with large heads, whose tiles leave a CU one workgroup, three (2 over 600 keys, head_dim 128, 36 and 46; 4
  // over 2000 20.0 and 17.9), fp32, whose matrix instructions are slow, four (4 over 600 keys, head_dim 128, 73 and 120)
  const bool b16 = a.type == CRNN_BF16;
  if (rows <= (!b16 ? 4 : a.head_dim > 64 ? 3 : 1)) {
    p.rw = 0;
    // few keys, many heads: a wave a head, nothing to join
    p.kw = a.kv_len <= 128 && bg >= 1024 ? 1 : 4;
    blocks = bg;
    const int64_t chunks = a.head_dim / (a.type == CRNN_BF16 ? 8 : 4);
    keys = 256 / (chunks <= 4 ? 4 : chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32) * p.kw;
  } else {
    p.rw = rows > 64 ? 4 : rows > 32 ? 2 : 1;
    blocks = bg * ((rows + 32 * p.rw - 1) / (32 * p.rw));
    // fp32 tiles take twice the LDS, so half the waves over the keys, but where at most two workgroups come to a CU: two waves
    // of each leave SIMDs idle.  48 queries over 71 states, head_dim 64: 64 lines 18.8 us with two waves over the keys, 21.2
    // with one; 96 lines 27.1 and 23.3.
    p.kw = a.type == CRNN_BF16 ? 4 / p.rw : p.rw == 1 || (p.rw == 2 && blocks <= 512 && a.head_dim <= 64) ? 2 : 1;
    const int kt = a.type == CRNN_BF16 && p.rw == 4 ? 64 : 32;
    if (p.rw == 1 && a.kv_len <= 4 * kt && bg >= 1024) p.kw = 1;
    keys = kt * p.kw;
  }
  const int64_t steps = (a.kv_len + keys - 1) / keys;
  // workgroups at a time: what the registers of a SIMD hold, two a CU, without matrix instructions four for one row and less for
  // more; steps that each has at least
  const int64_t slots = 256 * (p.rw != 0 ? 2 : rows == 1 ? 4 : (rows == 2 ? 4 : 3) - b16), least = p.rw == 0 ? 1 : 2;
  int64_t ns = 1;
  if (blocks < slots) {
    // rounds of a workgroup's steps and as many again as the least, for its way in and out, and for the join three and one more
    // for each 24 splits.  (Splits that just fill the chip, slots / blocks rounded up, start a round for their last few: fp32
    // 4 x 400 queries of 8 heads over 3992 keys, head_dim 128, 347 us, this 256; bf16 30 x 20 queries over 500 keys 20.5 and
    // 11.6, 1 over 300 of 100 lines 21.4 and 15.9.)
    double best = 0.;
    for (int64_t n = 1; n <= MAX_SPLIT && (n == 1 || n * least <= steps); n++) {
      const double cost = (double)((blocks * n + slots - 1) / slots) * (double)((steps + n - 1) / n + least) + (n > 1 ? 3. + (double)n / 24. : 0.);
      if (n == 1 || cost < best) best = cost, ns = n;
    }
  }
  p.nsplit = (int)ns;
  return p;
}
int64_t cross_attention_workspace(const crnn_cross_attention_args& a) {
  if (!attention_chunks(a)) return 0;
  const AttnPlan p = attention_plan(a);
  return p.nsplit <= 1 ? 0 : (int64_t)p.nsplit * a.batch * a.heads * a.q_len * (a.head_dim + 2) * 4;
}

template <int TYPE, int DP, int RW, int KW>
static void attention_tile(const crnn_cross_attention_args& a, int nsplit, hipStream_t s) {
  constexpr int KT = TYPE == CRNN_BF16 && RW == 4 ? 64 : 32;
  const int64_t rows = a.q_len * (a.heads / a.kv_heads), each = (rows + 32 * RW - 1) / (32 * RW) * nsplit;
  hipLaunchKernelGGL((attention_tile_kernel<TYPE, DP, RW, KW, KT>), dim3((unsigned)attention_grid(a.batch * a.kv_heads, each)), dim3(64 * RW * KW), 0, s, a, nsplit);
}
template <int TYPE, int DP>
static void attention_tile(const crnn_cross_attention_args& a, const AttnPlan& p, hipStream_t s) {
  constexpr bool B16 = TYPE == CRNN_BF16;   // (the waves over the keys are what attention_plan says)
  if (p.rw == 4) attention_tile<TYPE, DP, 4, 1>(a, p.nsplit, s);
  else if (p.rw == 2 && p.kw > 1) attention_tile<TYPE, DP, 2, B16 || DP <= 64 ? 2 : 1>(a, p.nsplit, s);
  else if (p.rw == 2) attention_tile<TYPE, DP, 2, B16 ? 2 : 1>(a, p.nsplit, s);
  else if (p.kw > 1) attention_tile<TYPE, DP, 1, B16 ? 4 : 2>(a, p.nsplit, s);
  else attention_tile<TYPE, DP, 1, 1>(a, p.nsplit, s);
}
template <int TYPE>
static void attention_tile(const crnn_cross_attention_args& a, const AttnPlan& p, hipStream_t s) {
  if (a.head_dim <= 32) attention_tile<TYPE, 32>(a, p, s);
  else if (a.head_dim <= 64) attention_tile<TYPE, 64>(a, p, s);
  else if (a.head_dim <= 96) attention_tile<TYPE, 96>(a, p, s);
  else attention_tile<TYPE, 128>(a, p, s);
}
template <int TYPE, int LPK, int R>
static void attention_few(const crnn_cross_attention_args& a, const AttnPlan& p, hipStream_t s) {
  constexpr int U = 4;   // loads of each in a chunk (eight: a wave less per SIMD, one query over 256 lines 11.0 us for 10.4)
  const dim3 g((unsigned)attention_grid(a.batch * a.kv_heads, p.nsplit));
  if (p.kw == 1) hipLaunchKernelGGL((attention_few_kernel<TYPE, LPK, U, R, 1>), g, dim3(64), 0, s, a, p.nsplit);
  else hipLaunchKernelGGL((attention_few_kernel<TYPE, LPK, U, R, 4>), g, dim3(256), 0, s, a, p.nsplit);
}
template <int TYPE, int LPK>
static void attention_few(const crnn_cross_attention_args& a, const AttnPlan& p, hipStream_t s) {
  const int64_t rows = a.q_len * (a.heads / a.kv_heads);
  if constexpr (TYPE == CRNN_FP32 || LPK > 8) {   // (bf16 up to head_dim 64: one row, attention_plan)
    if (rows > 2) return attention_few<TYPE, LPK, 4>(a, p, s);
    if (rows == 2) return attention_few<TYPE, LPK, 2>(a, p, s);
  }
  attention_few<TYPE, LPK, 1>(a, p, s);
}
template <int TYPE>
static void attention_few(const crnn_cross_attention_args& a, const AttnPlan& p, hipStream_t s) {
  const int chunks = a.head_dim / (TYPE == CRNN_BF16 ? 8 : 4);
  if (chunks <= 4) attention_few<TYPE, 4>(a, p, s);
  else if (chunks <= 8) attention_few<TYPE, 8>(a, p, s);
  else if (chunks <= 16) attention_few<TYPE, 16>(a, p, s);
  else if constexpr (TYPE == CRNN_FP32) attention_few<TYPE, 32>(a, p, s);
}

template <int TYPE, int LP>
static void attention_join(const crnn_cross_attention_args& a, int nsplit, hipStream_t s) {
  const int64_t all = a.batch * a.heads * a.q_len;
  // a workgroup a row hides the way to memory, a row a few lanes wastes none of it: 8 rows of 64 splits 16.1 and 23.2 us with
  // the attention, 4800 rows of 5 30.7 and 26.9, 24000 of 2 66 and 38
  if (all <= JOIN_ROWS) hipLaunchKernelGGL((attention_join_kernel<TYPE, LP>), grid_for(all), dim3(256), 0, s, a, nsplit);
  else hipLaunchKernelGGL((attention_join_rows_kernel<TYPE, LP>), grid_for((all * LP + 255) / 256), dim3(256), 0, s, a, nsplit);
}

void launch_cross_attention(const crnn_cross_attention_args& a, hipStream_t s) {
  const int64_t rows = a.q_len * (a.heads / a.kv_heads);
  const int64_t blocks = a.batch * a.kv_heads * ((rows + 31) / 32);
  if (attention_chunks(a) && attention_aligned(a) && (blocks < (1 << 22) || a.batch > 1)) {
    if (blocks >= 1 << 22) {   // a launch has fewer than 2^32 threads: half the batch at a time (so many blocks use no workspace)
      const int64_t e = a.type == CRNN_BF16 ? 2 : 4, n = a.batch / 2;
      crnn_cross_attention_args h[2] = {a, a};
      h[0].batch = n;
      h[1].batch = a.batch - n;
      h[1].q = (const char*)a.q + n * a.q_stride[0] * e;
      h[1].k = (const char*)a.k + n * a.k_stride[0] * e;
      h[1].v = (const char*)a.v + n * a.v_stride[0] * e;
      h[1].out = (char*)a.out + n * a.out_stride[0] * e;
      if (a.lengths) h[1].lengths = a.lengths + n;
      if (a.mask) h[1].mask = a.mask + n * a.mask_stride;
      launch_cross_attention(h[0], s);
      launch_cross_attention(h[1], s);
      return;
    }
    const AttnPlan p = attention_plan(a);
    if (p.rw == 0) a.type == CRNN_BF16 ? attention_few<CRNN_BF16>(a, p, s) : attention_few<CRNN_FP32>(a, p, s);
    else a.type == CRNN_BF16 ? attention_tile<CRNN_BF16>(a, p, s) : attention_tile<CRNN_FP32>(a, p, s);
    if (p.nsplit > 1) {
      if (a.type == CRNN_BF16) a.head_dim <= 64 ? attention_join<CRNN_BF16, 16>(a, p.nsplit, s) : attention_join<CRNN_BF16, 32>(a, p.nsplit, s);
      else a.head_dim <= 64 ? attention_join<CRNN_FP32, 16>(a, p.nsplit, s) : attention_join<CRNN_FP32, 32>(a, p.nsplit, s);
    }
    return;
  }
  const dim3 g = grid_for(a.batch * a.kv_heads * ((rows + 15) / 16)), b(256);
  if (a.type == CRNN_FP32) hipLaunchKernelGGL((attention_any_kernel<CRNN_FP32>), g, b, 0, s, a);
  else hipLaunchKernelGGL((attention_any_kernel<CRNN_BF16>), g, b, 0, s, a);
}

// ---------------------------------------------------------------------------
// the recogniser's states for the operators above: 16 bytes per thread, zeros behind a line's end.  Bound by HBM: 256 lines
// of 280 pixels, fp32, 12.5 us (72 MB)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void copy_states_kernel(const f32x4* __restrict__ rec, f32x4* __restrict__ out, int32_t* __restrict__ out_len,
                                                          const int32_t* __restrict__ tlen, int64_t total, int row, int T) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {   // chunk; `row` chunks a state
    const int64_t st = i / row, line = st / T;
    const int t = (int)(st - line * T), n = tlen ? tlen[line] : T;
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    out[i] = t < n ? rec[i] : z;
    if (out_len && t == 0 && i % row == 0) out_len[line] = n;
  }
}

void launch_copy_states(const void* rec, void* out, int32_t* out_len, const int32_t* tlen, int n, int T, bool b16, hipStream_t s) {
  const int row = b16 ? 64 : 128;
  const int64_t total = (int64_t)n * T * row;
  hipLaunchKernelGGL(copy_states_kernel, grid_for((total + 255) / 256), dim3(256), 0, s, (const f32x4*)rec, (f32x4*)out, out_len, tlen, total, row, T);
}

__global__ void warm_seq_kernel() {}
void launch_warm_seq(hipStream_t s) { hipLaunchKernelGGL(warm_seq_kernel, dim3(1), dim3(64), 0, s); }

}  // namespace crnn
