// Kernels of the sequence operators (include/crnn_hip.h: crnn_linear, crnn_rms_norm, crnn_cross_attention), gfx950.
// Compiled without packed fp32 (crnn_kernels_nopk.hip says why).
#include "crnn_seq.h"

#include <cmath>

namespace crnn {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
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

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case CRNN_ACT_RELU: return v > 0.f ? v : 0.f;
    case CRNN_ACT_LEAKY: return v > 0.f ? v : 0.2f * v;
    case CRNN_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    case CRNN_ACT_SILU: return v / (1.f + expf(-v));
    default: return v;
  }
}

// ---------------------------------------------------------------------------
// linear, any strides and sizes: 64 x 64 tile of y per workgroup, four waves with 32 x 32 each; tiles of 32 values of k go
// through LDS element by element, so nothing is asked of alignment.  x is the first operand: the 32 lanes of a half-wave
// hold neighbouring columns of y.  8-bit values go through as bfloat16, which holds them exactly: the 8-bit matrix
// instructions keep only 13 bits below the largest of each few products that they add first (measured: 2^8 + 2^-5 in one
// group is exact, 2^8 + 2^-6 is 2^8; between groups and with the accumulator all 24 bits are kept).
// ---------------------------------------------------------------------------
template <typename TL> __device__ __forceinline__ TL load(const float* p) { return *p; }
template <typename TL> __device__ __forceinline__ TL load(const __bf16* p) { return *p; }
template <typename TL> __device__ __forceinline__ TL load(const e4m3* p) { return (TL)__builtin_amdgcn_cvt_f32_fp8(*p, 0); }

template <int IN, int OUT>
__global__ __launch_bounds__(256, 2) void linear_any_kernel(const crnn_linear_args a) {
  typedef typename TypeOf<IN>::t T;
  typedef typename TypeOf<OUT>::t TO;
  typedef typename TypeOf<IN == CRNN_FP32 ? CRNN_FP32 : CRNN_BF16>::t TL;
  constexpr int KT = 32, LD = IN == CRNN_FP32 ? KT + 1 : KT + 8;
  __shared__ __attribute__((aligned(16))) TL xs[64 * LD], ws[64 * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int64_t ntn = (a.n + 63) / 64, tiles = (a.m + 63) / 64 * ntn;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const T* x = (const T*)a.x;
  const T* w = (const T*)a.w;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t m0 = tile / ntn * 64, n0 = tile % ntn * 64;
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; r++) acc[r] = 0.f;
    for (int64_t k0 = 0; k0 < a.k; k0 += KT) {
#pragma unroll
      for (int i = 0; i < 64 * KT / 256; i++) {
        const int e = tid + 256 * i, row = e / KT, c = e % KT;
        const bool kin = k0 + c < a.k;
        xs[row * LD + c] = kin && m0 + row < a.m ? load<TL>(x + (m0 + row) * a.ldx + k0 + c) : (TL)0;
        ws[row * LD + c] = kin && n0 + row < a.n ? load<TL>(w + (n0 + row) * a.ldw + k0 + c) : (TL)0;
      }
      __syncthreads();
      const TL* xr = xs + (wm + (lane & 31)) * LD;
      const TL* wr = ws + (wn + (lane & 31)) * LD;
      if constexpr (IN != CRNN_FP32) {
#pragma unroll
        for (int c = 0; c < KT; c += 16)
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(xr + c + 8 * half), *(const bf16x8*)(wr + c + 8 * half), acc, 0, 0, 0);
      } else {
#pragma unroll
        for (int c = 0; c < KT; c += 2) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(xr[c + half], wr[c + half], acc, 0, 0, 0);
      }
      __syncthreads();
    }
    const int64_t n = n0 + wn + (lane & 31);
    if (n >= a.n) continue;
    const float ws1 = a.w_scale ? a.w_scale[n] : 1.f, b = a.bias ? a.bias[n] : 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int64_t m = m0 + wm + acc_row(r, lane);
      if (m >= a.m) continue;
      float v = acc[r];
      if (IN == CRNN_E4M3) v = v * (a.x_scale ? a.x_scale[m] : 1.f) * ws1;
      v = activate(v + b, a.act);
      if (a.residual) v += (float)((const TO*)a.residual)[m * a.ldr + n];
      ((TO*)a.y)[m * a.ldy + n] = (TO)v;
    }
  }
}

void launch_linear(const crnn_linear_args& a, hipStream_t s) {
  const dim3 g = grid_for((a.m + 63) / 64 * ((a.n + 63) / 64)), b(256);
  if (a.in_type == CRNN_FP32) {
    if (a.out_type == CRNN_FP32) hipLaunchKernelGGL((linear_any_kernel<CRNN_FP32, CRNN_FP32>), g, b, 0, s, a);
    else hipLaunchKernelGGL((linear_any_kernel<CRNN_FP32, CRNN_BF16>), g, b, 0, s, a);
  } else if (a.in_type == CRNN_BF16) {
    if (a.out_type == CRNN_FP32) hipLaunchKernelGGL((linear_any_kernel<CRNN_BF16, CRNN_FP32>), g, b, 0, s, a);
    else hipLaunchKernelGGL((linear_any_kernel<CRNN_BF16, CRNN_BF16>), g, b, 0, s, a);
  } else {
    if (a.out_type == CRNN_FP32) hipLaunchKernelGGL((linear_any_kernel<CRNN_E4M3, CRNN_FP32>), g, b, 0, s, a);
    else hipLaunchKernelGGL((linear_any_kernel<CRNN_E4M3, CRNN_BF16>), g, b, 0, s, a);
  }
}

// ---------------------------------------------------------------------------
// rms_norm.  y = t r g with r = (sum t^2 / n + eps)^-1/2.  Where the sum of squares leaves the range in which a 32-bit one is
// exact (rows around 1e-20 or above 1e18) it is taken again in 64 bits, and r is applied as a power of two near 1 / |t| and
// the rest, so that no product on the way leaves the normal numbers.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
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
__device__ __forceinline__ e4m3 to_e4m3(float v) { return (e4m3)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xFF); }

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

// Any strides and sizes: one workgroup per row, the row read again for each of the passes (sum of squares, with 8-bit outputs
// the largest |y|, the outputs).  The outputs are written in the last pass by the thread that reads the same element, so they
// may be the inputs themselves.
template <int IN, int OUT>
__global__ __launch_bounds__(256) void rms_norm_any_kernel(const crnn_rms_norm_args a) {
  typedef typename TypeOf<IN>::t T;
  typedef typename TypeOf<OUT>::t TO;
  __shared__ float part[4];
  __shared__ double partd[4];
  __shared__ unsigned partu[4];
  const int tid = threadIdx.x;
  for (int64_t m = blockIdx.x; m < a.m; m += gridDim.x) {
    const T* x = (const T*)a.x + m * a.ldx;
    const T* r = a.residual ? (const T*)a.residual + m * a.ldr : nullptr;
    auto value = [&](int64_t i) { return r ? (float)x[i] + (float)r[i] : (float)x[i]; };
    float ss = 0.f, r1 = 1.f, r2;
    for (int64_t i = tid; i < a.n; i += 256) {
      const float t = value(i);
      ss += t * t;
    }
    ss = row_sum<256>(ss, part);
    if (squares_ok(ss)) {
      r2 = 1.f / sqrtf(ss / (float)a.n + a.eps);
    } else {
      double sd = 0.0;
      for (int64_t i = tid; i < a.n; i += 256) {
        const double t = value(i);
        sd += t * t;
      }
      row_factors(row_sum<256>(sd, partd), (double)a.n, a.eps, &r1, &r2);
    }
    float c = 1.f, ic = 1.f;
    if (OUT == CRNN_E4M3) {
      unsigned top = 0;
      for (int64_t i = tid; i < a.n; i += 256) top = max(top, abs_bits(value(i) * r1 * r2 * a.gain[i]));
      c = row_scale(row_max<256>(top, partu));
      ic = 1.f / c;
    }
    for (int64_t i = tid; i < a.n; i += 256) {
      const float t = value(i), y = t * r1 * r2 * a.gain[i];
      if (a.sum) ((T*)a.sum)[m * a.lds + i] = (T)t;
      if constexpr (OUT == CRNN_E4M3) ((e4m3*)a.y)[m * a.ldy + i] = to_e4m3(y * ic);
      else ((TO*)a.y)[m * a.ldy + i] = (TO)y;
    }
    if (OUT == CRNN_E4M3 && tid == 0) a.y_scale[m] = c;
    __syncthreads();   // (part)
  }
}

// Rows of 16-byte chunks that fit the registers of one wave (TPR 64: four rows a workgroup) or one workgroup (TPR 256): x and
// the residual are read once, everything else happens in registers.  A thread holds C groups of eight values; the gain stays in
// registers over the rows that a workgroup takes.  Bound by HBM.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const __bf16* p, float (&v)[8]) {
  const bf16x8 a = *(const bf16x8*)p;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (float)a[i];
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
  *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(__bf16* p, const float (&v)[8]) {
  bf16x8 a;
#pragma unroll
  for (int i = 0; i < 8; i++) a[i] = (__bf16)v[i];
  *(bf16x8*)p = a;
}
__device__ __forceinline__ void store8(e4m3* p, const float (&v)[8]) {
  i32x2 a;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
    a[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], u, true);
  }
  *(i32x2*)p = a;
}

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
    if (i < n) {
#pragma unroll
      for (int e = 0; e < 8; e++) g[c][e] = a.gain[i + e];
    }
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
      if (i < n) {
        load8(x + i, t[c]);
        if (a.residual) {
          float r[8];
          load8(res + i, r);
#pragma unroll
          for (int e = 0; e < 8; e++) t[c][e] += r[e];
        }
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
      for (int c = 0; c < C; c++) {
        const int i = (c * TPR + at) * 8;
        if (i < n) store8((T*)a.sum + m * a.lds + i, t[c]);
      }
    }
    unsigned top = 0;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        t[c][e] = t[c][e] * r1 * r2 * g[c][e];
        // (past the end of the row t is 0, but 0 times an infinite factor would be NaN)
        if (OUT == CRNN_E4M3) top = max(top, (c * TPR + at) * 8 < n ? abs_bits(t[c][e]) : 0u);
      }
    float ic = 1.f;
    if (OUT == CRNN_E4M3) {
      const float sc = row_scale(row_max<TPR>(top, partu));
      ic = 1.f / sc;
      if (at == 0) a.y_scale[m] = sc;
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int i = (c * TPR + at) * 8;
      if (OUT == CRNN_E4M3) {
#pragma unroll
        for (int e = 0; e < 8; e++) t[c][e] *= ic;
      }
      if (i < n) store8((TO*)a.y + m * a.ldy + i, t[c]);
    }
  }
}

template <int IN, int OUT>
static void rms_norm_of(const crnn_rms_norm_args& a, hipStream_t s) {
  // whole 16-byte chunks in every row (8 bytes where the output is 8 bits)
  const int64_t ei = IN == CRNN_FP32 ? 4 : 2, eo = OUT == CRNN_E4M3 ? 1 : ei, wo = OUT == CRNN_E4M3 ? 8 : 16;
  auto fits = [](const void* p, int64_t ld, int64_t e, int64_t w) { return !p || (((uintptr_t)p | (uintptr_t)(ld * e)) & (uintptr_t)(w - 1)) == 0; };
  const bool wide = a.n % 8 == 0 && a.n <= 8192 && fits(a.x, a.ldx, ei, 16) && fits(a.residual, a.ldr, ei, 16) && fits(a.sum, a.lds, ei, 16) && fits(a.y, a.ldy, eo, wo);
  // at most 8 workgroups a CU at a time: more rows are taken in turn, with the gain at hand
  auto grid = [&](int rows) { return dim3((unsigned)((a.m + rows - 1) / rows < 2048 ? (a.m + rows - 1) / rows : 2048)); };
  if (!wide) hipLaunchKernelGGL((rms_norm_any_kernel<IN, OUT>), grid_for(a.m), dim3(256), 0, s, a);
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
// Any strides, sizes and types: 16 rows per workgroup, tiles of 32 keys in LDS as fp32, scores and sums by fp32 FMAs.
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

int64_t cross_attention_workspace(const crnn_cross_attention_args&) { return 0; }

void launch_cross_attention(const crnn_cross_attention_args& a, hipStream_t s) {
  const int64_t rows = a.q_len * (a.heads / a.kv_heads);
  const dim3 g = grid_for(a.batch * a.kv_heads * ((rows + 15) / 16)), b(256);
  if (a.type == CRNN_FP32) hipLaunchKernelGGL((attention_any_kernel<CRNN_FP32>), g, b, 0, s, a);
  else hipLaunchKernelGGL((attention_any_kernel<CRNN_BF16>), g, b, 0, s, a);
}

// ---------------------------------------------------------------------------
// the recogniser's states for the operators above: 16 bytes per thread, zeros behind a line's end
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
