// 4-bit frozen weights: quantise, dequantise, embedding lookup and the linear products on them.
//
// Format: W [N, K] as e2m1 codes [N, K / 2] (two per byte, the even column in the low half) and one scale
// byte per 32 columns of a row, [N, K / 32]: value = e2m1(code) * 2^(byte - 127); byte 255 reads as NaN.
// e2m1 has a 1-bit mantissa and the scale is a power of two, so every value is exact in bf16: the products
// below multiply exact bf16 weights in MFMA with fp32 accumulation and round once, at the store.
// The scale byte stays in [2, 252]: the smallest non-zero value is 2^-126 (a normal bf16 number), the
// largest 6 * 2^125 (finite).
#include "common.h"
#include "kernels.h"
#include "mfma.h"

#include <cstdio>
#include <cstdlib>

namespace mft {

namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// scale byte -> the fp32 whose exponent field it is; 255 -> NaN
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// 8 codes (one 32-bit word, low half-byte first) -> 8 bf16 values
__device__ __forceinline__ bf16x8_t mx4_cvt8(uint32_t w, float s) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ------------------------------------------------------------------ quantise
// Four lanes share a group of 32 columns (8 each).  The scale: with a = max |w| = f 2^e, 1 <= f < 2, the
// byte is e + 127 - 2, one more when f > 1.75.  |w| 2^(127 - byte) is then at most 7; above 6 it saturates,
// off by at most 1 -- half a step at that size, as everywhere on the grid.  Nearest code, ties to even.
// A group that holds an infinity or a NaN gets byte 255 (it reads as NaN) and codes 0.
template <bool F32>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void* __restrict__ w, uint32_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales, long n8) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;  // 8 columns; n8 % 4 == 0, so a group is in or out whole
  if (i >= n8) return;
  float v[8];
  if constexpr (F32) {
    const f32x4_t a = reinterpret_cast<const f32x4_t*>(w)[2 * i], b = reinterpret_cast<const f32x4_t*>(w)[2 * i + 1];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
    load8(reinterpret_cast<const bf16_t*>(w) + 8 * i, v);
  }
  // |w| as integers order like the magnitudes, infinities and NaNs above every number
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
  const bool bad = m >= 0x7f800000u;
  int byte = (int)(m >> 23) - 2 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
  byte = min(max(byte, 2), 252);
  const float s = __uint_as_float((uint32_t)byte << 23);
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
  codes[i] = bad ? 0u : q;
  if ((threadIdx.x & 3) == 0) scales[i >> 2] = bad ? 255 : (uint8_t)byte;
}

// ------------------------------------------------------------------ dequantise, embedding
// out[r, 0 : K] = W[n0 + r] for r < rows; columns K .. kpad - 1 and rows past N are zeros (the padded
// operand of a GEMM).  One lane per 8 columns: 4 B of codes in, 16 B out.
__global__ __launch_bounds__(256) void mx4_dequant_kernel(const uint32_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, long n0, long N, int K,
                                                          bf16_t* __restrict__ out, long ldo, long rows, int kpad) {
  const int k8 = kpad / 8;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * k8) return;
  const long r = i / k8, n = n0 + r;
  const int c8 = (int)(i - r * k8);
  bf16x8_t v = {};
  if (n < N && c8 * 8 < K) v = mx4_cvt8(codes[n * (K / 8) + c8], mx4_scale(scales[n * (K / 32) + c8 / 4]));
  *reinterpret_cast<bf16x8_t*>(out + r * ldo + c8 * 8) = v;
}

// out[m] = W[ids[m]] * scale (+ wpe[m % S]), rounded once.  An id outside [0, N) gives a row of NaN.
__global__ __launch_bounds__(256) void mx4_embed_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ codes,
                                                        const uint8_t* __restrict__ scales, long N, int K,
                                                        const bf16_t* __restrict__ wpe, bf16_t* __restrict__ out, long M,
                                                        int S, float scale) {
  const int k8 = K / 8;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * k8) return;
  const long m = i / k8, id = ids[m];
  const int c8 = (int)(i - m * k8);
  const bool ok = id >= 0 && id < N;
  const long n = ok ? id : 0;
  const bf16x8_t v = mx4_cvt8(codes[n * k8 + c8], ok ? mx4_scale(scales[n * (K / 32) + c8 / 4]) : __uint_as_float(0x7fc00000u));
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)v[j] * scale;
  if (wpe) {
    float p[8];
    load8(wpe + (m % S) * (long)K + c8 * 8, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] += p[j];
  }
  store8(out + m * K + c8 * 8, f);
}

// ------------------------------------------------------------------ y = x W^T + b, rows by rows
// A wave owns 16 output columns (rows n of W) and MT * 16 rows of x.  Per 128 columns of K a lane loads 16 B
// of codes -- one scale group -- of row n = n0 + (l & 15), columns 32 (l >> 4) .. + 31, and turns it into the
// operands of four 16x16x32 MFMAs; step t multiplies columns 32 (l >> 4) + 8 t + j, so x is read with the
// same permutation.  S waves of a workgroup share a column tile and split K; they meet in LDS.
template <int MT, int S>
__global__ __launch_bounds__(64 * (S > 4 ? S : 4)) void mx4_rows_kernel(Mx4LinearArgs g) {
  constexpr int NW = S > 4 ? S : 4, TPB = NW / S;  // waves, column tiles per workgroup
  __shared__ float red[S > 1 ? NW * MT * 256 : 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ks = w % S, r16 = lane & 15, kq = lane >> 4;
  const int n0 = (blockIdx.x * TPB + w / S) * 16, m0 = blockIdx.y * (MT * 16);
  const int n = min(n0 + r16, g.N - 1);
  const uint4* crow = reinterpret_cast<const uint4*>(g.codes + (long)n * (g.K / 2));
  const uint8_t* srow = g.scales + (long)n * (g.K / 32);
  const bf16_t* xrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xrow[i] = g.x + (long)min(m0 + i * 16 + r16, g.M - 1) * g.ldx;
  const int ng = g.K / 32;  // groups of a row; chunk c holds groups 4 c .. 4 c + 3
  f32x4_t acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = zero4();
  if (n0 < g.N) {
    for (int c = ks; c * 4 < ng; c += S) {
      const int grp = c * 4 + kq;
      const bool in = grp < ng;
      uint4 q = {0, 0, 0, 0};
      float s = 1.f;
      if (in) q = crow[grp], s = mx4_scale(srow[grp]);
      const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bf16x8_t b = mx4_cvt8(qw[t], s);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          bf16x8_t a = {};
          if (in) a = *reinterpret_cast<const bf16x8_t*>(xrow[i] + grp * 32 + t * 8);
          acc[i] = mfma16(b, a, acc[i]);  // C^T: lane holds columns n0 + 4 kq + r of row m0 + 16 i + r16
        }
      }
    }
  }
  if constexpr (S > 1) {
    f32x4_t* p = reinterpret_cast<f32x4_t*>(red) + (long)w * MT * 64 + lane;
#pragma unroll
    for (int i = 0; i < MT; ++i) p[i * 64] = acc[i];
    __syncthreads();
    if (ks != 0) return;
#pragma unroll
    for (int i = 0; i < MT; ++i)
      for (int k = 1; k < S; ++k) acc[i] += p[(k * MT + i) * 64];
  }
  if (n0 >= g.N) return;
  const int nc = n0 + 4 * kq;
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  if (g.bias)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (nc + r < g.N) bias[r] = bf2f(g.bias[nc + r]);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + i * 16 + r16;
    if (m >= g.M) continue;
    bf16_t* y = g.y + (long)m * g.ldy + nc;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (nc + r < g.N) y[r] = f2bf(acc[i][r] + bias[r]);
  }
}

// ------------------------------------------------------------------ dx = dy W
// 64 rows x 128 columns per workgroup, 32 rows n of W per step: the workgroup turns the [32, 128] codes into a
// bf16 LDS image and reads it transposed (ds_read_b64_tr_b16), dy comes straight from memory.
constexpr int kDgLd = 128 + 8;
__global__ __launch_bounds__(256) void mx4_dgrad_kernel(Mx4LinearArgs g) {
  __shared__ __attribute__((aligned(16))) bf16_t img[32 * kDgLd];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int k0 = blockIdx.x * 128, m0 = blockIdx.y * 64;
  const int pr = threadIdx.x >> 3, pc = (threadIdx.x & 7) * 16;  // this thread's 16 codes of the step's image
  const bool pin = k0 + pc < g.K;
  f32x4_t acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = zero4();
  for (int n0 = 0; n0 < g.N; n0 += 32) {
    uint2 q = {0, 0};
    float s = 1.f;
    const int n = n0 + pr;
    if (n < g.N && pin) {
      q = *reinterpret_cast<const uint2*>(g.codes + (long)n * (g.K / 2) + (k0 + pc) / 2);
      s = mx4_scale(g.scales[(long)n * (g.K / 32) + (k0 + pc) / 32]);
    }
    __syncthreads();
    *reinterpret_cast<bf16x8_t*>(img + pr * kDgLd + pc) = mx4_cvt8(q.x, s);
    *reinterpret_cast<bf16x8_t*>(img + pr * kDgLd + pc + 8) = mx4_cvt8(q.y, s);
    __syncthreads();
    const bf16x8_t b0 = frag_tr(img, kDgLd, 0, w * 32), b1 = frag_tr(img, kDgLd, 0, w * 32 + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = min(m0 + i * 16 + r16, g.M - 1);
      bf16x8_t a = {};
      if (n0 + kq * 8 < g.N) a = *reinterpret_cast<const bf16x8_t*>(g.x + (long)m * g.ldx + n0 + kq * 8);
      acc[i][0] = mfma16(b0, a, acc[i][0]);
      acc[i][1] = mfma16(b1, a, acc[i][1]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + i * 16 + r16;
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = k0 + w * 32 + j * 16 + 4 * kq;
      if (c >= g.K) continue;
      u16x4_t v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = f2bf(acc[i][j][r]);
      *reinterpret_cast<u16x4_t*>(g.y + (long)m * g.ldy + c) = v;
    }
  }
}

void check_grid(long blocks, const char* what) {
  if (blocks > 0x7fffffffL) {
    fprintf(stderr, "mft::%s: %ld workgroups exceed a grid\n", what, blocks);
    abort();
  }
}

}  // namespace

void mx4_quantize(const void* w, int w_f32, uint8_t* codes, uint8_t* scales, long N, int K, hipStream_t st) {
  const long n8 = N * (K / 8), blocks = (n8 + 255) / 256;
  if (n8 <= 0) return;
  check_grid(blocks, "mx4_quantize");
  auto k = w_f32 ? mx4_quantize_kernel<true> : mx4_quantize_kernel<false>;
  k<<<(unsigned)blocks, 256, 0, st>>>(w, reinterpret_cast<uint32_t*>(codes), scales, n8);
}

void mx4_dequantize(const uint8_t* codes, const uint8_t* scales, long n0, long N, int K, bf16_t* out, long ldo, long rows,
                    int kpad, hipStream_t st) {
  const long n = rows * (kpad / 8), blocks = (n + 255) / 256;
  if (n <= 0) return;
  check_grid(blocks, "mx4_dequantize");
  mx4_dequant_kernel<<<(unsigned)blocks, 256, 0, st>>>(reinterpret_cast<const uint32_t*>(codes), scales, n0, N, K, out, ldo,
                                                       rows, kpad);
}

void mx4_embed(const int64_t* ids, const uint8_t* codes, const uint8_t* scales, long N, int K, const bf16_t* wpe,
               bf16_t* out, long M, int S, float scale, hipStream_t st) {
  const long n = M * (K / 8), blocks = (n + 255) / 256;
  if (n <= 0) return;
  check_grid(blocks, "mx4_embed");
  mx4_embed_kernel<<<(unsigned)blocks, 256, 0, st>>>(ids, reinterpret_cast<const uint32_t*>(codes), scales, N, K, wpe, out, M,
                                                     S, scale);
}

void mx4_linear(const Mx4LinearArgs& a, hipStream_t st) {
  if (a.M <= 0 || a.N <= 0) return;
  const int tiles = (a.N + 15) / 16;
  const dim3 grid1(tiles, (a.M + 15) / 16), grid4(tiles, (a.M + 63) / 64);
  if (a.M <= 16) mx4_rows_kernel<1, 4><<<grid1, 256, 0, st>>>(a);
  else mx4_rows_kernel<4, 4><<<grid4, 256, 0, st>>>(a);
}

void mx4_dgrad(const Mx4LinearArgs& a, hipStream_t st) {
  if (a.M <= 0 || a.K <= 0) return;
  mx4_dgrad_kernel<<<dim3((a.K + 127) / 128, (a.M + 63) / 64), 256, 0, st>>>(a);
}

}  // namespace mft
