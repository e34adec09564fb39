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
#include "mx4.h"

#include <cstdio>
#include <cstdlib>

namespace mft {

namespace {

// ------------------------------------------------------------------ quantise
// Four lanes share a group of 32 columns (8 each).  The scale: with a = max |w| = f 2^e, 1 <= f < 2, the
// byte is e + 127 - 2, one more when f > 1.75.  |w| 2^(127 - byte) is then at most 7; above 6 it saturates,
// off by at most 1 -- half a step at that size, as everywhere on the grid.  Nearest code, ties to even.
// A group that holds an infinity or a NaN gets byte 255 (it reads as NaN) and codes 0.
// Bound by memory, read once in 16- and 32-B loads, a lane's 8 columns its whole state: 262144 x 640 fp32 135 us
// (5.6 TB/s), 262144 x 1152 bf16 130 us (5.9 TB/s); 2304 x 768 is one launch, 5 us.
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
// operand of a GEMM).  One lane per 8 columns: 4 B of codes in, 16 B out.  Bound by the writes: 262144 x 640 87 us (4.9 TB/s).
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

// out[m] = W[ids[m]] * scale (+ wpe[m % S]), rounded once.  An id outside [0, N) gives a row of NaN.  Bound by the writes
// and, for ids all over the table, by rows of a few hundred bytes: 65536 x 640 20 us with the ids of text, 24 us at random.
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

// out[r, 0 : ldo] = in[r, 0 : width] and zeros, for rows of any 2-byte address and stride (ldo % 8 == 0, out aligned)
__global__ __launch_bounds__(256) void mx4_pad_rows_kernel(const bf16_t* __restrict__ in, long ldi, long rows, int width,
                                                           bf16_t* __restrict__ out, int ldo) {
  const int l8 = ldo / 8;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * l8) return;
  const long r = i / l8;
  const int c = (int)(i - r * l8) * 8;
  const bf16_t* p = in + r * ldi + c;
  u16x8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (c + 8 <= width) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < width) v[j] = p[j];
  }
  *reinterpret_cast<u16x8_t*>(out + r * ldo + c) = v;
}

// ------------------------------------------------------------------ y = x W^T + b, few rows
// A wave owns TN * 16 output columns (rows n of W) and MT * 16 rows of x.  Per 128 columns of K a lane loads 16 B
// of codes -- one scale group -- of row n = n0 + (l & 15), columns 32 (l >> 4) .. + 31, and turns it into the
// operands of four 16x16x32 MFMAs; step t multiplies columns 32 (l >> 4) + 8 t + j, so x is read with the
// same permutation.  Nothing is staged: codes and x go from memory into the operands, the loads of U such
// chunks in flight together.  S waves of a workgroup share a column tile and split K; they meet in LDS.
// Bound by a launch and one or two rounds of loads: 1 x 2304 x 768 3.2 us, 16 rows 4.2 us, 64 rows 5.5 us.
template <int MT, int TN, int S, int U>
__global__ __launch_bounds__(64 * (S > 4 ? S : 4)) void mx4_rows_kernel(Mx4LinearArgs g) {
  constexpr int NW = S > 4 ? S : 4, TPB = NW / S;  // waves, column tiles (of TN * 16) per workgroup
  __shared__ float red[S > 1 ? NW * MT * TN * 256 : 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ks = w % S, r16 = lane & 15, kq = lane >> 4;
  const int n0 = (blockIdx.x * TPB + w / S) * (16 * TN);
  const int ng = g.K / 32;  // groups of a row; chunk c holds groups 4 c .. 4 c + 3
  const uint4* crow[TN];
  const uint8_t* srow[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = min(n0 + j * 16 + r16, g.N - 1);
    crow[j] = reinterpret_cast<const uint4*>(g.codes + (long)n * (g.K / 2));
    srow[j] = g.scales + (long)n * ng;
  }
  const bf16_t* xrow[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xrow[i] = g.x + (long)min(i * 16 + r16, g.M - 1) * g.ldx;
  f32x4_t acc[MT][TN];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = zero4();
  if (n0 < g.N) {
    for (int c = ks; c * 4 < ng; c += S * U) {
      uint4 q[U][TN];
      uint32_t sb[U][TN];
      bf16x8_t a[U][MT][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // lanes past the row's end multiply zeros by zeros (their loads go to the last group)
        const int grp = (c + u * S) * 4 + kq, gc = min(grp, ng - 1);
        const bool in = grp < ng;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          q[u][j] = crow[j][gc];
          sb[u][j] = srow[j][gc];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) a[u][i][t] = *reinterpret_cast<const bf16x8_t*>(xrow[i] + gc * 32 + t * 8);
        if (!in) {
#pragma unroll
          for (int j = 0; j < TN; ++j) q[u][j] = uint4{0, 0, 0, 0}, sb[u][j] = 127;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) a[u][i][t] = bf16x8_t{};
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float s = mx4_scale(sb[u][j]);
          const uint32_t qw[4] = {q[u][j].x, q[u][j].y, q[u][j].z, q[u][j].w};
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const bf16x8_t b = mx4_cvt8(qw[t], s);
#pragma unroll
            for (int i = 0; i < MT; ++i)  // C^T: lane holds columns 16 j + 4 kq + r of row 16 i + r16
              acc[i][j] = mfma16(b, a[u][i][t], acc[i][j]);
          }
        }
      }
    }
  }
  if constexpr (S > 1) {
    // wave ks of a tile sums every S-th accumulator block over the tile's waves, in wave order, and stores it
    f32x4_t* p = reinterpret_cast<f32x4_t*>(red) + (w - ks) * (MT * TN * 64) + lane;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) p[(ks * MT * TN + i * TN + j) * 64] = acc[i][j];
    __syncthreads();
  }
  if (n0 >= g.N) return;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      f32x4_t v = acc[i][j];
      if constexpr (S > 1) {
        if ((i * TN + j) % S != ks) continue;
        const f32x4_t* p = reinterpret_cast<const f32x4_t*>(red) + (w - ks) * (MT * TN * 64) + (i * TN + j) * 64 + lane;
        v = p[0];
#pragma unroll
        for (int k = 1; k < S; ++k) v += p[k * MT * TN * 64];
      }
      const int m = i * 16 + r16, nc = n0 + j * 16 + 4 * kq;
      if (m >= g.M || nc >= g.N) continue;
      bf16_t* y = g.y + (long)m * g.ldy + nc;
      if (nc + 4 <= g.N) {
        if (g.bias) {
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += bf2f(g.bias[nc + r]);
        }
        store4_any(y, v);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (nc + r < g.N) y[r] = f2bf(v[r] + (g.bias ? bf2f(g.bias[nc + r]) : 0.f));
      }
    }
}

// ------------------------------------------------------------------ y = x W^T + b, up to 16 rows, many columns
// Streams the codes once: a wave owns 32 columns and walks K in steps of 256, a lane reading 32 B of its row (two
// scale groups: columns 256 s + 64 (l >> 4) .. + 63), so a step takes whole 128-B lines.  x sits in LDS, read with
// the same permutation; rows M .. 15 of the operand repeat row M - 1 and are never stored.  No barrier in the loop.
// 4 x 262144 x 1152: 35.7 us (4.5 TB/s of codes and scales; the same through the tiles of mx4_gemm 43 us, through mx4_rows
// 45 us).  Measured and not kept: waves that go on to further strips with x already in LDS (0.9 us more), 8 waves per SIMD
// (spills).
__global__ __launch_bounds__(256) void mx4_stream_kernel(Mx4LinearArgs g) {
  extern __shared__ __attribute__((aligned(16))) bf16_t xs[];
  constexpr int TN = 2;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kq = lane >> 4;
  const int ng = g.K / 32, kb = g.K / 2, ldxs = g.K + 8;
  const int n0 = blockIdx.x * (64 * TN) + w * (16 * TN);
  const uint8_t* cb = g.codes + (long)n0 * kb;
  const uint8_t* sb = g.scales + (long)n0 * ng;
  uint32_t co[TN], so[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = min(j * 16 + r16, max(g.N - 1 - n0, 0));
    co[j] = (uint32_t)(n * kb), so[j] = (uint32_t)(n * ng);
  }
  const bool live = n0 < g.N;  // (a wave past the last column only helps to fetch x)
  if (!live) cb = g.codes, sb = g.scales;
  struct Step {
    uint4 q[TN][2];
    uint32_t sw[TN];
  };
  auto load = [&](Step& t, int s) {
    const int g0 = s * 8 + kq * 2, c0 = min(g0, ng - 1) * 16, c1 = min(g0 + 1, ng - 1) * 16, gs = min(g0, ng - 4);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      t.q[j][0] = *reinterpret_cast<const uint4*>(cb + (co[j] + c0));
      t.q[j][1] = *reinterpret_cast<const uint4*>(cb + (co[j] + c1));
      __builtin_memcpy(&t.sw[j], sb + (so[j] + gs), 4);
    }
  };
  const int steps = (ng + 7) / 8;
  Step a, b;
  load(a, 0);
  {
    const int k8 = g.K / 8, n = g.M * k8;
    for (int i = tid; i < n; i += 256) {
      const int r = i / k8, c = i - r * k8;
      *reinterpret_cast<uint4*>(xs + r * ldxs + c * 8) = *reinterpret_cast<const uint4*>(g.x + (long)r * g.ldx + c * 8);
    }
  }
  __syncthreads();
  if (!live) return;
  const bf16_t* xr = xs + min(r16, g.M - 1) * ldxs;
  f32x4_t acc[TN] = {zero4(), zero4()};
  auto use = [&](Step& t, int s) {
    const int g0 = s * 8 + kq * 2, sh = (g0 - min(g0, ng - 4)) * 8;
    float sc[TN][2];
#pragma unroll
    for (int j = 0; j < TN; ++j) sc[j][0] = mx4_scale(t.sw[j] >> (sh & 31) & 255u), sc[j][1] = mx4_scale(t.sw[j] >> (sh + 8 & 31) & 255u);
    if (s * 8 + 8 > ng) {  // groups past the end of the row multiply zeros (their x reads repeat the last group)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (g0 + e >= ng)
#pragma unroll
          for (int j = 0; j < TN; ++j) t.q[j][e] = uint4{0, 0, 0, 0}, sc[j][e] = 1.f;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool in = s * 8 + 8 <= ng || g0 + e < ng;
      const bf16_t* xp = xr + min(g0 + e, ng - 1) * 32;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        bf16x8_t xv = *reinterpret_cast<const bf16x8_t*>(xp + u * 8);
        if (!in) xv = bf16x8_t{};
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const uint32_t c = u == 0 ? t.q[j][e].x : u == 1 ? t.q[j][e].y : u == 2 ? t.q[j][e].z : t.q[j][e].w;
          acc[j] = mfma16(mx4_cvt8(c, sc[j][e]), xv, acc[j]);
        }
      }
    }
  };
  int s = 0;
  for (; s + 1 < steps; s += 2) {
    load(b, s + 1);
    use(a, s);
    load(a, min(s + 2, steps - 1));
    use(b, s + 1);
  }
  if (s < steps) use(a, s);
  if (r16 >= g.M) return;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int nc = n0 + j * 16 + 4 * kq;
    if (nc >= g.N) continue;
    bf16_t* y = g.y + (long)r16 * g.ldy + nc;
    f32x4_t v = acc[j];
    if (nc + 4 <= g.N) {
      if (g.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += bf2f(g.bias[nc + r]);
      }
      store4_any(y, v);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (nc + r < g.N) y[r] = f2bf(v[r] + (g.bias ? bf2f(g.bias[nc + r]) : 0.f));
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

void mx4_pad_rows(const bf16_t* in, long ldi, long rows, int width, bf16_t* out, int ldo, hipStream_t st) {
  const long n = rows * (ldo / 8), blocks = (n + 255) / 256;
  if (n <= 0) return;
  check_grid(blocks, "mx4_pad_rows");
  mx4_pad_rows_kernel<<<(unsigned)blocks, 256, 0, st>>>(in, ldi, rows, width, out, ldo);
}

template <int MT, int TN, int S, int U>
static void launch_rows(const Mx4LinearArgs& a, hipStream_t st) {
  const int per = 16 * TN * (S > 4 ? 1 : 4 / S);
  mx4_rows_kernel<MT, TN, S, U><<<(a.N + per - 1) / per, 64 * (S > 4 ? S : 4), 0, st>>>(a);
}

// S: the waves that share a column tile, until tiles x S fill the SIMDs (each 1/S of K is at least one chunk)
template <int MT>
static void launch_rows_mt(const Mx4LinearArgs& a, hipStream_t st) {
  const int tiles = (a.N + 15) / 16, chunks = (a.K + 127) / 128;
  int S = 2;
  while (S < 16 && S < chunks && (long)tiles * S < 2048) S *= 2;
  constexpr int U = MT == 1 ? 2 : 1;
  switch (S) {
    case 2: launch_rows<MT, 1, 2, U>(a, st); break;
    case 4: launch_rows<MT, 1, 4, U>(a, st); break;
    case 8: launch_rows<MT, 1, 8, U>(a, st); break;
    default: launch_rows<MT, 1, 16, U>(a, st); break;
  }
}

// The kernel of a forward product of few rows: 1 mx4_rows, 2 mx4_stream, 0 the tiles of mx4_gemm.hip.  Measured (us,
// rows / stream / best tile): 1 x 2304 x 768 3.5 / 4.6 / 4.7; 4 x 13824 x 1152 7.6 / 6.2 / 7.4; 16 x 6400 x 1600 9.7 / 9.0 / 8.8;
// 16 x 1152 x 6912 12.4 / - / 9.8; 24 x 768 x 2304 7.2 / - / 8.5; 64 x 2304 x 768 6.4 / - / 7.0; 64 x 768 x 2304 12 / - / 8.9;
// 64 x 13824 x 1152 21.9 / - / 11.9.  The stream wins once its 128-column strips fill a good part of the chip; mx4_rows
// reads x once per column tile and loses when that is much, by length or by the number of tiles.
int mx4_few_rows(int M, int N, int K) {
  if (M > 64) return 0;
  if (M <= 16 && N >= 12800 && K >= 128 && (long)M * (K + 8) * 2 <= 65536) return 2;
  const int mt = (M + 15) / 16;
  if (mt == 1) return N < 12800 && M * K <= 80000 ? 1 : 0;
  return mt * K <= 5000 && N <= 8192 ? 1 : 0;
}

void mx4_rows(const Mx4LinearArgs& a, hipStream_t st) {
  if (mx4_few_rows(a.M, a.N, a.K) == 2) {
    mx4_stream_kernel<<<(a.N + 127) / 128, 256, (size_t)a.M * (a.K + 8) * 2, st>>>(a);
    return;
  }
  if (a.M <= 16) launch_rows_mt<1>(a, st);
  else if (a.M <= 32) launch_rows_mt<2>(a, st);
  else if (a.M <= 48) launch_rows_mt<3>(a, st);
  else launch_rows_mt<4>(a, st);
}

}  // namespace mft
