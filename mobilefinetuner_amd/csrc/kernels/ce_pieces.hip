// LM-head cross entropy swept in pieces of the vocabulary.
//
// One sweep, two products per piece of P columns:
//   1. the logits product with the CE_FWD epilogue: E = exp(logit - tile max) in bf16 ([M, P], the only
//      vocabulary-wide buffer), (max, sum) per row and 256-column tile, the label's logit;
//   2. ce_piece_finalize: the running row maximum M' and sum S' over the pieces so far, the factor
//      exp(M - M') that rescales what earlier pieces added, the dgrad's per-tile factors;
//   3. the gradient product A' = A exp(M - M') + sum_v exp(l_v - M') W_v in fp32.
// E is bf16 because the matrix cores multiply bf16: each softmax number is off by at most half a step (2^-8 of it).
// Maxima are held in units of log 2, m log2(e) rounded to fp32 as the epilogue rounds it: E and the sums are relative to that
// rounded number (at a logit of 1000 it is 6e-5 beside the maximum), so every factor between tiles uses it too.
// At the end, with p the label's probability and d = l_label log2(e) - M (one fma: exact where the label is the maximum),
//   loss = log S - d log 2,   dh = w (A / S - (1 - p) W_label),   w = 1 / valid rows,
// the label's own column being left out of A (its E is set to 0): a row that is sure of its label has p near 1,
// and (p - 1) W_label from a p rounded to bf16 would drown the small gradient that is left.
// A 4-bit table is turned into bf16 one piece at a time, in a workspace of P rows.
#include "common.h"
#include "kernels.h"
#include "mx4.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>

namespace mft {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// a logit in units of log 2, rounded by itself (the empty asm keeps a later subtraction from taking the product into an fma)
__device__ __forceinline__ float log2_units(float l) {
  float p = l * kLog2e;
  asm("" : "+v"(p));
  return p;
}

// a row's position inside its 256-row tile in the order the CE dgrad reads its row factors (gemm8.hip)
__device__ __forceinline__ long ratio_pos(int R) {
  const int rl = R & 255;
  return (R & ~255) + (rl >> 6) * 64 + (rl & 15) * 4 + ((rl >> 4) & 3);
}

// The running state cleared, the labels of the first piece (relative to it, -100 elsewhere), and the valid rows
// counted per workgroup (count_valid sums the counts: whole numbers, any order).
__global__ __launch_bounds__(1024) void ce_pieces_begin_kernel(const int64_t* __restrict__ labels, int M, int V, int w0,
                                                               int64_t* __restrict__ rel, float* __restrict__ run_m,
                                                               float* __restrict__ run_s, float* __restrict__ lbl,
                                                               float* __restrict__ zero, float* __restrict__ counts) {
  __shared__ float red[16];
  const int i = blockIdx.x * 1024 + threadIdx.x;
  float n = 0.f;
  if (i < M) {
    const int64_t l = labels[i];
    if (l >= 0 && l < V) n = 1.f;
    rel[i] = l >= 0 && l < w0 ? l : -100;
    run_m[i] = -INFINITY;
    run_s[i] = 0.f;
    lbl[i] = 0.f;
    zero[i] = 0.f;
  }
  n = block_sum(n, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// by a whole wave; M <= 2^24, so the sum is exact in fp32
__device__ __forceinline__ float count_valid(const float* counts, int M) {
  float n = 0.f;
  for (int i = threadIdx.x & 63; i < (M + 1023) / 1024; i += 64) n += counts[i];
  return wave_sum(n);
}

// RB rows per block.  Pass 1 (a wave per row, lanes over the piece's tiles): the piece's maximum and sum join the
// running ones.  Pass 2: ratio[t][row] = 2^(m'_{t-1} - m'_t) with m'_t = max(m_t, M' - 86): the clamp keeps every factor and
// partial sum finite in fp32, and a tile further below the maximum, weighted 2^-86, adds at most 256 x 2^-86 of its share
// -- staged through LDS so that reads run over tiles and writes over rows.
template <int RB>
__global__ __launch_bounds__(256) void ce_piece_finalize_kernel(const float2* __restrict__ stats, int M, int T, long mpad,
                                                                const int64_t* __restrict__ labels, int next0, int next_w,
                                                                int64_t* __restrict__ rel, float* __restrict__ run_m,
                                                                float* __restrict__ run_s, float* __restrict__ accscale,
                                                                bf16_t* __restrict__ E, long lde,
                                                                float* __restrict__ ratio, float* __restrict__ fin,
                                                                int nsplit, int tps) {
  __shared__ float s_mx[RB];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r0 = blockIdx.x * RB;
  for (int rr = w; rr < RB; rr += 4) {
    const int R = r0 + rr;
    if (R >= M) break;
    const float2* st = stats + (long)R * T;
    float m = -INFINITY;
    for (int t = lane; t < T; t += 64) m = fmaxf(m, log2_units(st[t].x));
    const float m0 = run_m[R];
    m = fmaxf(wave_max(m), m0);
    float s = 0.f;
    for (int t = lane; t < T; t += 64) {
      const float2 v = st[t];
      s += v.y == 0.f ? 0.f : v.y * fast_exp2(log2_units(v.x) - m);
    }
    s = wave_sum(s);
    const float back = m0 == -INFINITY ? 0.f : fast_exp2(m0 - m);
    if (fin)
      for (int sp = lane; sp < nsplit; sp += 64) {
        const int te = min((sp + 1) * tps, T) - 1;
        fin[(long)sp * M + R] = fast_exp2(fmaxf(log2_units(st[te].x), m - 86.f) - m);
      }
    if (lane == 0) {
      s_mx[rr] = m;
      run_m[R] = m;
      run_s[R] = run_s[R] * back + s;
      if (accscale) accscale[R] = back;
      const int64_t here = rel[R];
      if (E && here >= 0) E[(long)R * lde + here] = 0;
      const int64_t l = labels[R];
      rel[R] = l >= next0 && l < (int64_t)next0 + next_w ? l - next0 : -100;
    }
  }
  if (!ratio || T < 2) return;
  __shared__ float s_m[RB][65];
  __syncthreads();
  const int nrow = min(RB, M - r0);
  const int rr2 = threadIdx.x % RB, jg = threadIdx.x / RB;
  const long dst = ratio_pos(r0 + rr2);
  for (int c0 = 0; c0 < T - 1; c0 += 63) {
    const int cn = min(64, T - c0);
    for (int rr = w; rr < nrow; rr += 4)
      if (lane < cn) s_m[rr][lane] = fmaxf(log2_units(stats[(long)(r0 + rr) * T + c0 + lane].x), s_mx[rr] - 86.f);
    __syncthreads();
    if (rr2 < nrow)
      for (int j = 1 + jg; j < cn; j += 256 / RB) ratio[(long)(c0 + j) * mpad + dst] = fast_exp2(s_m[rr2][j - 1] - s_m[rr2][j]);
    __syncthreads();
  }
}

// acc = acc * accscale[row] (absent on the first piece) + the split slabs in split order
__global__ __launch_bounds__(256) void ce_piece_merge_kernel(const float* __restrict__ slab, int S, int M, int N,
                                                             const float* __restrict__ accscale, float* __restrict__ acc) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4, MN = (long)M * N;
  if (i >= MN) return;
  f32x4_t a = *reinterpret_cast<const f32x4_t*>(slab + i);
  for (int sp = 1; sp < S; ++sp) a += *reinterpret_cast<const f32x4_t*>(slab + sp * MN + i);
  if (accscale) a += *reinterpret_cast<const f32x4_t*>(acc + i) * accscale[i / N];
  *reinterpret_cast<f32x4_t*>(acc + i) = a;
}

// WPR waves per row: its loss and, with dh, its gradient.  The last piece's sum comes in here: S > 0 slabs of a split
// product (on top of acc * accscale when there were pieces before it), or acc alone.  WPR = 4 (few rows): the waves share
// the slabs out and wave 0 adds their four sums in order.
template <int WPR>
__global__ __launch_bounds__(256) void ce_pieces_rows_kernel(const float* __restrict__ run_m, const float* __restrict__ run_s,
                                                             const float* __restrict__ lbl, const int64_t* __restrict__ labels,
                                                             int M, int K, int V, const float* __restrict__ counts,
                                                             const float* __restrict__ acc, const float* __restrict__ accscale,
                                                             const float* __restrict__ slab, int S,
                                                             const bf16_t* __restrict__ W, long ldw,
                                                             const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, float* __restrict__ loss_rows,
                                                             bf16_t* __restrict__ dh) {
  __shared__ f32x4_t part[WPR > 1 ? 3 * 128 : 1];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int R = WPR > 1 ? blockIdx.x : blockIdx.x * 4 + w, ws = WPR > 1 ? w : 0;
  if (R >= M) return;
  const int64_t lab = labels[R];
  const bool valid = lab >= 0 && lab < V;
  // log S near 1 keeps the bits that a loss formed from numbers of the logits' size would drop (4e-6 at 64, 6e-5 at 1024)
  const float s = run_s[R], d = fmaf(lbl[R], kLog2e, -run_m[R]), nll = logf(s) - d * kLn2;
  if (lane == 0 && ws == 0) loss_rows[R] = valid ? nll : 0.f;
  if (!dh) return;
  const float wt = 1.f / fmaxf(count_valid(counts, M), 1.f), fa = wt / s, fl = wt * -expm1f(-nll);  // 1 - p = 1 - exp(l - lse)
  const float old = accscale ? accscale[R] : 1.f;
  for (int c0 = 0; c0 < K; c0 += 512) {
    const int c = c0 + lane * 8;
    f32x4_t a = zero4(), b = zero4();
    if (c < K && valid) {
#pragma unroll 4
      for (int sp = ws; sp < S; sp += WPR) {
        const f32x4_t* p = reinterpret_cast<const f32x4_t*>(slab + ((long)sp * M + R) * K + c);
        a += p[0];
        b += p[1];
      }
      if (acc && ws == 0) {
        const f32x4_t* p = reinterpret_cast<const f32x4_t*>(acc + (long)R * K + c);
        a += p[0] * old;
        b += p[1] * old;
      }
    }
    if constexpr (WPR > 1) {
      __syncthreads();
      if (ws) part[(ws - 1) * 128 + lane * 2] = a, part[(ws - 1) * 128 + lane * 2 + 1] = b;
      __syncthreads();
      if (ws) continue;
      for (int i = 0; i < 3; ++i) a += part[i * 128 + lane * 2], b += part[i * 128 + lane * 2 + 1];
    }
    if (c >= K) continue;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid) {
      float wl[8];
      if (W) load8(W + lab * ldw + c, wl);
      else {
        const bf16x8_t v = mx4_cvt8(*reinterpret_cast<const uint32_t*>(codes + lab * (K / 2) + c / 2), mx4_scale(scales[lab * (K / 32) + c / 32]));
#pragma unroll
        for (int j = 0; j < 8; ++j) wl[j] = (float)v[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = a[j] * fa - wl[j] * fl;
        o[4 + j] = b[j] * fa - wl[4 + j] * fl;
      }
    }
    store8(dh + (long)R * K + c, o);
  }
}

// one workgroup, fixed order: loss = sum of the rows' losses / valid rows
__global__ __launch_bounds__(1024) void ce_pieces_loss_kernel(const float* __restrict__ loss_rows, int M,
                                                              const float* __restrict__ counts, float* __restrict__ loss,
                                                              int64_t* __restrict__ n_valid) {
  __shared__ float red[16];
  float s = 0.f;
  for (int i = threadIdx.x; i < M; i += 1024) s += loss_rows[i];
  s = block_sum(s, red);
  const float n = count_valid(counts, M);
  if (threadIdx.x == 0) {
    *loss = s / fmaxf(n, 1.f);
    *n_valid = (int64_t)n;
  }
}

// ---- few rows on a 4-bit table: fp32 logits of a piece from the 4-bit tiles, these two kernels, the 4-bit gradient tiles.
// (row, 2,048 columns) per workgroup: maximum and sum of exp(l - maximum), relative to the maximum as log2_units rounds it
constexpr int kChunk = 2048;
__global__ __launch_bounds__(256) void ce_few_stats_kernel(const float* __restrict__ logits, int W,
                                                           float2* __restrict__ stats) {
  __shared__ float red[16];
  const float* l = logits + (long)blockIdx.y * W;
  const int c0 = blockIdx.x * kChunk;
  float v[kChunk / 256], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) {
    const int c = c0 + i * 256 + threadIdx.x;
    v[i] = c < W ? l[c] : -INFINITY;
    m = fmaxf(m, v[i]);
  }
  m = block_max(m, red);
  const float mb = log2_units(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kChunk / 256; ++i) s += v[i] == -INFINITY ? 0.f : fast_exp2(fmaf(v[i], kLog2e, -mb));
  s = block_sum(s, red);
  if (threadIdx.x == 0) stats[(long)blockIdx.y * gridDim.x + blockIdx.x] = float2{mb, s};
}

// The row's running maximum and sum over the pieces so far (old state -> new state, by the row's first workgroup), the
// label's logit, and with E: exp(l - maximum), 0 at the label's column and past the piece's end.
__global__ __launch_bounds__(256) void ce_few_exp_kernel(const float* __restrict__ logits, int W,
                                                         const float2* __restrict__ stats, const int64_t* __restrict__ labels,
                                                         int v0, const float* __restrict__ old_m, const float* __restrict__ old_s,
                                                         float* __restrict__ run_m, float* __restrict__ run_s,
                                                         float* __restrict__ lbl, float* __restrict__ accscale,
                                                         bf16_t* __restrict__ E, long lde) {
  __shared__ float red[16];
  const int R = blockIdx.y, C = gridDim.x;
  const float2* st = stats + (long)R * C;
  const float m0 = old_m[R];
  float m = m0;
  for (int i = threadIdx.x; i < C; i += 256) m = fmaxf(m, st[i].x);
  m = block_max(m, red);
  const long rel = labels[R] - v0;
  const float* l = logits + (long)R * W;
  if (blockIdx.x == 0) {
    float s = 0.f;
    for (int i = threadIdx.x; i < C; i += 256) s += st[i].y == 0.f ? 0.f : st[i].y * fast_exp2(st[i].x - m);
    s = block_sum(s, red);
    if (threadIdx.x == 0) {
      const float back = m0 == -INFINITY ? 0.f : fast_exp2(m0 - m);
      run_m[R] = m;
      run_s[R] = old_s[R] * back + s;
      accscale[R] = back;
      if (rel >= 0 && rel < W) lbl[R] = l[rel];
    }
  }
  if (!E) return;
  const int c0 = blockIdx.x * kChunk;
#pragma unroll
  for (int i = 0; i < kChunk / 512; ++i) {  // pairs of columns
    const int c = c0 + (i * 256 + threadIdx.x) * 2;
    if (c >= lde) continue;
    const float a = c < W && c != rel ? fast_exp2(fmaf(l[c], kLog2e, -m)) : 0.f,
                b = c + 1 < W && c + 1 != rel ? fast_exp2(fmaf(l[c + 1], kLog2e, -m)) : 0.f;
    *reinterpret_cast<uint32_t*>(E + R * lde + c) = pack_bf2(a, b);
  }
}

// rows of the operand copied with zero padding: in [rows_in, K] -> out [rows, kpad]
__global__ __launch_bounds__(256) void pad_rows_kernel(const bf16_t* __restrict__ in, long ldi, long rows_in, int K,
                                                       bf16_t* __restrict__ out, long rows, int kpad) {
  const int k8 = kpad / 8;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * k8) return;
  const long r = i / k8;
  const int c = (int)(i - r * k8) * 8;
  u16x8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (r < rows_in && c < K) v = *reinterpret_cast<const u16x8_t*>(in + r * ldi + c);
  *reinterpret_cast<u16x8_t*>(out + r * kpad + c) = v;
}

int num_cus() {
  static const int n = [] {
    int dev = 0, v = 0;
    MFT_HIP_CHECK(hipGetDevice(&dev));
    MFT_HIP_CHECK(hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev));
    return v > 0 ? v : 256;
  }();
  return n;
}

struct Layout {
  float *logits;
  float *run_m, *run_s, *lbl, *zero, *accscale, *counts, *stats, *ratio, *fin, *slab, *acc;
  int64_t* rel;
  bf16_t *E, *wb;
  long bytes;
};

struct Plan {
  int width;      // columns of a full piece, <= the padded vocabulary
  int last;       // columns of the last piece
  int n;          // pieces
  int splits;     // of a full piece's dgrad
  bool copy;      // the table's pieces pass through the bf16 workspace: a 4-bit table, C not a multiple of 64 or below 128
  bool few;       // few rows on a 4-bit table: no bf16 workspace, the 4-bit tiles
};

// Rows up to which a 4-bit table is multiplied as it is, loss and gradient in us there / through the bf16 workspace:
// 262144 x 640 1 row 83 / 349, 64 rows 138 / 351, 200 rows 341 / 380, 256 rows 414 / 381; 262144 x 1152 200 rows 449 / 560,
// 256 rows 522 / 566; 50257 x 768 64 rows 61 / 105, 200 rows 119 / 115, 256 rows 130 / 116.
constexpr int kFewRows = 192;

int up64(int x) { return (x + 63) / 64 * 64; }

// Slabs of the gradient product over w columns: K splits that hold whole 256-column tiles.  us = rounds of the 256 CUs x
// (5 + 2.1 per 64 columns) + the slabs written and read back at 4.5 TB/s, the least of it.  Product and sum at 768 channels,
// w = 50257: 512 rows 40 splits 66 (18: 91, 9: 147); 4096 rows 9 splits 405 (20: 432); 8192 rows 9 splits 815 (18: 860).
int dgrad_splits(int M, int K, int w) {
  const int nk = (w + 63) / 64, tiles = ((M + 255) / 256) * ((K + 255) / 256), cus = num_cus();
  int best = 1;
  double best_t = 1e30;
  for (int sp = 1; sp <= 64 && sp <= nk; ++sp) {
    const int kps = (nk + sp - 1) / sp;
    if (sp > 1 && (kps % 4 || (long)(sp - 1) * kps >= nk)) continue;
    const double t = (tiles * sp + cus - 1) / cus * (5 + 2.1 * kps) + (sp > 1 ? (double)sp * M * K * 8 / 4.5e6 : 0);
    if (t < best_t) best_t = t, best = sp;
  }
  return best;
}

// the slabs of a few-rows gradient product over w columns of the vocabulary (64 splits, with 32: 262144 x 640 1 row 97 us)
Mx4Plan few_plan(const CePiecesArgs& a, int w) { return mx4_plan(a.M, w, a.K, true, up64(w), 64, false); }

Plan make_plan(const CePiecesArgs& a) {
  Plan p{};
  p.width = lm_head_ce_pieces_width(a.M, a.V, a.piece);
  p.few = !a.W && a.M <= kFewRows && a.K >= 128;
  p.n = (a.V + p.width - 1) / p.width;
  p.last = a.V - (p.n - 1) * p.width;
  p.copy = !a.W || a.K != a.Kp || !gemm4_supported(a.M, p.width, a.Kp, false, false);
  p.splits = a.dh ? dgrad_splits(a.M, a.K, p.n > 1 ? p.width : up64(p.last)) : 1;
  return p;
}

// bump allocation in the workspace (base null: sizes only), 256-byte aligned
struct Bump {
  char* base;
  long o = 0;
  char* take(long bytes) {
    char* q = base ? base + o : nullptr;
    o += (bytes + 255) / 256 * 256;
    return q;
  }
  float* floats(long n) { return reinterpret_cast<float*>(take(n * 4)); }
};

Layout few_layout(const CePiecesArgs& a, const Plan& p) {
  const long M = a.M;
  Bump b{reinterpret_cast<char*>(a.ws)};
  Layout L{};
  L.run_m = b.floats(2 * M), L.run_s = b.floats(2 * M);  // old and new, by turns
  L.lbl = b.floats(M), L.zero = b.floats(M), L.accscale = b.floats(M), L.counts = b.floats((M + 1023) / 1024);
  L.rel = reinterpret_cast<int64_t*>(b.take(M * 8));
  L.stats = b.floats(2 * M * ((p.width + kChunk - 1) / kChunk));
  L.logits = b.floats(M * (long)p.width);
  if (a.dh) {
    const long S = std::max(few_plan(a, p.width).splits, few_plan(a, p.last).splits);
    L.slab = b.floats(S * M * a.K);
    L.acc = b.floats(M * a.K);
    L.E = reinterpret_cast<bf16_t*>(b.take(M * (long)p.width * 2));
  }
  L.bytes = b.o;
  return L;
}

Layout make_layout(const CePiecesArgs& a, const Plan& p) {
  const long M = a.M, T = p.width / 256, mpad = (M + 255) / 256 * 256;
  // the last piece may split otherwise than the full ones
  const long S = std::max(p.splits, a.dh ? dgrad_splits(a.M, a.K, up64(p.last)) : 1);
  Layout L{};
  if (p.few) return few_layout(a, p);
  Bump b{reinterpret_cast<char*>(a.ws)};
  auto take = [&](long bytes) { return b.take(bytes); };
  auto floats = [&](long n) { return b.floats(n); };
  L.run_m = floats(M), L.run_s = floats(M), L.lbl = floats(M), L.zero = floats(M), L.accscale = floats(M);
  L.counts = floats((M + 1023) / 1024);
  L.rel = reinterpret_cast<int64_t*>(take(M * 8));
  L.stats = floats(2 * M * T);
  if (a.dh) {
    L.ratio = floats(T * mpad);
    L.fin = floats(S * M);
    if (S > 1) L.slab = floats(S * M * a.K);
    L.acc = floats(M * a.K);
    L.E = reinterpret_cast<bf16_t*>(take(M * (long)p.width * 2));
  }
  if (p.copy) L.wb = reinterpret_cast<bf16_t*>(take((long)(p.n > 1 ? p.width : up64(p.last)) * a.Kp * 2));
  L.bytes = b.o;
  return L;
}

}  // namespace

int lm_head_ce_pieces_width(long M, int V, int piece) {
  // E [M, piece] bf16 of 2 GiB, at least 4,096 columns.  16384 x 262144 x 640 in ms by columns of a piece: 4,096 17.4,
  // 16,384 (512 MiB) 12.6, 65,536 (2 GiB) 11.5, the whole vocabulary (8 GiB) 11.5.
  M = std::max(M, 1L);
  long w = piece ? piece : std::max((2L << 30) / (2 * M) / 256 * 256, 4096L);
  // What the products address in 32 bits: 256 rows of E (2^21 columns: 1 GiB) and the statistics of all rows (8 B a tile).
  w = std::min({w, 1L << 21, 0x7fffffffL / (8 * M) * 256});
  return (int)std::min(w, (long)(V + 255) / 256 * 256);
}

long lm_head_ce_pieces_ws_bytes(const CePiecesArgs& a) {
  CePiecesArgs b = a;
  b.ws = nullptr;
  return make_layout(b, make_plan(b)).bytes;
}

void lm_head_ce_pieces(const CePiecesArgs& a, hipStream_t st) {
  if (a.M <= 0) return;
  const Plan p = make_plan(a);
  const Layout L = make_layout(a, p);
  const long mpad = (long)((a.M + 255) / 256) * 256;
  const bool grad = a.dh != nullptr;
  ce_pieces_begin_kernel<<<(a.M + 1023) / 1024, 1024, 0, st>>>(a.labels, a.M, a.V, p.n > 1 ? p.width : p.last, L.rel, L.run_m,
                                                               L.run_s, L.lbl, L.zero, L.counts);
  // rows per workgroup of the finalize: fewer while the workgroups do not fill the chip twice
  int rb = 64;
  for (; rb > 4 && (a.M + rb - 1) / rb < 2 * num_cus(); rb /= 2) {}
  int last_slabs = 0, state = 0;
  for (int i = 0; p.few && i < p.n; ++i) {
    const int v0 = i * p.width, w = i + 1 < p.n ? p.width : p.last, C = (w + kChunk - 1) / kChunk;
    Mx4LinearArgs f{};
    f.codes = a.codes + (long)v0 * (a.K / 2); f.scales = a.scales + (long)v0 * (a.K / 32);
    f.x = a.h; f.ldx = a.ldh;
    f.M = a.M; f.N = w; f.K = a.K;
    f.ws = L.logits;
    f.slabs_only = 1;
    mx4_tiles(f, mx4_plan(a.M, w, a.K, false, a.ldh, 1, false), false, st);
    ce_few_stats_kernel<<<dim3(C, a.M), 256, 0, st>>>(L.logits, w, reinterpret_cast<float2*>(L.stats));
    const long o = (long)state * a.M, n = (long)(state ^ 1) * a.M;
    state ^= 1;
    ce_few_exp_kernel<<<dim3(C, a.M), 256, 0, st>>>(L.logits, w, reinterpret_cast<const float2*>(L.stats), a.labels, v0, L.run_m + o,
                                                    L.run_s + o, L.run_m + n, L.run_s + n, L.lbl, L.accscale,
                                                    grad ? L.E : nullptr, up64(w));
    if (!grad) continue;
    f.x = L.E; f.ldx = up64(w);
    f.ws = L.slab;
    const Mx4Plan dp = few_plan(a, w);
    mx4_tiles(f, dp, true, st);
    if (i + 1 == p.n) {
      last_slabs = dp.splits;
      break;
    }
    const long n4 = (long)a.M * a.K / 4;
    ce_piece_merge_kernel<<<(unsigned)((n4 + 255) / 256), 256, 0, st>>>(L.slab, dp.splits, a.M, a.K, i ? L.accscale : nullptr, L.acc);
  }
  for (int i = 0; !p.few && i < p.n; ++i) {
    const int v0 = i * p.width, w = i + 1 < p.n ? p.width : p.last, wp = up64(w), T = (wp + 255) / 256;
    const bf16_t* W = a.W ? a.W + (long)v0 * a.ldw : nullptr;
    long ldw = a.ldw;
    if (p.copy) {
      if (a.W) {
        const long n8 = (long)wp * (a.Kp / 8);
        pad_rows_kernel<<<(unsigned)((n8 + 255) / 256), 256, 0, st>>>(W, a.ldw, w, a.K, L.wb, wp, a.Kp);
      } else {
        mx4_dequantize(a.codes, a.scales, v0, a.V, a.K, L.wb, a.Kp, wp, a.Kp, st);
      }
      W = L.wb;
      ldw = a.Kp;
    }
    GemmArgs f{};
    f.A = a.h; f.lda = a.ldh;
    f.B = W; f.ldb = ldw;
    f.C = grad ? L.E : nullptr; f.ldc = wp;
    f.M = a.M; f.N = wp; f.K = a.Kp; f.alpha = 1.f;
    f.ce_labels = L.rel; f.ce_stats = L.stats; f.ce_lbl = L.lbl; f.ce_V = w;
    f.b_rows = w;  // the table ends anywhere
    if (gemm4_supported(a.M, wp, a.Kp, false, false)) gemm4x(f, GEMM_EPI_CE_FWD, false, false, st);
    else gemm8x(f, GEMM_EPI_CE_FWD, false, false, st);
    const int S = grad ? dgrad_splits(a.M, a.K, wp) : 1;
    const int tps = S > 1 ? ((wp / 64 + S - 1) / S) / 4 : T;
    auto fk = rb == 64   ? ce_piece_finalize_kernel<64>
              : rb == 32 ? ce_piece_finalize_kernel<32>
              : rb == 16 ? ce_piece_finalize_kernel<16>
              : rb == 8  ? ce_piece_finalize_kernel<8>
                         : ce_piece_finalize_kernel<4>;
    const int next0 = v0 + w, next_w = i + 1 >= p.n ? 0 : i + 2 < p.n ? p.width : p.last;
    fk<<<(a.M + rb - 1) / rb, 256, 0, st>>>(reinterpret_cast<const float2*>(L.stats), a.M, T, mpad, a.labels, next0, next_w,
                                            L.rel, L.run_m, L.run_s, grad ? L.accscale : nullptr, grad ? L.E : nullptr, wp,
                                            L.ratio, L.fin, S, tps);
    if (!grad) continue;
    GemmArgs d{};
    d.A = L.E; d.lda = wp;
    d.B = W; d.ldb = ldw;
    d.M = a.M; d.N = a.K; d.K = wp; d.alpha = 1.f;
    d.ce_labels = L.rel; d.ce_ratio = L.ratio; d.ce_fin = L.fin; d.ce_wlab = L.zero;
    d.b_rows = w;
    if (S > 1) {
      d.ksplit = S;
      d.ws = L.slab;
      gemm8x(d, GEMM_EPI_CE_DGRAD, false, true, st);
      if (i + 1 == p.n) {
        last_slabs = S;
        break;
      }
      const long n4 = (long)a.M * a.K / 4;
      ce_piece_merge_kernel<<<(unsigned)((n4 + 255) / 256), 256, 0, st>>>(L.slab, S, a.M, a.K, i ? L.accscale : nullptr, L.acc);
    } else {
      d.ce_acc = L.acc;
      d.ce_accscale = i ? L.accscale : nullptr;
      gemm8x(d, GEMM_EPI_CE_DGRAD_ACC, false, true, st);
    }
  }
  const bool w4 = last_slabs >= 8 && a.M < 2048;
  auto rk = w4 ? ce_pieces_rows_kernel<4> : ce_pieces_rows_kernel<1>;
  rk<<<w4 ? a.M : (a.M + 3) / 4, 256, 0, st>>>(
      L.run_m + (long)state * a.M, L.run_s + (long)state * a.M, L.lbl, a.labels, a.M, a.K, a.V, L.counts, last_slabs && p.n == 1 ? nullptr : L.acc,
      last_slabs ? L.accscale : nullptr, L.slab, last_slabs, a.W, a.ldw, a.codes, a.scales, a.loss_rows, a.dh);
  ce_pieces_loss_kernel<<<1, 1024, 0, st>>>(a.loss_rows, a.M, L.counts, a.loss, a.n_valid);
}

}  // namespace mft
