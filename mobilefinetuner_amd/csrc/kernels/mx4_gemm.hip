// Products with 4-bit weights for more than a few rows: y = x W^T + b and dx = dy W.
//
// One skeleton: a workgroup of 4 waves owns BM rows and 64 * TN columns of the result, each wave all BM rows and
// 16 * TN columns.  The activation tile goes through LDS (global_load_lds, two buffers, one barrier a step) and is
// shared by the waves; the weight is never staged in bf16: each wave turns the codes of its own columns into MFMA
// operands in registers, so a step's LDS traffic is the activation's alone.
//   y  = x W^T: the reduction runs along the codes.  A lane loads 16 B -- one scale group -- of its column's row of
//        W, 128 columns of K a step, straight from memory.
//   dx = dy W: the reduction runs across the rows of W, 64 or 128 a step.  Their codes go through LDS as they are and come
//        back transposed (ds_read_b64_tr_b4: a lane gets 16 rows of its column); every row has its own scale, so a
//        byte (two rows) is converted under both scales and the halves are picked.
// The reduction may be split over workgroups (few tiles): fp32 slabs, summed in split order by mx4_join.
// Small products are bound by a step's latency (loads to LDS, barrier, products): 512 x 2304 x 768 y 9.9 us, dx 14.9 us;
// large ones by the conversions, which share the vector unit's issue with the MFMAs: 32768 x 13824 x 1152 y 895 us
// (1166 TF), dx 999 us (1045 TF).  Through a bf16 copy and gemm4 those take 747 us (1397 TF) and 822 us (1270 TF), which
// pays from about 2e10 multiplications on (8192 x 13824 x 1152 212 / 264 us against 231 / 302 us; 1999 x 6400 x 1600 y 49
// against 52 us; 8192 x 2304 x 768 by tiles, 39 / 42 us): mx4_plan models both.
#include "common.h"
#include "kernels.h"
#include "mx4.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <type_traits>

namespace mft {

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glb_void;
typedef int i32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void glds16(const void* src, void* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((glb_void*)src, (lds_void*)lds_wave_base, 16, 0, 0);
}

// every load of this wave arrived (those to LDS included), every LDS access of it done; then the workgroup's barrier
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 64-row blocks of W in a dx step: two in the small tiles, whose steps are bound by latency (2048 x 2304 x 768 22.7 us, with
// one 26.7 us; 128 x 128 tiles lose by it: 70.7 against 68.5 us on 1999 x 6400 x 1600).  256 columns a step of y gain nothing.
template <int BM, int TN>
constexpr int kBlocks = BM * TN <= 128 ? 2 : 1;

// reduction length of a step
template <int BM, int TN, bool DG>
constexpr int kStep = DG ? 64 * kBlocks<BM, TN> : 128;

template <int BM, int TN, bool DG>
constexpr int lds_bytes() {
  constexpr int st = kStep<BM, TN, DG>;
  return 2 * (BM * st * 2 + (DG ? st * (32 * TN + 16) + st * 4 * 2 * TN : 0));
}

// Scale bytes travel as unaligned 32-bit words of four neighbouring groups, the byte taken at its use: a byte kept in
// a register across steps is masked to 8 bits by the compiler right after its load, and that waits for every load
// in flight.  NARROW: rows of fewer than four groups (K < 128), byte loads.
__device__ __forceinline__ uint32_t load_u32(const uint8_t* p) {
  uint32_t v;
  __builtin_memcpy(&v, p, 4);
  return v;
}

template <int BM, int TN, bool DG, bool PART, bool NARROW>
__global__ __launch_bounds__(256, 2) void mx4_tile_kernel(Mx4LinearArgs g, int splits) {
  constexpr int MI = BM / 16, BN = 64 * TN;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kq = lane >> 4;
  const int cols = DG ? g.K : g.N, red = DG ? g.N : g.K;  // result columns, reduction length
  // tiles in groups of 8 row tiles, column by column inside a group, neighbours on one XCD: its L2 holds the
  // group's activation rows and a strip of codes
  const int tn = (cols + BN - 1) / BN, tm = (g.M + BM - 1) / BM;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int split = bid / (tn * tm), tile = bid - split * (tn * tm);
  const int grp0 = tile / (8 * tn) * 8, gsz = min(8, tm - grp0), in_grp = tile - grp0 * tn;
  const int m0 = (grp0 + in_grp % gsz) * BM, c0 = in_grp / gsz * BN;
  constexpr int STEP = kStep<BM, TN, DG>, H = kBlocks<BM, TN>;
  const int steps = (red + STEP - 1) / STEP, per = (steps + splits - 1) / splits;
  const int s0 = split * per, s1 = min(s0 + per, steps);

  f32x4_t acc[MI][TN];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = zero4();

  // ---- the activation tile: [BM][STEP] bf16 in 16-B chunks.  Lane group kq of an operand read takes chunk 4 kq + t of
  // 16 rows (dx: 8 (t / 2) + 2 kq + t % 2, as the transposed codes come); it is stored at slot (4 t + kq) ^ swz(row).
  // The hardware serves a 16-B read 16 lanes at a time, rows 0-3 and 12-15 of one lane group with rows 4-11 of the
  // next: with kq in the slot's low bits those 16 fall into different banks (in the chunk's own order they met in
  // pairs: half of all LDS cycles).
  // Rows past M repeat the last one (never stored); chunks past the reduction's end repeat the last one and are
  // zeroed in LDS by tail() before use.
  constexpr int CPR = STEP / 8, ALOADS = BM * CPR / 256;  // chunks per row, loads per thread
  const bf16_t* abase = g.x + (long)m0 * g.ldx;
  auto swz = [](int row) { return CPR == 8 ? (row >> 1) & 7 : row & 15; };
  const int chunks = DG ? (red + 7) / 8 : red / 8;  // chunks that exist in a row
  // thread tid loads slot tid % CPR of rows tid / CPR + t * 256 / CPR, all with the same swizzle
  constexpr int RPL = 256 / CPR;
  const int arow = tid / CPR, asl = (tid % CPR) ^ swz(arow);
  const int achk = DG ? (asl >> 3) * 8 + (asl & 3) * 2 + ((asl >> 2) & 1) : (asl & 3) * 4 + (asl >> 2);
  const int mlast = g.M - 1 - m0, lda = (int)g.ldx;
  auto abuf = [&](int buf) { return reinterpret_cast<bf16_t*>(smem) + buf * (BM * STEP); };
  auto load_a = [&](int buf, int s) {
    const int ch = min(s * CPR + achk, chunks - 1) * 8;
#pragma unroll
    for (int t = 0; t < ALOADS; ++t)
      glds16(abase + (uint32_t)(__mul24(min(arow + t * RPL, mlast), lda) + ch), abuf(buf) + (t * 256 + w * 64) * 8);
  };
  auto tail = [&](int buf, int s) {  // the last step when the reduction ends inside it
    if ((s + 1) * CPR <= chunks) return;
    if (s * CPR + achk >= chunks) {
#pragma unroll
      for (int t = 0; t < ALOADS; ++t) reinterpret_cast<uint4*>(abuf(buf))[t * 256 + tid] = uint4{0, 0, 0, 0};
    }
    __syncthreads();
  };
  // T sub-steps of 32 reduction columns, each MI x TN MFMAs, in blocks of HB row tiles: while a block multiplies, the
  // next one's activation operands are read, and in a sub-step's last block the next sub-step's weight operands are
  // converted (conv(b, t)).  The scheduling barriers keep the compiler from pulling each read down to its first use.
  constexpr int HB = MI == 1 ? 1 : MI < 4 || (!DG && MI * TN == 32) ? 2 : 4, T = STEP / 32, NB = T * MI / HB;  // (128 x 256: 4 would spill)
  auto frag_a = [&](int buf, int i, int t) {
    const int row = i * 16 + r16;
    return *reinterpret_cast<const bf16x8_t*>(abuf(buf) + (row * CPR + ((t * 4 + kq) ^ swz(row))) * 8);
  };

  auto products = [&](int buf, auto&& conv) {
    bf16x8_t a[2][HB], b[2][TN];
    conv(b[0], 0);
#pragma unroll
    for (int i = 0; i < HB; ++i) a[0][i] = frag_a(buf, i, 0);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int t = k / (MI / HB), i0 = k % (MI / HB) * HB;
      if (k + 1 < NB) {
        const int tn2 = (k + 1) / (MI / HB), in2 = (k + 1) % (MI / HB) * HB;
#pragma unroll
        for (int i = 0; i < HB; ++i) a[(k + 1) & 1][i] = frag_a(buf, in2 + i, tn2);
        if (tn2 != t) conv(b[tn2 & 1], tn2);
      }
#pragma unroll
      for (int i = 0; i < HB; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i0 + i][j] = mfma16(b[t & 1][j], a[k & 1][i], acc[i0 + i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if constexpr (!DG) {
    const int ng = g.K / 32;
    const uint8_t* cb = g.codes + (long)c0 * (g.K / 2);
    const uint8_t* sbp = g.scales + (long)c0 * ng;
    const int nlast = g.N - 1 - c0, nfirst = w * TN * 16 + r16, kb = g.K / 2;
    uint4 q[TN], qn[TN];
    uint32_t sw[TN], swn[TN];
    auto load_w = [&](uint4 (&qq)[TN], uint32_t (&ss)[TN], int s) {
      const int gc = min(s * 4 + kq, ng - 1);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = min(nfirst + j * 16, nlast);
        qq[j] = *reinterpret_cast<const uint4*>(cb + (uint32_t)(__mul24(n, kb) + gc * 16));
        if constexpr (NARROW) ss[j] = sbp[(uint32_t)(__mul24(n, ng) + gc)];
        else ss[j] = load_u32(sbp + (uint32_t)(__mul24(n, ng) + min(s * 4, ng - 4)));
      }
    };
    if (s0 < s1) {
      load_w(q, sw, s0);
      load_a(0, s0);
    }
    // One step: the next one's loads go out (past the end the last step's again, never used), then 4 x MI x TN MFMAs.
    // This step's codes are claimed before them: the compiler waits for all loads in flight at the first use of one
    // to a register while others go to LDS, and that wait has to fall where nothing newer is under way.
    for (int s = s0; s < s1; ++s) {
      const int buf = (s - s0) & 1;
      arrive();
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(q[j].x), "+v"(q[j].y), "+v"(q[j].z), "+v"(q[j].w), "+v"(sw[j]));
      tail(buf, s);
      load_w(qn, swn, min(s + 1, s1 - 1));
      load_a(buf ^ 1, min(s + 1, s1 - 1));
      float sc[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) sc[j] = mx4_scale(NARROW ? sw[j] : sw[j] >> ((s * 4 + kq - min(s * 4, ng - 4)) * 8 & 31) & 255u);
      if (s * 4 + 4 > ng && s * 4 + kq >= ng) {  // lanes past the end of a row multiply zeros
#pragma unroll
        for (int j = 0; j < TN; ++j) q[j] = uint4{0, 0, 0, 0}, sc[j] = 1.f;
      }
      products(buf, [&](bf16x8_t (&b)[TN], int t) {
#pragma unroll
        for (int j = 0; j < TN; ++j) b[j] = mx4_cvt8(t == 0 ? q[j].x : t == 1 ? q[j].y : t == 2 ? q[j].z : q[j].w, sc[j]);
      });
#pragma unroll
      for (int j = 0; j < TN; ++j) q[j] = qn[j], sw[j] = swn[j];
    }
  } else {
    constexpr int CLD = BN / 2 + 16;           // bytes of a staged code row: 16 rows of 8-B reads hit different banks
    constexpr int CBT = BN / 8;                // code bytes per thread: 8, 16 or 32
    constexpr int NG = BN / 32;                // scale groups of a code row: 2, 4 or 8; its four threads share them out
    char* cbase = smem + 2 * BM * STEP * 2;
    float* sbase = reinterpret_cast<float*>(cbase + 2 * STEP * CLD);
    const int crow = tid >> 2, cseg = (tid & 3) * CBT;
    const int ng = g.K / 32;
    uint2 q[H][CBT / 8];  // the next step's, on their way to LDS
    uint32_t sw[H];
    const int sgrp = NG == 8 ? (tid & 3) * 2 : (tid & 3) % NG;  // this thread's first group of the row
    const int sfirst = NARROW ? c0 / 32 + sgrp : min(c0 / 32 + (sgrp & ~3), g.K / 32 - 4);
    auto load_c = [&](int s) {
#pragma unroll
      for (int hb = 0; hb < H; ++hb) {
        const long n = min(s * STEP + hb * 64 + crow, g.N - 1);
        const uint8_t* p = g.codes + n * (g.K / 2);
#pragma unroll
        for (int e = 0; e < CBT / 8; ++e) q[hb][e] = *reinterpret_cast<const uint2*>(p + min(c0 / 2 + cseg + e * 8, g.K / 2 - 8));
        const uint8_t* sp = g.scales + n * ng;
        if constexpr (NARROW) sw[hb] = sp[min(sfirst, ng - 1)];
        else sw[hb] = load_u32(sp + sfirst);
      }
    };
    // rows past N become zeros; columns past K are never stored
    auto put_c = [&](int buf, int s) {
#pragma unroll
      for (int hb = 0; hb < H; ++hb) {
        const int row = hb * 64 + crow;
        const bool in = s * STEP + row < g.N;
        char* cb = cbase + buf * STEP * CLD + row * CLD + cseg;
#pragma unroll
        for (int e = 0; e < CBT / 8; ++e) *reinterpret_cast<uint2*>(cb + e * 8) = in ? q[hb][e] : uint2{0, 0};
        float* sb = sbase + buf * STEP * NG + row;
#pragma unroll
        for (int e = 0; e < (NG == 8 ? 2 : 1); ++e) {
          const uint32_t byte = NARROW ? sw[hb] : sw[hb] >> ((c0 / 32 + sgrp + e - sfirst) * 8 & 31) & 255u;
          sb[(sgrp + e) * STEP] = mx4_scale(in ? byte : 127u);
        }
      }
    };
    if (s0 < s1) {
      load_c(s0);
      load_a(0, s0);
      put_c(0, s0);
    }
    for (int s = s0; s < s1; ++s) {
      const int buf = (s - s0) & 1;
      arrive();
      // (before the next loads go out: the compiler makes a transposed read wait for every load to LDS in flight)
      i32x2_t raw[H][TN];
#pragma unroll
      for (int hb = 0; hb < H; ++hb)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          raw[hb][j] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)(
              cbase + (buf * STEP + hb * 64 + lane) * CLD + (w * TN + j) * 8));
      tail(buf, s);
      load_c(min(s + 1, s1 - 1));
      load_a(buf ^ 1, min(s + 1, s1 - 1));
      const float* sl = sbase + buf * STEP * NG + kq * 16;
      products(buf, [&](bf16x8_t (&b)[TN], int t) {  // rows 64 (t / 2) + 16 kq + 8 (t % 2) + 0 .. 7 of the step
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float* p = sl + ((w * TN + j) >> 1) * STEP + (t >> 1) * 64 + (t & 1) * 8;
          b[j] = mx4_cvt8((uint32_t)raw[t >> 1][j][t & 1], *reinterpret_cast<const f32x4_t*>(p), *reinterpret_cast<const f32x4_t*>(p + 4));
        }
      });
      put_c(buf ^ 1, s + 1);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup

  // ---- store.  Lane: row i * 16 + r16, columns j * 16 + 4 kq + 0 .. 3; two column tiles are exchanged between
  // neighbouring lane groups so that a lane holds 8 columns in a row.
  const int cw = c0 + w * TN * 16;
  if constexpr (PART) {
    float* P = g.ws + (long)split * g.M * cols;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int m = m0 + i * 16 + r16, c = cw + j * 16 + 4 * kq;
        if (m >= g.M) continue;
        float* p = P + (long)m * cols + c;
        if (c + 4 <= cols) __builtin_memcpy(p, &acc[i][j], 16);
        else
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c + r < cols) p[r] = acc[i][j][r];
      }
    return;
  }
  if constexpr (TN > 1) {
    const int cofs = (kq & 1) * 16 + (kq >> 1) * 8;
#pragma unroll
    for (int j = 0; j + 1 < TN; j += 2) {
      const int c = cw + j * 16 + cofs;
      float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const bool whole = c + 8 <= cols;
      if (!DG && g.bias) {
        if (whole) load8(g.bias + c, bias);
        else
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (c + r < cols) bias[r] = bf2f(g.bias[c + r]);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = m0 + i * 16 + r16;
        float o[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][r]), __float_as_uint(acc[i][j + 1][r]), false, false);
          o[r] = __uint_as_float(sw[0]) + bias[r];
          o[4 + r] = __uint_as_float(sw[1]) + bias[4 + r];
        }
        if (m >= g.M) continue;
        bf16_t* y = g.y + (long)m * g.ldy + c;
        if (whole) store8_any(y, o);
        else
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (c + r < cols) y[r] = f2bf(o[r]);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int c = cw + j * 16 + 4 * kq;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + i * 16 + r16;
      if (m >= g.M) continue;
      f32x4_t v = acc[i][j];
      if (!DG && g.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (c + r < cols) v[r] += bf2f(g.bias[c + r]);
      }
      bf16_t* y = g.y + (long)m * g.ldy + c;
      if (c + 4 <= cols) store4_any(y, v);
      else
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (c + r < cols) y[r] = f2bf(v[r]);
    }
  }
}

// y = the sum of the slabs in split order (+ bias), rounded once; y and the slabs are contiguous, 4 values a lane
__global__ __launch_bounds__(256) void mx4_join_kernel(const float* __restrict__ ws, int splits, long n, int cols,
                                                       const bf16_t* __restrict__ bias, bf16_t* __restrict__ y) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int have = (int)min(4L, n - i);
  f32x4_t v = zero4();
  for (int s = 0; s < splits; ++s) {
    const float* p = ws + s * n + i;
    f32x4_t a = zero4();
    if (have == 4) {
      __builtin_memcpy(&a, p, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < have) a[e] = p[e];
    }
    v += a;
  }
  if (bias) {
    const int c = (int)(i % cols);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < have) v[e] += bf2f(bias[(c + e) % cols]);
  }
  if (have == 4) {
    store4_any(y + i, v);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < have) y[i + e] = f2bf(v[e]);
  }
}

// W^T in bf16: out[k, n], n < Np = N rounded up to 64 (zeros past N), 64 rows of W x 256 columns per workgroup.  The codes
// go through LDS and come back transposed, as in the dx tiles; a lane writes 16 values of one row of W^T, four lanes 128 B.
__global__ __launch_bounds__(256) void mx4_dequant_t_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            int N, int Np, int K, bf16_t* __restrict__ out) {
  constexpr int CLD = 128 + 16;
  __shared__ __attribute__((aligned(16))) char img[64 * CLD];
  __shared__ __attribute__((aligned(16))) float sc[8 * 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r16 = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 64, c0 = blockIdx.y * 256, ng = K / 32;
  const bool in = n0 + (tid >> 2) < N;
  const uint8_t* p = codes + (long)min(n0 + (tid >> 2), N - 1) * (K / 2) + c0 / 2 + (tid & 3) * 32;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (c0 + (tid & 3) * 64 + e * 32 < K)
      *reinterpret_cast<uint4*>(img + (tid >> 2) * CLD + (tid & 3) * 32 + e * 16) =
          in ? *reinterpret_cast<const uint4*>(p + e * 16) : uint4{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int id = e * 256 + tid, gi = c0 / 32 + (id & 7), n = n0 + (id >> 3);
    if (gi < ng) sc[(id & 7) * 64 + (id >> 3)] = n < N ? mx4_scale(scales[(long)n * ng + gi]) : 1.f;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const i32x2_t raw = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)(
        img + lane * CLD + (w * 4 + j) * 8));
    const float* s = sc + ((w * 4 + j) >> 1) * 64 + kq * 16;
    const int k = c0 + (w * 4 + j) * 16 + r16;
    if (k >= K) continue;
    bf16x8_t* o = reinterpret_cast<bf16x8_t*>(out + (long)k * Np + n0 + kq * 16);
    o[0] = mx4_cvt8((uint32_t)raw[0], *reinterpret_cast<const f32x4_t*>(s), *reinterpret_cast<const f32x4_t*>(s + 4));
    o[1] = mx4_cvt8((uint32_t)raw[1], *reinterpret_cast<const f32x4_t*>(s + 8), *reinterpret_cast<const f32x4_t*>(s + 12));
  }
}

template <int BM, int TN, bool DG, bool PART, bool NARROW = false>
void launch_k(const Mx4LinearArgs& a, const Mx4Plan& p, hipStream_t st) {
  constexpr int shm = lds_bytes<BM, TN, DG>();
  static const bool once = [] {
    MFT_HIP_CHECK(hipFuncSetAttribute((const void*)mx4_tile_kernel<BM, TN, DG, PART, NARROW>, hipFuncAttributeMaxDynamicSharedMemorySize, shm));
    return true;
  }();
  (void)once;
  const int cols = DG ? a.K : a.N;
  const long tiles = (long)((a.M + BM - 1) / BM) * ((cols + 64 * TN - 1) / (64 * TN)) * p.splits;
  mx4_tile_kernel<BM, TN, DG, PART, NARROW><<<(unsigned)tiles, 256, shm, st>>>(a, p.splits);
}

template <int BM, int TN>
void launch(const Mx4LinearArgs& a, const Mx4Plan& p, bool dg, hipStream_t st) {
  const bool part = p.splits > 1 || a.slabs_only;
  if (dg) {
    if (part) launch_k<BM, TN, true, true>(a, p, st);
    else launch_k<BM, TN, true, false>(a, p, st);
  } else {
    if (part) launch_k<BM, TN, false, true>(a, p, st);
    else launch_k<BM, TN, false, false>(a, p, st);
  }
}

}  // namespace

namespace {

// Modelled time of a tile shape, in us: a0 + steps of a workgroup x max(lat, workgroups per CU x thr) + workgroups per
// CU x fix (+ the join: j0 + slab bytes at jb TB/s).  lat: a step alone on its CU, bound by a load's latency; thr: a step's
// share of a busy CU; fix: a workgroup's start and stores.  Fitted to 320 products (1 to 16,384 rows, 12 weights, every
// shape and split): the shape picked costs 3 % (y) and 2 % (dx) over the best one on average, at worst 22 % and 17 %.
struct TileCost {
  int bm, tn;
  float lat, thr, fix;
};
constexpr TileCost kCostY[] = {{128, 4, 2.07f, 1.32f, 4.4f}, {128, 2, 1.27f, 0.86f, 2.5f}, {64, 4, 1.37f, 0.90f, 2.8f},
                               {64, 2, 0.87f, 0.55f, 1.7f},  {64, 1, 0.64f, 0.43f, 1.2f},  {32, 2, 0.66f, 0.41f, 1.3f},
                               {32, 1, 0.47f, 0.30f, 0.85f}, {16, 1, 0.45f, 0.26f, 0.8f}};
constexpr TileCost kCostDx[] = {{128, 4, 1.32f, 0.81f, 2.1f}, {128, 2, 0.83f, 0.49f, 1.4f}, {64, 4, 1.01f, 0.56f, 1.5f},
                                {64, 2, 1.02f, 0.74f, 0.90f}, {64, 1, 0.85f, 0.58f, 0.47f}, {32, 2, 0.81f, 0.57f, 0.38f},
                                {32, 1, 0.71f, 0.43f, 0.30f}};

}  // namespace

Mx4Plan mx4_plan(int M, int N, int K, bool dgrad, int xcols, int max_splits, bool dense) {
  if (K < 128) return Mx4Plan{64, 2, 1, 0};  // the narrow kernel
  const long cols = dgrad ? K : N, red = dgrad ? N : K;
  Mx4Plan best{};
  double best_t = 1e30;
  auto consider = [&](const TileCost& c) {
    if (M <= c.bm / 2 && c.bm > 32) return;  // (32 rows: the smallest dx tile)
    const long tiles = (M + c.bm - 1L) / c.bm * ((cols + 64 * c.tn - 1) / (64 * c.tn));
    const long step = dgrad && c.bm * c.tn > 128 ? 64 : 128, steps = (red + step - 1) / step;
    for (int s = 1; s <= max_splits; s += s < 4 ? 1 : s < 8 ? 2 : s < 16 ? 4 : 8) {
      if (s > 1 && (steps / s < 2 || tiles * s > 2048)) break;
      const double n = (double)((tiles * s + 255) / 256), per = (double)((steps + s - 1) / s);
      double t = (dgrad ? 3.6 : 3.0) + per * std::max((double)c.lat, n * c.thr) + n * c.fix;
      if (s > 1) t += (dgrad ? 3.4 : 3.2) + (double)s * M * cols * 4 / (dgrad ? 2.8e6 : 3.2e6);
      if (t < best_t) best_t = t, best = Mx4Plan{c.bm, c.tn, s, 0};
    }
  };
  if (dgrad)
    for (const TileCost& c : kCostDx) consider(c);
  else
    for (const TileCost& c : kCostY) consider(c);
  // through a bf16 copy: its writing and reading at 4.5 TB/s, then 256 x 256 tiles of gemm4 in K steps of 64 -- 1.15 us alone
  // on a CU, 1.5 us when every CU is busy -- and about 4 us per round of tiles
  if (dense && mx4_dense_supported(M, N, K, dgrad, xcols)) {
    const double tiles = (double)((M + 255L) / 256 * ((cols + 255) / 256)), rounds = std::ceil(tiles / 256), st = red / 64.0;
    const double t = 5 + (double)N * K * 2.53 / 4.5e6 + std::max(rounds * (st * 1.15 + 4), tiles / 256 * (st * 1.5 + 1));
    if (t < best_t) best = Mx4Plan{0, 0, 1, 1};
  }
  return best;
}

long mx4_plan_ws_floats(const Mx4Plan& p, int M, int N, int K, bool dgrad) {
  return p.splits > 1 ? (long)p.splits * M * (dgrad ? K : N) : 0;
}

bool mx4_dense_supported(int M, int N, int K, bool dgrad, int xcols) {
  const int Np = (N + 63) / 64 * 64;
  return dgrad ? xcols >= Np && gemm4_supported(M, K, Np, false, false) : gemm4_supported(M, N, K, false, false);
}

long mx4_dense_ws_elems(int N, int K, bool dgrad) { return (long)(dgrad ? (N + 63) / 64 * 64 : N) * K; }

void mx4_dense(const Mx4LinearArgs& a, bf16_t* w, bool dgrad, hipStream_t st) {
  GemmArgs f{};
  f.A = a.x; f.lda = a.ldx;
  f.B = w;
  f.C = a.y; f.ldc = a.ldy;
  f.M = a.M; f.alpha = 1.f;
  if (dgrad) {
    const int Np = (a.N + 63) / 64 * 64;
    mx4_dequant_t_kernel<<<dim3(Np / 64, (a.K + 255) / 256), 256, 0, st>>>(a.codes, a.scales, a.N, Np, a.K, w);
    f.ldb = Np; f.N = a.K; f.K = Np;
    gemm4x(f, GEMM_EPI_NONE, false, false, st);
  } else {
    mx4_dequantize(a.codes, a.scales, 0, a.N, a.K, w, a.K, a.N, a.K, st);
    f.ldb = a.K; f.N = a.N; f.K = a.K;
    f.bias = a.bias;
    gemm4x(f, a.bias ? GEMM_EPI_BIAS : GEMM_EPI_NONE, false, false, st);
  }
}

void mx4_tiles(const Mx4LinearArgs& a, const Mx4Plan& p, bool dgrad, hipStream_t st) {
  const int shape = p.bm * 10 + p.tn;
  if (a.K < 128) {
    if (dgrad) launch_k<64, 2, true, false, true>(a, p, st);
    else launch_k<64, 2, false, false, true>(a, p, st);
  } else if (shape == 1284) launch<128, 4>(a, p, dgrad, st);
  else if (shape == 1282) launch<128, 2>(a, p, dgrad, st);
  else if (shape == 644) launch<64, 4>(a, p, dgrad, st);
  else if (shape == 642) launch<64, 2>(a, p, dgrad, st);
  else if (shape == 641) launch<64, 1>(a, p, dgrad, st);
  else if (shape == 322) launch<32, 2>(a, p, dgrad, st);
  else if (shape == 321) launch<32, 1>(a, p, dgrad, st);
  else if (shape == 161 && !dgrad && (p.splits > 1 || a.slabs_only)) launch_k<16, 1, false, true>(a, p, st);
  else if (shape == 161 && !dgrad) launch_k<16, 1, false, false>(a, p, st);
  else {
    fprintf(stderr, "mft::mx4_tiles: no kernel for tile %d x %d\n", p.bm, 64 * p.tn);
    abort();
  }
  if (p.splits > 1 && !a.slabs_only) {
    const int cols = dgrad ? a.K : a.N;
    const long n = (long)a.M * cols;
    const bf16_t* bias = dgrad ? nullptr : a.bias;
    mx4_join_kernel<<<(unsigned)((n + 1023) / 1024), 256, 0, st>>>(a.ws, p.splits, n, cols, bias, a.y);
  }
}

}  // namespace mft
