// Products with 4-bit weights for more than a few rows: y = x W^T + b and dx = dy W.
//
// One skeleton: a workgroup of 4 waves owns BM rows and 64 * TN columns of the result, each wave all BM rows and
// 16 * TN columns.  The activation tile goes through LDS (global_load_lds, two buffers, one barrier a step) and is
// shared by the waves; the weight is never staged in bf16: each wave turns the codes of its own columns into MFMA
// operands in registers, so a step's LDS traffic is the activation's alone.
//   y  = x W^T: the reduction runs along the codes.  A lane loads 16 B -- one scale group -- of its column's row of
//        W, 128 columns of K a step, straight from memory.
//   dx = dy W: the reduction runs across the rows of W, 64 a step.  Their codes go through LDS as they are and come
//        back transposed (ds_read_b64_tr_b4: a lane gets 16 rows of its column); every row has its own scale, so a
//        byte (two rows) is converted under both scales and the halves are picked.
// The reduction may be split over workgroups (few tiles): fp32 slabs, summed in split order by mx4_join.
#include "common.h"
#include "kernels.h"
#include "mx4.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>

namespace mft {

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glb_void;
typedef int i32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void glds16(const void* src, void* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((glb_void*)src, (lds_void*)lds_wave_base, 16, 0, 0);
}

// every load of this wave arrived (LDS ones included), every LDS write of it done; then the workgroup's barrier
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int BM, int TN, bool DG>
constexpr int lds_bytes() {
  return DG ? 2 * (BM * 128 + 64 * (32 * TN + 16) + 64 * 4 * 2 * TN) : 2 * BM * 256;
}

template <int BM, int TN, bool DG, bool PART>
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
  constexpr int STEP = DG ? 64 : 128;
  const int steps = (red + STEP - 1) / STEP, per = (steps + splits - 1) / splits;
  const int s0 = split * per, s1 = min(s0 + per, steps);

  f32x4_t acc[MI][TN];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = zero4();

  // ---- the activation tile: [BM][STEP] bf16 in 16-B chunks.  Lane group kq of an operand read takes chunk
  // kq * (CPR / 4) + t of 16 rows; it is stored at slot (4 t + kq) ^ swz(row).  The hardware serves a 16-B read 16
  // lanes at a time, rows 0-3 and 12-15 of one lane group with rows 4-11 of the next: with kq in the slot's low bits
  // those 16 fall into different banks (in the chunk's own order they met in pairs: half of all LDS cycles).
  // Rows past M repeat the last one (never stored); chunks past the reduction's end repeat the last one and are
  // zeroed in LDS by tail() before use.
  constexpr int CPR = STEP / 8, ALOADS = BM * CPR / 256;  // chunks per row, loads per thread
  const bf16_t* abase = g.x + (long)m0 * g.ldx;
  auto swz = [](int row) { return DG ? (row >> 1) & 7 : row & 15; };
  const int chunks = DG ? (red + 7) / 8 : red / 8;  // chunks that exist in a row
  // thread tid loads slot tid % CPR of rows tid / CPR + t * 256 / CPR, all with the same swizzle
  constexpr int RPL = 256 / CPR;
  const int arow = tid / CPR, asl = (tid % CPR) ^ swz(arow), achk = (asl & 3) * (CPR / 4) + (asl >> 2);
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
  constexpr int HB = MI < 4 ? MI : 4, T = STEP / 32, NB = T * MI / HB;
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
    uint32_t sb[TN], sbn[TN];
    auto load_w = [&](uint4 (&qq)[TN], uint32_t (&ss)[TN], int s) {
      const int grp = s * 4 + kq, gc = min(grp, ng - 1);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = min(nfirst + j * 16, nlast);
        qq[j] = *reinterpret_cast<const uint4*>(cb + (uint32_t)(__mul24(n, kb) + gc * 16));
        ss[j] = sbp[(uint32_t)(__mul24(n, ng) + gc)];
      }
      if (grp >= ng) {
#pragma unroll
        for (int j = 0; j < TN; ++j) qq[j] = uint4{0, 0, 0, 0}, ss[j] = 127;
      }
    };
    // one step: the next one's loads go out (into the other registers and the other buffer; past the end the last
    // step's again, never used), then 4 x MI x TN MFMAs
    auto step = [&](int buf, int s, uint4 (&qc)[TN], uint32_t (&sc)[TN], uint4 (&qo)[TN], uint32_t (&so)[TN]) {
      arrive();
      tail(buf, s);
      load_a(buf ^ 1, min(s + 1, s1 - 1));
      load_w(qo, so, min(s + 1, s1 - 1));
      products(buf, [&](bf16x8_t (&b)[TN], int t) {
#pragma unroll
        for (int j = 0; j < TN; ++j) b[j] = mx4_cvt8(t == 0 ? qc[j].x : t == 1 ? qc[j].y : t == 2 ? qc[j].z : qc[j].w, mx4_scale(sc[j]));
      });
    };
    if (s0 < s1) {
      load_a(0, s0);
      load_w(q, sb, s0);
    }
    for (int s = s0; s < s1; s += 2) {
      step(0, s, q, sb, qn, sbn);
      if (s + 1 < s1) step(1, s + 1, qn, sbn, q, sb);
    }
  } else {
    constexpr int CLD = BN / 2 + 16;           // bytes of a staged code row: 16 rows of 8-B reads hit different banks
    constexpr int CBT = BN / 8;                // code bytes per thread: 8, 16 or 32
    constexpr int NG = BN / 32, SPT = (64 * NG + 255) / 256;
    char* cbase = smem + 2 * BM * 128;
    float* sbase = reinterpret_cast<float*>(cbase + 2 * 64 * CLD);
    const int crow = tid >> 2, cseg = (tid & 3) * CBT;
    const int ng = g.K / 32;
    uint2 q[CBT / 8];
    float sc[SPT];
    auto load_c = [&](int s) {
      const int n = s * 64 + crow;
      const uint8_t* p = g.codes + (long)min(n, g.N - 1) * (g.K / 2) + c0 / 2 + cseg;
#pragma unroll
      for (int e = 0; e < CBT / 8; ++e) {
        q[e] = uint2{0, 0};
        if (n < g.N && c0 + (cseg + e * 8) * 2 < g.K) q[e] = *reinterpret_cast<const uint2*>(p + e * 8);
      }
#pragma unroll
      for (int e = 0; e < SPT; ++e) {
        const int id = e * 256 + tid, sn = s * 64 + id / NG, gi = c0 / 32 + id % NG;
        sc[e] = 1.f;
        if (id < 64 * NG && sn < g.N && gi < ng) sc[e] = mx4_scale(g.scales[(long)sn * ng + gi]);
      }
    };
    auto put_c = [&](int buf) {
#pragma unroll
      for (int e = 0; e < CBT / 8; ++e) *reinterpret_cast<uint2*>(cbase + buf * 64 * CLD + crow * CLD + cseg + e * 8) = q[e];
#pragma unroll
      for (int e = 0; e < SPT; ++e) {
        const int id = e * 256 + tid;
        if (id < 64 * NG) sbase[buf * 64 * NG + (id % NG) * 64 + id / NG] = sc[e];
      }
    };
    if (s0 < s1) {
      load_a(0, s0);
      load_c(s0);
      put_c(0);
    }
    for (int s = s0; s < s1; ++s) {
      const int buf = (s - s0) & 1;
      arrive();
      // the codes come out of LDS before the next step's loads start: the compiler would make a transposed read
      // wait for every load to LDS in flight
      i32x2_t raw[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        raw[j] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)(
            cbase + buf * 64 * CLD + lane * CLD + (w * TN + j) * 8));
      tail(buf, s);
      load_c(min(s + 1, s1 - 1));
      load_a(buf ^ 1, min(s + 1, s1 - 1));
      const float* sl = sbase + buf * 64 * NG + kq * 16;
      products(buf, [&](bf16x8_t (&b)[TN], int h) {  // rows 16 kq + 8 h + 0 .. 7 of the step
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const float* p = sl + ((w * TN + j) >> 1) * 64 + h * 8;
          b[j] = mx4_cvt8((uint32_t)raw[j][h], *reinterpret_cast<const f32x4_t*>(p), *reinterpret_cast<const f32x4_t*>(p + 4));
        }
      });
      put_c(buf ^ 1);
    }
  }

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
        if (c + 4 <= cols && cols % 4 == 0) *reinterpret_cast<f32x4_t*>(p) = acc[i][j];
        else
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c + r < cols) p[r] = acc[i][j][r];
      }
    return;
  }
  const bool wide = TN > 1 && cols % 8 == 0 && g.ldy % 8 == 0;
  if (wide) {
    const int cofs = (kq & 1) * 16 + (kq >> 1) * 8;
#pragma unroll
    for (int j = 0; j + 1 < TN; j += 2) {
      const int c = cw + j * 16 + cofs;
      float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (!DG && g.bias && c < cols) load8(g.bias + c, bias);
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
        if (m < g.M && c < cols) store8(g.y + (long)m * g.ldy + c, o);
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
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (c + r < cols) g.y[(long)m * g.ldy + c + r] = f2bf(acc[i][j][r] + (!DG && g.bias ? bf2f(g.bias[c + r]) : 0.f));
    }
  }
}

// y = the sum of the slabs in split order (+ bias), rounded once
template <int V>
__global__ __launch_bounds__(256) void mx4_join_kernel(const float* __restrict__ ws, int splits, long M, int cols,
                                                       const bf16_t* __restrict__ bias, bf16_t* __restrict__ y, long ldy) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * V, n = M * cols;
  if (i >= n) return;
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float* p = ws + s * n + i;
    if constexpr (V == 4) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += a[e];
    } else {
      v[0] += p[0];
    }
  }
  const long m = i / cols;
  const int c = (int)(i - m * cols);
#pragma unroll
  for (int e = 0; e < V; ++e) y[m * ldy + c + e] = f2bf(v[e] + (bias ? bf2f(bias[c + e]) : 0.f));
}

template <int BM, int TN, bool DG, bool PART>
void launch_k(const Mx4LinearArgs& a, const Mx4Plan& p, hipStream_t st) {
  constexpr int shm = lds_bytes<BM, TN, DG>();
  static const bool once = [] {
    MFT_HIP_CHECK(hipFuncSetAttribute((const void*)mx4_tile_kernel<BM, TN, DG, PART>, hipFuncAttributeMaxDynamicSharedMemorySize, shm));
    return true;
  }();
  (void)once;
  const int cols = DG ? a.K : a.N;
  const long tiles = (long)((a.M + BM - 1) / BM) * ((cols + 64 * TN - 1) / (64 * TN)) * p.splits;
  mx4_tile_kernel<BM, TN, DG, PART><<<(unsigned)tiles, 256, shm, st>>>(a, p.splits);
}

template <int BM, int TN>
void launch(const Mx4LinearArgs& a, const Mx4Plan& p, bool dg, hipStream_t st) {
  if (dg) {
    if (p.splits > 1) launch_k<BM, TN, true, true>(a, p, st);
    else launch_k<BM, TN, true, false>(a, p, st);
  } else {
    if (p.splits > 1) launch_k<BM, TN, false, true>(a, p, st);
    else launch_k<BM, TN, false, false>(a, p, st);
  }
}

}  // namespace

Mx4Plan mx4_plan(int M, int N, int K, bool dgrad) {
  Mx4Plan p{};
  p.bm = 128, p.tn = 4, p.splits = 1;
  if (const char* e = getenv("MX4_PLAN")) sscanf(e, "%d,%d,%d", &p.bm, &p.tn, &p.splits);
  return p;
}

long mx4_plan_ws_floats(const Mx4Plan& p, int M, int N, int K, bool dgrad) {
  return p.splits > 1 ? (long)p.splits * M * (dgrad ? K : N) : 0;
}

void mx4_tiles(const Mx4LinearArgs& a, const Mx4Plan& p, bool dgrad, hipStream_t st) {
  if (p.bm == 128 && p.tn == 4) launch<128, 4>(a, p, dgrad, st);
  else if (p.bm == 128 && p.tn == 2) launch<128, 2>(a, p, dgrad, st);
  else if (p.bm == 64 && p.tn == 4) launch<64, 4>(a, p, dgrad, st);
  else if (p.bm == 64 && p.tn == 2) launch<64, 2>(a, p, dgrad, st);
  else if (p.bm == 64 && p.tn == 1) launch<64, 1>(a, p, dgrad, st);
  else if (p.bm == 32 && p.tn == 2) launch<32, 2>(a, p, dgrad, st);
  else if (p.bm == 32 && p.tn == 1) launch<32, 1>(a, p, dgrad, st);
  else {
    fprintf(stderr, "mft::mx4_tiles: no kernel for tile %d x %d\n", p.bm, 64 * p.tn);
    abort();
  }
  if (p.splits > 1) {
    const int cols = dgrad ? a.K : a.N;
    const long n = (long)a.M * cols;
    const bf16_t* bias = dgrad ? nullptr : a.bias;
    if (cols % 4 == 0) mx4_join_kernel<4><<<(unsigned)((n / 4 + 255) / 256), 256, 0, st>>>(a.ws, p.splits, a.M, cols, bias, a.y, a.ldy);
    else mx4_join_kernel<1><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a.ws, p.splits, a.M, cols, bias, a.y, a.ldy);
  }
}

}  // namespace mft
