// gemm4: 256 x 256 x 64 bf16 MFMA GEMM with FOUR waves (one per SIMD) and a hand-scheduled K-tile body.
//
//   C[M, N] = epi(alpha * A . B^T)        A [M, K], B [N, K], both K-contiguous ("NT")
//
// Why four waves: gemm8 (8 waves, 128 accumulator VGPRs per wave) reads 1.67x the LDS bytes per FLOP
// of a kernel whose waves own 128 x 128 output tiles, and its ping-pong barrier pairs cost ~130 cycles
// per 256-cycle MFMA cluster (profiles/r4b_gemm8_deep_ab.txt, README round-4 item 1).  Here each wave
// owns a 128 x 128 tile -- 64 blocks of 16 x 16 (v_mfma_f32_16x16x32_bf16), 256 fp32 accumulators in
// AGPRs -- so per K-tile a wave issues 128 MFMAs against 32 ds_read_b128 and 16 LDS-DMA pieces, all
// from ONE instruction stream: the fragment reads of the next k-step and the DMA of the K-tile after
// next sit in the MFMA gaps, and the MFMA pipe of a SIMD never waits for another wave's segment.
//
// The K-tile body is one inline-asm statement generated by gen_gemm4.py (gemm4_sched.h: schedule and
// the reasons for it); this file holds the addressing, the pipeline prologue and the epilogues.
//   * LDS: 2 buffers x {A image [256][64], B image [256][64]} bf16 = 128 KB.  Rows are 128 B; the
//     16-B chunk c of row r sits in slot c ^ (r & 7), applied on the SOURCE address of the LDS-DMA
//     (lane-linear destination, CDNA HIP guide §5.4 rule 21) and on the ds_read address: every
//     ds_read_b128 lane group hits 16 distinct 16-B slots (conflict-free).
//   * LDS-DMA: buffer_load_dwordx4 ... lds through range-checked descriptors (rows past M / N read as
//     out of range: no clamping, no branch), one 1-KB piece = 8 rows per wave-instruction.  Past the
//     last K-tile the descriptors have 0 records: the loads keep the counted waits uniform and move
//     no bytes.
//   * Tile order: XCD remap (T1) + 8-row groups when the output has more than 8 column tiles, so the
//     32 tiles an XCD holds at once share A and B panels in its L2.
#include <algorithm>
#include <string>

#include "mfma.h"
#include "kernels.h"
#include "kernels/gemm4_sched.h"

namespace mft {

namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t rfl(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// raw buffer descriptor (stride 0, num_records bytes): every word provably wave-uniform (T20)
__device__ __forceinline__ i32x4_t make_srd(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  i32x4_t r;
  r[0] = (int)rfl((uint32_t)a);
  r[1] = (int)(rfl((uint32_t)(a >> 32)) & 0xffffu);
  r[2] = (int)rfl(bytes);
  r[3] = 0x00020000;
  return r;
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// one 1-KB LDS-DMA piece: 64 lanes x 16 B from srd + voff + koff to LDS [m0val, m0val + 1024)
__device__ __forceinline__ void dma_piece(const i32x4_t& srd, uint32_t voff, uint32_t koff, uint32_t m0val) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(m0val), "v"(voff), "s"(srd), "s"(koff)
               : "memory");
}

}  // namespace

// ------------------------------------------------------------------ kernel
// NOMEM (diagnostic build, MFT_G4_DIAG=nomem): every descriptor has 0 records -- the same instruction
// stream and waits with no operand traffic (outputs wrong), to separate memory stalls from issue
// SCHED: the K-tile schedule variant of gemm4_sched.h (0 = product; others diagnostic, MFT_G4_DIAG)
template <int EPI, int SCHED = 0, bool NOMEM = false, int STORE = 0>
__global__ __launch_bounds__(256, 1) void gemm4_nt_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) bf16_t smem[];
  const int tiles_m = (g.M + 255) / 256, tiles_n = (g.N + 255) / 256;
  const int ntiles = tiles_m * tiles_n;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  int tm, tn;
  if (tiles_n > 8) {  // groups of 8 row tiles sweep the columns
    const int GM = 8, per = GM * tiles_n;
    const int grp = bid / per, first = grp * GM, rows = min(tiles_m - first, GM);
    const int r = bid % per;
    tm = first + r % rows;
    tn = r / rows;
  } else {
    tm = bid / tiles_n;
    tn = bid % tiles_n;
  }
  (void)ntiles;
  const int m0 = tm * 256, n0 = tn * 256;
  const int lane = threadIdx.x & 63;
  const int w = (int)rfl(threadIdx.x >> 6);
  const int wm = w >> 1, wn = w & 1;
  const int nk = g.K / 64;

  // descriptors: this tile's 256-row panels of A and B (rows past M / N are out of range)
  const uint32_t a_bytes = NOMEM ? 0u : (uint32_t)min((long)(g.M - m0) * g.lda * 2, (long)0xffffffff);
  const uint32_t b_bytes = NOMEM ? 0u : (uint32_t)min((long)(g.N - n0) * g.ldb * 2, (long)0xffffffff);
  const i32x4_t srda = make_srd(g.A + (long)m0 * g.lda, a_bytes);
  const i32x4_t srdb = make_srd(g.B + (long)n0 * g.ldb, b_bytes);
  const i32x4_t srd0 = make_srd(g.A, 0);  // zero records: past the last K-tile

  // per-lane source offsets of the 8 pieces per operand: piece j of wave w = rows 32 j + 8 w + (lane >> 3),
  // 16-B slot lane & 7 holding logical chunk (lane & 7) ^ (row & 7)
  const int rr = lane >> 3, sl = lane & 7;
  uint32_t oa[8], ob[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = 32 * j + 8 * w + rr;
    oa[j] = (uint32_t)((r * g.lda + ((sl ^ rr) << 3)) * 2);
    ob[j] = (uint32_t)((r * g.ldb + ((sl ^ rr) << 3)) * 2);
  }
  const uint32_t lds0 = rfl(lds_addr(smem));
  // fragment read bases (buffer 0): lane holds T[row0 + (l & 15)][8 * (4 ks + (l >> 4)) + j]
  const int fr = lane & 15, fg = lane >> 4;
  uint32_t ra0 = lds0 + (uint32_t)((wm * 128 + fr) * 128 + ((fg ^ (lane & 7)) << 4));
  uint32_t ra1 = lds0 + (uint32_t)((wm * 128 + fr) * 128 + (((4 + fg) ^ (lane & 7)) << 4));
  uint32_t rb0 = ra0 - (uint32_t)(wm * 128 * 128) + 32768u + (uint32_t)(wn * 128 * 128);
  uint32_t rb1 = ra1 - (uint32_t)(wm * 128 * 128) + 32768u + (uint32_t)(wn * 128 * 128);

  // ---- pipeline prologue: K-tile 0 -> buffer 0, K-tile 1 -> buffer 1; set 0 <- (0, ks 0)
  {
    const uint32_t mw = lds0 + (uint32_t)w * 1024u;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const i32x4_t& sa = t < nk ? srda : srd0;
      const i32x4_t& sb = t < nk ? srdb : srd0;
#pragma unroll
      for (int j = 0; j < 8; ++j) dma_piece(sa, oa[j], t * 128u, mw + t * 65536u + j * 4096u);
#pragma unroll
      for (int j = 0; j < 8; ++j) dma_piece(sb, ob[j], t * 128u, mw + t * 65536u + 32768u + j * 4096u);
    }
    asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
  }
  bf16x8_t fa0[8], fb0[8], fa1[8], fb1[8];
  asm volatile(
      "ds_read_b128 %0, %16 offset:0\n\tds_read_b128 %1, %16 offset:2048\n\t"
      "ds_read_b128 %2, %16 offset:4096\n\tds_read_b128 %3, %16 offset:6144\n\t"
      "ds_read_b128 %4, %16 offset:8192\n\tds_read_b128 %5, %16 offset:10240\n\t"
      "ds_read_b128 %6, %16 offset:12288\n\tds_read_b128 %7, %16 offset:14336\n\t"
      "ds_read_b128 %8, %17 offset:0\n\tds_read_b128 %9, %17 offset:2048\n\t"
      "ds_read_b128 %10, %17 offset:4096\n\tds_read_b128 %11, %17 offset:6144\n\t"
      "ds_read_b128 %12, %17 offset:8192\n\tds_read_b128 %13, %17 offset:10240\n\t"
      "ds_read_b128 %14, %17 offset:12288\n\tds_read_b128 %15, %17 offset:14336\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(fa0[0]), "=&v"(fa0[1]), "=&v"(fa0[2]), "=&v"(fa0[3]), "=&v"(fa0[4]), "=&v"(fa0[5]), "=&v"(fa0[6]),
        "=&v"(fa0[7]), "=&v"(fb0[0]), "=&v"(fb0[1]), "=&v"(fb0[2]), "=&v"(fb0[3]), "=&v"(fb0[4]), "=&v"(fb0[5]),
        "=&v"(fb0[6]), "=&v"(fb0[7])
      : "v"(ra0), "v"(rb0)
      : "memory");

  f32x4_t acc[64];
#pragma unroll
  for (int i = 0; i < 64; ++i) acc[i] = zero4();

  for (int kt = 0; kt < nk; ++kt) {
    const bool more = kt + 2 < nk;
    const i32x4_t sa = more ? srda : srd0;
    const i32x4_t sb = more ? srdb : srd0;
    const uint32_t koff = rfl((uint32_t)(kt + 2) * 128u);
    const uint32_t ldsm = lds0 + (uint32_t)(kt & 1) * 65536u + (uint32_t)w * 1024u;
#define G4_CALL(M) M(acc, fa0, fb0, fa1, fb1, ra0, ra1, rb0, rb1, oa, ob, sa, sb, koff, ldsm)
    if constexpr (SCHED == 0) G4_CALL(GEMM4_KTILE_NT);
    else if constexpr (SCHED == 1) G4_CALL(GEMM4_KTILE_NT_NODMA);
    else if constexpr (SCHED == 2) G4_CALL(GEMM4_KTILE_NT_FAST_SPREAD4);
    else if constexpr (SCHED == 3) G4_CALL(GEMM4_KTILE_NT_FAST_SPREAD2);
    else G4_CALL(GEMM4_KTILE_NT_SPREAD6);
#undef G4_CALL
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no LDS-DMA outlives the workgroup

  // ---- epilogue: block (i, j) = rows wm*128 + 16 i + (l & 15), columns wn*128 + 16 j + 4 (l >> 4) + r
  // (the MFMAs ran with B as src0: each lane holds a row).  permlane16_swap pairs blocks 2c, 2c+1 so
  // lane group g owns 8 contiguous columns {0, 16, 8, 24}[g] of the 32-column pair.
  // STORE 0: 16-B stores straight from registers (16 rows x 64 B per wave instruction); 1: through the
  // (idle) LDS, each wave's 128 x 128 bf16 tile swizzled into its own 32 KB, read back as whole 256-B
  // rows (4 rows per store instruction); 2: no stores (diagnostic)
  if constexpr (STORE == 1) asm volatile("s_barrier" ::: "memory");  // every wave's last LDS reads done
  bf16_t* const img = smem + w * 16384;
  const int cofs = (fg & 1) * 16 + (fg >> 1) * 8;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int colt = wn * 128 + c * 32 + cofs;
    const int col = n0 + colt;
    const bool col_ok = col < g.N;
    float bias_v[8];
    if constexpr (EPI == GEMM_EPI_BIAS) load8(g.bias + min(col, g.N - 8), bias_v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i * 8 + 2 * c][r]),
                                                         __float_as_uint(acc[i * 8 + 2 * c + 1][r]), false, false);
        v[r] = __uint_as_float(sw[0]);
        v[4 + r] = __uint_as_float(sw[1]);
      }
      const int rowt = i * 16 + fr;  // row inside the wave's 128-row slab
      const int row = m0 + wm * 128 + rowt;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= g.alpha;
        if constexpr (EPI == GEMM_EPI_BIAS) v[e] += bias_v[e];
      }
      if constexpr (STORE == 0) {
        if (col_ok && row < g.M) store8(reinterpret_cast<bf16_t*>(g.C) + (long)row * g.ldc + col, v);
      } else if constexpr (STORE == 1) {
        const int ch = (c * 32 + cofs) >> 3;  // 16-B chunk of the wave's 256-B row
        *reinterpret_cast<uint4*>(img + rowt * 128 + ((ch ^ (rowt & 15)) << 3)) =
            uint4{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
      } else {
        asm volatile("" ::"v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]));
      }
    }
  }
  if constexpr (STORE == 1) {
    // a wave reads back only its own image: its LDS writes retired is all the ordering needed
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int ch = lane & 15;
    const int col = n0 + wn * 128 + ch * 8;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const int rowt = k * 4 + (lane >> 4);
      const uint4 pk = *reinterpret_cast<const uint4*>(img + rowt * 128 + ((ch ^ (rowt & 15)) << 3));
      const int row = m0 + wm * 128 + rowt;
      if (row < g.M && col < g.N) *reinterpret_cast<uint4*>(reinterpret_cast<bf16_t*>(g.C) + (long)row * g.ldc + col) = pk;
    }
  }
}

// ------------------------------------------------------------------ persistent form
// One workgroup per CU walks its tiles (logical ids bl, bl + grid, ..., grouped as above) as ONE stream
// of K-tiles: the LDS-DMA of stream position G + 2 is issued during position G whatever tile it belongs
// to, so a tile's first K-tiles are already in LDS (and its first k-step in registers) when the previous
// tile's epilogue runs -- no pipeline fill per tile.  The first K-tile of a tile accumulates onto 0 (the
// *_FIRST schedules), and its barrier-B wait leaves the previous tile's epilogue stores in flight
// (vm_extra): they must be exactly Epi4<EPI>::kStores buffer stores per wave (range-checked, never
// branched around), so the counted waits stay exact.

// the tile of logical id t: XCD remap already applied to the workgroup slot; 8-row groups
__device__ __forceinline__ void tile_origin4(int t, int tiles_m, int tiles_n, int& m0, int& n0) {
  int tm, tn;
  if (tiles_n > 8) {
    const int GM = 8, per = GM * tiles_n;
    const int grp = t / per, first = grp * GM, rows = min(tiles_m - first, GM);
    const int r = t % per;
    tm = first + r % rows;
    tn = r / rows;
  } else {
    tm = t / tiles_n;
    tn = t % tiles_n;
  }
  m0 = tm * 256;
  n0 = tn * 256;
}

// the persistent kernel keeps its accumulators in literal AGPRs (block (i, j) of a wave's 8 x 8 grid of
// 16 x 16 blocks at a[4 (8 i + j) .. + 3]) and its fragments in v[128:255]: the K-tile statements name
// them directly (gemm4_sched.h, *_X), so no register allocator touches them between statements
template <int A>
__device__ __forceinline__ float accr() {
  float x;
  // ("memory": keeps the reads in program order with the epilogue's LDS / global accesses, so the
  // compiler cannot hoist all 256 of them and run out of VGPRs)
  asm volatile("v_accvgpr_read_b32 %0, a%c1" : "=v"(x) : "i"(A) : "memory");
  return x;
}

// B-image swizzle of the persistent kernel: its B fragments read rows 32 c + 4 h + 8 (q >> 2) + (q & 3)
// (q = lane & 15; fragment j = 2c + h), so that lane group g of blocks 2c and 2c + 1 holds the 8
// CONTIGUOUS columns 32 c + 8 g .. + 7 (no permlane in the epilogue); this XOR keeps those ds_read_b128
// conflict-free (searched exhaustively over linear row-bit swizzles)
__device__ __forceinline__ int swz_b(int row) { return (row & 7) ^ ((row >> 1) & 4); }

// one 16-row x 32-column piece of the epilogue: row block I, column group C (blocks 2C, 2C + 1)
template <int EPI, int I, int C>
__device__ __forceinline__ void epi4_piece(const GemmArgs& g, const __amdgpu_buffer_rsrc_t& rc, int m0r, int col, int fr,
                                          const float (&bias_v)[8], bool scale) {
  constexpr int b0 = 4 * (8 * I + 2 * C), b1 = b0 + 4;
  float v[8] = {accr<b0>(), accr<b0 + 1>(), accr<b0 + 2>(), accr<b0 + 3>(),
                accr<b1>(), accr<b1 + 1>(), accr<b1 + 2>(), accr<b1 + 3>()};
  if (scale) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= g.alpha;
  }
  if constexpr (EPI == GEMM_EPI_BIAS) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias_v[e];
  }
  const int rowt = m0r + I * 16 + fr;
  const uint32_t off = col < g.N ? (uint32_t)((rowt * g.ldc + col) * 2) : 0x7ffffff0u;
  const uint4 pk{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, pk), rc, off, 0, 0);
}

template <int EPI, int C>
__device__ __forceinline__ void epi4_cols(const GemmArgs& g, const __amdgpu_buffer_rsrc_t& rc, int m0r, int col, int fr,
                                         bool scale) {
  float bias_v[8] = {};
  if constexpr (EPI == GEMM_EPI_BIAS) load8(g.bias + min(col, g.N - 8), bias_v);
  epi4_piece<EPI, 0, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 1, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 2, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 3, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 4, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 5, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 6, C>(g, rc, m0r, col, fr, bias_v, scale);
  epi4_piece<EPI, 7, C>(g, rc, m0r, col, fr, bias_v, scale);
}

// LDS-staged epilogue (persistent kernel).  A round R covers block row R = 16 rows of the wave's 128:
// the converted fragments go to the wave's own 4 KB image in the spare LDS (two images, 8 KB per wave,
// for the two outputs of BIAS_GELU_D; 16-B chunks XOR-swizzled by row & 7: the ds_write_b128 lane
// groups and the ds_read_b128 lane groups are conflict-free) and leave as 4 stores of 4 whole 256-B
// rows each (16-rows x 64-B stores straight from registers drain ~4x slower per CU:
// profiles/r5_gemm4_persistent.txt).  Nothing of a round is held in registers past it.
// Stores per wave and tile (exact: the next tile's first wait counts them): 32, 64 with two outputs.
template <int EPI>
struct Epi4 {
  static constexpr int kStores = EPI == GEMM_EPI_BIAS_GELU_D || EPI == GEMM_EPI_GEGLU_BWD ? 64
                               : EPI == GEMM_EPI_GEGLU_FWD ? 48 : EPI == GEMM_EPI_CE_FWD ? 40 : 32;
  static constexpr bool kAux = EPI == GEMM_EPI_MUL_AUX || EPI == GEMM_EPI_DGELU || EPI == GEMM_EPI_BIAS_ADD;
  static constexpr bool kBias = EPI == GEMM_EPI_BIAS || EPI == GEMM_EPI_BIAS_GELU_D || EPI == GEMM_EPI_BIAS_ADD;
};

// the 8 accumulators of blocks (R, 2c) and (R, 2c + 1): the lane's row 16 R + (l & 15), columns
// 32 c + 8 (l >> 4) .. + 7 (permuted B rows)
template <int R, int C>
__device__ __forceinline__ void acc8(float (&v)[8]) {
  constexpr int b0 = 4 * (8 * R + 2 * C), b1 = b0 + 4;
  v[0] = accr<b0>(), v[1] = accr<b0 + 1>(), v[2] = accr<b0 + 2>(), v[3] = accr<b0 + 3>();
  v[4] = accr<b1>(), v[5] = accr<b1 + 1>(), v[6] = accr<b1 + 2>(), v[7] = accr<b1 + 3>();
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return uint4{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
}

__device__ __forceinline__ void stage_put(bf16_t* img, int rowl, int ch, const uint4& pk) {
  *reinterpret_cast<uint4*>(img + rowl * 128 + ((ch ^ (rowl & 7)) << 3)) = pk;
}

// 4 stores: the staged 16 x 128 image -> rows m0r + 16 R .., columns n0w .. of the descriptor's matrix
template <int R, int POL = 0>
__device__ __forceinline__ void stage_flush(const __amdgpu_buffer_rsrc_t& rc, long ld, int N, int m0r, int n0w,
                                            int lane, const bf16_t* img) {
  const int ch = lane & 15;
  const int col = n0w + ch * 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int rowl = 4 * k + (lane >> 4);
    const uint4 pk = *reinterpret_cast<const uint4*>(img + rowl * 128 + ((ch ^ (rowl & 7)) << 3));
    const int rowt = m0r + 16 * R + rowl;
    const uint32_t off = col < N ? (uint32_t)((rowt * ld + col) * 2) : 0x7ffffff0u;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, pk), rc, off, 0, POL);
  }
}

template <int EPI, int R, int C>
__device__ __forceinline__ void epi4_frag(const GemmArgs& g, bf16_t* img, bf16_t* img2, int fr, int fg,
                                         const u16x8_t (&bias_p)[4], const u16x8_t (&auxv)[8][4], bool scale) {
  float v[8];
  acc8<R, C>(v);
  if (scale) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= g.alpha;
  }
  if constexpr (Epi4<EPI>::kBias) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bf2f(bias_p[C][e]);
  }
  if constexpr (EPI == GEMM_EPI_MUL_AUX) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= bf2f(auxv[R][C][e]);
  }
  if constexpr (EPI == GEMM_EPI_BIAS_ADD) {  // + the residual stream (aux may alias C: loaded before any store)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bf2f(auxv[R][C][e]);
  }
  if constexpr (EPI == GEMM_EPI_DGELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= gelu_tanh_grad(bf2f(auxv[R][C][e]));
  }
  if constexpr (EPI == GEMM_EPI_BIAS_GELU_D) {
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      f32x2_t y2, d2;
      gelu_tanh_and_grad2(f32x2_t{v[e], v[e + 1]}, y2, d2);
      v[e] = y2.x, v[e + 1] = y2.y, d[e] = d2.x, d[e + 1] = d2.y;
    }
    stage_put(img2, fr, 4 * C + fg, pack8(d));
  }
  stage_put(img, fr, 4 * C + fg, pack8(v));
}

template <int EPI, int R, int POL>
__device__ __forceinline__ void epi4_round(const GemmArgs& g, const __amdgpu_buffer_rsrc_t& rc,
                                          const __amdgpu_buffer_rsrc_t& rx, int m0r, int n0w, int fr, int fg, int lane,
                                          bf16_t* img, const u16x8_t (&bias_p)[4], const u16x8_t (&auxv)[8][4],
                                          bool scale) {
  bf16_t* img2 = img + 2048;  // second 4 KB image (BIAS_GELU_D's GELU' output)
  epi4_frag<EPI, R, 0>(g, img, img2, fr, fg, bias_p, auxv, scale);
  epi4_frag<EPI, R, 1>(g, img, img2, fr, fg, bias_p, auxv, scale);
  epi4_frag<EPI, R, 2>(g, img, img2, fr, fg, bias_p, auxv, scale);
  epi4_frag<EPI, R, 3>(g, img, img2, fr, fg, bias_p, auxv, scale);
  stage_flush<R, POL>(rc, g.ldc, g.N, m0r, n0w, lane, img);
  if constexpr (EPI == GEMM_EPI_BIAS_GELU_D) stage_flush<R, POL>(rx, g.ldaux, g.N, m0r, n0w, lane, img2);
}

// ---- LM-head cross-entropy forward (CE_FWD): the semantics of gemm8's epilogue_ce_fwd (gemm8.hip) --
// per row and 256-column vocab tile the max and sum of exp(logit - max) -> ce_stats [M][T] float2, the
// label's logit -> ce_lbl [M], and (C given) E = exp(logit - tile max) in bf16 for the dgrad; the
// logits themselves are never stored.  A row's 256 tile columns sit in 4 lanes (l & 15 equal) x 32
// values of two waves (wn = 0, 1): lane reductions by permlane, the wave pair through the spare half
// of each wave's LDS staging image (maxima at [0, 128), sums at [128, 256) floats).
// Stores per wave: 32 (E) + 8 (label, out of range where the lane holds no label) [+ 2 stats, wn = 0]
// >= Epi4<CE_FWD>::kStores = 40, so the next tile's first wait stays exact or stricter.
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;  // (asm: fmaxf on MFMA results makes hipcc canonicalise every operand)
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

template <int R, int C>
__device__ __forceinline__ void ce_vals(float (&v)[8], bool full, int col, int V) {
  acc8<R, C>(v);
  if (!full) {  // padding columns -> -inf: the max ignores them and exp2 makes them 0
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = col + 32 * C + e < V ? v[e] : -INFINITY;
  }
}

template <int R>
__device__ __forceinline__ float ce_rowmax(bool full, int col, int V) {
  float a[8], b[8];
  ce_vals<R, 0>(a, full, col, V);
  ce_vals<R, 1>(b, full, col, V);
  float m = max3f(a[0], a[1], a[2]);
  m = max3f(m, a[3], a[4]), m = max3f(m, a[5], a[6]), m = max3f(m, a[7], b[0]);
  m = max3f(m, b[1], b[2]), m = max3f(m, b[3], b[4]), m = max3f(m, b[5], b[6]), m = max3f(m, b[7], m);
  ce_vals<R, 2>(a, full, col, V);
  ce_vals<R, 3>(b, full, col, V);
  m = max3f(m, a[0], a[1]), m = max3f(m, a[2], a[3]), m = max3f(m, a[4], a[5]), m = max3f(m, a[6], a[7]);
  m = max3f(m, b[0], b[1]), m = max3f(m, b[2], b[3]), m = max3f(m, b[4], b[5]), m = max3f(m, b[6], b[7]);
  m = fmaxf(m, xor16_pl(m));
  return fmaxf(m, xor32_pl(m));
}

template <int R, int C>
__device__ __forceinline__ void ce_exp_piece(f32x2_t& s, float& xl, bool& hit, bf16_t* img, int fr, int fg, bool full,
                                             int col, int V, long lab, float mb) {
  float v[8];
  ce_vals<R, C>(v, full, col, V);
  const unsigned d = (unsigned)(lab - (col + 32 * C));  // -100 (ignored) never matches
  if (__builtin_expect(d < 8u, 0)) {
    float x = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) x = d == (unsigned)e ? v[e] : x;
    xl = x;
    hit = true;
  }
#pragma unroll
  for (int e = 0; e < 8; e += 2) {  // the scale-and-shift and the running sums as pairs: two sums, of the even and the odd columns
    const f32x2_t t = __builtin_elementwise_fma(f32x2_t{v[e], v[e + 1]}, f32x2_t{1.4426950408889634f, 1.4426950408889634f},
                                                f32x2_t{-mb, -mb});
    v[e] = fast_exp2(t.x), v[e + 1] = fast_exp2(t.y);
    s += f32x2_t{v[e], v[e + 1]};
  }
  stage_put(img, fr, 4 * C + fg, pack8(v));
}

template <int R, int POL>
__device__ __forceinline__ float ce_round(const GemmArgs& g, const __amdgpu_buffer_rsrc_t& rc,
                                          const __amdgpu_buffer_rsrc_t& rl, int m0, int wm, int n0w, int fr, int fg,
                                          int lane, bf16_t* img, bool full, long lab, float mrow) {
  const int col = n0w + 8 * fg;
  const float mb = (mrow == -INFINITY ? 0.f : mrow) * 1.4426950408889634f;  // all-padding tile: no NaN
  f32x2_t s2 = {0.f, 0.f};
  float xl = 0.f;
  bool hit = false;
  ce_exp_piece<R, 0>(s2, xl, hit, img, fr, fg, full, col, g.ce_V, lab, mb);
  ce_exp_piece<R, 1>(s2, xl, hit, img, fr, fg, full, col, g.ce_V, lab, mb);
  ce_exp_piece<R, 2>(s2, xl, hit, img, fr, fg, full, col, g.ce_V, lab, mb);
  ce_exp_piece<R, 3>(s2, xl, hit, img, fr, fg, full, col, g.ce_V, lab, mb);
  float s = s2.x + s2.y;
  stage_flush<R, POL>(rc, g.ldc, g.N, wm * 128, n0w, lane, img);
  const int row = m0 + wm * 128 + 16 * R + fr;
  __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(xl), rl, hit ? (uint32_t)row * 4u : 0x7ffffff0u, 0, 0);
  s += xor16_pl(s);
  return s + xor32_pl(s);
}

template <int POL>
__device__ __forceinline__ void epi4_ce_fwd(const GemmArgs& g, const __amdgpu_buffer_rsrc_t& rc, int m0, int n0, int wm,
                                            int wn, int w, int fr, int fg, int lane, bf16_t* smem) {
  const int n0w = n0 + wn * 128, col = n0w + 8 * fg;
  const bool full = n0 + 256 <= g.ce_V;
  bf16_t* img = smem + 65536 + w * 4096;
  float* red = reinterpret_cast<float*>(img + 2048);
  const float* redp = reinterpret_cast<const float*>(smem + 65536 + (w ^ 1) * 4096 + 2048);
  long lab[8];
#pragma unroll
  for (int R = 0; R < 8; ++R) lab[R] = g.ce_labels[min(m0 + wm * 128 + 16 * R + fr, g.M - 1)];
  float mx[8];
  mx[0] = ce_rowmax<0>(full, col, g.ce_V), mx[1] = ce_rowmax<1>(full, col, g.ce_V);
  mx[2] = ce_rowmax<2>(full, col, g.ce_V), mx[3] = ce_rowmax<3>(full, col, g.ce_V);
  mx[4] = ce_rowmax<4>(full, col, g.ce_V), mx[5] = ce_rowmax<5>(full, col, g.ce_V);
  mx[6] = ce_rowmax<6>(full, col, g.ce_V), mx[7] = ce_rowmax<7>(full, col, g.ce_V);
  if (fg == 0) {
#pragma unroll
    for (int R = 0; R < 8; ++R) red[16 * R + fr] = mx[R];
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int R = 0; R < 8; ++R) mx[R] = fmaxf(mx[R], redp[16 * R + fr]);
  const __amdgpu_buffer_rsrc_t rl = __builtin_amdgcn_make_buffer_rsrc(g.ce_lbl, (short)0, (int)rfl((uint32_t)(g.M * 4)), 0x00020000);
  float sm[8];
  sm[0] = ce_round<0, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[0], mx[0]);
  sm[1] = ce_round<1, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[1], mx[1]);
  sm[2] = ce_round<2, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[2], mx[2]);
  sm[3] = ce_round<3, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[3], mx[3]);
  sm[4] = ce_round<4, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[4], mx[4]);
  sm[5] = ce_round<5, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[5], mx[5]);
  sm[6] = ce_round<6, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[6], mx[6]);
  sm[7] = ce_round<7, POL>(g, rc, rl, m0, wm, n0w, fr, fg, lane, img, full, lab[7], mx[7]);
  if (fg == 0) {
#pragma unroll
    for (int R = 0; R < 8; ++R) red[128 + 16 * R + fr] = sm[R];
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if (wn == 0) {  // the pair's 128 rows: lane -> rows lane, lane + 64
    const int T = (g.N + 255) / 256, tn = n0 >> 8;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        g.ce_stats, (short)0, (int)rfl((uint32_t)std::min((long)g.M * T * 8, 0x7fffffffL)), 0x00020000);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = lane + 64 * h;
      const float m = fmaxf(red[r], redp[r]);
      const float sum = red[128 + r] + redp[128 + r];
      const uint32_t off = (uint32_t)(((long)(m0 + wm * 128 + r) * T + tn) * 8);
      typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
      __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(m), __float_as_uint(sum)}, rs, off, 0, 0);
    }
  }
}

// ---- Gemma-3 GeGLU MLP in the epilogues (the unfused gated_fwd / gated_bwd passes over [M, 2I] are gone).
// GEGLU_FWD: a tile's B panel is 128 gate rows + the matching 128 up rows (tile_b_row), so wave (wm, 0)
// holds gate columns and wave (wm, 1) the up columns of the same 128 h columns.  Round R: both waves stage
// their 16 x 128 bf16 image (one of two alternating 4 KB images per wave) and store it to gu as usual; one
// barrier; then each wave of the pair forms h = gelu(g) u for 8 of the round's 16 rows from the two images
// (the bf16 gu values the unfused kernel read) -- 4 + 2 stores per round, 48 per tile.  The barrier of
// round R + 1 orders the partner's reads of an image before its rewrite two rounds later.
template <int R, int POL>
__device__ __forceinline__ void geglu_fwd_round(const GemmArgs& g, const __amdgpu_buffer_rsrc_t& rc,
                                               const __amdgpu_buffer_rsrc_t& rh, int wm, int wn, int w, int n0h, int fr,
                                               int fg, int lane, bf16_t* smem, bool scale) {
  constexpr int kImg = (R & 1) * 2048;
  bf16_t* mine = smem + 65536 + w * 4096 + kImg;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float v[8];
    if (c == 0) acc8<R, 0>(v);
    else if (c == 1) acc8<R, 1>(v);
    else if (c == 2) acc8<R, 2>(v);
    else acc8<R, 3>(v);
    if (scale) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= g.alpha;
    }
    stage_put(mine, fr, 4 * c + fg, pack8(v));
  }
  stage_flush<R, POL>(rc, g.ldc, g.N, wm * 128, wn * g.geglu_I + n0h, lane, mine);  // gu
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  const bf16_t* gi = smem + 65536 + (w & ~1) * 4096 + kImg;
  const bf16_t* ui = smem + 65536 + (w | 1) * 4096 + kImg;
  const int ch = lane & 15, col = n0h + ch * 8;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int rowl = 8 * wn + 4 * k + (lane >> 4);
    const u16x8_t gp = *reinterpret_cast<const u16x8_t*>(gi + rowl * 128 + ((ch ^ (rowl & 7)) << 3));
    const u16x8_t up = *reinterpret_cast<const u16x8_t*>(ui + rowl * 128 + ((ch ^ (rowl & 7)) << 3));
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = gelu_tanh(bf2f(gp[e])) * bf2f(up[e]);
    const int rowt = wm * 128 + 16 * R + rowl;
    const uint32_t off = col < g.geglu_I ? (uint32_t)((rowt * g.ldaux + col) * 2) : 0x7ffffff0u;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, pack8(h)), rh, off, 0, POL);
  }
}

// GEGLU_BWD: the accumulator is dh for 8 h columns per lane; g / u of those columns are read from gu
// (aux, columns col and I + col), dgu written to C at the same two places: two staged images, 64 stores.
template <int R, int C>
__device__ __forceinline__ void geglu_bwd_frag(const GemmArgs& g, bf16_t* img, bf16_t* img2, int fr, int fg,
                                              const u16x8_t& gv, const u16x8_t& uv, bool scale) {
  float v[8];
  acc8<R, C>(v);
  float dg[8], du[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = scale ? v[e] * g.alpha : v[e];
    float a, ag;
    gelu_tanh_and_grad(bf2f(gv[e]), a, ag);
    const float u = bf2f(uv[e]);
    dg[e] = d * u * ag;
    du[e] = d * a;
  }
  stage_put(img, fr, 4 * C + fg, pack8(dg));
  stage_put(img2, fr, 4 * C + fg, pack8(du));
}

// PDIAG (diagnostic builds, MFT_G4_PDIAG): 1 = every epilogue store out of range (issued, dropped);
// 2 = operand descriptors with 0 records (DMAs issued, no traffic); outputs wrong in both.
// 3 = the epilogue stores through the default cache policy (A/B; outputs correct).  The product stores
// are non-temporal (nt): the 256 x 256 output tiles streaming through L2 otherwise evict the operand
// rows the neighbouring tiles re-read -- 8-12 % on the GPT-2 K = 768 shapes, the LM head now ahead of
// hipBLASLt (profiles/r5_gemm4_nt_stores.txt)
// SEG2: a second K segment after the main one, C = epi(A B^T + A2 B2^T) (K2 = 64 x k columns of A2 / B2,
// own row strides): the LoRA data gradient dx = dy W + (s dy B) A as ONE GEMM -- A2 = v = s dy B
// zero-padded to 64 columns, B2 = A^T zero-padded (engine/nn.cpp) -- one more K-tile per tile instead
// of a rank-r FMA epilogue
// the epilogue's [M, N] operand is read once: non-temporal (g.aux_pol = 1, MFT_G4_AUX=plain: default policy, A/B)
__device__ __forceinline__ u16x8_t aux_load(const u16x8_t* p, int pol) {
  return pol ? *p : __builtin_nontemporal_load(p);
}

template <int EPI, int PDIAG = 0, bool SEG2 = false>
__global__ __launch_bounds__(256, 1) void gemm4p_nt_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) bf16_t smem[];
  const int tiles_m = (g.M + 255) / 256, tiles_n = (g.N + 255) / 256;
  const int ntiles = tiles_m * tiles_n;
  const int grid = gridDim.x, bl = xcd_remap(blockIdx.x, grid);
  const int n_my = (ntiles - bl + grid - 1) / grid;  // >= 1: grid <= ntiles
  const int nk = g.K / 64;                           // >= 2 (gemm4x)
  const int nkt = nk + (SEG2 ? g.K2 / 64 : 0);       // K-tiles per output tile
  if (g.stagger > 0) {  // diagnostic (MFT_G4_STAGGER): delay workgroup slot (bl / 8) % 16 by that many x stagger cycles
    for (int c = ((bl >> 3) & 15) * g.stagger; c > 0; c -= 8000) __builtin_amdgcn_s_sleep(125);
  }
  const int lane_k = threadIdx.x & 63;
  const int w = (int)rfl(threadIdx.x >> 6);
  const int wm = w >> 1, wn = w & 1;

  auto srd_a = [&](int m0) {
    return make_srd(g.A + (long)m0 * g.lda, PDIAG == 2 ? 0u : (uint32_t)min((long)(g.M - m0) * g.lda * 2, 0xffffffffL));
  };
  auto srd_b = [&](int n0) {
    if constexpr (EPI == GEMM_EPI_GEGLU_FWD)  // rows n0 / 2 .. of the gate half, the up half I rows further
      return make_srd(g.B + (long)(n0 >> 1) * g.ldb, (uint32_t)min((long)(2 * g.geglu_I - (n0 >> 1)) * g.ldb * 2, 0xffffffffL));
    const int nr = EPI == GEMM_EPI_CE_FWD && g.b_rows ? g.b_rows : g.N;
    return make_srd(g.B + (long)n0 * g.ldb, PDIAG == 2 ? 0u : (uint32_t)min((long)(nr - n0) * g.ldb * 2, 0xffffffffL));
  };
  auto srd_a2 = [&](int m0) {
    return make_srd(g.A2 + (long)m0 * g.lda2, (uint32_t)min((long)(g.M - m0) * g.lda2 * 2, 0xffffffffL));
  };
  auto srd_b2 = [&](int n0) {
    return make_srd(g.B2 + (long)n0 * g.ldb2, (uint32_t)min((long)(g.N - n0) * g.ldb2 * 2, 0xffffffffL));
  };
  const i32x4_t srd0 = make_srd(g.A, 0);

  const int rr = lane_k >> 3, sl = lane_k & 7;
  uint32_t oa[8], ob[8], oa2[8], ob2[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = 32 * j + 8 * w + rr;
    oa[j] = (uint32_t)((r * g.lda + ((sl ^ rr) << 3)) * 2);
    // (GEGLU_FWD: LDS rows 128.. of the B image come from the up half, I rows after the gate rows)
    const int rsrc = EPI == GEMM_EPI_GEGLU_FWD && r >= 128 ? r - 128 + g.geglu_I : r;
    ob[j] = (uint32_t)((rsrc * g.ldb + ((sl ^ swz_b(r)) << 3)) * 2);
    if constexpr (SEG2) {
      oa2[j] = (uint32_t)((r * g.lda2 + ((sl ^ rr) << 3)) * 2);
      ob2[j] = (uint32_t)((r * g.ldb2 + ((sl ^ swz_b(r)) << 3)) * 2);
    }
  }
  const uint32_t lds0 = rfl(lds_addr(smem));
  const int fr_k = lane_k & 15, fg_k = lane_k >> 4;
  uint32_t ra0 = lds0 + (uint32_t)((wm * 128 + fr_k) * 128 + ((fg_k ^ (lane_k & 7)) << 4));
  uint32_t ra1 = lds0 + (uint32_t)((wm * 128 + fr_k) * 128 + (((4 + fg_k) ^ (lane_k & 7)) << 4));
  uint32_t rb[4];  // (ks, h): fragment 2c + h of k-step ks at rb[2 ks + h] + 4096 c
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = wn * 128 + 4 * h + 8 * (fr_k >> 2) + (fr_k & 3);
      rb[2 * ks + h] = lds0 + 32768u + (uint32_t)(row * 128 + (((4 * ks + fg_k) ^ swz_b(row)) << 4));
    }

  // DMA target: stream position (tile di, K-tile dk) and its descriptors
  int di = 0, dk = 0, dm0 = 0, dn0 = 0;
  tile_origin4(bl, tiles_m, tiles_n, dm0, dn0);
  i32x4_t dsa = srd_a(dm0), dsb = srd_b(dn0), dsa2 = srd0, dsb2 = srd0;
  if constexpr (SEG2) dsa2 = srd_a2(dm0), dsb2 = srd_b2(dn0);
  auto d_next = [&]() {
    if (++dk == nkt) {
      dk = 0;
      if (++di < n_my) {
        tile_origin4(bl + di * grid, tiles_m, tiles_n, dm0, dn0);
        dsa = srd_a(dm0);
        dsb = srd_b(dn0);
        if constexpr (SEG2) dsa2 = srd_a2(dm0), dsb2 = srd_b2(dn0);
      }
    }
  };
  {  // prologue: stream positions 0 and 1 (nk >= 2: both in tile 0)
    const uint32_t mw = lds0 + (uint32_t)w * 1024u;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t ko = rfl((uint32_t)dk * 128u);
#pragma unroll
      for (int j = 0; j < 8; ++j) dma_piece(dsa, oa[j], ko, mw + t * 65536u + j * 4096u);
#pragma unroll
      for (int j = 0; j < 8; ++j) dma_piece(dsb, ob[j], ko, mw + t * 65536u + 32768u + j * 4096u);
      d_next();
    }
    asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
  }

  int G = 0;
  for (int i = 0; i < n_my; ++i) {
    int m0, n0;
    tile_origin4(bl + i * grid, tiles_m, tiles_n, m0, n0);
    GEMM4_SET0_READ_X(ra0, rb);  // the tile's first k-step (its K-tile landed behind the last barrier B)
    for (int kt = 0; kt < nkt; ++kt, ++G) {
      const bool ok = di < n_my;
      const uint32_t mode = rfl(kt > 0 ? 0u : i == 0 ? 1u : 2u);
      const uint32_t ldsm = lds0 + (uint32_t)(G & 1) * 65536u + (uint32_t)w * 1024u;
      if constexpr (SEG2) {  // the DMA position (2 K-tiles ahead) may be in the second segment
        const bool s2 = dk >= nk;
        const i32x4_t sa = ok ? (s2 ? dsa2 : dsa) : srd0;
        const i32x4_t sb = ok ? (s2 ? dsb2 : dsb) : srd0;
        const uint32_t koff = rfl((uint32_t)(s2 ? dk - nk : dk) * 128u);
        uint32_t oas[8], obs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) oas[j] = s2 ? oa2[j] : oa[j], obs[j] = s2 ? ob2[j] : ob[j];
        if constexpr (Epi4<EPI>::kStores == 64) GEMM4_KTILE_V2_X64(ra0, ra1, rb, oas, obs, sa, sb, koff, ldsm, mode);
        else GEMM4_KTILE_V2_X32(ra0, ra1, rb, oas, obs, sa, sb, koff, ldsm, mode);
      } else {
        const i32x4_t sa = ok ? dsa : srd0;
        const i32x4_t sb = ok ? dsb : srd0;
        const uint32_t koff = rfl((uint32_t)dk * 128u);
        if constexpr (Epi4<EPI>::kStores == 64) GEMM4_KTILE_V2_X64(ra0, ra1, rb, oa, ob, sa, sb, koff, ldsm, mode);
        else if constexpr (Epi4<EPI>::kStores == 48) GEMM4_KTILE_V2_X48(ra0, ra1, rb, oa, ob, sa, sb, koff, ldsm, mode);
        else if constexpr (Epi4<EPI>::kStores == 40) GEMM4_KTILE_V2_X40(ra0, ra1, rb, oa, ob, sa, sb, koff, ldsm, mode);
        else GEMM4_KTILE_V2_X32(ra0, ra1, rb, oa, ob, sa, sb, koff, ldsm, mode);
      }
      d_next();
    }
    // the epilogue's addresses are computed here, not hoisted above the K-loop (where they would stay
    // live across the asm bodies in the 128 compiler-owned VGPRs and spill)
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // last MFMA -> v_accvgpr_read
    asm volatile("" : "+s"(m0), "+s"(n0));
    int fr = fr_k, fg = fg_k, lane = lane_k;  // (lane indices laundered for the same reason)
    asm volatile("" : "+v"(fr), "+v"(fg), "+v"(lane));
    // ---- epilogue of tile i: exactly Epi4<EPI>::kStores range-checked buffer stores per wave
    const long rows = min(g.M - m0, 256);
    const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<bf16_t*>(g.C) + (long)m0 * g.ldc, (short)0,
        PDIAG == 1 || !g.C ? 0 : (int)rfl((uint32_t)(rows * g.ldc * 2)), 0x00020000);
    const bool scale = g.alpha != 1.f;
    if constexpr (EPI == GEMM_EPI_CE_FWD) {
      epi4_ce_fwd<PDIAG == 3 ? 0 : 2>(g, rc, m0, n0, wm, wn, w, fr, fg, lane, smem);
      continue;
    }
    if constexpr (EPI == GEMM_EPI_GEGLU_FWD) {
      const __amdgpu_buffer_rsrc_t rh = __builtin_amdgcn_make_buffer_rsrc(
          g.aux + (long)m0 * g.ldaux, (short)0, PDIAG == 1 ? 0 : (int)rfl((uint32_t)(rows * g.ldaux * 2)), 0x00020000);
      const int n0h = n0 >> 1;
      geglu_fwd_round<0, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<1, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<2, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<3, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<4, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<5, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<6, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      geglu_fwd_round<7, 2>(g, rc, rh, wm, wn, w, n0h, fr, fg, lane, smem, scale);
      // (the last round's images are read by the partner before this wave's next epilogue rewrites them:
      // the next tile's K-tile barriers order it)
      continue;
    }
    if constexpr (EPI == GEMM_EPI_GEGLU_BWD) {
      const int n0w = n0 + wn * 128;
      bf16_t* img = smem + 65536 + w * 4096;
      bf16_t* img2 = img + 2048;
      // g / u fragments of a round: rows 16 R + fr, columns n0w + 32 c + 8 fg (+ I for u); one round ahead
      // (two ahead held 96 VGPRs and spilled)
      u16x8_t gq[2][4], uq[2][4];
      auto load_gu = [&](int r, int slot) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const long row = min(m0 + wm * 128 + 16 * r + fr, g.M - 1);
          const bf16_t* p = g.aux + row * g.ldaux + min(n0w + 32 * c + 8 * fg, g.N - 8);
          gq[slot][c] = aux_load(reinterpret_cast<const u16x8_t*>(p), g.aux_pol);
          uq[slot][c] = aux_load(reinterpret_cast<const u16x8_t*>(p + g.geglu_I), g.aux_pol);
        }
      };
      load_gu(0, 0);
#define G4_GEGLU_BWD_ROUND(R)                                                                   \
      {                                                                                         \
        if (R + 1 < 8) load_gu(R + 1, (R + 1) % 2);                                             \
        geglu_bwd_frag<R, 0>(g, img, img2, fr, fg, gq[R % 2][0], uq[R % 2][0], scale);          \
        geglu_bwd_frag<R, 1>(g, img, img2, fr, fg, gq[R % 2][1], uq[R % 2][1], scale);          \
        geglu_bwd_frag<R, 2>(g, img, img2, fr, fg, gq[R % 2][2], uq[R % 2][2], scale);          \
        geglu_bwd_frag<R, 3>(g, img, img2, fr, fg, gq[R % 2][3], uq[R % 2][3], scale);          \
        stage_flush<R, PDIAG == 3 ? 0 : 2>(rc, g.ldc, g.geglu_I, wm * 128, n0w, lane, img);  /* dg: cols < I */ \
        stage_flush<R, PDIAG == 3 ? 0 : 2>(rc, g.ldc, 2 * g.geglu_I, wm * 128, g.geglu_I + n0w, lane, img2); \
      }
      G4_GEGLU_BWD_ROUND(0) G4_GEGLU_BWD_ROUND(1) G4_GEGLU_BWD_ROUND(2) G4_GEGLU_BWD_ROUND(3)
      G4_GEGLU_BWD_ROUND(4) G4_GEGLU_BWD_ROUND(5) G4_GEGLU_BWD_ROUND(6) G4_GEGLU_BWD_ROUND(7)
#undef G4_GEGLU_BWD_ROUND
      continue;
    }
    if constexpr (EPI == GEMM_EPI_NONE || EPI == GEMM_EPI_BIAS) {
      if (g.ntail_full) {  // MFT_G4_EPI=reg: 16-B stores straight from registers (A/B)
        const int colw = n0 + wn * 128 + 8 * fg;
        epi4_cols<EPI, 0>(g, rc, wm * 128, colw, fr, scale);
        epi4_cols<EPI, 1>(g, rc, wm * 128, colw + 32, fr, scale);
        epi4_cols<EPI, 2>(g, rc, wm * 128, colw + 64, fr, scale);
        epi4_cols<EPI, 3>(g, rc, wm * 128, colw + 96, fr, scale);
        continue;
      }
    }
    {
      const int n0w = n0 + wn * 128;
      u16x8_t bias_p[4] = {};
      if constexpr (Epi4<EPI>::kBias) {
#pragma unroll
        for (int c = 0; c < 4; ++c) bias_p[c] = *reinterpret_cast<const u16x8_t*>(g.bias + min(n0w + 32 * c + 8 * fg, g.N - 8));
      }
      // [M, N] epilogue operand: a rolling prefetch three rounds deep (rounds 0-2 up front, round R + 3 after
      // round R; all 32 fragments at once held 128 VGPRs and spilled ~19 to scratch).  A round's loads never follow
      // a store of its own rows, so an aux that aliases C (the in-place residual) is read before written.
      u16x8_t auxv[8][4] = {};
      auto load_aux = [&](int r0, int r1) {
        if constexpr (Epi4<EPI>::kAux) {
#pragma unroll
          for (int r = r0; r < r1; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int row = min(m0 + wm * 128 + 16 * r + fr, g.M - 1);
              auxv[r][c] = aux_load(reinterpret_cast<const u16x8_t*>(g.aux + (long)row * g.ldaux + min(n0w + 32 * c + 8 * fg, g.N - 8)), g.aux_pol);
            }
        }
      };
      load_aux(0, 3);
      __amdgpu_buffer_rsrc_t rx = rc;
      if constexpr (EPI == GEMM_EPI_BIAS_GELU_D)
        rx = __builtin_amdgcn_make_buffer_rsrc(g.aux + (long)m0 * g.ldaux, (short)0,
                                               PDIAG == 1 ? 0 : (int)rfl((uint32_t)(rows * g.ldaux * 2)), 0x00020000);
      bf16_t* img = smem + 65536 + w * 4096;  // bytes [128 KB + 8 KB w, + 8 KB): two 4 KB images
      epi4_round<EPI, 0, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      load_aux(3, 4);
      epi4_round<EPI, 1, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      load_aux(4, 5);
      epi4_round<EPI, 2, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      load_aux(5, 6);
      epi4_round<EPI, 3, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      load_aux(6, 7);
      epi4_round<EPI, 4, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      load_aux(7, 8);
      epi4_round<EPI, 5, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      epi4_round<EPI, 6, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
      epi4_round<EPI, 7, PDIAG == 3 ? 0 : 2>(g, rc, rx, wm * 128, n0w, fr, fg, lane, img, bias_p, auxv, scale);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ------------------------------------------------------------------ TN weight gradient
// C[M, N] (+)= alpha A^T B summed over K tokens, A = dy stored [K, M] (lda), B = x stored [K, N] (ldb):
// the full fine-tune's dW = dy^T x (reference: operators/finetune_ops/core/backward_functions.cpp:94-138
// computes the same product on the CPU).  The 4-wave AGPR design of the NT kernels, with token-major
// K-tiles: each operand's K-tile is a [64 k][256 column] LDS image (512-B rows; the 16-B chunk c of row k
// sits at c ^ tsw5(k), applied on the LDS-DMA source address), read as MFMA fragments by pairs of
// ds_read_b64_tr_b16 (gen_gemm4.py ktile_tn: schedule and addressing).  One workgroup per (output tile,
// token split): the grid is tiles x ksplit <= the CU count, each split a contiguous token range; with
// ksplit > 1 (SLAB) the tile goes to its fp32 slab ws[split][M][N] and gemm_splitk_reduce adds the
// slabs into C in a fixed order (deterministic), else it is added into C directly.  The split index is
// the slow one of the XCD-remapped block id, so the ~tiles workgroups that stream one token range share
// an XCD's L2 (the same A and B K-tiles, read once from HBM).
__device__ __forceinline__ int tsw5(int k) { return ((k & 3) | (((k >> 3) & 1) << 2)) << 1; }

template <bool SLAB, int I>
__device__ __forceinline__ void tn_store_row(const GemmArgs& g, int row, int colb, float* out, long ld, bool ok_row) {
  // row block I: blocks (I, 0..7), lane columns colb + 16 J .. + 3
#define G4_TN_ST(J)                                                                                   \
  {                                                                                                   \
    constexpr int b = 4 * (8 * I + J);                                                                \
    const f32x4_t v = f32x4_t{accr<b>(), accr<b + 1>(), accr<b + 2>(), accr<b + 3>()};               \
    const int col = colb + 16 * J;                                                                    \
    if (ok_row && col < g.N) {                                                                        \
      f32x4_t* p = reinterpret_cast<f32x4_t*>(out + (long)row * ld + col);                            \
      if constexpr (SLAB) *p = v;                                                                     \
      else *p = *p + v * g.alpha;                                                                     \
    }                                                                                                 \
  }
  G4_TN_ST(0) G4_TN_ST(1) G4_TN_ST(2) G4_TN_ST(3) G4_TN_ST(4) G4_TN_ST(5) G4_TN_ST(6) G4_TN_ST(7)
#undef G4_TN_ST
}

template <bool SLAB, int SCHED = 0>
__global__ __launch_bounds__(256, 1) void gemm4_tn_kernel(GemmArgs g) {
  extern __shared__ __attribute__((aligned(16))) bf16_t smem[];
  const int tiles_n = (g.N + 255) / 256, tiles = ((g.M + 255) / 256) * tiles_n;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int split = bid / tiles, t = bid % tiles;
  const int m0 = (t / tiles_n) * 256, n0 = (t % tiles_n) * 256;
  const int nk_all = g.K / 64, ks = g.ksplit > 1 ? g.ksplit : 1;
  const int kps = (nk_all + ks - 1) / ks;
  const int kt0 = split * kps, nk = min(nk_all - kt0, kps);  // >= 2 (gemm4_tn_pick_ksplit)
  const int lane = threadIdx.x & 63;
  const int w = (int)rfl(threadIdx.x >> 6);
  const int wm = w >> 1, wn = w & 1;

  // descriptors of one K-tile: base = its first token row at the tile's first column, 64 rows of range
  // (so the 32-bit offsets never grow with the token count: the LM head's [T, V] operand is > 4 GB); a
  // lane whose 16-B chunk lies past column M (N) reads out of range (0) instead
  const long k0 = (long)kt0 * 64;
  const uint32_t rec_a = (uint32_t)(64 * g.lda * 2), rec_b = (uint32_t)(64 * g.ldb * 2);
  auto srd_ka = [&](int kt) { return make_srd(g.A + (k0 + 64L * kt) * g.lda + m0, rec_a); };
  auto srd_kb = [&](int kt) { return make_srd(g.B + (k0 + 64L * kt) * g.ldb + n0, rec_b); };
  const i32x4_t srd0 = make_srd(g.A, 0);
  // piece j of wave w: LDS rows 8 j + 2 w + (lane >> 5), physical chunk lane & 31
  uint32_t oa[8], ob[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int kr = 8 * j + 2 * w + (lane >> 5);
    const int lc = (lane & 31) ^ tsw5(kr);
    oa[j] = m0 + lc * 8 < g.M ? (uint32_t)((kr * g.lda + lc * 8) * 2) : 0x80000000u;
    ob[j] = n0 + lc * 8 < g.N ? (uint32_t)((kr * g.ldb + lc * 8) * 2) : 0x80000000u;
  }
  const uint32_t lds0 = rfl(lds_addr(smem));
  // fragment addresses (buffer 0, k-step 0, rows k .. k + 3): lane 4q + p of 16-lane group g supplies row
  // 8 g + q, columns 4p .. 4p + 3 of fragment i's 16 columns -> chunk 16 wm + 2 i + (p >> 1) ^ tsw5(row)
  const int gq = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
  const int t3 = q | ((gq & 1) << 2);
  const uint32_t rbase = (uint32_t)((8 * gq + q) * 512 + (p >> 1) * 16 + (p & 1) * 8);
  uint32_t ra[8], rb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ra[i] = lds0 + rbase + (uint32_t)(wm * 256 + 32 * (i ^ t3));
    rb[i] = lds0 + 32768u + rbase + (uint32_t)(wn * 256 + 32 * (i ^ t3));
  }
  {  // prologue: K-tiles 0 and 1 of the split -> buffers 0 and 1
    const uint32_t mw = lds0 + (uint32_t)w * 1024u;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const i32x4_t sa = srd_ka(tt), sb = srd_kb(tt);
#pragma unroll
      for (int j = 0; j < 8; ++j) dma_piece(sa, oa[j], 0u, mw + tt * 65536u + j * 4096u);
#pragma unroll
      for (int j = 0; j < 8; ++j) dma_piece(sb, ob[j], 0u, mw + tt * 65536u + 32768u + j * 4096u);
    }
    asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
  }
  GEMM4_ZERO_ACC_X();
  GEMM4_TN_SET0_READ_X(ra, rb);
  for (int kt = 0; kt < nk; ++kt) {
    const bool more = kt + 2 < nk;
    const i32x4_t sa = more ? srd_ka(kt + 2) : srd0;
    const i32x4_t sb = more ? srd_kb(kt + 2) : srd0;
    const uint32_t zero = 0u, ldsm = lds0 + (uint32_t)(kt & 1) * 65536u + (uint32_t)w * 1024u;
    if constexpr (SCHED == 1) GEMM4_KTILE_TN_X1(ra, rb, oa, ob, sa, sb, zero, zero, ldsm);
    else if constexpr (SCHED == 2) GEMM4_KTILE_TN_X2(ra, rb, oa, ob, sa, sb, zero, zero, ldsm);
    else GEMM4_KTILE_TN_X(ra, rb, oa, ob, sa, sb, zero, zero, ldsm);
  }
  asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");  // last MFMA -> v_accvgpr_read
  // block (i, j): row m0 + wm 128 + 16 i + (lane & 15), columns n0 + wn 128 + 16 j + 4 (lane >> 4) .. + 3
  float* out = SLAB ? g.ws + (long)split * g.M * g.N : reinterpret_cast<float*>(g.C);
  const long ld = SLAB ? (long)g.N : g.ldc;
  int fr = lane & 15, colb = n0 + wn * 128 + 4 * (lane >> 4);
  asm volatile("" : "+v"(fr), "+v"(colb));
  const int rowb = m0 + wm * 128 + fr;
  tn_store_row<SLAB, 0>(g, rowb, colb, out, ld, rowb < g.M);
  tn_store_row<SLAB, 1>(g, rowb + 16, colb, out, ld, rowb + 16 < g.M);
  tn_store_row<SLAB, 2>(g, rowb + 32, colb, out, ld, rowb + 32 < g.M);
  tn_store_row<SLAB, 3>(g, rowb + 48, colb, out, ld, rowb + 48 < g.M);
  tn_store_row<SLAB, 4>(g, rowb + 64, colb, out, ld, rowb + 64 < g.M);
  tn_store_row<SLAB, 5>(g, rowb + 80, colb, out, ld, rowb + 80 < g.M);
  tn_store_row<SLAB, 6>(g, rowb + 96, colb, out, ld, rowb + 96 < g.M);
  tn_store_row<SLAB, 7>(g, rowb + 112, colb, out, ld, rowb + 112 < g.M);
}

// ------------------------------------------------------------------ host
bool gemm4_supported(int M, int N, int K, bool a_t, bool b_t) {
  if (a_t || b_t) return false;
  return K % 64 == 0 && K >= 128 && M > 0 && N >= 8 && N % 8 == 0;
}

// MFT_G4_DIAG (A/B and diagnosis only): nomem | nodma | spread4 | spread2 | spread6
static int g4_diag() {
  static const int v = [] {
    const char* e = getenv("MFT_G4_DIAG");
    if (!e) return 0;
    const std::string d(e);
    return d == "nomem" ? 100 : d == "nodma" ? 1 : d == "spread4" ? 2 : d == "spread2" ? 3 : d == "spread6" ? 4
         : d == "ldsepi" ? 101 : d == "nostore" ? 102 : d == "tiles" ? 103 : 0;
  }();
  return v;
}

template <int EPI, int SCHED, bool NOMEM, int STORE = 0>
static void launch4_k(const GemmArgs& g, hipStream_t st) {
  constexpr size_t shm = 131072;
  static bool attr = false;
  if (!attr) {
    MFT_HIP_CHECK(hipFuncSetAttribute((const void*)gemm4_nt_kernel<EPI, SCHED, NOMEM, STORE>,
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)shm));
    attr = true;
  }
  const int tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  gemm4_nt_kernel<EPI, SCHED, NOMEM, STORE><<<tiles, 256, shm, st>>>(g);
}

static int num_cus4() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    MFT_HIP_CHECK(hipGetDevice(&dev));
    MFT_HIP_CHECK(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
    if (n <= 0) n = 256;
  }
  return n;
}

// CUs left to a concurrent side-stream kernel (gemm4_reserve_cus): a persistent grid assigns its tiles
// statically, so one workgroup queued behind a long-running kernel on its CU delays the whole product
static int g_reserved_cus = 0;
void gemm4_reserve_cus(int n) { g_reserved_cus = n < 0 ? 0 : n; }

template <int EPI, int PDIAG, bool SEG2 = false>
static void launch4p_k(const GemmArgs& g, hipStream_t st) {
  constexpr size_t shm = 163840;  // 2 x 64 KB operand buffers + 4 x 8 KB epilogue staging
  static bool attr = false;
  if (!attr) {
    MFT_HIP_CHECK(hipFuncSetAttribute((const void*)gemm4p_nt_kernel<EPI, PDIAG, SEG2>,
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)shm));
    attr = true;
  }
  const int tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  const int cus = std::max(num_cus4() / 2, num_cus4() - g_reserved_cus);
  gemm4p_nt_kernel<EPI, PDIAG, SEG2><<<std::min(tiles, cus), 256, shm, st>>>(g);
}

template <int EPI>
static void launch4p(const GemmArgs& g0, hipStream_t st) {
  GemmArgs g = g0;
  static const int stag = getenv("MFT_G4_STAGGER") ? atoi(getenv("MFT_G4_STAGGER")) : 0;
  static const int pd = getenv("MFT_G4_PDIAG") ? atoi(getenv("MFT_G4_PDIAG")) : 0;
  g.stagger = stag;
  static const int epi_reg = getenv("MFT_G4_EPI") && std::string(getenv("MFT_G4_EPI")) == "reg";
  g.ntail_full = epi_reg;
  static const int aux_plain = getenv("MFT_G4_AUX") && std::string(getenv("MFT_G4_AUX")) == "plain";
  g.aux_pol = aux_plain;
  if (pd == 1) return launch4p_k<EPI, 1>(g, st);
  if (pd == 2) return launch4p_k<EPI, 2>(g, st);
  if (pd == 3) return launch4p_k<EPI, 3>(g, st);
  launch4p_k<EPI, 0>(g, st);
}

template <int EPI>
static void launch4(const GemmArgs& g, hipStream_t st) {
  if (g4_diag() == 0 && g.K >= 128) return launch4p<EPI>(g, st);
  if constexpr (EPI == GEMM_EPI_BIAS) {
    switch (g4_diag()) {
      case 100: return launch4_k<EPI, 0, true>(g, st);
      case 1: return launch4_k<EPI, 1, false>(g, st);
      case 2: return launch4_k<EPI, 2, false>(g, st);
      case 3: return launch4_k<EPI, 3, false>(g, st);
      case 4: return launch4_k<EPI, 4, false>(g, st);
      case 101: return launch4_k<EPI, 0, false, 1>(g, st);
      case 102: return launch4_k<EPI, 0, false, 2>(g, st);
      default: break;
    }
  }
  launch4_k<EPI, 0, false>(g, st);
}

void gemm4x(const GemmArgs& g, int epi, bool a_t, bool b_t, hipStream_t st) {
  if (!gemm4_supported(g.M, g.N, g.K, a_t, b_t) || g.lda % 8 || g.ldb % 8 || (long)255 * g.lda * 2 + 256 > 0x7fffffffL ||
      (long)255 * g.ldb * 2 + 256 > 0x7fffffffL) {
    fprintf(stderr, "mft::gemm4: unsupported shape M=%d N=%d K=%d (a_t=%d b_t=%d)\n", g.M, g.N, g.K, a_t, b_t);
    abort();
  }
  if (epi == GEMM_EPI_GEGLU_FWD || epi == GEMM_EPI_GEGLU_BWD) {
    const int I = g.geglu_I;
    const bool ok = I > 0 && I % 128 == 0 && g.aux && g.ldaux % 8 == 0 && g.ldc % 8 == 0 &&
                    (epi == GEMM_EPI_GEGLU_FWD ? g.N == 2 * I && g.ldaux >= I && g.ldc >= 2 * I
                                               : g.N == I && g.ldaux >= 2 * I && g.ldc >= 2 * I);
    if (!ok || (epi == GEMM_EPI_GEGLU_FWD && g.K2 > 0)) {
      fprintf(stderr, "mft::gemm4: bad GeGLU epilogue arguments (epi=%d N=%d I=%d ldaux=%ld ldc=%ld K2=%d)\n", epi, g.N, I,
              g.ldaux, g.ldc, g.K2);
      abort();
    }
  }
  if (g.K2 > 0) {  // second K segment: plain output, or the GeGLU backward
    if ((epi != GEMM_EPI_NONE && epi != GEMM_EPI_GEGLU_BWD) || g.K2 % 64 || !g.A2 || !g.B2 || g.lda2 % 8 || g.ldb2 % 8 ||
        g.lda2 < g.K2 || g.ldb2 < g.K2) {
      fprintf(stderr, "mft::gemm4: unsupported second K segment (epi=%d K2=%d lda2=%ld ldb2=%ld)\n", epi, g.K2, g.lda2,
              g.ldb2);
      abort();
    }
    if (epi == GEMM_EPI_GEGLU_BWD) launch4p_k<GEMM_EPI_GEGLU_BWD, 0, true>(g, st);
    else launch4p_k<GEMM_EPI_NONE, 0, true>(g, st);
    return;
  }
  switch (epi) {
    case GEMM_EPI_NONE: launch4<GEMM_EPI_NONE>(g, st); break;
    case GEMM_EPI_BIAS: launch4<GEMM_EPI_BIAS>(g, st); break;
    case GEMM_EPI_BIAS_GELU_D: launch4p<GEMM_EPI_BIAS_GELU_D>(g, st); break;
    case GEMM_EPI_MUL_AUX: launch4p<GEMM_EPI_MUL_AUX>(g, st); break;
    case GEMM_EPI_DGELU: launch4p<GEMM_EPI_DGELU>(g, st); break;
    case GEMM_EPI_BIAS_ADD: launch4p<GEMM_EPI_BIAS_ADD>(g, st); break;
    case GEMM_EPI_CE_FWD: launch4p<GEMM_EPI_CE_FWD>(g, st); break;
    case GEMM_EPI_GEGLU_FWD: launch4p<GEMM_EPI_GEGLU_FWD>(g, st); break;
    case GEMM_EPI_GEGLU_BWD: launch4p<GEMM_EPI_GEGLU_BWD>(g, st); break;
    default: fprintf(stderr, "mft::gemm4: epilogue %d not supported yet\n", epi); abort();
  }
}

// ---- TN weight gradient (gemm4_tn_kernel)
bool gemm4_tn_supported(int M, int N, int K, long lda, long ldb) {
  // 32-bit byte offsets inside one K-tile's 64 rows
  return M >= 8 && N >= 8 && M % 8 == 0 && N % 8 == 0 && K % 64 == 0 && K >= 128 && lda % 8 == 0 && ldb % 8 == 0 &&
         lda >= M && ldb >= N && 64L * lda * 2 < 0x7fff0000L && 64L * ldb * 2 < 0x7fff0000L;
}

int gemm4_tn_pick_ksplit(int M, int N, int K) {
  const int tiles = ((M + 255) / 256) * ((N + 255) / 256);
  const int nk = K / 64, cus = num_cus4();
  static const int cap = getenv("MFT_WGRAD_MAXSPLIT") ? atoi(getenv("MFT_WGRAD_MAXSPLIT")) : 64;
  // modelled time in us: rounds of workgroups x K-tiles per split (~1.4 us per 256 x 256 x 64 K-tile
  // per CU) + the fp32 slabs written and reduced (8 B per element per split at ~5 TB/s); >= 16
  // K-tiles per split, every split >= 2 K-tiles
  int best = 1;
  double best_t = 1e30;
  for (int ks = 1; ks <= cap && (ks == 1 || nk / ks >= 16); ++ks) {
    const int kps = (nk + ks - 1) / ks;
    if (nk - (ks - 1) * kps < 2) continue;
    const int rounds = (tiles * ks + cus - 1) / cus;
    const double t = rounds * kps * 1.4 + (ks > 1 ? (double)ks * M * N * 8 / 5e6 : 0.0);
    if (t < best_t * 0.97) best_t = t, best = ks;
  }
  return best;
}

template <bool SLAB, int SCHED>
static void launch4tn_k(const GemmArgs& g, int grid, hipStream_t st) {
  constexpr size_t shm = 131072;  // 2 buffers x {A, B} [64][256] bf16
  static bool attr = false;
  if (!attr) {
    MFT_HIP_CHECK(hipFuncSetAttribute((const void*)gemm4_tn_kernel<SLAB, SCHED>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)shm));
    attr = true;
  }
  gemm4_tn_kernel<SLAB, SCHED><<<grid, 256, shm, st>>>(g);
}

template <int SCHED>
static void launch4tn(const GemmArgs& g, int tiles, int ks, hipStream_t st) {
  if (ks > 1) launch4tn_k<true, SCHED>(g, tiles * ks, st);
  else launch4tn_k<false, SCHED>(g, tiles, st);
}

void gemm4_tn(const GemmArgs& g, hipStream_t st) {
  if (!gemm4_tn_supported(g.M, g.N, g.K, g.lda, g.ldb) || (g.ksplit > 1 && !g.ws)) {
    fprintf(stderr, "mft::gemm4_tn: unsupported shape M=%d N=%d K=%d lda=%ld ldb=%ld ksplit=%d\n", g.M, g.N, g.K, g.lda,
            g.ldb, g.ksplit);
    abort();
  }
  const int ks = g.ksplit > 1 ? g.ksplit : 1;
  const int nk = g.K / 64, kps = (nk + ks - 1) / ks;
  if (nk - (ks - 1) * kps < 2) {
    fprintf(stderr, "mft::gemm4_tn: split %d of K=%d leaves a split under 2 K-tiles\n", ks, g.K);
    abort();
  }
  const int tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  static const int sched = getenv("MFT_WGRAD_SCHED") ? atoi(getenv("MFT_WGRAD_SCHED")) : 0;  // A/B
  if (sched == 1) launch4tn<1>(g, tiles, ks, st);
  else if (sched == 2) launch4tn<2>(g, tiles, ks, st);
  else launch4tn<0>(g, tiles, ks, st);
  if (ks > 1) gemm_splitk_reduce(g.ws, ks, g.M, g.N, reinterpret_cast<float*>(g.C), g.ldc, g.alpha, 1, st);
}

}  // namespace mft
