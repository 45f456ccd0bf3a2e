// Wide dense GEMM of the plain nn.Linear layers whose two dimensions are both large: the ZINB zero-inflation layer
// G x G (reference model.py:228,255-256) and the VAE's 900 <-> G layers (pairedVAE.py:111-119), precision mode 'bf16'.
//
//   C[m][n] = sum_k A(m,k) B(n,k)  (+ bias[n])  (zero where mask[m][n] <= 0)       bf16 operands, fp32 accumulate / output
//
// Each operand is either stored "row" ([rows][ld], k contiguous) or "col" ([K][ld], rows contiguous), so the three
// products of a Linear layer run on the operands as they lie in memory, without a transposed copy:
//   y  = x W^T   : A = x  row, B = W row        dx = dy W : A = dy row, B = W col        dW = dy^T x : A = dy col, B = x col
//
// Workgroup: tile 256 x 256 x 64 on 512 threads = 2 x 4 waves of 128 x 64 (4 x 2 accumulators of the 32x32x16 bf16
// MFMA, two waves per SIMD) or on 256 threads = 2 x 2 waves of 128 x 128 (one wave per SIMD).  Operand tiles come with
// 16-byte buffer loads, the range check supplying the zeros of ragged edges, straight into LDS (eight waves) or through
// registers (four), two LDS stages of 64 KB, one barrier per K-step: the next step's global loads are in flight while this
// step's 64 MFMAs run.
//   row image  [256][64]  : 128-byte rows, 16-byte chunk c of row r at chunk c ^ ((r >> 1) & 7); read with ds_read_b128
//   col image  [64][256]  : 512-byte rows, 64-byte segment s of row k at segment s ^ (k & 3); read with the
//                           transposing ds_read_b64_tr_b16 (4 k-rows x 16 columns per 16 lanes), conflict-free
// Work split: tiles x nsplit K-ranges so that the launch fills the 256 CUs evenly (1024 x 20 k is 316 tiles = 1.23
// rounds; four K-ranges make it 4.94 rounds of a quarter each); the K-ranges write fp32 slabs which a second kernel
// adds in a fixed order, together with bias and mask (bitwise reproducible: no atomics).  Consecutive workgroup ids
// go round-robin over the 8 XCDs, so the id is remapped to give each XCD a contiguous run of tiles (the tiles that
// share a B tile sit next to each other in one L2).
#include <stdlib.h>
#include "ckpt8.h"
#include "common.h"
#include "scpair_hip.h"

namespace {

constexpr int TM = 256, TN = 256, TK = 64;
constexpr int STAGE_BYTES = (TM + TN) * TK * 2;   // 64 KB

struct WgArgs {
  const __bf16* A;
  const __bf16* B;
  float* C;            // output, or slabs [nsplit][M][ldc] when nsplit > 1
  const float* bias;   // direct mode only
  const __bf16* mask;  // direct mode only
  long lda, ldb, ldc, ldm;
  int M, N, K;
  int tiles_m, tiles_n, nsplit, ksteps_per_split;
  int group;           // order of the tiles: 0 along m, else in blocks of that many tile rows
  unsigned a_bytes, b_bytes;
  unsigned c_bytes, m_bytes;   // extent of C (one slab) and of the mask when both are below 2 GiB, else 0 (guarded global stores)
  // weight gradient with the AdamW step applied in the epilogue (EPI_ADAMW): C = fp32 master weights, updated in place
  float* adam_m; float* adam_v; __bf16* adam_sh; long adam_ldsh;
  float lr, wd, b1, b2, eps, bc1, bc2, gscale;
  const float* bc_dev;       // optional device words {bias_corr1, bias_corr2} (HIP-graph replays), else bc1 / bc2
  const uint8_t* steps;      // B in 8-bit checkpoint form: its step bytes [K][ldb / 64]
  unsigned dbg_oor;    // experiments only (SCPAIR_WGEMM_DBG=1): every load in the K loop out of range -> no memory traffic
};

typedef __attribute__((ext_vector_type(4))) short short4_;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;

__device__ __forceinline__ u32x4 ld128(__amdgpu_buffer_rsrc_t rsrc, unsigned voff) {
  return __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)voff, 0, 0);
}

// 16 bytes per lane from memory into LDS, lane l's at lds + 16 l (lds: the same in all lanes).  In assembly because the compiler
// lets no transposing LDS read pass such a load in flight (it waits for it, whichever buffer either one works on); whoever
// issues it waits (vmcnt) and passes a barrier before the bytes are read.  The load has no output register.  The wait states in
// front of it: one behind m0, five behind a vector instruction that wrote the descriptor (the compiler sees neither).
__device__ __forceinline__ void ld128_lds(u32x4 rsrc, unsigned lds, unsigned voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ u32x4 rsrc_of(const void* p, unsigned bytes) {
  const uint64_t a = (uint64_t)p;
  return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(a >> 32)),
               (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// LDS byte offsets inside an operand image
// (rows r and r + 1 lie in the two halves of a 256-byte bank row, so the swizzle runs over r >> 1: the 16 lanes that
// a ds_read_b128 serves together then touch 16 distinct 16-byte slots)
__device__ __forceinline__ int row_off(int r, int ch) { return r * 128 + ((ch ^ ((r >> 1) & 7)) << 4); }
__device__ __forceinline__ int col_off(int k, int m) { return k * 512 + ((((m >> 5) ^ (k & 3))) << 6) + ((m & 31) << 1); }

template <bool COL>
__device__ __forceinline__ bf16x8 read_frag(const unsigned char* img, int r0, int s, int lane) {
  if (!COL) {
    const int r = r0 + (lane & 31), ch = 2 * s + (lane >> 5);
    return *(const bf16x8*)(img + row_off(r, ch));
  } else {
    // lane 4q+p of a 16-lane group addresses row q, columns 4p..4p+3 of a 4 x 16 block; lane i receives column i
    const int g = lane >> 5, mb = ((lane >> 4) & 1) * 16, q = (lane & 15) >> 2, p = lane & 3;
    const int k = 16 * s + 8 * g + q, m = r0 + mb + 4 * p;
    typedef __attribute__((address_space(3))) short4_ lds_s4;
    short4_ lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(img + col_off(k, m)));
    short4_ hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(img + col_off(k + 4, m)));
    union { short4_ h[2]; bf16x8 v; } u;
    u.h[0] = lo;
    u.h[1] = hi;
    return u.v;
  }
}

enum { EPI_SLAB = 0, EPI_DIRECT = 1, EPI_ADAMW = 2 };

// NW = 8 (default for the plain products): two waves per SIMD, wave tile 128 x 64; one wave's MFMA groups cover the other's
// waits, and the tiles go from memory to LDS without passing through registers (a lane's 16 bytes land at LDS slot `lane` of
// its wave's KB, so the swizzle is applied to what the lane fetches).  16384 x 4096 x 4096 bf16: 425-485 us by box and clock
// (1130-1290 TFLOP/s) with rows or columns for B; 516 and 512 us through registers, 437 and 499 us with the barrier at the step's end.  NW = 4 (the AdamW form; SCPAIR_WGEMM_NW=4
// elsewhere): one wave per SIMD, wave tile 128 x 128, two register sets (loads two K-steps ahead).
// BQ: the B operand (col) is an 8-bit activation checkpoint (ckpt8.hip): codes [K][ldb] int8 and one step byte per 64
// columns.  A thread takes 16 codes with one 16-byte load, half the bytes of the bf16 operand, and takes them apart on the
// way into LDS (a byte conversion and an fma per element, exact in bf16), where the image is that of a bf16 operand.  The
// K-ranges are addressed from their own first row, so the operands of a long batch may pass 2 GiB as long as one range does not.
// CT: type of the output (slabs are fp32 whatever it is).
template <bool A_COL, bool B_COL, int EPI, int NW = 4, bool BQ = false, typename CT = float>
__global__ __launch_bounds__(64 * NW) void wgemm_kernel(WgArgs g) {
  constexpr bool DIRECT = EPI == EPI_DIRECT;
  constexpr bool DMA = NW == 8;
  constexpr int NJ = NW == 4 ? 4 : 2, WN = 32 * NJ, CH = 32 / NW, LSTEP = 1024 * NW, NSET = NW == 4 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  // two objects: the compiler then sees that a stage's reads need not wait for the loads on their way into the other
  __shared__ __attribute__((aligned(1024))) unsigned char stage0[DMA ? STAGE_BYTES : 1], stage1[DMA ? STAGE_BYTES : 1];
  auto stage_of = [&](int stage) -> unsigned char* {
    if constexpr (DMA) return stage ? stage1 : stage0;
    return smem + stage * STAGE_BYTES;
  };
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = NW == 4 ? wave >> 1 : wave >> 2, wn = NW == 4 ? wave & 1 : wave & 3;

  // XCD-aware id: ids b, b+8, b+16.. run on one XCD -> give them consecutive tiles
  const int total = g.tiles_m * g.tiles_n * g.nsplit;
  const int per_xcd = (total + 7) >> 3;
  const int lid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (lid >= total) return;
  const int per_z = g.tiles_m * g.tiles_n, z = lid / per_z;
  int tm = lid % g.tiles_m, tn = (lid / g.tiles_m) % g.tiles_n;
  if (g.group) {                        // blocks of `group` tile rows, walked column by column
    const int t = lid - z * per_z, b = t / (g.group * g.tiles_n), r = t - b * g.group * g.tiles_n;
    const int h = min(g.group, g.tiles_m - g.group * b);
    tn = r / h;
    tm = g.group * b + r - tn * h;
  }
  const int m0 = tm * TM, n0 = tn * TN;
  const int nk_all = (g.K + TK - 1) / TK;
  const int kt0 = z * g.ksteps_per_split;
  const int kt1 = min(nk_all, kt0 + g.ksteps_per_split);

  static_assert(!BQ || (A_COL && B_COL && NW == 8 && EPI != EPI_ADAMW), "8-bit operands: the weight gradient's form only");
  // BQ: first row and rows of this K-range
  const long krow0 = BQ ? (long)kt0 * TK : 0;
  const long krows = min((long)g.K - krow0, (long)(kt1 - kt0) * TK);
  const void* pA = g.A + krow0 * g.lda;
  const unsigned bytesA = BQ ? (unsigned)(((krows - 1) * g.lda + ((g.M + 7) & ~7)) * 2) : g.a_bytes;
  const __amdgpu_buffer_rsrc_t rsA = __builtin_amdgcn_make_buffer_rsrc((void*)pA, 0, (int)bytesA, 0x00020000);
  const __amdgpu_buffer_rsrc_t rsB = __builtin_amdgcn_make_buffer_rsrc(
      BQ ? (void*)((const int8_t*)g.B + krow0 * g.ldb) : (void*)g.B, 0, BQ ? (int)(krows * g.ldb) : (int)g.b_bytes, 0x00020000);
  const u32x4 dmaA = rsrc_of(pA, bytesA), dmaB = rsrc_of(g.B, g.b_bytes);
  const __amdgpu_buffer_rsrc_t rsS = __builtin_amdgcn_make_buffer_rsrc(
      BQ ? (void*)(g.steps + krow0 * (g.ldb >> 6)) : (void*)g.B, 0, BQ ? (int)(krows * (g.ldb >> 6)) : 0, 0x00020000);
  constexpr unsigned OOR = 0x80000000u;     // beyond any operand (host checks bytes < 2 GiB): the load returns zeros

  // chunk c = tid + 256 i.  row image: row (tid >> 3) + 32 i, chunk tid & 7; col image: k row (tid >> 5) + 8 i,
  // chunk tid & 31: the global offset and the LDS offset of chunk i are those of chunk 0 plus i times a constant
  const int Kp = (g.K + 7) & ~7;
  // DMA: the chunk that belongs at LDS slot tid of the image, which the swizzle maps from the slot
  const int rA = A_COL ? (tid >> 5) : (tid >> 3), rB = B_COL ? (tid >> 5) : (tid >> 3);
  const int dR = (tid & 7) ^ ((tid >> 4) & 7), dC = (tid & 31) ^ (((tid >> 5) & 3) << 2);
  const int cA = A_COL ? (DMA ? dC : tid & 31) : (DMA ? dR : tid & 7);
  const int cB = B_COL ? (DMA ? dC : tid & 31) : (DMA ? dR : tid & 7);
  const unsigned baseA = A_COL ? (unsigned)(((long)rA * g.lda + m0 + 8 * cA) * 2) : (unsigned)(((long)(m0 + rA) * g.lda + 8 * cA) * 2);
  const unsigned baseB = B_COL ? (unsigned)(((long)rB * g.ldb + n0 + 8 * cB) * 2) : (unsigned)(((long)(n0 + rB) * g.ldb + 8 * cB) * 2);
  const unsigned stepA = (unsigned)((A_COL ? 8 : 32) * (NW / 4) * g.lda * 2), stepB = (unsigned)((B_COL ? 8 : 32) * (NW / 4) * g.ldb * 2);
  const int ldsA0 = A_COL ? col_off(rA, 8 * cA) : row_off(rA, cA);
  const int ldsB0 = B_COL ? col_off(rB, 8 * cB) : row_off(rB, cB);
  // Ragged edges come from the buffer's range check: a row image's rows >= M and a col image's k rows >= K start at
  // or beyond the operand's last byte and load as zeros.  Only the k tail of a row image needs a test (it would run
  // into the next row): those chunks get the top offset bit.  A col image's columns beyond ld wrap into the next k
  // row; they only feed output rows >= M, which are not stored.
  unsigned offA[CH], offB[CH];
#pragma unroll
  for (int i = 0; i < CH; i++) {
    offA[i] = baseA + stepA * i;
    offB[i] = baseB + stepB * i;
  }

  // BQ: 16-code chunk i of this thread: row (tid >> 4) + 32 i of the K-step, columns 16 (tid & 15)
  const int rQ = tid >> 4, cQ = tid & 15;
  const unsigned baseQ = (unsigned)((long)rQ * g.ldb + n0 + 16 * cQ), baseS = (unsigned)((long)rQ * (g.ldb >> 6) + ((n0 + 16 * cQ) >> 6));
  unsigned qs[2];

  // NW 4, two register sets: the loads of K-step kt + 2 are issued during step kt and stored to LDS during step kt + 1,
  // so a load has more than a whole K-step (64 MFMAs) to arrive
  u32x4 ra[NSET][CH], rb[NSET][CH];
  const unsigned wave_kb = (unsigned)__builtin_amdgcn_readfirstlane(tid >> 6) * 1024u;
  auto lds_of = [&](int stage) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)stage_of(stage) + wave_kb; };
  auto k_off = [&](int kt, unsigned& kA, unsigned& kB) {       // kt >= kt1: out of range, zeros
    const int k0 = (BQ ? kt - kt0 : kt) * TK;
    const unsigned dead = (kt < kt1 ? 0u : OOR) | g.dbg_oor;
    kA = (A_COL ? (unsigned)((long)k0 * g.lda * 2) : ((k0 + 8 * cA < Kp) ? (unsigned)k0 * 2u : OOR)) | dead;
    kB = (B_COL ? (unsigned)((long)k0 * g.ldb * 2) : ((k0 + 8 * cB < Kp) ? (unsigned)k0 * 2u : OOR)) | dead;
  };
  // chunk i of both operands into a stage
  auto dma = [&](int stage, int i, unsigned kA, unsigned kB) {
    const unsigned to = lds_of(stage) + LSTEP * i;
    ld128_lds(dmaA, to, offA[i] + kA);
    if constexpr (!BQ) ld128_lds(dmaB, to + TM * TK * 2, offB[i] + kB);
  };
  auto load_tiles = [&](int kt, int set) {       // into registers
    const int k0 = (BQ ? kt - kt0 : kt) * TK;
    const unsigned dead = (kt < kt1 ? 0u : OOR) | g.dbg_oor;
    unsigned kA, kB;
    k_off(kt, kA, kB);
    if constexpr (BQ) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const unsigned kq = (unsigned)(k0 + 32 * i);
        rb[set][i] = ld128(rsB, baseQ + kq * (unsigned)g.ldb | dead);
        qs[i] = __builtin_amdgcn_raw_buffer_load_b8(rsS, (int)(baseS + kq * (unsigned)(g.ldb >> 6) | dead), 0, 0);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < CH; i++) {
      ra[set][i] = ld128(rsA, offA[i] + kA);
      rb[set][i] = ld128(rsB, offB[i] + kB);
    }
  };
  auto store_tiles = [&](int stage, int set) {
    unsigned char* ia = stage_of(stage);
    unsigned char* ib = ia + TM * TK * 2;
    if constexpr (BQ) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float step = q8_step(qs[i]);
        bf16x8 v[2];
#pragma unroll
        for (int w = 0; w < 4; w++) {
          __bf16 f[4];
          q8_values(rb[set][i][w], step, f);
#pragma unroll
          for (int b = 0; b < 4; b++) v[w >> 1][(w & 1) * 4 + b] = f[b];
        }
        unsigned char* p = ib + col_off(rQ + 32 * i, 16 * cQ);
        *(bf16x8*)p = v[0];
        *(bf16x8*)(p + 16) = v[1];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < CH; i++) {
      *(u32x4*)(ia + ldsA0 + LSTEP * i) = ra[set][i];
      *(u32x4*)(ib + ldsB0 + LSTEP * i) = rb[set][i];
    }
  };

  f32x16 acc[4][NJ];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

  bf16x8 fa[2][4], fb[2][NJ];
  auto read_frags = [&](int stage, int s, int set) {
    const unsigned char* ia = stage_of(stage);
    const unsigned char* ib = ia + TM * TK * 2;
    auto read_b = [&] {
#pragma unroll
      for (int j = 0; j < NJ; j++) fb[set][j] = read_frag<B_COL>(ib, wn * WN + 32 * j, s, lane);
    };
    if (NW == 8) read_b();        // in the order of their use
#pragma unroll
    for (int i = 0; i < 4; i++) fa[set][i] = read_frag<A_COL>(ia, wm * 128 + 32 * i, s, lane);
    if (NW == 4) read_b();
  };
  auto product = [&](int set, int q) { acc[q / NJ][q % NJ] = mfma32(fa[set][q / NJ], fb[set][q % NJ], acc[q / NJ][q % NJ]); };
  auto products = [&](int set) {
#pragma unroll
    for (int q = 0; q < 4 * NJ; q++) product(set, q);
  };
  // instruction classes of __builtin_amdgcn_sched_group_barrier
  constexpr int MFMA = 0x008, VMEM_RD = 0x020, DS_RD = 0x100, DS_WR = 0x200;
  constexpr int RD_A = A_COL ? 2 : 1, RD_B = B_COL ? 2 : 1;     // LDS reads per fragment

  constexpr int VMCNT0 = 0x0f70;      // s_waitcnt vmcnt(0): this wave's part of the other stage has arrived
  if constexpr (!DMA || BQ) {
    load_tiles(kt0, 0);
    store_tiles(0, 0);
  }
  if constexpr (DMA) {
    unsigned kA, kB;
    k_off(kt0, kA, kB);
#pragma unroll
    for (int i = 0; i < CH; i++) dma(0, i, kA, kB);
    __builtin_amdgcn_s_waitcnt(VMCNT0);
  } else {
    load_tiles(kt0 + 1, 1);
  }
  __syncthreads();
  if constexpr (DMA) {
    unsigned kA, kB;
    k_off(kt0 + 1, kA, kB);
#pragma unroll
    for (int i = 0; i < CH; i++) dma(1, i, kA, kB);
    if constexpr (BQ) load_tiles(kt0 + 1, 0);
    read_frags(0, 0, 0);
  }
  // One K-step = four MFMA groups of 4 x NJ products, the fragments of the next group being read while a group multiplies.
  // Two steps per trip; an odd range runs one step on zero tiles.
  // NW 4: the global loads of step kt + 2 are spread over group 0 and the LDS stores of step kt + 1's tiles over group 3 (the
  // other stage: nobody reads it before the barrier at the step's end).
  // NW 8: the barrier stands before group 3, whose fragments are in registers by then: step kt + 1's tiles have arrived and
  // nobody reads step kt's any more, so group 3 hides the first reads of the one and the loads of step kt + 2 into the other.
  // A group's reads go out over its first three products: spread over all eight, the next group's first product waits for them.
#define WG_SCHED(VM)                                                                 \
  _Pragma("unroll") for (int t = 0; t < 4; t++) {                                    \
    if (VM) __builtin_amdgcn_sched_group_barrier(VMEM_RD, 2, 0);                     \
    __builtin_amdgcn_sched_group_barrier(DS_RD, RD_A, 0);                            \
    __builtin_amdgcn_sched_group_barrier(MFMA, 2, 0);                                \
  }                                                                                  \
  _Pragma("unroll") for (int t = 0; t < NJ; t++) {                                   \
    if (VM) __builtin_amdgcn_sched_group_barrier(VMEM_RD, 2, 0);                     \
    __builtin_amdgcn_sched_group_barrier(DS_RD, RD_B, 0);                            \
    __builtin_amdgcn_sched_group_barrier(MFMA, 2, 0);                                \
  }                                                                                  \
  __builtin_amdgcn_sched_barrier(0);
  constexpr int RD = (4 * RD_A + NJ * RD_B + 2) / 3;
#define WG_SCHED8                                                                    \
  _Pragma("unroll") for (int t = 0; t < 3; t++) {                                    \
    __builtin_amdgcn_sched_group_barrier(DS_RD, RD, 0);                              \
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);                                \
  }                                                                                  \
  _Pragma("unroll") for (int t = 0; t < 4; t++) {                                    \
    if (BQ) __builtin_amdgcn_sched_group_barrier(DS_WR, 1, 0);                       \
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);                                \
  }                                                                                  \
  __builtin_amdgcn_sched_barrier(0);
  auto k_step = [&](int kt, int stage, int set_ld, int set_st) {
    if constexpr (DMA) {
      read_frags(stage, 1, 1);
      products(0);
      WG_SCHED8
      read_frags(stage, 2, 0);
      products(1);
      WG_SCHED8
      if constexpr (BQ) store_tiles(stage ^ 1, 0);
      read_frags(stage, 3, 1);
      products(0);
      WG_SCHED8
      __builtin_amdgcn_s_waitcnt(VMCNT0);
      __syncthreads();
      unsigned kA, kB;
      k_off(kt + 2, kA, kB);
      read_frags(stage ^ 1, 0, 0);
      if constexpr (BQ) load_tiles(kt + 2, 0);
#pragma unroll
      for (int q = 0; q < 3; q++) product(1, q);
#pragma unroll
      for (int t = 0; t < 3; t++) {
        __builtin_amdgcn_sched_group_barrier(DS_RD, RD, 0);
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < CH; i++) {
        dma(stage, i, kA, kB);
        product(1, 3 + i);
        __builtin_amdgcn_sched_barrier(0);
      }
      product(1, 7);
      __builtin_amdgcn_sched_barrier(0);
      return;
    }
    read_frags(stage, 0, 0);
    load_tiles(kt + NSET, set_ld);
    read_frags(stage, 1, 1);
    products(0);
    WG_SCHED(true)
    read_frags(stage, 2, 0);
    products(1);
    WG_SCHED(false)
    read_frags(stage, 3, 1);
    products(0);
    WG_SCHED(false)
    store_tiles(stage ^ 1, set_st);
    products(1);
#pragma unroll
    for (int t = 0; t < 2 * CH; t++) {
      __builtin_amdgcn_sched_group_barrier(DS_WR, 1, 0);
      __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    }
    __syncthreads();
  };
#undef WG_SCHED
#undef WG_SCHED8
  for (int kt = kt0; kt < kt1; kt += 2) {
    k_step(kt, 0, 0, NSET - 1);
    k_step(kt + 1, 1, NSET - 1, 0);
  }

  if (DMA) {       // the loads past the last step, before the stages get another use or another owner
    __builtin_amdgcn_s_waitcnt(VMCNT0);
    __syncthreads();
  }
  // epilogue: accumulator element e of lane l is row acc_row(e, l), column l & 31 of its 32 x 32 tile
  if constexpr (EPI == EPI_ADAMW) {
    static_assert(NW == 4, "the AdamW epilogue is written for the four-wave tile");
    // The tile is a block of the weight gradient: apply torch.optim.AdamW's update to the master weights, the moments
    // and the bf16 shadow right here; the gradient never reaches HBM.  Every wave passes its 32-row strips through a
    // private LDS buffer [32][132] (the operand stages are free after the loop's last barrier; same-wave LDS accesses
    // need no barrier) and walks them row-wise: half a wave per 512-byte row segment, float4 loads and stores.
    typedef float f4 __attribute__((ext_vector_type(4)));
    float* wt = (float*)smem + wave * (32 * 132);
    const float bc1 = g.bc_dev ? g.bc_dev[0] : g.bc1, bc2 = g.bc_dev ? g.bc_dev[1] : g.bc2;
    const AdamHyper hy = adam_hyper(g.lr, g.wd, g.b1, g.b2, g.eps, bc1, bc2, g.gscale);
    const int c4 = (lane & 31) * 4;
    const int n = n0 + wn * 128 + c4;
    const bool col_ok = n + 4 <= g.N;             // N % 4 == 0 (host-checked): a float4 is all in or all out
    const bool interior = m0 + TM <= g.M && n0 + TN <= g.N;
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) wt[acc_row(e, lane) * 132 + 32 * j + (lane & 31)] = acc[i][j][e];
      __builtin_amdgcn_wave_barrier();
      const int mrow = m0 + wm * 128 + 32 * i + (lane >> 5);
      if (interior) {
        // no tests: the loads of four row pairs are issued before the first update, twelve float4 in flight per lane
#pragma unroll
        for (int it0 = 0; it0 < 16; it0 += 4) {
          f4 pv[4], mv[4], vv[4];
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const long idx = (long)(mrow + 2 * (it0 + u)) * g.ldc + n;
            // read once and written once per step, 10 GB in all: streaming accesses, nothing to keep in the caches
            pv[u] = __builtin_nontemporal_load((const f4*)(g.C + idx));
            mv[u] = __builtin_nontemporal_load((const f4*)(g.adam_m + idx));
            vv[u] = __builtin_nontemporal_load((const f4*)(g.adam_v + idx));
          }
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const int row = 2 * (it0 + u) + (lane >> 5);
            const f4 gv = *(const f4*)(wt + row * 132 + c4);
            const long idx = (long)(mrow + 2 * (it0 + u)) * g.ldc + n;
            bf16x4 sh4;
#pragma unroll
            for (int t = 0; t < 4; t++) {
              float p_ = pv[u][t], m_ = mv[u][t], v_ = vv[u][t];
              adamw_update_fast(hy, p_, gv[t], m_, v_);
              pv[u][t] = p_;
              mv[u][t] = m_;
              vv[u][t] = v_;
              sh4[t] = (__bf16)p_;
            }
            __builtin_nontemporal_store(pv[u], (f4*)(g.C + idx));
            __builtin_nontemporal_store(mv[u], (f4*)(g.adam_m + idx));
            __builtin_nontemporal_store(vv[u], (f4*)(g.adam_v + idx));
            *(bf16x4*)(g.adam_sh + (long)(mrow + 2 * (it0 + u)) * g.adam_ldsh + n) = sh4;
          }
        }
      } else {
#pragma unroll 2
        for (int it = 0; it < 16; it++) {
          const int row = 2 * it + (lane >> 5);
          const f4 gv = *(const f4*)(wt + row * 132 + c4);
          const int m = m0 + wm * 128 + 32 * i + row;
          if (col_ok && m < g.M) {
            const long idx = (long)m * g.ldc + n;
            f4 pv = *(const f4*)(g.C + idx), mv = *(const f4*)(g.adam_m + idx), vv = *(const f4*)(g.adam_v + idx);
            bf16x4 sh4;
#pragma unroll
            for (int t = 0; t < 4; t++) {
              float p_ = pv[t], m_ = mv[t], v_ = vv[t];
              adamw_update_fast(hy, p_, gv[t], m_, v_);
              pv[t] = p_;
              mv[t] = m_;
              vv[t] = v_;
              sh4[t] = (__bf16)p_;
            }
            *(f4*)(g.C + idx) = pv;
            *(f4*)(g.adam_m + idx) = mv;
            *(f4*)(g.adam_v + idx) = vv;
            *(bf16x4*)(g.adam_sh + (long)m * g.adam_ldsh + n) = sh4;
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
    return;
  }
  if constexpr (NW == 8) {
    // A wave's 32-row strips go through a private LDS buffer (the operand stages are free by now), so that 16 lanes write a row
    // segment of 64 columns: an accumulator's own layout makes 2- or 4-byte stores, 128 of them a lane, and registers spill over
    // their addresses (weight gradient 900 x 20 k over 1024 rows, fp32: 62 against 89 us).
    if (sizeof(CT) == 2 || !(DIRECT && g.mask)) {
      static_assert(sizeof(CT) == 4 || DIRECT, "slabs are fp32");
      constexpr int LD = 72;                      // lanes 32 .. 63 write four rows further down, to the other 32 banks
      typedef CT ct4 __attribute__((ext_vector_type(4), aligned(sizeof(CT))));
      typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
      CT* Cs = (CT*)(void*)g.C + (DIRECT ? 0 : (long)z * g.M * g.ldc);
      float* wt = (float*)stage_of(wave >> 2) + (wave & 3) * (32 * LD);
      const int c4 = (lane & 15) * 4, n = n0 + wn * WN + c4;
      const bool whole = n + 4 <= g.N;
      f32x4 bn = {0.f, 0.f, 0.f, 0.f};
      if (DIRECT && g.bias) {
        if (whole) bn = *(const f4u*)(g.bias + n);
        else
#pragma unroll
          for (int t = 0; t < 4; t++) bn[t] = n + t < g.N ? g.bias[n + t] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
          for (int e = 0; e < 16; e++) wt[acc_row(e, lane) * LD + 32 * j + (lane & 31)] = acc[i][j][e];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < 8; it++) {
          const int row = 4 * it + (lane >> 4), m = m0 + wm * 128 + 32 * i + row;
          const f32x4 v = *(const f32x4*)(wt + row * LD + c4) + bn;
          if (m >= g.M) continue;
          CT* p = Cs + (long)m * g.ldc + n;
          if (whole) {
            ct4 o;
#pragma unroll
            for (int t = 0; t < 4; t++) o[t] = (CT)v[t];
            *(ct4*)p = o;
          } else {
#pragma unroll
            for (int t = 0; t < 4; t++)
              if (n + t < g.N) p[t] = (CT)v[t];
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
      return;
    }
  }
  if constexpr (sizeof(CT) == 2) return;
  float* Cz = g.C + (DIRECT ? 0 : (long)z * g.M * g.ldc);
  if (m0 + TM <= g.M && n0 + TN <= g.N && !(DIRECT && g.mask)) {
    // interior tile: no tests; one store instruction writes two 128-byte row segments
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int n = n0 + wn * WN + 32 * j + (lane & 31);
      const float bn = (DIRECT && g.bias) ? g.bias[n] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float* p = Cz + (long)(m0 + wm * 128 + 32 * i + 4 * (lane >> 5)) * g.ldc + n;
#pragma unroll
        for (int e = 0; e < 16; e++) p[(long)((e & 3) + 8 * (e >> 2)) * g.ldc] = acc[i][j][e] + bn;
      }
    }
    return;
  }
  if (g.c_bytes) {
    // edge tile or masked output, C (and mask) below 2 GiB: buffer stores, no branches.  Rows >= M start at or beyond
    // the buffer's last byte, so the range check drops them; columns >= N get the top offset bit.
    const __amdgpu_buffer_rsrc_t rsC = __builtin_amdgcn_make_buffer_rsrc((void*)Cz, 0, (int)g.c_bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t rsM =
        __builtin_amdgcn_make_buffer_rsrc((void*)(DIRECT && g.mask ? g.mask : g.A), 0, (int)g.m_bytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int n = n0 + wn * WN + 32 * j + (lane & 31);
      const unsigned colbad = n < g.N ? 0u : OOR;
      const float bn = (DIRECT && g.bias && n < g.N) ? g.bias[n] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int mb = m0 + wm * 128 + 32 * i + 4 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int r = (e & 3) + 8 * (e >> 2);
          // The out-of-range mark REPLACES the offset (a top bit OR-ed into a base would be carried out again by the
          // row term when C ends just below 2 GiB); offsets are formed in 64 bits and compared with the extent.
          const long co = ((long)(mb + r) * g.ldc + n) * 4, mo = ((long)(mb + r) * g.ldm + n) * 2;
          const unsigned coff = (colbad || co >= (long)g.c_bytes) ? OOR : (unsigned)co;
          float v = acc[i][j][e] + bn;
          if (DIRECT && g.mask) {
            const unsigned moff = (colbad || mo >= (long)g.m_bytes) ? OOR : (unsigned)mo;
            const unsigned short mk = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rsM, (int)moff, 0, 0);
            const float mf = __uint_as_float((unsigned)mk << 16);
            if (!(mf > 0.f)) v = 0.f;
          }
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rsC, (int)coff, 0, 0);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int n = n0 + wn * WN + 32 * j + (lane & 31);
    if (n >= g.N) continue;
    const float bn = (DIRECT && g.bias) ? g.bias[n] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int m = m0 + wm * 128 + 32 * i + acc_row(e, lane);
        if (m < g.M) {
          float v = acc[i][j][e] + bn;
          if (DIRECT && g.mask && !((float)g.mask[(long)m * g.ldm + n] > 0.f)) v = 0.f;
          Cz[(long)m * g.ldc + n] = v;
        }
      }
    }
  }
}

// C = sum of the K-range slabs in slab order, + bias, masked
// (slabs and output share the row stride ldc)
template <typename CT>
__global__ __launch_bounds__(256) void wgemm_reduce_kernel(const float* __restrict__ slabs, int nsplit, int M, int N, long ldc,
                                                            const float* __restrict__ bias, const __bf16* __restrict__ mask,
                                                            long ldm, CT* __restrict__ C) {
  const long n4 = (N + 3) / 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)M * n4) return;
  const int m = (int)(i / n4), c = (int)(i % n4) * 4;
  const long slab = (long)M * ldc;
  const float* p = slabs + (long)m * ldc + c;
  if (c + 3 < N && (ldc & 3) == 0) {
    f32x4 s = *(const f32x4*)p;
    for (int zz = 1; zz < nsplit; zz++) s += *(const f32x4*)(p + zz * slab);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if (bias) s[t] += bias[c + t];
      if (mask && !((float)mask[(long)m * ldm + c + t] > 0.f)) s[t] = 0.f;
    }
    if constexpr (sizeof(CT) == 4) {
      *(f32x4*)(C + (long)m * ldc + c) = s;
    } else {
#pragma unroll
      for (int t = 0; t < 4; t++) C[(long)m * ldc + c + t] = (CT)s[t];
    }
  } else {
    for (int t = 0; t < 4 && c + t < N; t++) {
      float s = p[t];
      for (int zz = 1; zz < nsplit; zz++) s += p[t + zz * slab];
      if (bias) s += bias[c + t];
      if (mask && !((float)mask[(long)m * ldm + c + t] > 0.f)) s = 0.f;
      C[(long)m * ldc + c + t] = (CT)s;
    }
  }
}

// K-ranges so that tiles x ranges fill the 256 CUs evenly; a function of the shape only (results do not depend on
// the machine's state).  Cost model in units of one full-K tile: rounds / nsplit for the product, plus the slab
// traffic of the reduction priced against the tile's MFMA time.
int pick_nsplit(int M, int N, int K) {
  if (const char* e = getenv("SCPAIR_WGEMM_NSPLIT")) {      // experiments only
    const int v = atoi(e);
    if (v >= 1 && v <= 16 && v <= (K + TK - 1) / TK) return v;
  }
  const long tiles = (long)((M + TM - 1) / TM) * ((N + TN - 1) / TN);
  const int nk = (K + TK - 1) / TK;
  const double tile_s = 2.0 * TM * TN * (double)K / (2.5e15 / 256 * 0.5);       // one tile at half of the MFMA peak
  double best = 1e30;
  int best_ns = 1;
  for (int ns = 1; ns <= 16; ns++) {
    if (ns > 1 && nk / ns < 8) break;
    const double rounds = (double)((tiles * ns + 255) / 256) / ns;
    double cost = rounds * tile_s;
    if (ns > 1) cost += (double)(ns + 2) * M * N * 4.0 / 4.0e12 + 4e-6;
    if (cost < best * 0.97) {
      best = cost;
      best_ns = ns;
    }
  }
  return best_ns;
}

template <bool AC, bool BC>
int launch(const WgArgs& g, hipStream_t st) {
  static uint64_t done_d = 0, done_s = 0;
  const int total = g.tiles_m * g.tiles_n * g.nsplit;
  const unsigned grid = (unsigned)(((total + 7) / 8) * 8);
  // eight waves by default (measured 2-10 % faster than four on every shape of the wide layers, same box, back to
  // back); SCPAIR_WGEMM_NW=4 selects the four-wave form for comparison
  const char* e8 = getenv("SCPAIR_WGEMM_NW");
  const bool nw8 = !(e8 && atoi(e8) == 4);
  if (g.nsplit == 1 && !nw8) {
    int rc = scp_set_smem((const void*)wgemm_kernel<AC, BC, EPI_DIRECT>, 2 * STAGE_BYTES, &done_d);
    if (rc) return rc;
    hipLaunchKernelGGL((wgemm_kernel<AC, BC, EPI_DIRECT>), dim3(grid), dim3(256), 2 * STAGE_BYTES, st, g);
  } else if (!nw8) {
    int rc = scp_set_smem((const void*)wgemm_kernel<AC, BC, EPI_SLAB>, 2 * STAGE_BYTES, &done_s);
    if (rc) return rc;
    hipLaunchKernelGGL((wgemm_kernel<AC, BC, EPI_SLAB>), dim3(grid), dim3(256), 2 * STAGE_BYTES, st, g);
  } else if (g.nsplit == 1) {
    hipLaunchKernelGGL((wgemm_kernel<AC, BC, EPI_DIRECT, 8>), dim3(grid), dim3(512), 0, st, g);
  } else {
    hipLaunchKernelGGL((wgemm_kernel<AC, BC, EPI_SLAB, 8>), dim3(grid), dim3(512), 0, st, g);
  }
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

// eight-wave forms with a bf16 output and / or an 8-bit B operand
template <bool AC, bool BC, int EPI, bool BQ, typename CT>
int launch8(const WgArgs& g, hipStream_t st) {
  const int total = g.tiles_m * g.tiles_n * g.nsplit;
  hipLaunchKernelGGL((wgemm_kernel<AC, BC, EPI, 8, BQ, CT>), dim3((unsigned)(((total + 7) / 8) * 8)), dim3(512), 0, st, g);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

template <typename CT>
int reduce_slabs(const WgArgs& g, const float* ws, const float* bias, CT* C, hipStream_t st) {
  const long n = (long)g.M * ((g.N + 3) / 4);
  hipLaunchKernelGGL((wgemm_reduce_kernel<CT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, ws, g.nsplit, g.M, g.N,
                     g.ldc, bias, nullptr, 0L, C);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

// Order of the tiles for the products of linear8: with long K-ranges, blocks of 8 tile rows, so that the 32 tiles at work on an
// XCD share 8 + 4 operand tiles instead of 32 + 1 (16384 x 4096 x 4096: 575 -> 520 us)
int tile_group(const WgArgs& g) { return g.ksteps_per_split >= 32 ? 8 : 0; }

// K-ranges of a product with an 8-bit operand: at least as many as keep a range's bytes below 1 GiB
int q8_nsplit(int M, int N, int K, long lda) {
  const int nk = (K + TK - 1) / TK;
  long ns = pick_nsplit(M, N, K);
  const long need = ((long)nk * TK * lda * 2 + (1L << 30) - 1) >> 30;
  if (need > ns) ns = need;
  // whole K-steps per range, no empty range
  const long per = (nk + ns - 1) / ns;
  return (int)((nk + per - 1) / per);
}

}  // namespace

extern "C" int scp_gemm_bf16_nsplit(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 1;
  return pick_nsplit(M, N, K);
}

extern "C" long scp_gemm_bf16_ws_floats(int M, int N, int K, long ldc) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const int ns = pick_nsplit(M, N, K);
  return ns > 1 ? (long)ns * M * ldc : 0;
}

// dW = A^T-style product of two k-major operands with the AdamW step of W in the epilogue (see the header)
extern "C" int scp_gemm_bf16_adamw(int M, int N, int K, const void* A, long lda, const void* B, long ldb, float* W, long ldw,
                                   float* exp_avg, float* exp_avg_sq, void* W_bf16, long ld_bf16, float lr, float weight_decay,
                                   float beta1, float beta2, float eps, float bias_corr1, float bias_corr2, float grad_scale,
                                   const float* bc_dev, void* stream_) {
  SCP_CHECK(M > 0 && N > 0 && K > 0, SCP_ERR_ARG, "scp_gemm_bf16_adamw: M, N, K must be positive (%d, %d, %d)", M, N, K);
  SCP_CHECK(A && B && W && exp_avg && exp_avg_sq && W_bf16, SCP_ERR_ARG, "scp_gemm_bf16_adamw: null pointer");
  SCP_CHECK(lda >= ((M + 7) & ~7L) && ldb >= ((N + 7) & ~7L) && ldw >= N && ld_bf16 >= N, SCP_ERR_ARG,
            "scp_gemm_bf16_adamw: leading dimension too small");
  SCP_CHECK(lda % 8 == 0 && ldb % 8 == 0 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0, SCP_ERR_ARG,
            "scp_gemm_bf16_adamw: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  SCP_CHECK(((long)K + 3 * TK) * lda * 2 + 4096 < (1L << 31) && ((long)K + 3 * TK) * ldb * 2 + 4096 < (1L << 31), SCP_ERR_SHAPE,
            "scp_gemm_bf16_adamw: an operand within 3 K-steps of 2 GiB (or larger) is not supported (see scp_gemm_bf16)");
  SCP_CHECK(N % 4 == 0 && ldw % 4 == 0 && ld_bf16 % 4 == 0 &&
                (((uintptr_t)W | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) % 16) == 0 && ((uintptr_t)W_bf16 % 8) == 0,
            SCP_ERR_SHAPE, "scp_gemm_bf16_adamw: needs N %% 4 == 0, leading dimensions %% 4 == 0 and 16-byte aligned W / moments");
  SCP_CHECK(bc_dev || (bias_corr1 > 0.f && bias_corr2 > 0.f), SCP_ERR_ARG, "scp_gemm_bf16_adamw: bias corrections must be > 0");
  WgArgs g = {};
  g.A = (const __bf16*)A;
  g.B = (const __bf16*)B;
  g.C = W;
  g.lda = lda;
  g.ldb = ldb;
  g.ldc = ldw;
  g.M = M;
  g.N = N;
  g.K = K;
  g.tiles_m = (M + TM - 1) / TM;
  g.tiles_n = (N + TN - 1) / TN;
  g.nsplit = 1;                                   // the update needs the complete sum: one K-range
  g.ksteps_per_split = (K + TK - 1) / TK;
  g.a_bytes = (unsigned)((long)K * lda * 2);
  g.b_bytes = (unsigned)((long)K * ldb * 2);
  g.adam_m = exp_avg; g.adam_v = exp_avg_sq; g.adam_sh = (__bf16*)W_bf16; g.adam_ldsh = ld_bf16;
  g.lr = lr; g.wd = weight_decay; g.b1 = beta1; g.b2 = beta2; g.eps = eps; g.bc1 = bias_corr1; g.bc2 = bias_corr2;
  g.gscale = grad_scale; g.bc_dev = bc_dev;
  SCP_CHECK((long)g.tiles_m * g.tiles_n < (1L << 30), SCP_ERR_SHAPE, "scp_gemm_bf16_adamw: too many tiles");
  static uint64_t done_a = 0;
  int rc = scp_set_smem((const void*)wgemm_kernel<true, true, EPI_ADAMW>, 2 * STAGE_BYTES, &done_a);
  if (rc) return rc;
  const int total = g.tiles_m * g.tiles_n;
  hipLaunchKernelGGL((wgemm_kernel<true, true, EPI_ADAMW>), dim3((unsigned)(((total + 7) / 8) * 8)), dim3(256), 2 * STAGE_BYTES,
                     (hipStream_t)stream_, g);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

extern "C" int scp_gemm_bf16(int a_col, int b_col, int M, int N, int K, const void* A, long lda, const void* B, long ldb,
                             float* C, long ldc, const float* bias, const void* mask, long ldm, float* ws, void* stream_) {
  SCP_CHECK(M > 0 && N > 0 && K > 0, SCP_ERR_ARG, "scp_gemm_bf16: M, N, K must be positive (%d, %d, %d)", M, N, K);
  SCP_CHECK(A && B && C, SCP_ERR_ARG, "scp_gemm_bf16: null pointer");
  SCP_CHECK((a_col == 0 || a_col == 1) && (b_col == 0 || b_col == 1), SCP_ERR_ARG, "scp_gemm_bf16: a_col / b_col must be 0 or 1");
  const long a_rows = a_col ? K : M, a_cols = a_col ? M : K, b_rows = b_col ? K : N, b_cols = b_col ? N : K;
  SCP_CHECK(lda >= ((a_cols + 7) & ~7L) && ldb >= ((b_cols + 7) & ~7L) && ldc >= N, SCP_ERR_ARG,
            "scp_gemm_bf16: leading dimension too small (operands are padded to a multiple of 8 columns)");
  SCP_CHECK(lda % 8 == 0 && ldb % 8 == 0 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0, SCP_ERR_ARG,
            "scp_gemm_bf16: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  // The K loop marks dead loads by OR-ing the top offset bit into the per-step term and then adds the per-chunk offset:
  // the sum must stay below 2^31 for every (step <= last + 2, chunk), or the mark would be carried out and real data
  // read.  Hence the slack of two K-steps (k-major operand: whole k rows) on top of the operand's own extent.
  SCP_CHECK((a_rows + (a_col ? 3 * TK : 0)) * lda * 2 + 4096 < (1L << 31) &&
                (b_rows + (b_col ? 3 * TK : 0)) * ldb * 2 + 4096 < (1L << 31), SCP_ERR_SHAPE,
            "scp_gemm_bf16: an operand within 3 K-steps of 2 GiB (or larger) is not supported");
  SCP_CHECK(!mask || ldm >= N, SCP_ERR_ARG, "scp_gemm_bf16: mask leading dimension too small");
  WgArgs g = {};
  g.A = (const __bf16*)A;
  g.B = (const __bf16*)B;
  g.lda = lda;
  g.ldb = ldb;
  g.ldc = ldc;
  g.ldm = ldm;
  g.M = M;
  g.N = N;
  g.K = K;
  g.tiles_m = (M + TM - 1) / TM;
  g.tiles_n = (N + TN - 1) / TN;
  g.nsplit = pick_nsplit(M, N, K);
  const int nk = (K + TK - 1) / TK;
  g.ksteps_per_split = (nk + g.nsplit - 1) / g.nsplit;
  g.a_bytes = (unsigned)(a_rows * lda * 2);
  g.b_bytes = (unsigned)(b_rows * ldb * 2);
  g.dbg_oor = (getenv("SCPAIR_WGEMM_DBG") && atoi(getenv("SCPAIR_WGEMM_DBG")) == 1) ? 0x80000000u : 0u;
  SCP_CHECK((long)g.tiles_m * g.tiles_n * g.nsplit < (1L << 30), SCP_ERR_SHAPE, "scp_gemm_bf16: too many tiles");
  {
    const long cb = (long)M * ldc * 4, mb = mask ? (long)M * ldm * 2 : 2;
    const bool small = cb < (1L << 31) && mb < (1L << 31);
    g.c_bytes = small ? (unsigned)cb : 0u;
    g.m_bytes = small ? (unsigned)mb : 0u;
  }
  hipStream_t st = (hipStream_t)stream_;
  if (g.nsplit == 1) {
    g.C = C;
    g.bias = bias;
    g.mask = (const __bf16*)mask;
  } else {
    SCP_CHECK(ws, SCP_ERR_ARG, "scp_gemm_bf16: this shape runs as %d K-ranges and needs the workspace of scp_gemm_bf16_ws_floats",
              g.nsplit);
    g.C = ws;
    g.bias = nullptr;
    g.mask = nullptr;
  }
  int rc = a_col ? (b_col ? launch<true, true>(g, st) : launch<true, false>(g, st))
                 : (b_col ? launch<false, true>(g, st) : launch<false, false>(g, st));
  if (rc) return rc;
  if (g.nsplit > 1) {
    const long n = (long)M * ((N + 3) / 4);
    hipLaunchKernelGGL((wgemm_reduce_kernel<float>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, ws, g.nsplit, M, N, ldc, bias,
                       (const __bf16*)mask, ldm, C);
    SCP_LAUNCH_CHECK();
  }
  return SCP_OK;
}

extern "C" int scp_gemm_rows(int b_col, int M, int N, int K, const void* A, long lda, const void* B, long ldb, void* C,
                             int c_bf16, long ldc, const float* bias, float* ws, void* stream_) {
  SCP_CHECK(M > 0 && N > 0 && K > 0, SCP_ERR_ARG, "scp_gemm_rows: M, N, K must be positive (%d, %d, %d)", M, N, K);
  SCP_CHECK(A && B && C, SCP_ERR_ARG, "scp_gemm_rows: null pointer");
  SCP_CHECK(b_col == 0 || b_col == 1, SCP_ERR_ARG, "scp_gemm_rows: b_col must be 0 or 1");
  const long b_rows = b_col ? K : N, b_cols = b_col ? N : K;
  SCP_CHECK(lda >= ((K + 7) & ~7L) && ldb >= ((b_cols + 7) & ~7L) && ldc >= N, SCP_ERR_ARG,
            "scp_gemm_rows: leading dimension too small (operands are padded to a multiple of 8 columns)");
  SCP_CHECK(lda % 8 == 0 && ldb % 8 == 0 && ((uintptr_t)A & 15) == 0 && ((uintptr_t)B & 15) == 0, SCP_ERR_ARG,
            "scp_gemm_rows: operands must be 16-byte aligned with leading dimensions that are multiples of 8");
  // the slack of scp_gemm_bf16: offset + dead-load mark must not carry out of 32 bits
  SCP_CHECK((long)M * lda * 2 + 4096 < (1L << 31) && (b_rows + (b_col ? 3 * TK : 0)) * ldb * 2 + 4096 < (1L << 31), SCP_ERR_SHAPE,
            "scp_gemm_rows: an operand within 3 K-steps of 2 GiB (or larger) is not supported");
  WgArgs g = {};
  g.A = (const __bf16*)A; g.B = (const __bf16*)B;
  g.lda = lda; g.ldb = ldb; g.ldc = ldc;
  g.M = M; g.N = N; g.K = K;
  g.tiles_m = (M + TM - 1) / TM; g.tiles_n = (N + TN - 1) / TN;
  g.nsplit = pick_nsplit(M, N, K);
  g.ksteps_per_split = ((K + TK - 1) / TK + g.nsplit - 1) / g.nsplit;
  g.a_bytes = (unsigned)((long)M * lda * 2);
  g.b_bytes = (unsigned)(b_rows * ldb * 2);
  SCP_CHECK((long)g.tiles_m * g.tiles_n * g.nsplit < (1L << 30), SCP_ERR_SHAPE, "scp_gemm_rows: too many tiles");
  g.group = tile_group(g);
  const long cb = (long)M * ldc * 4;
  g.c_bytes = cb < (1L << 31) ? (unsigned)cb : 0u;
  g.m_bytes = 2;
  hipStream_t st = (hipStream_t)stream_;
  if (g.nsplit == 1) {
    g.C = (float*)C;
    g.bias = bias;
    if (!c_bf16) return b_col ? launch<false, true>(g, st) : launch<false, false>(g, st);
    return b_col ? launch8<false, true, EPI_DIRECT, false, __bf16>(g, st) : launch8<false, false, EPI_DIRECT, false, __bf16>(g, st);
  }
  SCP_CHECK(ws, SCP_ERR_ARG, "scp_gemm_rows: this shape runs as %d K-ranges and needs the workspace of scp_gemm_bf16_ws_floats",
            g.nsplit);
  g.C = ws;
  const int rc = b_col ? launch8<false, true, EPI_SLAB, false, float>(g, st) : launch8<false, false, EPI_SLAB, false, float>(g, st);
  if (rc) return rc;
  return c_bf16 ? reduce_slabs(g, ws, bias, (__bf16*)C, st) : reduce_slabs(g, ws, bias, (float*)C, st);
}

extern "C" long scp_gemm_q8_ws_floats(int M, int N, int K, long lda, long ldc) {
  if (M <= 0 || N <= 0 || K <= 0 || lda <= 0) return 0;
  const int ns = q8_nsplit(M, N, K, lda);
  return ns > 1 ? (long)ns * M * ldc : 0;
}

extern "C" int scp_gemm_q8(int M, int N, int K, const void* A, long lda, const int8_t* codes, const uint8_t* steps, void* C,
                           int c_bf16, long ldc, float* ws, void* stream_) {
  SCP_CHECK(M > 0 && N > 0 && K > 0, SCP_ERR_ARG, "scp_gemm_q8: M, N, K must be positive (%d, %d, %d)", M, N, K);
  SCP_CHECK(A && codes && steps && C, SCP_ERR_ARG, "scp_gemm_q8: null pointer");
  const long ldb = (N + 63) / 64 * 64L;
  SCP_CHECK(lda >= ((M + 7) & ~7L) && lda % 8 == 0 && ldc >= N, SCP_ERR_ARG,
            "scp_gemm_q8: leading dimension too small or not a multiple of 8");
  SCP_CHECK((((uintptr_t)A | (uintptr_t)codes) & 15) == 0, SCP_ERR_ARG, "scp_gemm_q8: operands must be 16-byte aligned");
  WgArgs g = {};
  g.A = (const __bf16*)A; g.B = (const __bf16*)(const void*)codes; g.steps = steps;
  g.lda = lda; g.ldb = ldb; g.ldc = ldc;
  g.M = M; g.N = N; g.K = K;
  g.tiles_m = (M + TM - 1) / TM; g.tiles_n = (N + TN - 1) / TN;
  g.nsplit = q8_nsplit(M, N, K, lda > ldb ? lda : ldb);
  g.ksteps_per_split = ((K + TK - 1) / TK + g.nsplit - 1) / g.nsplit;
  // offsets are formed in 32 bits within a K-range, up to three K-steps past its end, and the dead-load mark is bit 31
  const long range = ((long)g.ksteps_per_split + 3) * TK;
  SCP_CHECK(range * lda * 2 + 4096 < (1L << 31) && range * ldb + 4096 < (1L << 31), SCP_ERR_SHAPE,
            "scp_gemm_q8: a K-range of %ld rows of %ld columns passes 2 GiB", range, lda > ldb ? lda : ldb);
  SCP_CHECK((long)g.tiles_m * g.tiles_n * g.nsplit < (1L << 30), SCP_ERR_SHAPE, "scp_gemm_q8: too many tiles");
  g.group = tile_group(g);
  hipStream_t st = (hipStream_t)stream_;
  if (g.nsplit == 1) {
    g.C = (float*)C;
    if (c_bf16) return launch8<true, true, EPI_DIRECT, true, __bf16>(g, st);
    return launch8<true, true, EPI_DIRECT, true, float>(g, st);
  }
  SCP_CHECK(ws, SCP_ERR_ARG, "scp_gemm_q8: this shape runs as %d K-ranges and needs the workspace of scp_gemm_q8_ws_floats", g.nsplit);
  g.C = ws;
  const int rc = launch8<true, true, EPI_SLAB, true, float>(g, st);
  if (rc) return rc;
  return c_bf16 ? reduce_slabs(g, ws, nullptr, (__bf16*)C, st) : reduce_slabs(g, ws, nullptr, (float*)C, st);
}
