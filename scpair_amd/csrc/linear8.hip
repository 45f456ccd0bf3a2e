// A Linear layer that keeps its input as an 8-bit checkpoint (ckpt8.hip): everything a call launches, one C entry forward
// and one backward.
//
//   y = x W^T + b          dx = dy W          dW = dy^T v,  v the values of x's codes          db = sum over the rows of dy
//
// Operands are bf16, sums fp32.  fp32 tensors in the fp32-equivalent precision (ns 3) are taken apart into three bf16 terms
// each, f = h + m + l (24 bits), and a product keeps the six term pairs of weight 2^-16 and more.  The pairs are laid out as
// six column blocks of one long product -- first operand (h h m h m l), second (h m h l m h) -- so the matrix kernels know
// nothing of them.  v is exact in one term: dW takes three pairs, read out of dy's blocks 0, 2 and 5.
//
// Two matrix kernels: the wide one (wgemm.hip, 256 x 256 tiles) where its tiles fill the chip, and the one below (64 x 64 or
// 128 x 128 tiles, several K-ranges) for the minibatch sizes, where 256 x 256 leaves most CUs idle.
#include <stdlib.h>
#include "ckpt8.h"
#include "common.h"
#include "scpair_hip.h"

namespace {

typedef __attribute__((ext_vector_type(4))) short short4_;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;

// ---------------------------------------------------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------------------------------------------------
// term of each of the six blocks, first and second operand
__device__ constexpr int BLK_A[6] = {0, 0, 1, 0, 1, 2};
__device__ constexpr int BLK_B[6] = {0, 1, 0, 2, 1, 0};

enum { LAY_ONE = 0, LAY_COLS_A = 1, LAY_COLS_B = 2, LAY_ROWS_B = 3 };

// 8 columns of one row written as bf16: one copy, or six blocks side by side ([rows][6 w]) or below each other ([6 hb][w])
template <int LAY>
__device__ __forceinline__ void put8(__bf16* __restrict__ dst, long row, int col, int w, long hb, const float* f) {
  if constexpr (LAY == LAY_ONE) {
    store8<__bf16>(dst + row * w, col, w, f);
  } else {
    float t[3][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      __bf16 s[3];
      bf16_split<3>(f[i], s);
#pragma unroll
      for (int p = 0; p < 3; p++) t[p][i] = (float)s[p];
    }
#pragma unroll
    for (int b = 0; b < 6; b++) {
      const int p = LAY == LAY_COLS_A ? BLK_A[b] : BLK_B[b];
      if constexpr (LAY == LAY_ROWS_B)
        store8<__bf16>(dst + (b * hb + row) * w, col, w, t[p]);
      else
        store8<__bf16>(dst + row * (6L * w) + b * w, col, w, t[p]);
    }
  }
}

// src [rows][lds] -> dst in the given layout, w = cols rounded up to 8, zeros behind cols; rows .. hb are zero rows
// (LAY_ROWS_B).  PACK: also the 8-bit checkpoint of src.
template <typename T, int LAY, bool PACK>
__global__ __launch_bounds__(256) void lin_prep_kernel(const T* __restrict__ src, long lds, Shape8 s, long src_rows,
                                                       __bf16* __restrict__ dst, int w, long hb, int8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ steps) {
  FOR_CHUNKS(s) {
    const int col = ch * 8;
    float f[8];
    load8<T>(src + (row < src_rows ? row : 0) * lds, col, row < src_rows ? s.cols : 0, f);
    if constexpr (PACK) {
      unsigned step;
      const uint2 c = quantise(f, step);
      *(uint2*)(codes + row * s.ld + col) = c;
      if ((ch & 7) == 0) steps[row * (s.ld >> 6) + (ch >> 3)] = (uint8_t)step;
    }
    if (col < w) put8<LAY>(dst, row, col, w, hb, f);
  }
}

// dy: bf16 blocks (DST) and partial column sums part[gridDim.y][cols] (null: none) in one pass.  A workgroup takes 512 columns,
// 8 per lane, and every gridDim.y-th group of four rows, a row a wave, four rows in flight.
template <typename T, int LAY, bool DST>
__global__ __launch_bounds__(256) void lin_dy_kernel(const T* __restrict__ x, long ldx, long rows, int cols,
                                                     __bf16* __restrict__ dst, int w, float* __restrict__ part) {
  __shared__ float buf[3][8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 512 + lane * 8;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < cols) {
    const long step = (long)gridDim.y * 4;
    long r = (long)blockIdx.y * 4 + wave;
    for (; r + 3 * step < rows; r += 4 * step) {
      float f[4][8];
#pragma unroll
      for (int u = 0; u < 4; u++) load8<T>(x + (r + u * step) * ldx, col, cols, f[u]);
#pragma unroll
      for (int u = 0; u < 4; u++) {
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] += f[u][i];
        if (DST) put8<LAY>(dst, r + u * step, col, w, 0, f[u]);
      }
    }
    for (; r < rows; r += step) {
      float f[8];
      load8<T>(x + r * ldx, col, cols, f);
#pragma unroll
      for (int i = 0; i < 8; i++) acc[i] += f[i];
      if (DST) put8<LAY>(dst, r, col, w, 0, f);
    }
  }
  if (!part) return;
  if (wave) {
#pragma unroll
    for (int i = 0; i < 8; i++) buf[wave - 1][i][lane] = acc[i];
  }
  __syncthreads();
  if (wave == 0 && col < cols) {
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] += buf[0][i][lane] + buf[1][i][lane] + buf[2][i][lane];
    store8<float>(part + (long)blockIdx.y * cols, col, cols, acc);
  }
}
__global__ __launch_bounds__(256) void lin_db_kernel(const float* __restrict__ part, int n, int cols, float* __restrict__ out) {
  __shared__ double buf[16][17];
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4, col = blockIdx.x * 16 + cx;
  double s = 0.0;
  if (col < cols)
    for (int r = ry; r < n; r += 16) s += (double)part[(long)r * cols + col];
  buf[ry][cx] = s;
  __syncthreads();
  if (ry || col >= cols) return;
  for (int y = 1; y < 16; y++) s += buf[y][cx];
  out[col] = (float)s;
}

// ---------------------------------------------------------------------------------------------------------------------
// the matrix kernel of the smaller shapes
// ---------------------------------------------------------------------------------------------------------------------
// C[m][n] = sum_k A(m,k) B(n,k) (+ bias[n]).  "row" operands [rows][ld] with k contiguous, "col" operands [K][ld] with the
// rows contiguous, B also as an 8-bit checkpoint (col).  A workgroup of four waves (2 x 2) computes TS x TS over its K-range,
// 64 k per step.  Tiles come with 16-byte buffer loads, DEPTH steps ahead, into registers, then LDS (two stages, one barrier
// a step); images as in wgemm.hip: row image 128-byte rows with the 16-byte chunks swizzled, col image read with the
// transposing ds_read_b64_tr_b16.  Every buffer descriptor covers one tile's rows (row operands) or one K-step's rows (col
// operands): offsets stay small whatever the operand's size, and the range check supplies the zeros behind the last k row.
struct LgArgs {
  const __bf16* A;
  const void* B;
  const uint8_t* steps;
  void* C;             // [M][ldc], or slabs [planes * nsplit][M][ldc] fp32
  const float* bias;
  long lda, ldb, ldc;
  int M, N, K;
  int tiles_m, tiles_n, nsplit, per_split;   // K-ranges of per_split steps
  int planes, plane_off[3];                  // A's column blocks that are summed up
};

template <int TS> __device__ __forceinline__ int lg_col_off(int k, int m) {
  constexpr int SEG = TS / 32;       // 64-byte segments of an image row
  const int sw = TS == 128 ? (k & 3) : ((k >> 1) & 1);
  return k * (TS * 2) + (((m >> 5) ^ sw) & (SEG - 1)) * 64 + ((m & 31) << 1);
}
__device__ __forceinline__ int lg_row_off(int r, int ch) { return r * 128 + ((ch ^ ((r >> 1) & 7)) << 4); }

template <int TS, bool COL>
__device__ __forceinline__ bf16x8 lg_frag(const unsigned char* img, int r0, int s, int lane) {
  if constexpr (!COL) {
    return *(const bf16x8*)(img + lg_row_off(r0 + (lane & 31), 2 * s + (lane >> 5)));
  } else {
    const int g = lane >> 5, mb = ((lane >> 4) & 1) * 16, q = (lane & 15) >> 2, p = lane & 3;
    const int k = 16 * s + 8 * g + q, m = r0 + mb + 4 * p;
    typedef __attribute__((address_space(3))) short4_ lds_s4;
    union { short4_ h[2]; bf16x8 v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(img + lg_col_off<TS>(k, m)));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(img + lg_col_off<TS>(k + 4, m)));
    return u.v;
  }
}

enum { OP_ROW = 0, OP_COL = 1, OP_Q8 = 2 };

// One operand's tiles: global -> registers -> LDS.  What a lane adds to the descriptor's base does not change from step to
// step; the step itself moves the scalar offset (row operands) or the descriptor (col operands).
template <int TS, int OP>
struct Tile {
  static constexpr int EB = OP == OP_Q8 ? 1 : 2;                   // bytes per element
  static constexpr int NC = TS * 64 * EB / 16 / 256;               // 16-byte chunks per thread and step
  static constexpr int CPR = OP == OP_ROW ? 8 : TS * EB / 16;      // chunks per image row
  static constexpr int RPI = 256 / CPR;                            // image rows per round of the 256 threads
  struct Reg {
    u32x4 v[NC];
    unsigned step[OP == OP_Q8 ? NC : 1];
  };
  const unsigned char* base;     // first byte of the tile's rows (row) / of k row 0 (col)
  const uint8_t* steps;
  long ld;
  int kp, K, tail;               // K rounded up to 8 / K / bytes of a last k row, from the tile's first column on
  int bytes;                     // row operands: extent of the tile's rows
  int voff[NC], soff[OP == OP_Q8 ? NC : 1], lds[NC];

  __device__ __forceinline__ void init(const void* p, const uint8_t* st, long ld_, int origin, int extent, int K_) {
    ld = ld_;
    K = K_;
    kp = (K + 7) & ~7;
    steps = st;
    base = (const unsigned char*)p + (OP == OP_ROW ? (long)origin * ld * 2 : (long)origin * EB);
    bytes = (int)(min(TS, extent - origin) * ld * 2);
    // a k row is read up to its last column rounded up to a chunk, the last one of the operand no further
    tail = (int)((OP == OP_Q8 ? ld : (long)((extent + 7) & ~7)) - origin) * EB;
    const int r = threadIdx.x / CPR, c = threadIdx.x % CPR;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      voff[i] = (int)((r + RPI * i) * ld * EB) + 16 * c;
      lds[i] = OP == OP_ROW ? lg_row_off(r + RPI * i, c) : lg_col_off<TS>(r + RPI * i, 16 / EB * c);
      if constexpr (OP == OP_Q8) soff[i] = (int)((r + RPI * i) * (ld >> 6)) + ((origin + 16 * c) >> 6);
    }
  }
  __device__ __forceinline__ void load(Reg& r, int kt, bool live) const {
    const int k0 = kt * 64;
    if constexpr (OP == OP_ROW) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, live ? bytes : 0, 0x00020000);
      if (k0 + 64 <= kp) {
#pragma unroll
        for (int i = 0; i < NC; i++) r.v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, voff[i], 2 * k0, 0);
      } else {         // the step that K ends in: chunks behind it would run into the next row
        const bool in = k0 + 8 * (int)(threadIdx.x % CPR) < kp;
#pragma unroll
        for (int i = 0; i < NC; i++)
          r.v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, in ? voff[i] + 2 * k0 : (int)0x80000000u, 0, 0);
      }
    } else {
      const int kr = live ? min(64, K - k0) : 0;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(base + (long)k0 * ld * EB), 0, kr > 0 ? (int)((kr - 1) * ld * EB) + tail : 0, 0x00020000);
#pragma unroll
      for (int i = 0; i < NC; i++) r.v[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, voff[i], 0, 0);
      if constexpr (OP == OP_Q8) {
        const long ls = ld >> 6;
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(steps + k0 * ls), 0, kr > 0 ? (int)(kr * ls) : 0, 0x00020000);
#pragma unroll
        for (int i = 0; i < NC; i++) r.step[i] = __builtin_amdgcn_raw_buffer_load_b8(rq, soff[i], 0, 0);
      }
    }
  }
  __device__ __forceinline__ void store(const Reg& r, unsigned char* img) const {
#pragma unroll
    for (int i = 0; i < NC; i++) {
      if constexpr (OP != OP_Q8) {
        *(u32x4*)(img + lds[i]) = r.v[i];
      } else {
        const float step = q8_step(r.step[i]), off = -128.f * step;
        bf16x8 v[2];
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const unsigned u = r.v[i][w] ^ 0x80808080u;      // code + 128: unsigned bytes convert in one instruction
#pragma unroll
          for (int b = 0; b < 4; b++) v[w >> 1][(w & 1) * 4 + b] = (__bf16)fmaf((float)((u >> (8 * b)) & 0xffu), step, off);
        }
        *(bf16x8*)(img + lds[i]) = v[0];
        *(bf16x8*)(img + lds[i] + 16) = v[1];
      }
    }
  }
};

template <int TS, int OPA, int OPB, typename CT>
__global__ __launch_bounds__(256, TS == 64 ? 4 : 2) void lgemm_kernel(LgArgs g) {
  constexpr int NI = TS / 64, WT = TS / 2, IMG = TS * 128, DEPTH = TS == 64 ? 4 : 2;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  // ids b, b + 8, b + 16 .. share an XCD: give them neighbouring tiles
  const int per_z = g.tiles_m * g.tiles_n, total = per_z * g.nsplit * g.planes, per_xcd = (total + 7) >> 3;
  const int lid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (lid >= total || (int)(blockIdx.x >> 3) >= per_xcd) return;
  // and those in blocks of 8 tile rows, walked column by column: the tiles at work on an XCD share a few rows and columns
  const int z = lid / per_z, t = lid - z * per_z, grp = t / (8 * g.tiles_n), in = t - grp * 8 * g.tiles_n;
  const int gh = min(8, g.tiles_m - 8 * grp), tn = in / gh, tm = 8 * grp + in - tn * gh;
  const int m0 = tm * TS, n0 = tn * TS, plane = z / g.nsplit;
  const int kt0 = (z % g.nsplit) * g.per_split, kt1 = min((g.K + 63) / 64, kt0 + g.per_split);

  Tile<TS, OPA> ta;
  Tile<TS, OPB> tb;
  ta.init(g.A + g.plane_off[plane], nullptr, g.lda, m0, g.M, g.K);
  tb.init(g.B, g.steps, g.ldb, n0, g.N, g.K);
  typename Tile<TS, OPA>::Reg ra[DEPTH];
  typename Tile<TS, OPB>::Reg rb[DEPTH];
  f32x16 acc[NI][NI];
#pragma unroll
  for (int i = 0; i < NI; i++)
#pragma unroll
    for (int j = 0; j < NI; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

#pragma unroll
  for (int d = 0; d < DEPTH; d++) {
    ta.load(ra[d], kt0 + d, kt0 + d < kt1);
    tb.load(rb[d], kt0 + d, kt0 + d < kt1);
  }
  ta.store(ra[0], smem);
  tb.store(rb[0], smem + IMG);
  __syncthreads();
  for (int kt = kt0; kt < kt1; kt += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      if (kt + d < kt1) {            // uniform
        const unsigned char* ia = smem + (d & 1) * 2 * IMG;
        const unsigned char* ib = ia + IMG;
        ta.load(ra[d], kt + d + DEPTH, kt + d + DEPTH < kt1);
        tb.load(rb[d], kt + d + DEPTH, kt + d + DEPTH < kt1);
#pragma unroll
        for (int s = 0; s < 4; s++) {
          bf16x8 fa[NI], fb[NI];
#pragma unroll
          for (int i = 0; i < NI; i++) fa[i] = lg_frag<TS, OPA != OP_ROW>(ia, wm * WT + 32 * i, s, lane);
#pragma unroll
          for (int j = 0; j < NI; j++) fb[j] = lg_frag<TS, OPB != OP_ROW>(ib, wn * WT + 32 * j, s, lane);
#pragma unroll
          for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < NI; j++) acc[i][j] = mfma32(fa[i], fb[j], acc[i][j]);
        }
        unsigned char* na = smem + ((d + 1) & 1) * 2 * IMG;
        ta.store(ra[(d + 1) % DEPTH], na);
        tb.store(rb[(d + 1) % DEPTH], na + IMG);
        __syncthreads();
      }
    }
  }

  CT* C = (CT*)g.C + (long)z * g.M * g.ldc;
#pragma unroll
  for (int j = 0; j < NI; j++) {
    const int n = n0 + wn * WT + 32 * j + (lane & 31);
    if (n >= g.N) continue;
    const float bn = g.bias ? g.bias[n] : 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int m = m0 + wm * WT + 32 * i + acc_row(e, lane);
        if (m < g.M) C[(long)m * g.ldc + n] = (CT)(acc[i][j][e] + bn);
      }
  }
}

// C = sum of n slabs in slab order, + bias.  Slabs and C are [M][N], contiguous: 4 elements a thread.
template <typename CT>
__global__ __launch_bounds__(256) void lin_sum_kernel(const float* __restrict__ slabs, int n, long MN, int N,
                                                      const float* __restrict__ bias, CT* __restrict__ C) {
  const long i0 = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i0 >= MN) return;
  float s[4];
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  if (i0 + 4 <= MN) {
    f4u a = *(const f4u*)(slabs + i0);
    for (int z = 1; z < n; z++) a += *(const f4u*)(slabs + z * MN + i0);
#pragma unroll
    for (int t = 0; t < 4; t++) s[t] = a[t];
  } else {
    for (int t = 0; t < 4; t++) {
      s[t] = 0.f;
      for (int z = 0; z < n && i0 + t < MN; z++) s[t] += slabs[z * MN + i0 + t];
    }
  }
#pragma unroll
  for (int t = 0; t < 4; t++)
    if (i0 + t < MN) C[i0 + t] = (CT)(bias ? s[t] + bias[(i0 + t) % N] : s[t]);
}

// ---------------------------------------------------------------------------------------------------------------------
// plans: what a call launches and where its workspace lies, a function of the shape alone
// ---------------------------------------------------------------------------------------------------------------------
constexpr long WIDE_BYTES = (1L << 31) - 65536;      // operand extent that the wide kernel addresses

long align256(long b) { return (b + 255) & ~255L; }
int up8(int n) { return (n + 7) & ~7; }

struct Gemm {
  int ts;              // 64 or 128: lgemm tiles; 256: the wide kernel
  int nsplit, slabs;   // K-ranges; slabs of the result in the workspace (0: written directly)
  long ws;             // workspace bytes
};

// Tile and K-ranges of one product of `planes` column blocks: the cheapest by a model in microseconds.  A step of 64 k with
// w workgroups per CU took, measured over products from 300^3 to 16384 x 4096^2: 0.25 + 0.2 w at 64 x 64, 1.15 (w = 1) or
// 0.70 w at 128 x 128, 2.3 w at 256 x 256; slabs are written and read at 7.5 TB/s, and a launch costs 3.5 us.
Gemm pick(long M, int N, long K, int planes, bool wide_ok, int wide_ns, long wide_ws) {
  Gemm best = {256, 1, 0, wide_ws};
  const long nk = (K + 63) / 64;
  const double mn = (double)M * N;
  double best_us = 1e30;
  if (wide_ok) {
    const long tiles = ((M + 255) / 256) * ((N + 255) / 256) * wide_ns;
    best_us = planes * ((tiles + 255) / 256 * 2.3 * ((nk + wide_ns - 1) / wide_ns) + 3.5);
    if (wide_ns > 1) best_us += planes * (mn * 4 * (2 * wide_ns + 1) / 7.5e6 + 3.5);
    if (planes > 1) best_us += mn * 4 * (2 * planes + 1) / 7.5e6 + 3.5;
  }
  for (int ts = 64; ts <= 128; ts += 64) {
    const long tiles = ((M + ts - 1) / ts) * ((N + ts - 1) / ts) * planes;
    if (tiles >= 1L << 24) continue;
    for (int ns = 1; ns <= 64; ns *= 2) {
      if (ns > 1 && nk / ns < 4) break;
      const double w = (double)((tiles * ns + 255) / 256);
      double us = 3.5 + (nk + ns - 1) / ns * (ts == 64 ? 0.25 + 0.2 * w : w == 1 ? 1.15 : 0.7 * w);
      if (ns * planes > 1) us += mn * 4 * (2 * ns * planes + 1) / 7.5e6 + 3.5;
      if (us < best_us) {
        best_us = us;
        best.ts = ts;
        best.nsplit = ns;
        best.slabs = ns * planes > 1 ? ns * planes : 0;
        best.ws = (long)best.slabs * M * N * 4;
      }
    }
  }
#ifdef LIN8_TUNE
  if (const char* e = getenv("LIN8_TS")) {
    best.ts = atoi(e);
    best.nsplit = best.ts == 256 ? 1 : atoi(getenv("LIN8_NS"));
    best.slabs = best.ts != 256 && best.nsplit * planes > 1 ? best.nsplit * planes : 0;
    best.ws = best.ts == 256 ? wide_ws : (long)best.slabs * M * N * 4;
  }
#endif
  return best;
}

struct Plan {
  int np;                    // column blocks of an fp32 operand: 6 (ns 3), else 1
  int Kp, Np;
  bool x_direct, w_direct, dy_direct;
  long a_off, b_off, part_off, g_off, total;   // workspace: prepared operands, column sums, slabs
  int parts;
  Gemm y, dx, dw;
};

int colsum_parts(long rows, int cols) {
  const long groups = (rows + 3) / 4, cols_wg = (cols + 511) / 512, cap = cols_wg < 32 ? 1024 / cols_wg : 32;
  return (int)(groups < cap ? groups : cap);
}

void common_plan(const ScpLinear8& a, Plan& p) {
  p.np = !a.x_bf16 && a.ns == 3 ? 6 : 1;
  p.Kp = up8(a.K);
  p.Np = up8(a.N);
  p.w_direct = a.w_bf16 && a.K % 8 == 0 && ((uintptr_t)a.W & 15) == 0;
}

int wide_splits(long M, int N, long K) { return scp_gemm_bf16_nsplit((int)M, N, (int)K); }

long wide_ws_rows(const Plan& p, long M, int N, long K, long lda) {
  const long piece = WIDE_BYTES / (2 * lda);
  const long a = scp_gemm_bf16_ws_floats((int)(M < piece ? M : piece), N, (int)K, N);
  const long b = M > piece ? scp_gemm_bf16_ws_floats((int)(M % piece), N, (int)K, N) : 0;    // the last piece may split K
  return (a > b ? a : b) * 4;
}

Plan plan_fwd(const ScpLinear8& a) {
  Plan p = {};
  common_plan(a, p);
  p.x_direct = a.x_bf16 && a.K % 8 == 0 && a.ldx % 8 == 0 && a.ldx >= a.K && ((uintptr_t)a.x & 15) == 0;
  const long KK = (long)p.np * p.Kp;
  long o = 0;
  p.a_off = o;
  if (!p.x_direct) o += align256(a.M * KK * 2);
  p.b_off = o;
  if (!p.w_direct) o += align256((long)a.N * KK * 2);
  const bool ok = ((long)a.N + 192) * KK * 2 < WIDE_BYTES;
  p.y = pick(a.M, a.N, KK, 1, ok, wide_splits(a.M, a.N, KK), ok ? wide_ws_rows(p, a.M, a.N, KK, p.x_direct ? a.ldx : KK) : 0);
  p.g_off = o;
  p.total = o + align256(p.y.ws);
  return p;
}

Plan plan_bwd(const ScpLinear8& a) {
  Plan p = {};
  common_plan(a, p);
  p.dy_direct = a.x_bf16 && a.N % 8 == 0 && a.lddy == a.N && ((uintptr_t)a.dy & 15) == 0;
  const long NN = (long)p.np * p.Np;
  const bool need_dy = a.dx || a.dW;
  long o = 0;
  p.a_off = o;
  if (need_dy && !p.dy_direct) o += align256(a.M * NN * 2);
  p.b_off = o;
  if (a.dx && !p.w_direct) o += align256((p.np == 1 ? (long)a.N : NN) * p.Kp * 2);
  p.part_off = o;
  p.parts = colsum_parts(a.M, a.N);
  if (a.db) o += align256((long)p.parts * a.N * 4);
  p.g_off = o;
  long g = 0;
  if (a.dx) {
    const long K2 = p.np == 1 ? a.N : NN;
    const bool ok = (K2 + 192) * p.Kp * 2 < WIDE_BYTES;
    p.dx = pick(a.M, a.K, K2, 1, ok, wide_splits(a.M, a.K, K2), ok ? wide_ws_rows(p, a.M, a.K, K2, p.dy_direct ? a.N : NN) : 0);
    g = p.dx.ws;
  }
  if (a.dW) {
    const int planes = p.np == 6 ? 3 : 1;
    const long ld8 = (a.K + 63) / 64 * 64L, lda = p.dy_direct ? a.N : NN;
    // the wide form runs once per plane, each into a slab of its own
    const long ws = scp_gemm_q8_ws_floats(a.N, a.K, (int)a.M, lda > ld8 ? lda : ld8, a.K) * 4;
    p.dw = pick(a.N, a.K, a.M, planes, true, wide_splits(a.N, a.K, a.M), align256(ws) + (planes > 1 ? 3L * a.N * a.K * 4 : 0));
    if (p.dw.ws > g) g = p.dw.ws;
  }
  p.total = p.g_off + align256(g);
  return p;
}

template <typename T, int LAY, bool PACK>
int prep(const void* src, long lds, long rows, int cols, long pad_rows, __bf16* dst, int w, int8_t* codes, uint8_t* steps,
         hipStream_t st) {
  Shape8 s;
  s.rows = pad_rows > rows ? pad_rows : rows;
  s.cols = cols;
  s.ld = (cols + 63) / 64 * 64;
  s.cpr = (PACK ? s.ld : w) / 8;
  const unsigned grid = grid_of(s);
  hipLaunchKernelGGL((lin_prep_kernel<T, LAY, PACK>), dim3(grid), dim3(256), 0, st, (const T*)src, lds, s, rows, dst, w, pad_rows,
                     codes, steps);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

int prep_w(const ScpLinear8& a, const Plan& p, bool rows_below, __bf16* dst, hipStream_t st) {
  if (a.w_bf16) return prep<__bf16, LAY_ONE, false>(a.W, a.K, a.N, a.K, 0, dst, p.Kp, nullptr, nullptr, st);
  if (p.np == 1) return prep<float, LAY_ONE, false>(a.W, a.K, a.N, a.K, 0, dst, p.Kp, nullptr, nullptr, st);
  if (rows_below) return prep<float, LAY_ROWS_B, false>(a.W, a.K, a.N, a.K, p.Np, dst, p.Kp, nullptr, nullptr, st);
  return prep<float, LAY_COLS_B, false>(a.W, a.K, a.N, a.K, 0, dst, p.Kp, nullptr, nullptr, st);
}

template <int TS, int OPA, int OPB, typename CT>
int launch_lg(const LgArgs& g, hipStream_t st) {
  constexpr size_t smem = 4 * TS * 128;
  static uint64_t done = 0;
  if (int rc = scp_set_smem((const void*)lgemm_kernel<TS, OPA, OPB, CT>, smem, &done)) return rc;
  const long total = (long)g.tiles_m * g.tiles_n * g.nsplit * g.planes;
  hipLaunchKernelGGL((lgemm_kernel<TS, OPA, OPB, CT>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(256), smem, st, g);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

// a product on the smaller tiles, C contiguous [M][N]
template <int OPA, int OPB>
int small_gemm(const Gemm& q, LgArgs g, int c_bf16, const float* bias, float* ws, hipStream_t st) {
  void* C = g.C;
  g.tiles_m = (g.M + q.ts - 1) / q.ts;
  g.tiles_n = (g.N + q.ts - 1) / q.ts;
  const int nk = (g.K + 63) / 64;
  g.per_split = (nk + q.nsplit - 1) / q.nsplit;
  g.nsplit = (nk + g.per_split - 1) / g.per_split;
  g.ldc = g.N;
  const int slabs = g.nsplit * g.planes;
  if (slabs > 1) g.C = ws;
  else g.bias = bias;
  const bool b16 = slabs == 1 && c_bf16;
  int rc = q.ts == 64 ? (b16 ? launch_lg<64, OPA, OPB, __bf16>(g, st) : launch_lg<64, OPA, OPB, float>(g, st))
                      : (b16 ? launch_lg<128, OPA, OPB, __bf16>(g, st) : launch_lg<128, OPA, OPB, float>(g, st));
  if (rc || slabs == 1) return rc;
  const long MN = (long)g.M * g.N;
  const dim3 grid((unsigned)((MN + 1023) / 1024));
  if (c_bf16) hipLaunchKernelGGL((lin_sum_kernel<__bf16>), grid, dim3(256), 0, st, ws, slabs, MN, g.N, bias, (__bf16*)C);
  else hipLaunchKernelGGL((lin_sum_kernel<float>), grid, dim3(256), 0, st, ws, slabs, MN, g.N, bias, (float*)C);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

// out[M][N] = A B^T (b_col 0) or A B (b_col 1), + bias.  The wide kernel addresses its operands with 31 bits: a longer batch
// runs in pieces.
int rows_product(const Gemm& q, int b_col, long M, int N, long K, const __bf16* A, long lda, const __bf16* B, long ldb, void* C,
                 int c_bf16, const float* bias, float* ws, hipStream_t st) {
  const long piece = q.ts == 256 ? WIDE_BYTES / (2 * lda) : 1L << 30;
  for (long r = 0; r < M; r += piece) {
    const int m = (int)(M - r < piece ? M - r : piece);
    void* c = c_bf16 ? (void*)((__bf16*)C + r * N) : (void*)((float*)C + r * N);
    int rc;
    if (q.ts == 256) {
      rc = scp_gemm_rows(b_col, m, N, (int)K, A + r * lda, lda, B, ldb, c, c_bf16, N, bias, ws, st);
    } else {
      LgArgs g = {};
      g.A = A + r * lda; g.B = B; g.C = c;
      g.lda = lda; g.ldb = ldb;
      g.M = m; g.N = N; g.K = (int)K;
      g.planes = 1;
      rc = b_col ? small_gemm<OP_ROW, OP_COL>(q, g, c_bf16, bias, ws, st) : small_gemm<OP_ROW, OP_ROW>(q, g, c_bf16, bias, ws, st);
    }
    if (rc) return rc;
  }
  return SCP_OK;
}

// dy's blocks (write) and, if asked for, its column sums
int dy_pass(const ScpLinear8& a, const Plan& p, bool write, hipStream_t st) {
  char* ws = (char*)a.ws;
  __bf16* dst = write ? (__bf16*)(ws + p.a_off) : nullptr;
  float* part = a.db ? (float*)(ws + p.part_off) : nullptr;
  const dim3 grid((a.N + 511) / 512, p.parts);
#define DY(T, LAY, DST) \
  hipLaunchKernelGGL((lin_dy_kernel<T, LAY, DST>), grid, dim3(256), 0, st, (const T*)a.dy, a.lddy, a.M, a.N, dst, p.Np, part)
  if (a.x_bf16 && !write) DY(__bf16, LAY_ONE, false);
  else if (a.x_bf16) DY(__bf16, LAY_ONE, true);
  else if (!write) DY(float, LAY_ONE, false);
  else if (p.np == 1) DY(float, LAY_ONE, true);
  else DY(float, LAY_COLS_A, true);
#undef DY
  SCP_LAUNCH_CHECK();
  if (a.db) {
    hipLaunchKernelGGL(lin_db_kernel, dim3((a.N + 15) / 16), dim3(256), 0, st, part, p.parts, a.N, a.db);
    SCP_LAUNCH_CHECK();
  }
  return SCP_OK;
}

// dW = dy^T v; A: dy's blocks
int weight_product(const ScpLinear8& a, const Plan& p, const __bf16* A, long lda, float* ws, hipStream_t st) {
  const int planes = p.np == 6 ? 3 : 1;
  const int off[3] = {0, 2 * p.Np, 5 * p.Np};
  if (p.dw.ts == 256) {
    if (planes == 1) return scp_gemm_q8(a.N, a.K, (int)a.M, A, lda, a.codes, a.steps, a.dW, a.w_bf16, a.K, ws, st);
    const long NK = (long)a.N * a.K;
    float* slabs = ws + (p.dw.ws - 3 * NK * 4) / 4;
    for (int i = 0; i < 3; i++)
      if (int rc = scp_gemm_q8(a.N, a.K, (int)a.M, A + off[i], lda, a.codes, a.steps, slabs + i * NK, 0, a.K, ws, st)) return rc;
    hipLaunchKernelGGL((lin_sum_kernel<float>), dim3((unsigned)((NK + 1023) / 1024)), dim3(256), 0, st, slabs, 3, NK, a.K, nullptr,
                       (float*)a.dW);
    SCP_LAUNCH_CHECK();
    return SCP_OK;
  }
  LgArgs g = {};
  g.A = A; g.B = a.codes; g.steps = a.steps; g.C = a.dW;
  g.lda = lda; g.ldb = (a.K + 63) / 64 * 64;
  g.M = a.N; g.N = a.K; g.K = (int)a.M;
  g.planes = planes;
  for (int i = 0; i < 3; i++) g.plane_off[i] = off[i];
  return small_gemm<OP_COL, OP_Q8>(p.dw, g, a.w_bf16, nullptr, ws, st);
}

int check_args(const ScpLinear8* a, const char* who) {
  SCP_CHECK(a, SCP_ERR_ARG, "%s: null argument block", who);
  SCP_CHECK(a->M > 0 && a->N > 0 && a->K > 0, SCP_ERR_ARG, "%s: M, N, K must be positive (%ld, %d, %d)", who, a->M, a->N, a->K);
  SCP_CHECK(a->M < (1L << 30) && a->K <= (1 << 20) && a->N <= (1 << 20), SCP_ERR_SHAPE,
            "%s: at most 2^30 - 1 rows and 2^20 inputs or outputs (got %ld, %d, %d)", who, a->M, a->K, a->N);
  SCP_CHECK(((long)(a->N > a->K ? a->N : a->K) + 256) * ((long)(a->N > a->K ? a->K : a->N) + 256) * 2 < (1L << 31) - 65536,
            SCP_ERR_SHAPE, "%s: a weight of %d x %d passes 2 GiB in bf16", who, a->N, a->K);
  SCP_CHECK(a->x_bf16 || !a->w_bf16, SCP_ERR_ARG, "%s: an fp32 input needs an fp32 weight", who);
  SCP_CHECK(a->ns == 1 || a->ns == 3, SCP_ERR_ARG, "%s: ns must be 1 or 3", who);
  SCP_CHECK(!a->codes == !a->steps && ((uintptr_t)a->codes & 15) == 0, SCP_ERR_ARG, "%s: codes (16-byte aligned) and steps belong together", who);
  return SCP_OK;
}

}  // namespace

extern "C" long scp_linear8_fwd_ws(const ScpLinear8* a) { return check_args(a, "scp_linear8_fwd") ? -1 : plan_fwd(*a).total; }
extern "C" long scp_linear8_bwd_ws(const ScpLinear8* a) { return check_args(a, "scp_linear8_bwd") ? -1 : plan_bwd(*a).total; }

extern "C" int scp_linear8_fwd(const ScpLinear8* a_, void* stream) {
  if (int rc = check_args(a_, "scp_linear8_fwd")) return rc;
  const ScpLinear8& a = *a_;
  SCP_CHECK(a.x && a.W && a.y && a.ldx >= 0, SCP_ERR_ARG, "scp_linear8_fwd: null pointer or negative row stride");
  const Plan p = plan_fwd(a);
  SCP_CHECK(a.ws || !p.total, SCP_ERR_ARG, "scp_linear8_fwd: needs the workspace of scp_linear8_fwd_ws");
  SCP_CHECK(((uintptr_t)a.ws & 255) == 0, SCP_ERR_ARG, "scp_linear8_fwd: the workspace must be 256-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)a.ws;
  const long KK = (long)p.np * p.Kp;
  int rc;
  const __bf16* A = (const __bf16*)a.x;
  long lda = a.ldx;
  if (p.x_direct) {
    rc = a.codes ? scp_pack8(a.x, 1, a.ldx, a.M, a.K, a.codes, a.steps, stream) : SCP_OK;
  } else {
    __bf16* dst = (__bf16*)(ws + p.a_off);
    A = dst;
    lda = KK;
#define PREP_X(T, LAY)                                                                                     \
  (a.codes ? prep<T, LAY, true>(a.x, a.ldx, a.M, a.K, 0, dst, p.Kp, a.codes, a.steps, st)                   \
           : prep<T, LAY, false>(a.x, a.ldx, a.M, a.K, 0, dst, p.Kp, nullptr, nullptr, st))
    rc = a.x_bf16 ? PREP_X(__bf16, LAY_ONE) : p.np == 1 ? PREP_X(float, LAY_ONE) : PREP_X(float, LAY_COLS_A);
#undef PREP_X
  }
  if (rc) return rc;
  const __bf16* B = (const __bf16*)a.W;
  if (!p.w_direct) {
    B = (const __bf16*)(ws + p.b_off);
    if ((rc = prep_w(a, p, false, (__bf16*)(ws + p.b_off), st))) return rc;
  }
  return rows_product(p.y, 0, a.M, a.N, p.np == 1 ? a.K : KK, A, lda, B, p.w_direct ? a.K : KK, a.y, a.x_bf16, a.b,
                      (float*)(ws + p.g_off), st);
}

extern "C" int scp_linear8_bwd(const ScpLinear8* a_, void* stream) {
  if (int rc = check_args(a_, "scp_linear8_bwd")) return rc;
  const ScpLinear8& a = *a_;
  SCP_CHECK(a.dy && a.lddy >= 0 && (!a.dx || a.W) && (!a.dW || a.codes), SCP_ERR_ARG,
            "scp_linear8_bwd: null pointer or negative row stride");
  const Plan p = plan_bwd(a);
  SCP_CHECK(a.ws || !p.total, SCP_ERR_ARG, "scp_linear8_bwd: needs the workspace of scp_linear8_bwd_ws");
  SCP_CHECK(((uintptr_t)a.ws & 255) == 0, SCP_ERR_ARG, "scp_linear8_bwd: the workspace must be 256-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)a.ws;
  float* gws = (float*)(ws + p.g_off);
  const long NN = (long)p.np * p.Np;
  const bool need_dy = a.dx || a.dW, write_dy = need_dy && !p.dy_direct;
  int rc;
  const __bf16* A = (const __bf16*)a.dy;
  long lda = a.N;
  if (write_dy) {
    A = (const __bf16*)(ws + p.a_off);
    lda = NN;
  }
  // The column sums come out of the pass that writes the operand's blocks; where none is needed, they come last, when the
  // products have left dy in the last-level cache (16384 x 4096 bf16: 43 us before them, 20 us after).
  if (write_dy && (rc = dy_pass(a, p, true, st))) return rc;
  if (a.dx) {
    const __bf16* B = (const __bf16*)a.W;
    if (!p.w_direct) {
      B = (const __bf16*)(ws + p.b_off);
      if ((rc = prep_w(a, p, true, (__bf16*)(ws + p.b_off), st))) return rc;
    }
    if ((rc = rows_product(p.dx, 1, a.M, a.K, p.np == 1 ? a.N : NN, A, lda, B, p.w_direct ? a.K : p.Kp, a.dx, a.x_bf16, nullptr, gws, st)))
      return rc;
  }
  if (a.dW && (rc = weight_product(a, p, A, lda, gws, st))) return rc;
  return a.db && !write_dy ? dy_pass(a, p, false, st) : SCP_OK;
}
