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
// Three matrix kernels: the wide one (wgemm.hip, 256 x 256 tiles) where its tiles fill the chip; 128 x 128 tiles below that;
// 64 x 64 tiles straight from the tensors, without prepared copies, for the minibatch sizes, where a launch counts as much as
// the product.  A cost model with measured rates chooses (step_us).
//
// Measured (products alone; in parentheses the library's on operands laid out for it): 16384 x 4096 x 4096 bf16 y 425-480
// (441), dx 425-485 (436), dW 427-510 us (554 with a bf16 operand), by box and clock; 1024 x 900 x 1800 fp32 39, 37 and 29 us (32, 31, 35, in fp32 without the
// checkpoint); 777 x 1801 x 901 bf16 25, 18, 16 us (19, 19, 19); 4096 x 4096 x 4096 fp32 y 806 (918).  The large ones are bound by the
// matrix pipes at the clock they hold (busy 70-73 % of the cycles, dW 67 %, at 1.5-1.8 GHz), the small ones by the latency of a tile's K-steps with one or two workgroups a CU.
#include <limits.h>
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
  // dgemm, beside the product: A's 8-bit checkpoint (row A), A's column sums [nsplit][M] (col A); null: not asked for
  int8_t* pack_codes;
  uint8_t* pack_steps;
  float* colsum;
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
        const float step = q8_step(r.step[i]);
        bf16x8 v[2];
#pragma unroll
        for (int w = 0; w < 4; w++) {
          __bf16 f[4];
          q8_values(r.v[i][w], step, f);
#pragma unroll
          for (int b = 0; b < 4; b++) v[w >> 1][(w & 1) * 4 + b] = f[b];
        }
        *(bf16x8*)(img + lds[i]) = v[0];
        *(bf16x8*)(img + lds[i] + 16) = v[1];
      }
    }
  }
};

// The workgroup's tile and K-range.  Ids b, b + 8, b + 16 .. share an XCD: they get neighbouring tiles, and those in blocks of
// 8 tile rows walked column by column, so that the tiles at work on an XCD share a few rows and columns.
__device__ __forceinline__ bool lg_tile(const LgArgs& g, int& tm, int& tn, int& z) {
  const int per_z = g.tiles_m * g.tiles_n, total = per_z * g.nsplit * g.planes, per_xcd = (total + 7) >> 3;
  const int lid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (lid >= total || (int)(blockIdx.x >> 3) >= per_xcd) return false;
  z = lid / per_z;
  const int t = lid - z * per_z, grp = t / (8 * g.tiles_n), in = t - grp * 8 * g.tiles_n, gh = min(8, g.tiles_m - 8 * grp);
  tn = in / gh;
  tm = 8 * grp + in - tn * gh;
  return true;
}

template <int OPA, int OPB, typename CT>
__global__ __launch_bounds__(256, 2) void lgemm_kernel(LgArgs g) {
  constexpr int TS = 128, NI = TS / 64, WT = TS / 2, IMG = TS * 128, DEPTH = 2;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  int tm, tn, z;
  if (!lg_tile(g, tm, tn, z)) return;
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

// ---------------------------------------------------------------------------------------------------------------------
// 64 x 64 tiles straight from the tensors
// ---------------------------------------------------------------------------------------------------------------------
// The same product on 64 x 64 tiles for what one call of minibatch size is made of.  The operands are read as they are --
// fp32 or bf16, any row stride, any alignment, any length -- and rounded (NP 1) or taken apart into three terms (NP 3) on the
// way into LDS: no prepared copies, a third of the bytes of the six-block layout through the caches, and a fragment that is
// in LDS serves every pair it belongs to.  Accesses are vectors of 8 elements without a test.  The step that K ends in is
// made apart, after the others, where a K that is no multiple of 64 or the last columns of a col operand need care: a vector
// that would pass the end goes element by element.  (In earlier steps a vector may run over the end of a k row, into the
// next one: rows are 8 elements at least and no closer than their length, checked on the host.  Those columns are not stored.)
template <typename T, int NP, bool COL>
struct DTile {
  typedef typename Vec8<T>::v V;
  typedef typename Vec8<T>::vu VU;
  struct Reg { V v[2]; };
  const T* base;
  long ld;
  int K, n;                 // n: columns from the tile's origin on (col operands)
  int start;                // first column or k of the lane's chunks
  unsigned voff[2];
  int lds[2];

  __device__ __forceinline__ void init(const void* p, const uint8_t*, long ld_, int origin, int extent, int K_) {
    ld = ld_;
    K = K_;
    n = extent - origin;
    base = (const T*)p + (COL ? (long)origin : (long)origin * ld);
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
    start = COL && 8 * c >= n ? 0 : 8 * c;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int q = r + 32 * i;
      voff[i] = (unsigned)((COL ? q : min(q, n - 1)) * ld) + start;      // rows behind the last: the last again
      lds[i] = COL ? lg_col_off<64>(q, 8 * c) : lg_row_off(q, c);
    }
  }
  __device__ __forceinline__ bool care() const { return (K & 63) || (COL && n < 64); }
  __device__ __forceinline__ void load(Reg& r, int kt, bool live) const {
    if (!live) return;        // uniform; r is not used then
    const T* p = base + (COL ? (long)kt * 64 * ld : (long)kt * 64);
#pragma unroll
    for (int i = 0; i < 2; i++) r.v[i] = *(const VU*)(p + voff[i]);
  }
  __device__ __forceinline__ void load_end(Reg& r, int kt) const {
    const int k0 = kt * 64;
    const T* p = base + (COL ? k0 * ld : (long)k0);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int have = COL ? (k0 + (int)(threadIdx.x >> 3) + 32 * i < K ? n - start : 0) : K - k0 - start;
      V v;
      if (have >= 8) {
        v = *(const VU*)(p + voff[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < have ? p[voff[i] + j] : (T)0.f;
      }
      r.v[i] = v;
    }
  }
  __device__ __forceinline__ void store(const Reg& r, unsigned char* img) const {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if constexpr (sizeof(T) == 2) {
        *(V*)(img + lds[i]) = r.v[i];
      } else {
        // the terms of bf16_split, two values at a time: a conversion instruction rounds and packs a pair
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        union { bf16x2 p[4]; bf16x8 v; } t[NP];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f32x2 f = {r.v[i][2 * j], r.v[i][2 * j + 1]};
#pragma unroll
          for (int q = 0; q < NP; q++) {
            t[q].p[j] = __builtin_convertvector(f, bf16x2);
            if (q + 1 < NP) f -= __builtin_convertvector(t[q].p[j], f32x2);
          }
        }
#pragma unroll
        for (int q = 0; q < NP; q++) *(bf16x8*)(img + q * 8192 + lds[i]) = t[q].v;
      }
    }
  }
};

// operand B: a DTile or an 8-bit checkpoint
template <typename TB, int PB, int OPB> struct BTile { typedef DTile<TB, PB, OPB == OP_COL> t; };
template <typename TB, int PB> struct BTile<TB, PB, OP_Q8> { typedef Tile<64, OP_Q8> t; };

// Two by-products come out of A's tiles while they are in registers, and save a launch and a pass each: a step of 64 k of a row
// operand is 8 lanes a group of the checkpoint, packed by the tile column kt mod tiles_n, so that no workgroup does it all; and
// the column sums of a col operand (db), by the first tile column.
template <typename TA, int PA, bool ACOL, typename TB, int PB, int OPB, typename CT>
__global__ __launch_bounds__(256, PA + PB > 2 || OPB == OP_ROW ? 3 : 4) void dgemm_kernel(LgArgs g) {
  typedef DTile<TA, PA, ACOL> TileA;
  typedef typename BTile<TB, PB, OPB>::t TileB;
  // one term each: two LDS stages, one barrier a step; three terms: one stage, so that three workgroups share a CU
  constexpr int STAGES = PA + PB == 2 ? 2 : 1, STAGE = (PA + PB) * 8192;
  constexpr int DEPTH = PA + PB > 2 ? 2 : sizeof(TA) + (OPB == OP_Q8 ? 1 : sizeof(TB)) <= 4 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) unsigned char smem[STAGES * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  int tm, tn, z;
  if (!lg_tile(g, tm, tn, z)) return;
  const int m0 = tm * 64, n0 = tn * 64;
  const int nk = (g.K + 63) / 64, kt0 = z * g.per_split, kt1 = min(nk, kt0 + g.per_split);

  TileA ta;
  TileB tb;
  ta.init(g.A, nullptr, g.lda, m0, g.M, g.K);
  tb.init(g.B, g.steps, g.ldb, n0, g.N, g.K);
  bool care = ta.care();
  if constexpr (OPB != OP_Q8) care = care || tb.care();      // (a checkpoint's rows are padded: its loads check themselves)
  const int ktv = kt1 - (care && kt1 == nk);                 // steps [kt0, ktv) in vectors
  // the pairs below the leading one are summed apart: their sum keeps its low bits
  f32x16 acc[PA == 3 ? 2 : 1];
#pragma unroll
  for (auto& q : acc)
#pragma unroll
    for (int e = 0; e < 16; e++) q[e] = 0.f;
  auto multiply = [&](const unsigned char* ia) {
    const unsigned char* ib = ia + PA * 8192;
#pragma unroll
    for (int s = 0; s < 4; s++) {
      bf16x8 fa[PA], fb[PB];
#pragma unroll
      for (int q = 0; q < PA; q++) fa[q] = lg_frag<64, ACOL>(ia + q * 8192, wm * 32, s, lane);
#pragma unroll
      for (int q = 0; q < PB; q++) fb[q] = lg_frag<64, OPB != OP_ROW>(ib + q * 8192, wn * 32, s, lane);
      if constexpr (PA == 3) {
#pragma unroll
        for (int w = 2; w > 0; w--)          // pairs of weight 2^-16, then 2^-8
#pragma unroll
          for (int q = 0; q < PB; q++)
            if (w - q >= 0 && w - q < PA) acc[1] = mfma32(fa[w - q], fb[q], acc[1]);
      }
      acc[0] = mfma32(fa[0], fb[0], acc[0]);
    }
  };

  const bool sums = ACOL && g.colsum && tn == 0;
  float cs[ACOL ? 8 : 1] = {};
  int next_pack = !ACOL && g.pack_codes ? kt0 + (tn - kt0 % g.tiles_n + g.tiles_n) % g.tiles_n : INT_MAX;
  // A's tile of step kt on its way into LDS
  auto put_a = [&](const typename TileA::Reg& r, int kt, unsigned char* img) {
    ta.store(r, img);
    if constexpr (ACOL) {
      if (sums) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < 8; j++) cs[j] += (float)r.v[i][j];
      }
    } else if (OPB == OP_ROW && kt == next_pack) {
      next_pack += g.tiles_n;
      const long ld8 = (long)nk * 64;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = (float)r.v[i][j];
        unsigned step;
        const uint2 c = quantise(f, step);
        const long m = m0 + (int)(threadIdx.x >> 3) + 32 * i;
        if (m < g.M) {
          *(uint2*)(g.pack_codes + m * ld8 + kt * 64 + 8 * (threadIdx.x & 7)) = c;
          if ((threadIdx.x & 7) == 0) g.pack_steps[m * nk + kt] = (uint8_t)step;
        }
      }
    }
  };

  if (kt0 < ktv) {
    typename TileA::Reg ra[DEPTH];
    typename TileB::Reg rb[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      ta.load(ra[d], kt0 + d, kt0 + d < ktv);
      tb.load(rb[d], kt0 + d, kt0 + d < ktv);
    }
    put_a(ra[0], kt0, smem);
    tb.store(rb[0], smem + PA * 8192);
    __syncthreads();
    for (int kt = kt0; kt < ktv; kt += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        if (kt + d < ktv) {            // uniform
          ta.load(ra[d], kt + d + DEPTH, kt + d + DEPTH < ktv);
          tb.load(rb[d], kt + d + DEPTH, kt + d + DEPTH < ktv);
          multiply(smem + (d % STAGES) * STAGE);
          if constexpr (STAGES == 1) __syncthreads();
          if (kt + d + 1 < ktv) {
            unsigned char* na = smem + ((d + 1) % STAGES) * STAGE;
            put_a(ra[(d + 1) % DEPTH], kt + d + 1, na);
            tb.store(rb[(d + 1) % DEPTH], na + PA * 8192);
          }
          __syncthreads();
        }
      }
    }
  }
  if (ktv < kt1) {
    typename TileA::Reg ra;
    typename TileB::Reg rb;
    ta.load_end(ra, ktv);
    if constexpr (OPB == OP_Q8) tb.load(rb, ktv, true);
    else tb.load_end(rb, ktv);
    put_a(ra, ktv, smem);
    tb.store(rb, smem + PA * 8192);
    __syncthreads();
    multiply(smem);
  }
  if constexpr (ACOL) {
    if (sums) {                  // uniform
      __syncthreads();
      float* p = (float*)smem;   // [32 rows of the tile][64 columns]
#pragma unroll
      for (int j = 0; j < 8; j++) p[(threadIdx.x >> 3) * 64 + 8 * (threadIdx.x & 7) + j] = cs[j];
      __syncthreads();
      if (threadIdx.x < 64 && m0 + (int)threadIdx.x < g.M) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; r++) t += p[r * 64 + threadIdx.x];
        g.colsum[(long)z * g.M + m0 + threadIdx.x] = t;
      }
    }
  }

  CT* C = (CT*)g.C + (long)z * g.M * g.ldc;
  const int n = n0 + wn * 32 + (lane & 31);
  if (n >= g.N) return;
  const float bn = g.bias ? g.bias[n] : 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const int m = m0 + wm * 32 + acc_row(e, lane);
    const float v = PA == 3 ? acc[0][e] + acc[PA == 3 ? 1 : 0][e] : acc[0][e];
    if (m < g.M) C[(long)m * g.ldc + n] = (CT)(v + bn);
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
// Rows of a prepared operand are no further apart: 128 of them stay within the 32-bit offsets of lgemm's tiles, and a piece of
// WIDE_BYTES holds hundreds.  Rows of x further apart are copied (to rows of K, at most 2^20 columns, six times that in fp32).
constexpr long MAX_LD = 1L << 20;

long align256(long b) { return (b + 255) & ~255L; }
int up8(int n) { return (n + 7) & ~7; }

struct Gemm {
  int ts;              // 64: dgemm straight from the tensors; 128: lgemm, 256: the wide kernel, on prepared operands
  int nsplit, slabs;   // K-ranges; slabs of the result in the workspace (0: written directly)
  long ws;             // workspace bytes
  double us;           // estimate
};

// Costs in microseconds of a step of 64 k with w workgroups per CU, measured over products from 300^3 to 16384 x 4096^2 (the
// product's own time only; a launch 3.5, slabs written and read at 7.5 TB/s, prepared operands at 5).
double step_us(int ts, int pairs, double w) {
  if (ts == 64) return pairs == 1 ? 0.25 + 0.2 * w : pairs == 3 ? 0.5 + 0.48 * w : 0.5 + 0.85 * w;
  return w == 1 ? 1.15 : 0.7 * w;
}
// the wide kernel's: rows of both operands or columns of W; the weight gradient, which takes codes apart
const double WIDE_ROWS_US = 1.7, WIDE_Q8_US = 1.9;
const double LAUNCH_US = 3.5;

void consider(Gemm& best, int ts, int pairs, long M, int N, long K, int planes) {
  const long nk = (K + 63) / 64, tiles = ((M + ts - 1) / ts) * ((N + ts - 1) / ts) * planes;
  const double mn = (double)M * N;
  if (tiles >= 1L << 24) return;
  for (int ns = 1; ns <= 64; ns *= 2) {
    if (ns > 1 && nk / ns < 4) break;
    double us = LAUNCH_US + (nk + ns - 1) / ns * step_us(ts, pairs, (double)((tiles * ns + 255) / 256));
    if (ns * planes > 1) us += mn * 4 * (2 * ns * planes + 1) / 7.5e6 + LAUNCH_US;
    if (us >= best.us) continue;
    best.ts = ts;
    best.nsplit = ns;
    best.slabs = ns * planes > 1 ? ns * planes : 0;
    best.ws = (long)best.slabs * M * N * 4;
    best.us = us;
  }
}

// straight from the tensors; pairs: term pairs per product
Gemm pick_direct(long M, int N, long K, int pairs) {
  Gemm best = {0, 1, 0, 0, 1e30};
  consider(best, 64, pairs, M, N, K, 1);
  return best;
}

// on prepared operands, of which `planes` column blocks are summed up apart
Gemm pick_blocks(long M, int N, long K, int planes, bool wide_ok, long wide_ws, double wide_us) {
  Gemm best = {0, 1, 0, 0, 1e30};
  if (wide_ok) {
    const long nk = (K + 63) / 64;
    const int ns = scp_gemm_bf16_nsplit((int)M, N, (int)K);
    const double mn = (double)M * N, w = (double)((((M + 255) / 256) * ((N + 255) / 256) * ns + 255) / 256);
    double us = planes * (LAUNCH_US + wide_us * w * ((nk + ns - 1) / ns));
    if (ns > 1) us += planes * (mn * 4 * (2 * ns + 1) / 7.5e6 + LAUNCH_US);
    if (planes > 1) us += mn * 4 * (2 * planes + 1) / 7.5e6 + LAUNCH_US;
    best = {256, 1, 0, wide_ws, us};
  }
  consider(best, 128, 1, M, N, K, planes);
  return best;
}

double prep_us(double elements, int in_bytes, int blocks) { return LAUNCH_US + elements * (in_bytes + 2 * blocks) / 5e6; }

struct Plan {
  int np;                    // column blocks of an fp32 operand: 6 (ns 3), else 1
  int Kp, Np;
  bool x_direct, w_direct, dy_direct;          // usable as prepared operands as they are
  bool prep_x, prep_w, prep_dy;                // copies to make
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

long wide_ws_rows(long M, int N, long K, long lda) {
  const long piece = WIDE_BYTES / (2 * lda);
  const long a = scp_gemm_bf16_ws_floats((int)(M < piece ? M : piece), N, (int)K, N);
  const long b = M > piece ? scp_gemm_bf16_ws_floats((int)(M % piece), N, (int)K, N) : 0;    // the last piece may split K
  return (a > b ? a : b) * 4;
}

// dgemm forms the offsets inside a tile in 32 bits; its col operands (W for dx, dy for dW) also have rows of 8 elements at
// least, no closer than their length
bool direct_rows_ok(long ld) { return ld < 1L << 25; }

Plan plan_fwd(const ScpLinear8& a) {
  Plan p = {};
  common_plan(a, p);
  p.x_direct = a.x_bf16 && a.K % 8 == 0 && a.ldx % 8 == 0 && a.ldx >= a.K && a.ldx <= MAX_LD && ((uintptr_t)a.x & 15) == 0;
  const int xb = a.x_bf16 ? 2 : 4, wb = a.w_bf16 ? 2 : 4;
  const long KK = p.np == 1 ? a.K : (long)p.np * p.Kp, ld = (long)p.np * p.Kp;
  const bool ok = ((long)a.N + 192) * ld * 2 < WIDE_BYTES;
  Gemm blocks = pick_blocks(a.M, a.N, KK, 1, ok, ok ? wide_ws_rows(a.M, a.N, KK, p.x_direct ? a.ldx : ld) : 0, WIDE_ROWS_US);
  if (!p.x_direct) blocks.us += prep_us((double)a.M * a.K, xb, p.np) - LAUNCH_US;    // else packing is a launch of its own
  if (!p.w_direct) blocks.us += prep_us((double)a.N * a.K, wb, p.np);
  Gemm direct = pick_direct(a.M, a.N, a.K, p.np);
  if (!direct_rows_ok(a.ldx)) direct.us = 1e30;
  p.y = direct.us < blocks.us ? direct : blocks;
  p.prep_x = p.y.ts != 64 && !p.x_direct;
  p.prep_w = p.y.ts != 64 && !p.w_direct;
  long o = 0;
  p.a_off = o;
  if (p.prep_x) o += align256(a.M * ld * 2);
  p.b_off = o;
  if (p.prep_w) o += align256((long)a.N * ld * 2);
  p.g_off = o;
  p.total = o + align256(p.y.ws);
  return p;
}

int ranges(const Gemm& q, long K);
bool fused_db(const ScpLinear8& a, const Plan& p);

Plan plan_bwd(const ScpLinear8& a) {
  Plan p = {};
  common_plan(a, p);
  p.dy_direct = a.x_bf16 && a.N % 8 == 0 && a.lddy == a.N && ((uintptr_t)a.dy & 15) == 0;
  const int xb = a.x_bf16 ? 2 : 4, wb = a.w_bf16 ? 2 : 4, planes = p.np == 6 ? 3 : 1;
  const long ld = (long)p.np * p.Np, K2 = p.np == 1 ? a.N : ld, lda = p.dy_direct ? a.N : ld;
  const double dy_us = p.dy_direct ? 0 : prep_us((double)a.M * a.N, xb, p.np) - LAUNCH_US;   // else the column sums are a launch of their own
  // Each product straight from the tensors or on prepared operands: the cheapest combination, dy being prepared once for both.
  // Chosen as if all gradients were asked for, so that none depends on the others being wanted.
  const bool ok = (K2 + 192) * p.Kp * 2 < WIDE_BYTES;
  Gemm xb_ = pick_blocks(a.M, a.K, K2, 1, ok, ok ? wide_ws_rows(a.M, a.K, K2, lda) : 0, WIDE_ROWS_US);
  if (!p.w_direct) xb_.us += prep_us((double)a.N * a.K, wb, p.np);
  Gemm xd = pick_direct(a.M, a.K, a.N, p.np);
  if (!direct_rows_ok(a.lddy) || a.K < 8) xd.us = 1e30;
  // the wide form of dW runs once per plane, each into a slab of its own
  const long ld8 = (a.K + 63) / 64 * 64L, wide_ws = scp_gemm_q8_ws_floats(a.N, a.K, (int)a.M, lda > ld8 ? lda : ld8, a.K) * 4;
  const Gemm wb_ = pick_blocks(a.N, a.K, a.M, planes, lda <= MAX_LD, align256(wide_ws) + (planes > 1 ? 3L * a.N * a.K * 4 : 0),
                               WIDE_Q8_US);
  Gemm wd = pick_direct(a.N, a.K, a.M, planes);
  if (!direct_rows_ok(a.lddy) || a.lddy < a.N || a.N < 8) wd.us = 1e30;
  double best = 1e300;
  for (int c = 0; c < 4; c++) {
    const Gemm &x = c & 1 ? xb_ : xd, &w = c & 2 ? wb_ : wd;
    const double us = x.us + w.us + (c ? dy_us : 0);
    if (us >= best) continue;
    best = us;
    p.dx = x;
    p.dw = w;
  }
  p.prep_w = a.dx && p.dx.ts != 64 && !p.w_direct;
  p.prep_dy = ((a.dx && p.dx.ts != 64) || (a.dW && p.dw.ts != 64)) && !p.dy_direct;
  long o = 0;
  p.a_off = o;
  if (p.prep_dy) o += align256(a.M * ld * 2);
  p.b_off = o;
  if (p.prep_w) o += align256((p.np == 1 ? (long)a.N : ld) * p.Kp * 2);
  p.part_off = o;
  p.parts = fused_db(a, p) ? ranges(p.dw, a.M) : colsum_parts(a.M, a.N);
  if (a.db && !(fused_db(a, p) && p.parts == 1)) o += align256((long)p.parts * a.N * 4);
  p.g_off = o;
  const long gx = a.dx ? p.dx.ws : 0, gw = a.dW ? p.dw.ws : 0;
  p.total = o + align256(gx > gw ? gx : gw);
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

// K-ranges that are left when a range takes whole steps
int ranges(const Gemm& q, long K) {
  const int nk = (int)((K + 63) / 64), per = (nk + q.nsplit - 1) / q.nsplit;
  return (nk + per - 1) / per;
}

// tiles, K-ranges and the sum of the slabs around one of the two kernels; C contiguous [M][N]
template <typename Launch>
int tiled(const Gemm& q, LgArgs g, int c_bf16, const float* bias, float* ws, hipStream_t st, Launch launch) {
  void* C = g.C;
  g.tiles_m = (g.M + q.ts - 1) / q.ts;
  g.tiles_n = (g.N + q.ts - 1) / q.ts;
  const int nk = (g.K + 63) / 64;
  g.per_split = (nk + q.nsplit - 1) / q.nsplit;
  g.nsplit = ranges(q, g.K);
  g.ldc = g.N;
  const int slabs = g.nsplit * g.planes;
  if (slabs > 1) g.C = ws;
  else g.bias = bias;
  const dim3 grid((unsigned)(((long)g.tiles_m * g.tiles_n * slabs + 7) / 8 * 8));
  if (int rc = launch(g, grid, slabs == 1 && c_bf16)) return rc;
  if (slabs == 1) return SCP_OK;
  const long MN = (long)g.M * g.N;
  const dim3 sum((unsigned)((MN + 1023) / 1024));
  if (c_bf16) hipLaunchKernelGGL((lin_sum_kernel<__bf16>), sum, dim3(256), 0, st, ws, slabs, MN, g.N, bias, (__bf16*)C);
  else hipLaunchKernelGGL((lin_sum_kernel<float>), sum, dim3(256), 0, st, ws, slabs, MN, g.N, bias, (float*)C);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

template <int OPA, int OPB, typename CT>
int launch_lg(const LgArgs& g, dim3 grid, hipStream_t st) {
  constexpr size_t smem = 4 * 128 * 128;
  static uint64_t done = 0;
  if (int rc = scp_set_smem((const void*)lgemm_kernel<OPA, OPB, CT>, smem, &done)) return rc;
  hipLaunchKernelGGL((lgemm_kernel<OPA, OPB, CT>), grid, dim3(256), smem, st, g);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}
template <int OPA, int OPB>
int block_gemm(const Gemm& q, const LgArgs& g, int c_bf16, const float* bias, float* ws, hipStream_t st) {
  return tiled(q, g, c_bf16, bias, ws, st, [st](const LgArgs& a, dim3 grid, bool b16) {
    return b16 ? launch_lg<OPA, OPB, __bf16>(a, grid, st) : launch_lg<OPA, OPB, float>(a, grid, st);
  });
}

// terms of a product straight from the tensors: x (or dy) of TA, W of TB or x's checkpoint
template <typename TA, int PA, bool ACOL, typename TB, int PB, int OPB>
int direct_gemm(const Gemm& q, LgArgs g, int c_bf16, const float* bias, float* ws, hipStream_t st) {
  g.planes = 1;
  return tiled(q, g, c_bf16, bias, ws, st, [st](const LgArgs& a, dim3 grid, bool b16) -> int {
    if constexpr (sizeof(TA) == 2) {       // (fp32 tensors have fp32 products)
      if (b16) {
        hipLaunchKernelGGL((dgemm_kernel<TA, PA, ACOL, TB, PB, OPB, __bf16>), grid, dim3(256), 0, st, a);
        SCP_LAUNCH_CHECK();
        return SCP_OK;
      }
    }
    hipLaunchKernelGGL((dgemm_kernel<TA, PA, ACOL, TB, PB, OPB, float>), grid, dim3(256), 0, st, a);
    SCP_LAUNCH_CHECK();
    return SCP_OK;
  });
}
template <int OPB>
int direct_rows(const ScpLinear8& a, const Plan& p, const Gemm& q, const LgArgs& g, const float* bias, float* ws, hipStream_t st) {
  if (a.x_bf16 && a.w_bf16) return direct_gemm<__bf16, 1, false, __bf16, 1, OPB>(q, g, 1, bias, ws, st);
  if (a.x_bf16) return direct_gemm<__bf16, 1, false, float, 1, OPB>(q, g, 1, bias, ws, st);
  if (p.np == 1) return direct_gemm<float, 1, false, float, 1, OPB>(q, g, 0, bias, ws, st);
  return direct_gemm<float, 3, false, float, 3, OPB>(q, g, 0, bias, ws, st);
}

// out[M][N] = A B^T (b_col 0) or A B (b_col 1), + bias, on prepared operands.  The wide kernel addresses its operands with 31
// bits: a longer batch runs in pieces.
int rows_product(const Gemm& q, int b_col, long M, int N, long K, const __bf16* A, long lda, const __bf16* B, long ldb, void* C,
                 int c_bf16, const float* bias, float* ws, hipStream_t st) {
  if (q.ts == 128) {
    LgArgs g = {};
    g.A = A; g.B = B; g.C = C;
    g.lda = lda; g.ldb = ldb;
    g.M = (int)M; g.N = N; g.K = (int)K;
    g.planes = 1;
    return b_col ? block_gemm<OP_ROW, OP_COL>(q, g, c_bf16, bias, ws, st) : block_gemm<OP_ROW, OP_ROW>(q, g, c_bf16, bias, ws, st);
  }
  const long piece = WIDE_BYTES / (2 * lda);
  for (long r = 0; r < M; r += piece) {
    const int m = (int)(M - r < piece ? M - r : piece);
    void* c = c_bf16 ? (void*)((__bf16*)C + r * N) : (void*)((float*)C + r * N);
    if (int rc = scp_gemm_rows(b_col, m, N, (int)K, A + r * lda, lda, B, ldb, c, c_bf16, N, bias, ws, st)) return rc;
  }
  return SCP_OK;
}

// db from n partial rows
int finish_db(const ScpLinear8& a, const float* part, int n, hipStream_t st) {
  hipLaunchKernelGGL(lin_db_kernel, dim3((a.N + 15) / 16), dim3(256), 0, st, part, n, a.N, a.db);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

// db comes out of dW's product where that reads dy itself, unless the pass that prepares dy has it already
bool fused_db(const ScpLinear8& a, const Plan& p) { return a.db && a.dW && p.dw.ts == 64 && !p.prep_dy; }

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
  return a.db ? finish_db(a, part, p.parts, st) : SCP_OK;
}

// dW = dy^T v; A: dy's blocks (unused straight from the tensors)
int weight_product(const ScpLinear8& a, const Plan& p, const __bf16* A, long lda, float* ws, hipStream_t st) {
  LgArgs g = {};
  g.B = a.codes; g.steps = a.steps; g.C = a.dW;
  g.ldb = (a.K + 63) / 64 * 64;
  g.M = a.N; g.N = a.K; g.K = (int)a.M;
  if (p.dw.ts == 64) {
    g.A = (const __bf16*)a.dy;
    g.lda = a.lddy;
    const int n = ranges(p.dw, a.M);
    float* part = (float*)((char*)a.ws + p.part_off);
    if (fused_db(a, p)) g.colsum = n == 1 ? a.db : part;
    const int rc = a.x_bf16 ? direct_gemm<__bf16, 1, true, __bf16, 1, OP_Q8>(p.dw, g, a.w_bf16, nullptr, ws, st)
                   : p.np == 1 ? direct_gemm<float, 1, true, __bf16, 1, OP_Q8>(p.dw, g, 0, nullptr, ws, st)
                               : direct_gemm<float, 3, true, __bf16, 1, OP_Q8>(p.dw, g, 0, nullptr, ws, st);
    return rc || !g.colsum || n == 1 ? rc : finish_db(a, part, n, st);
  }
  const int off[3] = {0, 2 * p.Np, 5 * p.Np};
  g.planes = p.np == 6 ? 3 : 1;
  if (p.dw.ts == 128) {
    g.A = A;
    g.lda = lda;
    for (int i = 0; i < 3; i++) g.plane_off[i] = off[i];
    return block_gemm<OP_COL, OP_Q8>(p.dw, g, a.w_bf16, nullptr, ws, st);
  }
  if (g.planes == 1) return scp_gemm_q8(a.N, a.K, (int)a.M, A, lda, a.codes, a.steps, a.dW, a.w_bf16, a.K, ws, st);
  const long NK = (long)a.N * a.K;
  float* slabs = ws + (p.dw.ws - 3 * NK * 4) / 4;
  for (int i = 0; i < 3; i++)
    if (int rc = scp_gemm_q8(a.N, a.K, (int)a.M, A + off[i], lda, a.codes, a.steps, slabs + i * NK, 0, a.K, ws, st)) return rc;
  hipLaunchKernelGGL((lin_sum_kernel<float>), dim3((unsigned)((NK + 1023) / 1024)), dim3(256), 0, st, slabs, 3, NK, a.K, nullptr,
                     (float*)a.dW);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
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

extern "C" int scp_linear8_tiles(const ScpLinear8* a, int* tiles) {
  if (int rc = check_args(a, "scp_linear8_tiles")) return rc;
  SCP_CHECK(tiles, SCP_ERR_ARG, "scp_linear8_tiles: null pointer");
  const Plan b = plan_bwd(*a);
  tiles[0] = plan_fwd(*a).y.ts;
  tiles[1] = b.dx.ts;
  tiles[2] = b.dw.ts;
  return SCP_OK;
}

extern "C" int scp_linear8_fwd(const ScpLinear8* a_, void* stream) {
  if (int rc = check_args(a_, "scp_linear8_fwd")) return rc;
  const ScpLinear8& a = *a_;
  SCP_CHECK(a.x && a.W && a.y && a.ldx >= 0, SCP_ERR_ARG, "scp_linear8_fwd: null pointer or negative row stride");
  const Plan p = plan_fwd(a);
  SCP_CHECK(a.ws || !p.total, SCP_ERR_ARG, "scp_linear8_fwd: needs the workspace of scp_linear8_fwd_ws");
  SCP_CHECK(((uintptr_t)a.ws & 255) == 0, SCP_ERR_ARG, "scp_linear8_fwd: the workspace must be 256-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)a.ws;
  float* gws = (float*)(ws + p.g_off);
  const long ld = (long)p.np * p.Kp;
  int rc = SCP_OK;
  const __bf16 *A = (const __bf16*)a.x, *B = (const __bf16*)a.W;
  if (p.prep_x) {
    __bf16* dst = (__bf16*)(ws + p.a_off);
    A = dst;
#define PREP_X(T, LAY)                                                                                     \
  (a.codes ? prep<T, LAY, true>(a.x, a.ldx, a.M, a.K, 0, dst, p.Kp, a.codes, a.steps, st)                   \
           : prep<T, LAY, false>(a.x, a.ldx, a.M, a.K, 0, dst, p.Kp, nullptr, nullptr, st))
    rc = a.x_bf16 ? PREP_X(__bf16, LAY_ONE) : p.np == 1 ? PREP_X(float, LAY_ONE) : PREP_X(float, LAY_COLS_A);
#undef PREP_X
  } else if (a.codes && p.y.ts != 64) {
    rc = scp_pack8(a.x, a.x_bf16, a.ldx, a.M, a.K, a.codes, a.steps, stream);
  }
  if (rc) return rc;
  if (p.y.ts == 64) {
    LgArgs g = {};
    g.A = A; g.B = B; g.C = a.y;
    g.lda = a.ldx; g.ldb = a.K;
    g.M = (int)a.M; g.N = a.N; g.K = a.K;
    g.pack_codes = a.codes; g.pack_steps = a.steps;
    return direct_rows<OP_ROW>(a, p, p.y, g, a.b, gws, st);
  }
  if (p.prep_w) {
    B = (const __bf16*)(ws + p.b_off);
    if ((rc = prep_w(a, p, false, (__bf16*)(ws + p.b_off), st))) return rc;
  }
  return rows_product(p.y, 0, a.M, a.N, p.np == 1 ? a.K : ld, A, p.prep_x ? ld : a.ldx, B, p.prep_w ? ld : a.K, a.y, a.x_bf16, a.b,
                      gws, st);
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
  const long ld = (long)p.np * p.Np, lda = p.prep_dy ? ld : a.N;
  const __bf16* A = p.prep_dy ? (const __bf16*)(ws + p.a_off) : (const __bf16*)a.dy;
  int rc;
  // The column sums come out of the pass that writes the operand's blocks; where none is needed, they come last, when the
  // products have left dy in the last-level cache (16384 x 4096 bf16: 43 us before them, 20 us after).
  if (p.prep_dy && (rc = dy_pass(a, p, true, st))) return rc;
  if (a.dx && p.dx.ts == 64) {
    LgArgs g = {};
    g.A = (const __bf16*)a.dy; g.B = a.W; g.C = a.dx;
    g.lda = a.lddy; g.ldb = a.K;
    g.M = (int)a.M; g.N = a.K; g.K = a.N;
    if ((rc = direct_rows<OP_COL>(a, p, p.dx, g, nullptr, gws, st))) return rc;
  } else if (a.dx) {
    const __bf16* B = (const __bf16*)a.W;
    if (p.prep_w) {
      B = (const __bf16*)(ws + p.b_off);
      if ((rc = prep_w(a, p, true, (__bf16*)(ws + p.b_off), st))) return rc;
    }
    if ((rc = rows_product(p.dx, 1, a.M, a.K, p.np == 1 ? a.N : ld, A, lda, B, p.prep_w ? p.Kp : a.K, a.dx, a.x_bf16, nullptr, gws, st)))
      return rc;
  }
  if (a.dW && (rc = weight_product(a, p, A, lda, gws, st))) return rc;
  return a.db && !p.prep_dy && !fused_db(a, p) ? dy_pass(a, p, false, st) : SCP_OK;
}
