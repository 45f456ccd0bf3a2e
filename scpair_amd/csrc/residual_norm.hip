// Norms around a block of a residual trunk, fused with the block's gate and residual scale.
//
//   n = Norm_post(h)   u = s * act(g) * n   r = x + u   y = Norm_pre(r)        one row = one cell
//   Norm: "layer" (t - mean) * rstd * w + b, "rms" t * rstd * w, post "none": n = h
//   g per element, per row or per column; s a value, one learned number or one per column
//
// Everything that is constant along the rows is folded once per thread:  S = s * act(g_col), A1 = w1 S, B1 = b1 S, so
//   u = (hhat A1 + B1) G          hhat = (h - mean1) rstd1,  G = act(g) of a full or a row gate, else 1
// Backward, per row (r and rhat are recomputed from x, h and the four saved statistics, not read back rounded):
//   a = dy w2     du = dr + rstd2 (a - mean(a) - rhat mean(a rhat))     dx = du
//   b = du G A1   dh = rstd1 (b - mean(b) - hhat mean(b hhat))          dG = du (hhat A1 + B1)
// (the mean(.) terms only for "layer", none of them for post "none"), and per column over all rows
//   P = sum du G hhat,  Q = sum du G,  sum dy rhat,  sum dy:
//   dw1 = S P, db1 = S Q, ds = act(g_col) (w1 P + b1 Q), dg_col = s act'(g_col) (w1 P + b1 Q), dw2, db2.
//
// All sums and statistics are fp32 (the column sums' last stage fp64); every output is rounded once.  The variance is
// taken about the mean in a second pass over registers: no cancellation for rows far from zero.
//
// Bound: HBM.  One pass over the data in each direction: a row lives in registers, 8 consecutive columns per lane and
// chunk (16 bytes of bf16, 32 of fp32), and a workgroup walks rows with the column constants and column sums in
// registers.  Up to 1024 columns a row belongs to one wave (no barriers), above that to a workgroup.  Rows need no
// alignment: the vector accesses are declared with the element's alignment, which the hardware takes as they are.
// Column sums leave a workgroup as one partial row each; a second launch adds them in a fixed order (no atomics).
#include "common.h"
#include "scpair_hip.h"

namespace {

typedef float vf8 __attribute__((ext_vector_type(8)));
typedef __bf16 vb8 __attribute__((ext_vector_type(8)));
template <typename T> struct Vec8;
template <> struct Vec8<float> { typedef vf8 v; typedef vf8 vu __attribute__((aligned(4))); };
template <> struct Vec8<__bf16> { typedef vb8 v; typedef vb8 vu __attribute__((aligned(2))); };

enum { GATE_NONE = 0, GATE_FULL = 1, GATE_ROW = 2, GATE_COL = 3 };
enum { ACT_NONE = 0, ACT_SIGMOID = 1, ACT_TANH = 2 };
enum { SCALE_VALUE = 0, SCALE_ONE = 1, SCALE_COL = 2 };
enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

// 8 columns from `col` of a row of D; columns behind the row's end are zero
template <typename T>
__device__ __forceinline__ typename Vec8<T>::v ld8(const T* __restrict__ p, int col, int D) {
  typename Vec8<T>::v v;
  if (col + 8 <= D) {
    v = *(const typename Vec8<T>::vu*)(p + col);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (col + i < D) ? p[col + i] : (T)0.f;
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void st8(T* __restrict__ p, int col, int D, const float* f) {
  typename Vec8<T>::v v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (T)f[i];
  if (col + 8 <= D) {
    *(typename Vec8<T>::vu*)(p + col) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (col + i < D) p[col + i] = v[i];
  }
}

__device__ __forceinline__ float gate_value(float g, int act) {
  if (act == ACT_SIGMOID) {
    const float t = expf(-fabsf(g)), q = __builtin_amdgcn_rcpf(1.f + t);
    return g >= 0.f ? q : t * q;
  }
  return act == ACT_TANH ? tanhf(g) : g;
}
// value and derivative; exp of a non-positive argument only, so neither end overflows
__device__ __forceinline__ float gate_both(float g, int act, float& d) {
  if (act == ACT_SIGMOID) {
    const float t = expf(-fabsf(g)), q = __builtin_amdgcn_rcpf(1.f + t);
    d = t * q * q;
    return g >= 0.f ? q : t * q;
  }
  if (act == ACT_TANH) {
    const float t = expf(-2.f * fabsf(g)), q = __builtin_amdgcn_rcpf(1.f + t);
    d = 4.f * t * q * q;
    return tanhf(g);
  }
  d = 1.f;
  return g;
}

// sum over the wave, in every lane
__device__ __forceinline__ float wsum(float v) {
  v += dppf<0xB1>(v);
  v += dppf<0x4E>(v);
  v += dppf<0x124>(v);
  v += dppf<0x128>(v);
  v = xor16_sum(v);
  return xor32_sum(v);
}
// Sums of NV values over the TPR threads of a row, in every thread.  Above one wave: one barrier per call; calls
// alternate between two LDS slots, and a slot's next write comes after the barrier of the call between.
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float* red, int& turn) {
#pragma unroll
  for (int i = 0; i < NV; i++) v[i] = wsum(v[i]);
  if constexpr (TPR > 64) {
    constexpr int NWV = TPR / 64;
    float* s = red + (turn & 1) * (4 * NWV);
    turn++;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < NV; i++) s[i * NWV + (threadIdx.x >> 6)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < NWV; w++) t += s[i * NWV + w];
      v[i] = t;
    }
  }
}

// mean and 1 / spread of a row held as v[NCH][8] (columns >= D hold zeros)
template <int TPR, int NCH>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][8], int kind, int t, int D, float inv_d, float eps,
                                          float* red, int& turn, float& mean, float& rstd) {
  mean = 0.f;
  if (kind == NORM_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NCH; c++)
#pragma unroll
      for (int i = 0; i < 8; i++) s[0] += v[c][i];
    row_sum<TPR, 1>(s, red, turn);
    mean = s[0] * inv_d;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    const int col = (t + TPR * c) * 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float e = col + i < D ? v[c][i] - mean : 0.f;
      q[0] += e * e;
    }
  }
  row_sum<TPR, 1>(q, red, turn);
  rstd = 1.f / sqrtf(q[0] * inv_d + eps);
}

// threads per workgroup: rows of one wave are handled by several independent waves
template <int TPR> constexpr int fwd_threads() { return TPR == 64 ? 256 : TPR; }
template <int TPR> constexpr int bwd_threads() { return TPR == 64 ? 512 : TPR; }

// column constants of one chunk
template <int FWD>
__device__ __forceinline__ void fold(const ScpResidualNorm& a, int col, float* A1, float* B1, float* W2, float* B2) {
  const int D = a.cols;
  float s = a.scale_mode == SCALE_ONE ? a.scale[0] : a.scale_value;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const bool ok = col + i < D;
    float S = s;
    if (a.scale_mode == SCALE_COL) S = ok ? a.scale[col + i] : 0.f;
    if (a.gate_mode == GATE_COL) S *= ok ? gate_value(((const float*)a.gate)[col + i], a.gate_act) : 0.f;
    A1[i] = !ok ? 0.f : a.w1 ? a.w1[col + i] * S : S;
    B1[i] = ok && a.b1 ? a.b1[col + i] * S : 0.f;
    W2[i] = !ok ? 0.f : a.w2 ? a.w2[col + i] : 1.f;
    if (FWD) B2[i] = ok && a.b2 ? a.b2[col + i] : 0.f;
  }
}

template <typename XT, typename HT, int TPR, int NCH>
__global__ __launch_bounds__(fwd_threads<TPR>()) void rnorm_fwd_kernel(ScpResidualNorm a) {
  constexpr int RPW = fwd_threads<TPR>() / TPR;
  __shared__ float red[TPR > 64 ? 2 * 4 * (TPR / 64) : 1];
  const int t = threadIdx.x % TPR, D = a.cols;
  const float inv_d = 1.f / (float)D;
  int turn = 0;
  float A1[NCH][8], B1[NCH][8], W2[NCH][8], B2[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; c++) fold<1>(a, (t + TPR * c) * 8, A1[c], B1[c], W2[c], B2[c]);

  for (long row = (long)blockIdx.x * RPW + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * RPW) {
    float r[NCH][8];
    const XT* xp = (const XT*)a.x + row * a.ldx;
    float m1 = 0.f, s1 = 1.f, m2, s2;
    if (a.h) {
      const HT* hp = (const HT*)a.h + row * a.ldh;
      float h[NCH][8];
      typename Vec8<XT>::v xv[NCH];
      typename Vec8<HT>::v gv[NCH];
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int col = (t + TPR * c) * 8;
        const auto hv = ld8<HT>(hp, col, D);
        xv[c] = ld8<XT>(xp, col, D);
        if (a.gate_mode == GATE_FULL) gv[c] = ld8<HT>((const HT*)a.gate + row * a.ldg, col, D);
#pragma unroll
        for (int i = 0; i < 8; i++) h[c][i] = (float)hv[i];
      }
      const float grow = a.gate_mode == GATE_ROW ? gate_value(((const float*)a.gate)[row], a.gate_act) : 1.f;
      if (a.post != NORM_NONE) row_stats<TPR, NCH>(h, a.post, t, D, inv_d, a.eps, red, turn, m1, s1);
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int col = (t + TPR * c) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float g = a.gate_mode == GATE_FULL ? gate_value((float)gv[c][i], a.gate_act) : grow;
          const float u = ((h[c][i] - m1) * s1 * A1[c][i] + B1[c][i]) * g;
          r[c][i] = col + i < D ? (float)xv[c][i] + u : 0.f;
        }
        if (col < D) st8<XT>((XT*)a.r + row * D, col, D, r[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const auto xv = ld8<XT>(xp, (t + TPR * c) * 8, D);
#pragma unroll
        for (int i = 0; i < 8; i++) r[c][i] = (float)xv[i];
      }
    }
    row_stats<TPR, NCH>(r, a.pre, t, D, inv_d, a.eps, red, turn, m2, s2);
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      const int col = (t + TPR * c) * 8;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = (r[c][i] - m2) * s2 * W2[c][i] + B2[c][i];
      if (col < D) st8<HT>((HT*)a.y + row * D, col, D, y);
    }
    if (a.stats && t == 0) {
      f32x4 s = {m1, s1, m2, s2};
      *(f32x4*)(a.stats + row * 4) = s;
    }
  }
}

// partial column sums: ws[block][4][cols], order P, Q, sum dy rhat, sum dy
template <typename XT, typename HT, int TPR, int NCH>
__global__ __launch_bounds__(bwd_threads<TPR>()) void rnorm_bwd_kernel(ScpResidualNorm a) {
  constexpr int RPW = bwd_threads<TPR>() / TPR;
  __shared__ float red[TPR > 64 ? 2 * 4 * (TPR / 64) : 1];
  __shared__ float colbuf[RPW > 1 ? NCH * 512 : 1];
  const int t = threadIdx.x % TPR, D = a.cols;
  const float inv_d = 1.f / (float)D;
  int turn = 0;
  float A1[NCH][8], B1[NCH][8], W2[NCH][8];
  float acc[4][NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    fold<0>(a, (t + TPR * c) * 8, A1[c], B1[c], W2[c], nullptr);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int i = 0; i < 8; i++) acc[k][c][i] = 0.f;
  }
  const float lay1 = a.post == NORM_LAYER ? inv_d : 0.f, cor1 = a.post == NORM_NONE ? 0.f : inv_d;
  const float lay2 = a.pre == NORM_LAYER ? inv_d : 0.f;

  for (long row = (long)blockIdx.x * RPW + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * RPW) {
    const f32x4 st = *(const f32x4*)(a.stats + row * 4);
    const float m1 = st[0], s1 = st[1], m2 = st[2], s2 = st[3];
    float hh[NCH][8], G[NCH][8], dG[NCH][8], rh[NCH][8], du[NCH][8];
    const float grow = a.h && a.gate_mode == GATE_ROW ? gate_value(((const float*)a.gate)[row], a.gate_act) : 1.f;
    float c12[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      const int col = (t + TPR * c) * 8;
      const auto xv = ld8<XT>((const XT*)a.x + row * a.ldx, col, D);
      typename Vec8<HT>::v hv, gv, yv;
      typename Vec8<XT>::v rv;
      if (a.h) hv = ld8<HT>((const HT*)a.h + row * a.ldh, col, D);
      if (a.gate_mode == GATE_FULL) gv = ld8<HT>((const HT*)a.gate + row * a.ldg, col, D);
      if (a.dy) yv = ld8<HT>((const HT*)a.dy + row * a.lddy, col, D);
      if (a.dr) rv = ld8<XT>((const XT*)a.dr + row * a.lddr, col, D);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        G[c][i] = grow;
        dG[c][i] = 1.f;
        float r = (float)xv[i];
        if (a.h) {
          if (a.gate_mode == GATE_FULL) G[c][i] = gate_both((float)gv[i], a.gate_act, dG[c][i]);
          hh[c][i] = ((float)hv[i] - m1) * s1;
          r += (hh[c][i] * A1[c][i] + B1[c][i]) * G[c][i];
        }
        rh[c][i] = col + i < D ? (r - m2) * s2 : 0.f;
        const float dy = a.dy ? (float)yv[i] : 0.f;
        du[c][i] = a.dr ? (float)rv[i] : 0.f;
        const float av = dy * W2[c][i];
        du[c][i] += s2 * av;
        c12[0] += av;
        c12[1] += av * rh[c][i];
        acc[2][c][i] += dy * rh[c][i];
        acc[3][c][i] += dy;
      }
    }
    if (a.dy) row_sum<TPR, 2>(c12, red, turn);
    const float c1 = c12[0] * lay2, c2 = c12[1] * inv_d;
    float e[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      const int col = (t + TPR * c) * 8;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        du[c][i] -= s2 * (c1 + rh[c][i] * c2);
        if (col + i >= D) du[c][i] = 0.f;
        if (a.h) {
          const float dg = du[c][i] * G[c][i], b = dg * A1[c][i];
          acc[0][c][i] += dg * hh[c][i];
          acc[1][c][i] += dg;
          e[0] += b;
          e[1] += b * hh[c][i];
          e[2] += du[c][i] * (hh[c][i] * A1[c][i] + B1[c][i]);
        }
      }
      if (a.dx && col < D) st8<XT>((XT*)a.dx + row * D, col, D, du[c]);
    }
    if (a.h) {
      row_sum<TPR, 3>(e, red, turn);
      const float e1 = e[0] * lay1, e2 = e[1] * cor1;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int col = (t + TPR * c) * 8;
        float dh[8], dg[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          dh[i] = s1 * (du[c][i] * G[c][i] * A1[c][i] - e1 - hh[c][i] * e2);
          dg[i] = du[c][i] * (hh[c][i] * A1[c][i] + B1[c][i]) * dG[c][i];
        }
        if (a.dh && col < D) st8<HT>((HT*)a.dh + row * D, col, D, dh);
        if (a.dgate && a.gate_mode == GATE_FULL && col < D) st8<HT>((HT*)a.dgate + row * D, col, D, dg);
      }
      if (a.dgate && a.gate_mode == GATE_ROW && t == 0) {
        float d;
        gate_both(((const float*)a.gate)[row], a.gate_act, d);
        ((float*)a.dgate)[row] = e[2] * d;
      }
    }
  }

  if (!a.ws) return;
  float* wsb = a.ws + (long)blockIdx.x * 4 * D;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if (k < 2 ? !a.want1 : !a.want2) continue;
    if constexpr (RPW > 1) {
      // add the waves of the workgroup in wave order
      for (int w = 0; w < RPW; w++) {
        if ((int)(threadIdx.x / 64) == w) {
#pragma unroll
          for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
              float* p = colbuf + (c * 8 + i) * 64 + t;
              *p = w ? *p + acc[k][c][i] : acc[k][c][i];
            }
        }
        __syncthreads();
      }
      for (int j = threadIdx.x; j < D; j += bwd_threads<TPR>()) {
        const int ch = j >> 3;
        wsb[(long)k * D + j] = colbuf[((ch >> 6) * 8 + (j & 7)) * 64 + (ch & 63)];
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const int col = (t + TPR * c) * 8;
        if (col < D) st8<float>(wsb + (long)k * D, col, D, acc[k][c]);
      }
    }
  }
}

// columns' sums of the partial rows (fixed order), and from them the parameters' gradients.  A workgroup takes 16
// columns; 16 threads share a column.
__global__ __launch_bounds__(256) void rnorm_cols_kernel(ScpResidualNorm a, int nblk, float* each) {
  __shared__ double part[4][16][17];
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + cx, D = a.cols;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    double s = 0.0;
    if (col < D && (k < 2 ? a.want1 : a.want2))
      for (int b = ry; b < nblk; b += 16) s += (double)a.ws[((long)b * 4 + k) * D + col];
    part[k][ry][cx] = s;
  }
  __syncthreads();
  if (ry || col >= D) return;
  double sum[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    sum[k] = 0.0;
    for (int y = 0; y < 16; y++) sum[k] += part[k][y][cx];
  }
  if (a.want2) {
    if (a.dw2) a.dw2[col] = (float)sum[2];
    if (a.db2) a.db2[col] = (float)sum[3];
  }
  if (a.want1) {
    const float s = a.scale_mode == SCALE_COL ? a.scale[col] : a.scale_mode == SCALE_ONE ? a.scale[0] : a.scale_value;
    float g = 1.f, d = 1.f;
    if (a.gate_mode == GATE_COL) g = gate_both(((const float*)a.gate)[col], a.gate_act, d);
    const double n = (a.w1 ? a.w1[col] : 1.f) * sum[0] + (a.b1 ? a.b1[col] * sum[1] : 0.0);
    if (a.dw1) a.dw1[col] = (float)(s * g * sum[0]);
    if (a.db1) a.db1[col] = (float)(s * g * sum[1]);
    if (a.gate_mode == GATE_COL && a.dgate) ((float*)a.dgate)[col] = (float)(s * d * n);
    if (a.dscale && a.scale_mode == SCALE_COL) a.dscale[col] = (float)(g * n);
    if (each) each[col] = (float)(g * n);
  }
}

// gradient of a single residual scale: the columns' shares added up by one workgroup
__global__ __launch_bounds__(256) void rnorm_scale_kernel(const float* each, int D, float* out) {
  __shared__ double red[16];
  double s = 0.0;
  for (int j = threadIdx.x; j < D; j += 256) s += (double)each[j];
  s = block_sum_d(s, red);
  if (threadIdx.x == 0) out[0] = (float)s;
}

constexpr int MAX_COLS = 16384;

// threads per row by width: a wave up to 1024 columns, above that a workgroup with 8 or 16 columns per thread
int tpr_of(int cols) { return cols <= 1024 ? 64 : cols <= 4096 ? 256 : cols <= 8192 ? 512 : 1024; }

int bwd_grid(long rows, int cols) {
  const int tpr = tpr_of(cols), rpw = tpr == 64 ? 8 : 1;
  const long need = (rows + rpw - 1) / rpw;
  const long cap = tpr == 64 ? 512 : tpr == 256 ? 1024 : 512;
  return (int)(need < cap ? need : cap);
}

template <typename XT, typename HT, int TPR, int NCH>
int go(const ScpResidualNorm& a, bool bwd, hipStream_t st) {
  if (!bwd) {
    const int rpw = fwd_threads<TPR>() / TPR;
    const long need = (a.rows + rpw - 1) / rpw, cap = 256L * (2048 / fwd_threads<TPR>());
    hipLaunchKernelGGL((rnorm_fwd_kernel<XT, HT, TPR, NCH>), dim3((unsigned)(need < cap ? need : cap)),
                       dim3(fwd_threads<TPR>()), 0, st, a);
  } else {
    hipLaunchKernelGGL((rnorm_bwd_kernel<XT, HT, TPR, NCH>), dim3((unsigned)bwd_grid(a.rows, a.cols)),
                       dim3(bwd_threads<TPR>()), 0, st, a);
  }
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

template <typename XT, typename HT>
int by_width(const ScpResidualNorm& a, bool bwd, hipStream_t st) {
  if (a.cols <= 512) return go<XT, HT, 64, 1>(a, bwd, st);
  if (a.cols <= 1024) return go<XT, HT, 64, 2>(a, bwd, st);
  if (a.cols <= 2048) return go<XT, HT, 256, 1>(a, bwd, st);
  if (a.cols <= 4096) return go<XT, HT, 256, 2>(a, bwd, st);
  if (a.cols <= 8192) return go<XT, HT, 512, 2>(a, bwd, st);
  return go<XT, HT, 1024, 2>(a, bwd, st);
}

int by_type(const ScpResidualNorm& a, bool bwd, hipStream_t st) {
  if (!a.x_bf16 && !a.h_bf16) return by_width<float, float>(a, bwd, st);
  if (!a.x_bf16) return by_width<float, __bf16>(a, bwd, st);
  return by_width<__bf16, __bf16>(a, bwd, st);
}

int check_args(const ScpResidualNorm* a, const char* who) {
  SCP_CHECK(a, SCP_ERR_ARG, "%s: null argument block", who);
  SCP_CHECK(a->rows > 0 && a->cols > 0, SCP_ERR_ARG, "%s: rows and cols must be positive (%ld, %d)", who, (long)a->rows,
            a->cols);
  SCP_CHECK(a->cols <= MAX_COLS, SCP_ERR_SHAPE, "%s: at most %d columns (got %d)", who, MAX_COLS, a->cols);
  SCP_CHECK(!(a->x_bf16 && !a->h_bf16), SCP_ERR_ARG, "%s: a bf16 residual stream needs bf16 blocks", who);
  SCP_CHECK(a->x && a->ldx >= 0 && a->ldh >= 0 && a->ldg >= 0, SCP_ERR_ARG, "%s: null x or negative row stride", who);
  SCP_CHECK(a->pre == NORM_RMS || a->pre == NORM_LAYER, SCP_ERR_ARG, "%s: pre must be rms (1) or layer (2)", who);
  SCP_CHECK(a->post >= NORM_NONE && a->post <= NORM_LAYER, SCP_ERR_ARG, "%s: post must be 0, 1 or 2", who);
  SCP_CHECK(a->gate_mode >= GATE_NONE && a->gate_mode <= GATE_COL && a->gate_act >= ACT_NONE && a->gate_act <= ACT_TANH &&
                a->scale_mode >= SCALE_VALUE && a->scale_mode <= SCALE_COL, SCP_ERR_ARG, "%s: unknown gate or scale mode", who);
  SCP_CHECK((a->gate_mode == GATE_NONE || a->gate) && (a->scale_mode == SCALE_VALUE || a->scale), SCP_ERR_ARG,
            "%s: gate or scale mode without its values", who);
  SCP_CHECK(a->h || (a->gate_mode == GATE_NONE && a->post == NORM_NONE), SCP_ERR_ARG, "%s: gate or post norm without a block", who);
  return SCP_OK;
}

}  // namespace

extern "C" int scp_residual_norm_max_cols(void) { return MAX_COLS; }

extern "C" int scp_residual_norm_fwd(const ScpResidualNorm* a, void* stream) {
  int rc = check_args(a, "scp_residual_norm_fwd");
  if (rc) return rc;
  SCP_CHECK(a->y && (!a->h || a->r), SCP_ERR_ARG, "scp_residual_norm_fwd: null output");
  return by_type(*a, false, (hipStream_t)stream);
}

extern "C" long scp_residual_norm_bwd_ws_floats(long rows, int cols) {
  if (rows <= 0 || cols <= 0 || cols > MAX_COLS) return 0;
  return (long)bwd_grid(rows, cols) * 4 * cols + cols;
}

extern "C" int scp_residual_norm_bwd(const ScpResidualNorm* a_, void* stream) {
  int rc = check_args(a_, "scp_residual_norm_bwd");
  if (rc) return rc;
  ScpResidualNorm a = *a_;
  SCP_CHECK(a.stats, SCP_ERR_ARG, "scp_residual_norm_bwd: null statistics");
  SCP_CHECK((!a.dr || a.lddr >= 0) && (!a.dy || a.lddy >= 0), SCP_ERR_ARG, "scp_residual_norm_bwd: negative row stride");
  a.want1 = a.h && (a.dw1 || a.db1 || a.dscale || (a.gate_mode == GATE_COL && a.dgate));
  a.want2 = a.dw2 || a.db2;
  SCP_CHECK(!(a.want1 || a.want2) || a.ws, SCP_ERR_ARG, "scp_residual_norm_bwd: parameter gradients need the workspace");
  SCP_CHECK((!a.dw1 || a.w1) && (!a.db1 || a.b1) && (!a.dscale || a.scale_mode != SCALE_VALUE) &&
                (!a.dgate || a.gate_mode != GATE_NONE), SCP_ERR_ARG, "scp_residual_norm_bwd: gradient of an absent parameter");
  if (!(a.want1 || a.want2)) a.ws = nullptr;
  hipStream_t st = (hipStream_t)stream;
  rc = by_type(a, true, st);
  if (rc || !a.ws) return rc;
  const int nblk = bwd_grid(a.rows, a.cols);
  float* each = a.dscale && a.scale_mode == SCALE_ONE ? a.ws + (long)nblk * 4 * a.cols : nullptr;
  hipLaunchKernelGGL(rnorm_cols_kernel, dim3((a.cols + 15) / 16), dim3(256), 0, st, a, nblk, each);
  SCP_LAUNCH_CHECK();
  if (each) {
    hipLaunchKernelGGL(rnorm_scale_kernel, dim3(1), dim3(256), 0, st, each, a.cols, a.dscale);
    SCP_LAUNCH_CHECK();
  }
  return SCP_OK;
}
