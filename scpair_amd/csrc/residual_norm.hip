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
// chunk (16 bytes of bf16, 32 of fp32), and a workgroup walks rows with the column constants and column sums in registers
// and the next row's values on their way.  Narrow rows share a wave (8 to 64 lanes each, no barriers), wide ones have a workgroup.  Rows need no
// alignment: the vector accesses are declared with the element's alignment, which the hardware takes as they are.
// Column sums leave a workgroup as one partial row each; a second launch adds them in a fixed order (no atomics).
//
// Measured (32768 x 4096 bf16, rms norms, a gate per column): forward 200 us for 1.07 GB, 5.3 TB/s; backward 291-320 us
// for 1.61 GB, 5.0-5.5 TB/s; a large copy reaches 5.1 TB/s.  4096 x 2048, fp32 stream beside bf16 blocks with a full gate: 22 and
// 33 us, 5.4 and 5.6 TB/s.  1024 x 900 fp32, full gate: 9 and 12 us, and 9 us for the column sums: bound by latency.
// 8192 x 6144 bf16, full gate: 93 and 155 us, 5.4 and 5.2 TB/s; 8192 x 8192 with biases: 132 and 227 us, 5.1 and 4.7 TB/s.
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

// A lane's chunk: 8 columns from `base` of a row of D.  Chunk q covers columns 8q ..; the one that would run over the
// row's end starts at D - 8 instead, so every access is one vector access without a test.  Its first `8 q - base` columns
// are its neighbour's: both lanes compute (and write) the same values there, and only the row's sums leave them out.
// Rows shorter than a chunk (SMALL) go element by element.
__device__ __forceinline__ int chunk_base(int q, int D) { return max(0, min(8 * q, D - 8)); }
__device__ __forceinline__ bool chunk_owns(int q, int i, int D) {
  return 8 * q < D && chunk_base(q, D) + i >= 8 * q && chunk_base(q, D) + i < D;
}
template <bool SMALL, typename T>
__device__ __forceinline__ typename Vec8<T>::v ld8(const T* __restrict__ p, int base, int D) {
  if constexpr (!SMALL) return *(const typename Vec8<T>::vu*)(p + base);
  typename Vec8<T>::v v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = i < D ? p[i] : (T)0.f;
  return v;
}
template <bool SMALL, typename T>
__device__ __forceinline__ void st8(T* __restrict__ p, int base, int D, const float* f) {
  typename Vec8<T>::v v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (T)f[i];
  if constexpr (!SMALL) {
    *(typename Vec8<T>::vu*)(p + base) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < D) p[i] = v[i];
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

// sum over the wave (or, G < 64, over groups of G neighbouring lanes), in every lane
template <int G = 64>
__device__ __forceinline__ float wsum(float v) {
  v += dppf<0xB1>(v);
  v += dppf<0x4E>(v);
  if constexpr (G == 8) return v + dppf<0x141>(v);
  v += dppf<0x124>(v);
  v += dppf<0x128>(v);
  if constexpr (G >= 32) v = xor16_sum(v);
  if constexpr (G == 64) v = xor32_sum(v);
  return v;
}
// columns of wave w of a workgroup that holds a row in NCH rounds of blockDim.x chunks
template <int NCH>
__device__ __forceinline__ int wave_cols(int w, int D) {
  int n = 0;
  if (64 * w >= (int)blockDim.x) return 0;
#pragma unroll
  for (int c = 0; c < NCH; c++) n += max(0, min(512, D - 8 * (int)blockDim.x * c - 512 * w));
  return n;
}
// sum over groups of 16 neighbouring lanes, in each of them
__device__ __forceinline__ float sum16(float v) {
  v += dppf<0xB1>(v);
  v += dppf<0x4E>(v);
  v += dppf<0x124>(v);
  return v + dppf<0x128>(v);
}
// Sums of NV values over the threads of a row, in every thread.  TPR > 64 (a workgroup of at most TPR threads): one barrier
// per call; the lanes of every wave read the waves' sums side by side (slots of absent waves hold zeros) and add them up.
// Calls alternate between two halves of `red`, and a half's next write comes after the barrier of the call between.
constexpr int RED = 4 * 16;
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float* red, int& turn) {
#pragma unroll
  for (int i = 0; i < NV; i++) v[i] = wsum<(TPR < 64 ? TPR : 64)>(v[i]);
  if constexpr (TPR > 64) {
    float* s = red + (turn & 1) * RED;
    turn++;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < NV; i++) s[i * 16 + (threadIdx.x >> 6)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; i++) v[i] = sum16(s[i * 16 + (threadIdx.x & 15)]);
  }
}

// Mean and 1 / spread of a row held as v[NCH][8]; own: the columns of the last chunk that are this lane's.  The others are left out
// by a select: multiplied by 0, an infinity would become NaN.
// The squares are taken about a mean, never about zero.  A workgroup's row needs one exchange for both: each wave takes its
// squares about its own mean, and M2 = sum_w M2_w + (sum_w - n_w mean)^2 / n_w, n_w the columns of wave w.
template <int TPR, int NCH>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][8], const bool (&own)[8], int kind, int D, float inv_d, float eps,
                                          float* red, int& turn, float& mean, float& rstd) {
  mean = 0.f;
  float s = 0.f;
  if (kind == NORM_LAYER) {
#pragma unroll
    for (int c = 0; c < NCH; c++)
#pragma unroll
      for (int i = 0; i < 8; i++) s += c < NCH - 1 || own[i] ? v[c][i] : 0.f;
    s = wsum<(TPR < 64 ? TPR : 64)>(s);
    if constexpr (TPR > 64) {
      mean = s * __builtin_amdgcn_rcpf((float)max(wave_cols<NCH>(threadIdx.x >> 6, D), 1));
    } else {
      mean = s * inv_d;
    }
  }
  float q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < NCH; c++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float e = c < NCH - 1 || own[i] ? v[c][i] - mean : 0.f;
      q[0] += e * e;
    }
  if (TPR > 64 && kind == NORM_LAYER) {
    q[0] = wsum(q[0]);
    float* r = red + (turn & 1) * RED;
    turn++;
    if ((threadIdx.x & 63) == 0) {
      r[threadIdx.x >> 6] = s;
      r[16 + (threadIdx.x >> 6)] = q[0];
    }
    __syncthreads();
    const int w = threadIdx.x & 15, n = wave_cols<NCH>(w, D);
    const float sw = r[w];
    mean = sum16(sw) * inv_d;
    const float d = sw - (float)n * mean;
    q[0] = sum16(r[16 + w] + (n > 0 ? d * d * __builtin_amdgcn_rcpf((float)n) : 0.f));
  } else {
    row_sum<TPR, 1>(q, red, turn);
  }
  rstd = 1.f / sqrtf(q[0] * inv_d + eps);
}

// Rows of TPR <= 64 lanes share a workgroup of four waves (independent in the forward; in the backward they add their column
// sums); wider rows have a workgroup each, of at most TPR threads.
template <int TPR> constexpr int threads() { return TPR <= 64 ? 256 : TPR; }
template <int TPR> __device__ __forceinline__ long first_row() {
  if constexpr (TPR > 64) return blockIdx.x;
  // a wave's row is uniform: its address goes into scalar registers
  const int in = TPR == 64 ? (int)__builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / TPR;
  return (long)blockIdx.x * (256 / TPR) + in;
}

// column constants of one chunk: vector loads behind uniform tests
template <bool SMALL>
__device__ __forceinline__ void fold(const ScpResidualNorm& a, int base, float* A1, float* B1, float* W2) {
  const int D = a.cols;
  float S[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    S[i] = a.scale_value;
    B1[i] = 0.f;
    W2[i] = 1.f;
  }
  if (a.scale_mode == SCALE_ONE) {
    const float s = a.scale[0];
#pragma unroll
    for (int i = 0; i < 8; i++) S[i] = s;
  } else if (a.scale_mode == SCALE_COL) {
    const vf8 s = ld8<SMALL, float>(a.scale, base, D);
#pragma unroll
    for (int i = 0; i < 8; i++) S[i] = s[i];
  }
  if (a.gate_mode == GATE_COL) {
    const vf8 g = ld8<SMALL, float>((const float*)a.gate, base, D);
#pragma unroll
    for (int i = 0; i < 8; i++) S[i] *= gate_value(g[i], a.gate_act);
  }
  if (a.b1) {
    const vf8 b = ld8<SMALL, float>(a.b1, base, D);
#pragma unroll
    for (int i = 0; i < 8; i++) B1[i] = b[i] * S[i];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) A1[i] = S[i];
  if (a.w1) {
    const vf8 w = ld8<SMALL, float>(a.w1, base, D);
#pragma unroll
    for (int i = 0; i < 8; i++) A1[i] = w[i] * S[i];
  }
  if (a.w2) {
    const vf8 w = ld8<SMALL, float>(a.w2, base, D);
#pragma unroll
    for (int i = 0; i < 8; i++) W2[i] = w[i];
  }
}

// GF: a gate for every element
template <typename XT, typename HT, int TPR, int NCH, bool GF, bool SMALL>
__global__ __launch_bounds__(threads<TPR>()) void rnorm_fwd_kernel(ScpResidualNorm a) {
  constexpr int RPW = TPR <= 64 ? 256 / TPR : 1;
  __shared__ float red[TPR > 64 ? 2 * RED : 1];
  const int t = RPW > 1 ? threadIdx.x & (TPR - 1) : threadIdx.x, D = a.cols;
  const int nt = RPW > 1 ? TPR : blockDim.x;      // threads of a row
  const float inv_d = 1.f / (float)D;
  int turn = 0;
  if constexpr (TPR > 64) {
    for (int i = threadIdx.x; i < 2 * RED; i += blockDim.x) red[i] = 0.f;
    __syncthreads();
  }
  long row = first_row<TPR>();
  const long stride = (long)gridDim.x * RPW;
  int base[NCH];
#pragma unroll
  for (int c = 0; c < NCH; c++) base[c] = chunk_base(t + nt * c, D);
  const bool last = 8 * (t + nt * (NCH - 1)) < D;     // this lane's last chunk exists; the others always do
  bool own[8];
#pragma unroll
  for (int i = 0; i < 8; i++) own[i] = chunk_owns(t + nt * (NCH - 1), i, D);

  // the next row's values are fetched while this one's sums run
  struct Raw {
    typename Vec8<XT>::v x[NCH];
    typename Vec8<HT>::v h[NCH], g[GF ? NCH : 1];
    float grow;
  };
  auto load = [&](long r) {
    Raw v;
    v.grow = a.gate_mode == GATE_ROW ? ((const float*)a.gate)[r] : 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      v.x[c] = ld8<SMALL, XT>((const XT*)a.x + r * a.ldx, base[c], D);
      if (a.h) v.h[c] = ld8<SMALL, HT>((const HT*)a.h + r * a.ldh, base[c], D);
      if constexpr (GF) v.g[c] = ld8<SMALL, HT>((const HT*)a.gate + r * a.ldg, base[c], D);
    }
    return v;
  };
  if (row >= a.rows) return;
  constexpr bool EARLY = !(TPR == 1024 && NCH == 2);      // (there the next row's values would spill)
  Raw cur;
  if (EARLY) cur = load(row);

  float A1[NCH][8], B1[NCH][8], W2[NCH][8], B2[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    fold<SMALL>(a, base[c], A1[c], B1[c], W2[c]);
#pragma unroll
    for (int i = 0; i < 8; i++) B2[c][i] = 0.f;
    if (a.b2) {
      const vf8 b = ld8<SMALL, float>(a.b2, base[c], D);
#pragma unroll
      for (int i = 0; i < 8; i++) B2[c][i] = b[i];
    }
  }

  for (; row < a.rows; row += stride) {
    const Raw v = EARLY ? cur : load(row);
    if (EARLY && row + stride < a.rows) cur = load(row + stride);
    float r[NCH][8];
    float m1 = 0.f, s1 = 1.f, m2, s2;
    if (a.h) {
      float h[NCH][8];
#pragma unroll
      for (int c = 0; c < NCH; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) h[c][i] = (float)v.h[c][i];
      const float grow = a.gate_mode == GATE_ROW ? gate_value(v.grow, a.gate_act) : 1.f;
      if (a.post != NORM_NONE) row_stats<TPR, NCH>(h, own, a.post, D, inv_d, a.eps, red, turn, m1, s1);
#pragma unroll
      for (int c = 0; c < NCH; c++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          float g = grow;
          if constexpr (GF) g = gate_value((float)v.g[c][i], a.gate_act);
          r[c][i] = (float)v.x[c][i] + ((h[c][i] - m1) * s1 * A1[c][i] + B1[c][i]) * g;
        }
        if (c < NCH - 1 || last) st8<SMALL, XT>((XT*)a.r + row * D, base[c], D, r[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NCH; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) r[c][i] = (float)v.x[c][i];
    }
    row_stats<TPR, NCH>(r, own, a.pre, D, inv_d, a.eps, red, turn, m2, s2);
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = (r[c][i] - m2) * s2 * W2[c][i] + B2[c][i];
      if (c < NCH - 1 || last) st8<SMALL, HT>((HT*)a.y + row * D, base[c], D, y);
    }
    if (a.stats && t == 0) {
      f32x4 s = {m1, s1, m2, s2};
      *(f32x4*)(a.stats + row * 4) = s;
    }
  }
}

// waves per SIMD that the registers have to leave room for (second argument of __launch_bounds__)
constexpr int bwd_waves(int tpr) { return tpr == 1024 ? 4 : tpr == 768 ? 3 : 2; }

// Partial column sums: ws[block][4][cols], order P, sum dy rhat, Q, sum dy; without BIAS (no post bias, no gradient of a pre
// bias) the last two stay unwritten.
// Rows above 8192 columns (WIDE) have no registers left for column sums: the row's two means are kept in rowc[rows][2] and
// rnorm_colpass_kernel reads the tensors once more.
template <typename XT, typename HT, int TPR, int NCH, bool GF, bool BIAS, bool SMALL>
__global__ __launch_bounds__(threads<TPR>(), bwd_waves(TPR)) void rnorm_bwd_kernel(ScpResidualNorm a, float* rowc) {
  constexpr int RPW = TPR <= 64 ? 256 / TPR : 1, NA = BIAS ? 4 : 2;
  __shared__ float red[TPR > 64 ? 2 * RED : 1];
  __shared__ float colbuf[RPW > 1 ? 2 * 256 * NCH * 8 : 1];
  const int t = RPW > 1 ? threadIdx.x & (TPR - 1) : threadIdx.x, D = a.cols;
  const int nt = RPW > 1 ? TPR : blockDim.x;      // threads of a row
  const float inv_d = 1.f / (float)D;
  int turn = 0;
  if constexpr (TPR > 64) {
    for (int i = threadIdx.x; i < 2 * RED; i += blockDim.x) red[i] = 0.f;
    __syncthreads();
  }
  long row = first_row<TPR>();
  const long stride = (long)gridDim.x * RPW;
  int base[NCH];
#pragma unroll
  for (int c = 0; c < NCH; c++) base[c] = chunk_base(t + nt * c, D);
  const bool last = 8 * (t + nt * (NCH - 1)) < D;
  bool own[8];
#pragma unroll
  for (int i = 0; i < 8; i++) own[i] = chunk_owns(t + nt * (NCH - 1), i, D);

  struct Raw {
    typename Vec8<XT>::v x[NCH], dr[NCH];
    typename Vec8<HT>::v h[NCH], g[GF ? NCH : 1], dy[NCH];
    f32x4 st;
    float grow;
  };
  auto load = [&](long r) {
    Raw v;
    v.st = *(const f32x4*)(a.stats + r * 4);
    v.grow = a.gate_mode == GATE_ROW ? ((const float*)a.gate)[r] : 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      v.x[c] = ld8<SMALL, XT>((const XT*)a.x + r * a.ldx, base[c], D);
      if (a.h) v.h[c] = ld8<SMALL, HT>((const HT*)a.h + r * a.ldh, base[c], D);
      else
#pragma unroll
        for (int i = 0; i < 8; i++) v.h[c][i] = (HT)0.f;
      if constexpr (GF) v.g[c] = ld8<SMALL, HT>((const HT*)a.gate + r * a.ldg, base[c], D);
      if (a.dy) v.dy[c] = ld8<SMALL, HT>((const HT*)a.dy + r * a.lddy, base[c], D);
      else
#pragma unroll
        for (int i = 0; i < 8; i++) v.dy[c][i] = (HT)0.f;
      if (a.dr) v.dr[c] = ld8<SMALL, XT>((const XT*)a.dr + r * a.lddr, base[c], D);
      else
#pragma unroll
        for (int i = 0; i < 8; i++) v.dr[c][i] = (XT)0.f;
    }
    return v;
  };
  float A1[NCH][8], B1[NCH][8], W2[NCH][8];
  constexpr bool WIDE = TPR == 1024;
  float acc[WIDE ? 1 : NA][WIDE ? 1 : NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; c++) {
    fold<SMALL>(a, base[c], A1[c], B1[c], W2[c]);
    if constexpr (!BIAS)
#pragma unroll
      for (int i = 0; i < 8; i++) B1[c][i] = 0.f;
#pragma unroll
    for (int k = 0; k < (WIDE ? 0 : NA); k++)
#pragma unroll
      for (int i = 0; i < 8; i++) acc[k][c][i] = 0.f;
  }
  const bool layer1 = a.post == NORM_LAYER, norm1 = a.post != NORM_NONE, layer2 = a.pre == NORM_LAYER;

  // Fetching the next row early is worth half of the waves where the registers allow it (32768 x 4096 bf16: 305 us against
  // 396 us with four waves per SIMD and no early fetch); with 16 columns per lane it spills (1024 x 900 fp32: 21 against 17 us).
  constexpr bool EARLY = NCH == 1 && TPR < 1024;
  Raw cur;
  if (EARLY && row < a.rows) cur = load(row);
  for (; row < a.rows; row += stride) {
    const Raw v = EARLY ? cur : load(row);
    if (EARLY && row + stride < a.rows) cur = load(row + stride);
    // y not used: its norm has no share in du, not even where the row has none (an infinity)
    const float m1 = v.st[0], s1 = v.st[1], m2 = v.st[2], s2 = a.dy ? v.st[3] : 0.f;
    float hh[NCH][8], rh[NCH][8], du[NCH][8], G[GF ? NCH : 1][8], dG[GF ? NCH : 1][8];
    const float grow = a.gate_mode == GATE_ROW ? gate_value(v.grow, a.gate_act) : 1.f;
    float c12[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; c++) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float g = grow;
        if constexpr (GF) g = G[c][i] = gate_both((float)v.g[c][i], a.gate_act, dG[c][i]);
        hh[c][i] = ((float)v.h[c][i] - m1) * s1;
        // without a block A1 is the scale's default, but the statistics are 0 and 1 and h is zero: nothing is added
        const float r = (float)v.x[c][i] + (hh[c][i] * A1[c][i] + B1[c][i]) * g;
        rh[c][i] = a.dy ? (r - m2) * s2 : 0.f;
        const float dy = (float)v.dy[c][i], av = dy * W2[c][i];
        du[c][i] = (float)v.dr[c][i] + s2 * av;
        const bool in = c < NCH - 1 || own[i];
        c12[0] += in ? av : 0.f;
        c12[1] += in ? av * rh[c][i] : 0.f;
        if constexpr (!WIDE) {
          acc[1][c][i] += dy * rh[c][i];
          if constexpr (BIAS) acc[3][c][i] += dy;
        }
      }
    }
    if (a.dy) row_sum<TPR, 2>(c12, red, turn);
    // means that the norm does not have stay 0, whatever their sums are
    const float c1 = layer2 ? s2 * c12[0] * inv_d : 0.f, c2 = s2 * c12[1] * inv_d;
    if (WIDE && a.ws && t == 0) {
      rowc[row * 2] = c1;
      rowc[row * 2 + 1] = c2;
    }
    float e[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; c++) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        du[c][i] -= c1 + rh[c][i] * c2;
        float g = grow;
        if constexpr (GF) g = G[c][i];
        const float dg = du[c][i] * g;
        if constexpr (!WIDE) {
          acc[0][c][i] += dg * hh[c][i];
          if constexpr (BIAS) acc[2][c][i] += dg;
        }
        const bool in = c < NCH - 1 || own[i];
        const float b = dg * A1[c][i];
        e[0] += in ? b : 0.f;
        e[1] += in ? b * hh[c][i] : 0.f;
        if constexpr (!GF) e[2] += in ? du[c][i] * (hh[c][i] * A1[c][i] + B1[c][i]) : 0.f;
      }
      if (a.dx && (c < NCH - 1 || last)) st8<SMALL, XT>((XT*)a.dx + row * D, base[c], D, du[c]);
    }
    if (!a.h) continue;
    row_sum<TPR, GF ? 2 : 3>((float(&)[GF ? 2 : 3])e, red, turn);
    const float e1 = layer1 ? e[0] * inv_d : 0.f, e2 = norm1 ? e[1] * inv_d : 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      if (c == NCH - 1 && !last) continue;
      float dh[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float g = grow;
        if constexpr (GF) g = G[c][i];
        dh[i] = s1 * (du[c][i] * g * A1[c][i] - e1 - (norm1 ? hh[c][i] * e2 : 0.f));
      }
      if (a.dh) st8<SMALL, HT>((HT*)a.dh + row * D, base[c], D, dh);
      if constexpr (GF) {
        float dg[8];
#pragma unroll
        for (int i = 0; i < 8; i++) dg[i] = du[c][i] * (hh[c][i] * A1[c][i] + B1[c][i]) * dG[c][i];
        if (a.dgate) st8<SMALL, HT>((HT*)a.dgate + row * D, base[c], D, dg);
      }
    }
    if (!GF && a.dgate && a.gate_mode == GATE_ROW && t == 0) {
      float d;
      gate_both(v.grow, a.gate_act, d);
      ((float*)a.dgate)[row] = e[2] * d;
    }
  }

  if (WIDE || !a.ws) return;
  float* wsb = a.ws + (long)blockIdx.x * 4 * D;
  if constexpr (RPW > 1) {
    // two sums at a time: every row's lanes lay their own into LDS, then the workgroup adds them in order
    const int w = threadIdx.x / TPR;
#pragma unroll
    for (int k0 = 0; k0 < NA; k0 += 2) {
      if (k0) __syncthreads();
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
          for (int i = 0; i < 8; i++) colbuf[((k * RPW + w) * NCH * 8 + c * 8 + i) * TPR + t] = acc[k0 + k][c][i];
      __syncthreads();
      for (int j = threadIdx.x; j < 2 * D; j += 256) {
        const int k = j >= D, col = j - k * D, q = col >> 3, ch = q / TPR;
        const int i = col - chunk_base(q, D);
        float s = 0.f;
#pragma unroll
        for (int ww = 0; ww < RPW; ww++) s += colbuf[((k * RPW + ww) * NCH * 8 + ch * 8 + i) * TPR + (q & (TPR - 1))];
        wsb[(long)(k0 + k) * D + col] = s;
      }
    }
  } else if constexpr (!WIDE) {
#pragma unroll
    for (int k = 0; k < NA; k++)
#pragma unroll
      for (int c = 0; c < NCH; c++)
        if (c < NCH - 1 || last) st8<SMALL, float>(wsb + (long)k * D, base[c], D, acc[k][c]);
  }
}

// The column sums of rows above 8192 columns: a thread takes 8 columns and every gridDim.y-th row, with the rows' statistics
// and means at hand; ws as rnorm_bwd_kernel leaves it, one partial row per blockIdx.y.
template <typename XT, typename HT, bool GF, bool BIAS>
__global__ __launch_bounds__(256) void rnorm_colpass_kernel(ScpResidualNorm a, const float* __restrict__ rowc) {
  const int D = a.cols, q = blockIdx.x * 256 + threadIdx.x, base = chunk_base(q, D);
  if (8 * q >= D) return;
  float A1[8], B1[8], W2[8], acc[BIAS ? 4 : 2][8];
  fold<false>(a, base, A1, B1, W2);
#pragma unroll
  for (auto& k : acc)
#pragma unroll
    for (int i = 0; i < 8; i++) k[i] = 0.f;
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const f32x4 st = *(const f32x4*)(a.stats + row * 4);
    const float c1 = rowc[row * 2], c2 = rowc[row * 2 + 1], s2 = a.dy ? st[3] : 0.f;
    const auto xv = ld8<false, XT>((const XT*)a.x + row * a.ldx, base, D);
    typename Vec8<HT>::v hv, gv, yv;
    typename Vec8<XT>::v rv;
    if (a.h) hv = ld8<false, HT>((const HT*)a.h + row * a.ldh, base, D);
    if constexpr (GF) gv = ld8<false, HT>((const HT*)a.gate + row * a.ldg, base, D);
    if (a.dy) yv = ld8<false, HT>((const HT*)a.dy + row * a.lddy, base, D);
    if (a.dr) rv = ld8<false, XT>((const XT*)a.dr + row * a.lddr, base, D);
    const float grow = a.gate_mode == GATE_ROW ? gate_value(((const float*)a.gate)[row], a.gate_act) : 1.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float g = grow;
      if constexpr (GF) g = gate_value((float)gv[i], a.gate_act);
      const float hh = a.h ? ((float)hv[i] - st[0]) * st[1] : 0.f;
      const float rh = a.dy ? ((float)xv[i] + (hh * A1[i] + B1[i]) * g - st[2]) * s2 : 0.f;
      const float dy = a.dy ? (float)yv[i] : 0.f;
      const float dg = ((a.dr ? (float)rv[i] : 0.f) + s2 * dy * W2[i] - (c1 + rh * c2)) * g;
      acc[0][i] += dg * hh;
      acc[1][i] += dy * rh;
      if constexpr (BIAS) {
        acc[2][i] += dg;
        acc[3][i] += dy;
      }
    }
  }
  float* p = a.ws + (long)blockIdx.y * 4 * D;
#pragma unroll
  for (int k = 0; k < (BIAS ? 4 : 2); k++) st8<false, float>(p + (long)k * D, base, D, acc[k]);
}

// The columns' sums of the partial rows (fixed order, fp64), and from them the parameters' gradients.  A workgroup takes 32
// columns; 32 threads share a column, four rows of all sums in flight each.
template <bool BIAS>
__global__ __launch_bounds__(1024) void rnorm_cols_kernel(ScpResidualNorm a, int nblk, float* each) {
  constexpr int NA = BIAS ? 4 : 2;
  __shared__ double part[NA][32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + cx, D = a.cols;
  double s[NA];
#pragma unroll
  for (int k = 0; k < NA; k++) s[k] = 0.0;
  if (col < D) {
    const float* p = a.ws + col;
    int b = ry;
    for (; b + 96 < nblk; b += 128) {
      float v[4][NA];
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int k = 0; k < NA; k++) v[u][k] = p[((long)(b + 32 * u) * 4 + k) * D];
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int k = 0; k < NA; k++) s[k] += (double)v[u][k];
    }
    for (; b < nblk; b += 32)
#pragma unroll
      for (int k = 0; k < NA; k++) s[k] += (double)p[((long)b * 4 + k) * D];
  }
#pragma unroll
  for (int k = 0; k < NA; k++) part[k][ry][cx] = s[k];
  __syncthreads();
  // 32 x NA sums of 32: one per thread of the first NA half-waves
  if (ry < NA) {
    double q = 0.0;
#pragma unroll
    for (int y = 0; y < 32; y++) q += part[ry][y][cx];
    part[ry][0][cx] = q;      // read by this thread only before the barrier
  }
  __syncthreads();
  if (ry || col >= D) return;
  const double P = part[0][0][cx], Q = BIAS ? part[NA / 2][0][cx] : 0.0;
  if (a.dw2) a.dw2[col] = (float)part[1][0][cx];
  if constexpr (BIAS)
    if (a.db2) a.db2[col] = (float)part[3][0][cx];
  if (a.want1) {
    const float sc = a.scale_mode == SCALE_COL ? a.scale[col] : a.scale_mode == SCALE_ONE ? a.scale[0] : a.scale_value;
    float g = 1.f, d = 1.f;
    if (a.gate_mode == GATE_COL) g = gate_both(((const float*)a.gate)[col], a.gate_act, d);
    const double n = (a.w1 ? a.w1[col] : 1.f) * P + (BIAS && a.b1 ? a.b1[col] * Q : 0.0);
    if (a.dw1) a.dw1[col] = (float)(sc * g * P);
    if (a.db1) a.db1[col] = (float)(sc * g * Q);
    if (a.gate_mode == GATE_COL && a.dgate) ((float*)a.dgate)[col] = (float)(sc * d * n);
    if (a.dscale && a.scale_mode == SCALE_COL) a.dscale[col] = (float)(g * n);
    if (each) each[col] = (float)(g * n);
  }
}

// gradient of a single residual scale: the columns' shares added up by one workgroup
__global__ __launch_bounds__(1024) void rnorm_scale_kernel(const float* each, int D, float* out) {
  __shared__ double red[16];
  double s = 0.0;
  for (int j = threadIdx.x; j < D; j += 1024) s += (double)each[j];
  s = block_sum_d(s, red);
  if (threadIdx.x == 0) out[0] = (float)s;
}

constexpr int MAX_COLS = 16384;

// Lanes of a row in a shared workgroup, 8 columns each; wider rows have a workgroup each, of as many waves as they need.
int row_lanes(int cols) { return cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : 64; }
unsigned wide_threads(int cols, int nch) { return 64u * ((cols + 512 * nch - 1) / (512 * nch)); }

// Workgroups of the backward: about those that are resident at once, since each leaves a partial row per column sum (above 8192
// columns: the partial rows of the column pass)
int bwd_grid(long rows, int cols) {
  const int rpw = cols <= 512 ? 256 / row_lanes(cols) : 1;
  const long need = (rows + rpw - 1) / rpw;
  // (513 .. 1024 columns: two waves to a workgroup; few rows leave fewer partial rows, whose sum then costs as much as they do)
  const long cap = cols <= 512 ? 512 : cols <= 1024 ? (rows < 16384 ? 512 : 1024) : cols <= 2048 ? 512 : cols <= 8192 ? 256 : 128;
  return (int)(need < cap ? need : cap);
}

template <typename XT, typename HT, int TPR, int NCH, bool GF, bool SMALL = false>
int go_fwd(const ScpResidualNorm& a, hipStream_t st) {
  const unsigned T = TPR <= 64 ? 256 : wide_threads(a.cols, NCH);
  // About as many workgroups as are resident at once, each walking its rows with the next one on its way: beyond that a
  // workgroup's column constants come again for every row (777 rows of 4999 bf16: 14 us against 17 us with three times as many,
  // 777 x 8000 fp32 with a full gate 31 against 42 us, 4096 x 1024 fp32 with a full gate 20 against 24 us).  One-chunk rows
  // have 16 waves a CU; rows of at most 512 columns have few constants, and a minibatch of them is spread as widely as it goes.
  const long rpw = TPR <= 64 ? 256 / TPR : 1, need = (a.rows + rpw - 1) / rpw;
  const long cap = 256L * (a.cols <= 512 ? 8 : a.cols <= 1024 ? 2 : NCH == 2 ? 1 : 1024 / T);
  hipLaunchKernelGGL((rnorm_fwd_kernel<XT, HT, TPR, NCH, GF, SMALL>), dim3((unsigned)(need < cap ? need : cap)), dim3(T), 0, st, a);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}
template <typename XT, typename HT, int TPR, int NCH, bool GF, bool SMALL = false>
int go_bwd(const ScpResidualNorm& a, bool bias, hipStream_t st) {
  const int nblk = bwd_grid(a.rows, a.cols);
  const dim3 T(TPR <= 64 ? 256 : wide_threads(a.cols, NCH));
  if constexpr (TPR == 1024) {
    float* rowc = a.ws ? a.ws + (long)nblk * 4 * a.cols + a.cols : nullptr;
    hipLaunchKernelGGL((rnorm_bwd_kernel<XT, HT, TPR, NCH, GF, true, SMALL>), dim3((unsigned)(a.rows < 512 ? a.rows : 512)), T, 0, st,
                       a, rowc);
    SCP_LAUNCH_CHECK();
    if (!a.ws) return SCP_OK;
    const dim3 grid((a.cols + 2047) / 2048, nblk);
    if (bias) hipLaunchKernelGGL((rnorm_colpass_kernel<XT, HT, GF, true>), grid, dim3(256), 0, st, a, rowc);
    else hipLaunchKernelGGL((rnorm_colpass_kernel<XT, HT, GF, false>), grid, dim3(256), 0, st, a, rowc);
  } else {
    if (bias) hipLaunchKernelGGL((rnorm_bwd_kernel<XT, HT, TPR, NCH, GF, true, SMALL>), dim3(nblk), T, 0, st, a, nullptr);
    else hipLaunchKernelGGL((rnorm_bwd_kernel<XT, HT, TPR, NCH, GF, false, SMALL>), dim3(nblk), T, 0, st, a, nullptr);
  }
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

// bwd: 0 forward, 1 backward without bias sums, 2 with them
template <typename XT, typename HT, bool GF>
int by_width(const ScpResidualNorm& a, int bwd, hipStream_t st) {
  const int D = a.cols;
  if (bwd) {
    const bool bias = bwd == 2;
    if (D < 8) return go_bwd<XT, HT, 8, 1, GF, true>(a, bias, st);
    if (D <= 64) return go_bwd<XT, HT, 8, 1, GF>(a, bias, st);
    if (D <= 128) return go_bwd<XT, HT, 16, 1, GF>(a, bias, st);
    if (D <= 256) return go_bwd<XT, HT, 32, 1, GF>(a, bias, st);
    if (D <= 512) return go_bwd<XT, HT, 64, 1, GF>(a, bias, st);
    if (D <= 1024) return go_bwd<XT, HT, 128, 1, GF>(a, bias, st);
    if (D <= 2048) return go_bwd<XT, HT, 256, 1, GF>(a, bias, st);
    if (D <= 4096) return go_bwd<XT, HT, 512, 1, GF>(a, bias, st);
    if (D <= 6144) return go_bwd<XT, HT, 768, 1, GF>(a, bias, st);
    if (D <= 8192) return go_bwd<XT, HT, 512, 2, GF>(a, bias, st);
    return go_bwd<XT, HT, 1024, 2, GF>(a, bias, st);
  }
  if (D < 8) return go_fwd<XT, HT, 8, 1, GF, true>(a, st);
  if (D <= 64) return go_fwd<XT, HT, 8, 1, GF>(a, st);
  if (D <= 128) return go_fwd<XT, HT, 16, 1, GF>(a, st);
  if (D <= 256) return go_fwd<XT, HT, 32, 1, GF>(a, st);
  if (D <= 512) return go_fwd<XT, HT, 64, 1, GF>(a, st);
  if (D <= 1024) return go_fwd<XT, HT, 64, 2, GF>(a, st);
  if (D <= 4096) return go_fwd<XT, HT, 512, 1, GF>(a, st);
  if (D <= 6144) return go_fwd<XT, HT, 1024, 1, GF>(a, st);
  if (D <= 8192) return go_fwd<XT, HT, 512, 2, GF>(a, st);
  return go_fwd<XT, HT, 1024, 2, GF>(a, st);
}

template <bool GF>
int by_type(const ScpResidualNorm& a, int bwd, hipStream_t st) {
  if (!a.x_bf16 && !a.h_bf16) return by_width<float, float, GF>(a, bwd, st);
  if (!a.x_bf16) return by_width<float, __bf16, GF>(a, bwd, st);
  return by_width<__bf16, __bf16, GF>(a, bwd, st);
}

int launch_rows(const ScpResidualNorm& a, int bwd, hipStream_t st) {
  return a.gate_mode == GATE_FULL ? by_type<true>(a, bwd, st) : by_type<false>(a, bwd, st);
}

int check_args(const ScpResidualNorm* a, const char* who) {
  SCP_CHECK(a, SCP_ERR_ARG, "%s: null argument block", who);
  SCP_CHECK(a->rows > 0 && a->cols > 0, SCP_ERR_ARG, "%s: rows and cols must be positive (%ld, %d)", who, (long)a->rows,
            a->cols);
  SCP_CHECK(a->cols <= MAX_COLS, SCP_ERR_SHAPE, "%s: at most %d columns (got %d)", who, MAX_COLS, a->cols);
  SCP_CHECK(!(a->x_bf16 && !a->h_bf16), SCP_ERR_ARG, "%s: a bf16 residual stream needs bf16 blocks", who);
  SCP_CHECK(a->x && a->ldx >= 0 && a->ldh >= 0 && a->ldg >= 0, SCP_ERR_ARG, "%s: null x or negative row stride", who);
  SCP_CHECK(a->eps > 0.f && a->eps < __builtin_inff(), SCP_ERR_ARG, "%s: eps must be positive and finite", who);
  SCP_CHECK(a->pre == NORM_RMS || a->pre == NORM_LAYER, SCP_ERR_ARG, "%s: pre must be rms (1) or layer (2)", who);
  SCP_CHECK(a->post >= NORM_NONE && a->post <= NORM_LAYER, SCP_ERR_ARG, "%s: post must be 0, 1 or 2", who);
  SCP_CHECK(a->gate_mode >= GATE_NONE && a->gate_mode <= GATE_COL && a->gate_act >= ACT_NONE && a->gate_act <= ACT_TANH &&
                a->scale_mode >= SCALE_VALUE && a->scale_mode <= SCALE_COL, SCP_ERR_ARG, "%s: unknown gate or scale mode", who);
  SCP_CHECK((a->gate_mode == GATE_NONE || a->gate) && (a->scale_mode == SCALE_VALUE || a->scale), SCP_ERR_ARG,
            "%s: gate or scale mode without its values", who);
  SCP_CHECK(a->h || (a->gate_mode == GATE_NONE && a->post == NORM_NONE && a->scale_mode == SCALE_VALUE && !a->w1 && !a->b1),
            SCP_ERR_ARG, "%s: gate, scale or post norm without a block", who);
  return SCP_OK;
}

}  // namespace

extern "C" int scp_residual_norm_max_cols(void) { return MAX_COLS; }

extern "C" int scp_residual_norm_fwd(const ScpResidualNorm* a, void* stream) {
  int rc = check_args(a, "scp_residual_norm_fwd");
  if (rc) return rc;
  SCP_CHECK(a->y && (!a->h || a->r), SCP_ERR_ARG, "scp_residual_norm_fwd: null output");
  return launch_rows(*a, 0, (hipStream_t)stream);
}

extern "C" long scp_residual_norm_bwd_ws_floats(long rows, int cols) {
  if (rows <= 0 || cols <= 0 || cols > MAX_COLS) return 0;
  return (long)bwd_grid(rows, cols) * 4 * cols + cols + (cols > 8192 ? 2 * rows : 0);
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
  SCP_CHECK((!a.dh || a.h) && (!a.dw1 || a.w1) && (!a.db1 || a.b1) && (!a.dscale || a.scale_mode != SCALE_VALUE) &&
                (!a.dgate || a.gate_mode != GATE_NONE), SCP_ERR_ARG, "scp_residual_norm_bwd: gradient of an absent parameter");
  if (!(a.want1 || a.want2)) a.ws = nullptr;
  hipStream_t st = (hipStream_t)stream;
  const bool bias = a.b1 || a.db2;
  rc = launch_rows(a, bias ? 2 : 1, st);
  if (rc || !a.ws) return rc;
  const int nblk = bwd_grid(a.rows, a.cols);
  float* each = a.dscale && a.scale_mode == SCALE_ONE ? a.ws + (long)nblk * 4 * a.cols : nullptr;
  if (bias)
    hipLaunchKernelGGL((rnorm_cols_kernel<true>), dim3((a.cols + 31) / 32), dim3(1024), 0, st, a, nblk, each);
  else
    hipLaunchKernelGGL((rnorm_cols_kernel<false>), dim3((a.cols + 31) / 32), dim3(1024), 0, st, a, nblk, each);
  SCP_LAUNCH_CHECK();
  if (each) {
    hipLaunchKernelGGL(rnorm_scale_kernel, dim3(1), dim3(1024), 0, st, each, a.cols, a.dscale);
    SCP_LAUNCH_CHECK();
  }
  return SCP_OK;
}
