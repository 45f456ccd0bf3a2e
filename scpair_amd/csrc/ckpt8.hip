// 8-bit activation checkpoints: what a backward pass needs of an activation, in 1 + 1/64 byte per element.
//
// 64 consecutive columns of a row share a step 2^k, the smallest power of two with max|x| <= 127 * 2^k and -126 <= k <= 121;
// a code is x / 2^k rounded to the nearest whole number (ties to even), c in [-127, 127], and stands for c * 2^k (beyond
// 127 * 2^121 = 3.38e38 the codes saturate: 64 * 2^122 would be no fp32 number any more).  The step
// being a power of two, x / 2^k and c * 2^k are exact: the code is THE nearest one whatever the order of operations, and
// every value is exact in bf16 (7 significant bits), so a product that takes the codes apart loses nothing further.  The
// price against a step of max|x| / 127 is at most one bit.  Layout: codes int8 [rows][ld], ld = cols rounded up to 64,
// zeros behind cols; steps uint8 [rows][ld / 64], k + 127.  255 marks a group that held an infinity or a NaN: all its
// values read as NaN, so that a bad activation is seen in the gradients as it is without the checkpoint.
//
// Bound of every kernel here: HBM.  A lane holds 8 consecutive columns, 8 lanes a group; the group's maximum is a maximum
// of integers (the magnitudes' bit patterns, which also shows infinities and NaN) over three lane exchanges.  Measured,
// 16384 x 8192 bf16: packing 71 us, unpacking 67 us (0.40 GB each, 5.7 and 6.0 TB/s), silu 117-125 us forward with the packing
// (0.67 GB, 5.4-5.8 TB/s), 129-137 us backward (0.67 GB, 4.9-5.2 TB/s: two streams of reads and the arithmetic of the derivative).
#include "common.h"
#include "ckpt8.h"
#include "scpair_hip.h"

namespace {

enum { ACT_GELU = 0, ACT_SILU = 1, ACT_LEAKY = 2 };

// FAST (bf16 tensors): the hardware exponential and reciprocal; with libm's functions the bf16 kernels were bound by instruction
// issue (16384 x 8192 silu: 165 us forward).  gelu's values far left of zero are small but not zero, and a bf16 has its step
// relative to them, so the normal distribution function is fitted for relative error: exp(x^2 / 2) Phi(-|x|) = t P(t),
// t = 1 / (1 + 0.36 |x|), P of degree 6 by linear programming for the least weighted error on [0, 60].  Relative error below 1.4e-5
// (half a step is 3.9e-3), absolute error of Phi below 1.9e-7.  The exponential is shared with the derivative.  fp32 tensors: libm's
// functions, Phi = (1 + erf) / 2, whose error is absolute (6e-8).
__device__ __forceinline__ float normal_cdf_fast(float x, float gauss) {      // gauss = exp(-x^2 / 2)
  const float t = __builtin_amdgcn_rcpf(fmaf(0.36f, fabsf(x), 1.f));
  float p = fmaf(t, 0.0433475859f, -0.165669665f);
  p = fmaf(t, p, 0.159787104f);
  p = fmaf(t, p, 0.0424004421f);
  p = fmaf(t, p, 0.133603156f);
  p = fmaf(t, p, 0.142892405f);
  p = fmaf(t, p, 0.143639043f);
  const float tail = t * p * gauss;
  return x < 0.f ? tail : 1.f - tail;
}
// exp of a non-positive argument only, so that a Newton step on the reciprocal (1 .. 2) is safe.  The step makes silu of every bf16
// down to -87 the nearest bf16 to its value (the hardware's reciprocal alone: not at 5.9375, 5.6e-7 below the middle of two).
__device__ __forceinline__ float sigmoid_fast(float x) {
  const float e = __expf(-fabsf(x)), d = 1.f + e, r = __builtin_amdgcn_rcpf(d), q = fmaf(fmaf(-d, r, 1.f), r, r);
  return x < 0.f ? e * q : q;
}
template <bool FAST> __device__ __forceinline__ float act_value(float x, int kind, float slope) {
  if (kind == ACT_GELU) {
    if (FAST) return x * normal_cdf_fast(x, __expf(-0.5f * x * x));
    return 0.5f * x * (1.f + erff(x * 0.70710678f));
  }
  if (kind == ACT_SILU) return FAST ? x * sigmoid_fast(x) : x / (1.f + expf(-x));
  return x > 0.f ? x : slope == 0.f && x < 0.f ? 0.f : slope * x;      // (relu of -infinity is 0)
}
template <bool FAST> __device__ __forceinline__ float act_slope(float x, int kind, float slope) {
  if (kind == ACT_GELU) {
    if (FAST) {
      const float gauss = __expf(-0.5f * x * x);
      return fmaf(x * 0.39894228f, gauss, normal_cdf_fast(x, gauss));
    }
    return 0.5f * (1.f + erff(x * 0.70710678f)) + x * 0.39894228f * expf(-0.5f * x * x);
  }
  if (kind == ACT_SILU) {
    const float s = FAST ? __builtin_amdgcn_rcpf(1.f + __expf(-x)) : 1.f / (1.f + expf(-x));
    return s * (1.f + x * (1.f - s));
  }
  return x > 0.f ? 1.f : x <= 0.f ? slope : x;      // (a NaN group has no sign: NaN, like the others)
}

// ACT: also out = act(x), and codes may be null (no backward pass to come)
template <typename T, bool ACT>
__global__ __launch_bounds__(256) void pack8_kernel(const T* __restrict__ x, long ldx, Shape8 s, int8_t* __restrict__ codes,
                                                    uint8_t* __restrict__ steps, T* __restrict__ out, int kind, float slope) {
  FOR_CHUNKS(s) {
    const int col = ch * 8;
    float f[8];
    load8<T>(x + row * ldx, col, s.cols, f);
    if (codes) {
      unsigned step;
      const uint2 c = quantise(f, step);
      *(uint2*)(codes + row * s.ld + col) = c;
      if ((ch & 7) == 0) steps[row * (s.ld >> 6) + (ch >> 3)] = (uint8_t)step;
    }
    if (ACT) {
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = act_value<sizeof(T) == 2>(f[j], kind, slope);
      if (col < s.cols) store8<T>(out + row * s.cols, col, s.cols, f);
    }
  }
}

// GRAD: out = d * act'(values), else out = values
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ steps,
                                                      Shape8 s, const T* __restrict__ d, long ldd, T* __restrict__ out,
                                                      int kind, float slope) {
  FOR_CHUNKS(s) {
    const int col = ch * 8;
    if (col >= s.cols) continue;
    const uint2 c = *(const uint2*)(codes + row * s.ld + col);
    const float step = q8_step(steps[row * (s.ld >> 6) + (ch >> 3)]);
    float f[8], g[8];
    if (GRAD) load8<T>(d + row * ldd, col, s.cols, g);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      f[j] = (float)(int8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3))) * step;
      if (GRAD) f[j] = g[j] * act_slope<sizeof(T) == 2>(f[j], kind, slope);
    }
    store8<T>(out + row * s.cols, col, s.cols, f);
  }
}

int check_shape(const char* who, long rows, int cols, Shape8* s, unsigned* grid) {
  SCP_CHECK(rows > 0 && cols > 0, SCP_ERR_ARG, "%s: rows and cols must be positive (%ld, %d)", who, rows, cols);
  SCP_CHECK(cols <= SCP_Q8_MAX_COLS, SCP_ERR_SHAPE, "%s: at most %d columns (got %d)", who, SCP_Q8_MAX_COLS, cols);
  s->rows = rows;
  s->cols = cols;
  s->ld = (cols + 63) / 64 * 64;
  s->cpr = s->ld / 8;
  *grid = grid_of(*s);
  return SCP_OK;
}

}  // namespace

extern "C" int scp_pack8(const void* x, int bf16, long ldx, long rows, int cols, int8_t* codes, uint8_t* steps, void* stream) {
  Shape8 s;
  unsigned grid;
  if (int rc = check_shape("scp_pack8", rows, cols, &s, &grid)) return rc;
  SCP_CHECK(x && codes && steps && ldx >= 0, SCP_ERR_ARG, "scp_pack8: null pointer or negative row stride");
  SCP_CHECK(((uintptr_t)codes & 15) == 0, SCP_ERR_ARG, "scp_pack8: codes must be 16-byte aligned");
  if (bf16)
    hipLaunchKernelGGL((pack8_kernel<__bf16, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, (const __bf16*)x,
                       ldx, s, codes, steps, nullptr, 0, 0.f);
  else
    hipLaunchKernelGGL((pack8_kernel<float, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, (const float*)x, ldx,
                       s, codes, steps, nullptr, 0, 0.f);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

extern "C" int scp_unpack8(const int8_t* codes, const uint8_t* steps, long rows, int cols, void* out, int bf16, void* stream) {
  Shape8 s;
  unsigned grid;
  if (int rc = check_shape("scp_unpack8", rows, cols, &s, &grid)) return rc;
  SCP_CHECK(out && codes && steps, SCP_ERR_ARG, "scp_unpack8: null pointer");
  SCP_CHECK(((uintptr_t)codes & 15) == 0, SCP_ERR_ARG, "scp_unpack8: codes must be 16-byte aligned");
  if (bf16)
    hipLaunchKernelGGL((unpack8_kernel<__bf16, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, codes, steps, s,
                       nullptr, 0, (__bf16*)out, 0, 0.f);
  else
    hipLaunchKernelGGL((unpack8_kernel<float, false>), dim3(grid), dim3(256), 0, (hipStream_t)stream, codes, steps, s,
                       nullptr, 0, (float*)out, 0, 0.f);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

extern "C" int scp_act8_fwd(const void* x, int bf16, long ldx, long rows, int cols, int kind, float slope, void* out,
                            int8_t* codes, uint8_t* steps, void* stream) {
  Shape8 s;
  unsigned grid;
  if (int rc = check_shape("scp_act8_fwd", rows, cols, &s, &grid)) return rc;
  SCP_CHECK(x && out && !codes == !steps && ldx >= 0, SCP_ERR_ARG, "scp_act8_fwd: null pointer or negative row stride");
  SCP_CHECK(kind >= ACT_GELU && kind <= ACT_LEAKY, SCP_ERR_ARG, "scp_act8_fwd: unknown activation %d", kind);
  SCP_CHECK(((uintptr_t)codes & 15) == 0, SCP_ERR_ARG, "scp_act8_fwd: codes must be 16-byte aligned");
  if (bf16)
    hipLaunchKernelGGL((pack8_kernel<__bf16, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, (const __bf16*)x, ldx,
                       s, codes, steps, (__bf16*)out, kind, slope);
  else
    hipLaunchKernelGGL((pack8_kernel<float, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, (const float*)x, ldx,
                       s, codes, steps, (float*)out, kind, slope);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

extern "C" int scp_act8_bwd(const int8_t* codes, const uint8_t* steps, long rows, int cols, int kind, float slope,
                            const void* dout, int bf16, long ldd, void* dx, void* stream) {
  Shape8 s;
  unsigned grid;
  if (int rc = check_shape("scp_act8_bwd", rows, cols, &s, &grid)) return rc;
  SCP_CHECK(dout && dx && codes && steps && ldd >= 0, SCP_ERR_ARG, "scp_act8_bwd: null pointer or negative row stride");
  SCP_CHECK(kind >= ACT_GELU && kind <= ACT_LEAKY, SCP_ERR_ARG, "scp_act8_bwd: unknown activation %d", kind);
  SCP_CHECK(((uintptr_t)codes & 15) == 0, SCP_ERR_ARG, "scp_act8_bwd: codes must be 16-byte aligned");
  if (bf16)
    hipLaunchKernelGGL((unpack8_kernel<__bf16, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, codes, steps, s,
                       (const __bf16*)dout, ldd, (__bf16*)dx, kind, slope);
  else
    hipLaunchKernelGGL((unpack8_kernel<float, true>), dim3(grid), dim3(256), 0, (hipStream_t)stream, codes, steps, s,
                       (const float*)dout, ldd, (float*)dx, kind, slope);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}
