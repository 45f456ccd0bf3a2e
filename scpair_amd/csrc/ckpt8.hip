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
// of integers (the magnitudes' bit patterns, which also shows infinities and NaN) over three lane exchanges.
#include "common.h"
#include "ckpt8.h"
#include "scpair_hip.h"

namespace {

typedef float vf8 __attribute__((ext_vector_type(8)));
typedef __bf16 vb8 __attribute__((ext_vector_type(8)));
template <typename T> struct Vec8;
template <> struct Vec8<float> { typedef vf8 v; typedef vf8 vu __attribute__((aligned(4))); };
template <> struct Vec8<__bf16> { typedef vb8 v; typedef vb8 vu __attribute__((aligned(2))); };

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int col, int D, float* f) {
  if (col + 8 <= D) {
    const typename Vec8<T>::v v = *(const typename Vec8<T>::vu*)(p + col);
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = col + i < D ? (float)p[col + i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int col, int D, const float* f) {
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

template <int CTRL> __device__ __forceinline__ unsigned dpp_umax(unsigned v) {
  const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
  return v > o ? v : o;
}

// codes and step of the group that 8 neighbouring lanes hold, 8 values each
__device__ __forceinline__ uint2 quantise(const float* f, unsigned& step) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const unsigned b = __float_as_uint(f[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  top = dpp_umax<0xB1>(top);     // lane ^ 1
  top = dpp_umax<0x4E>(top);     // lane ^ 2
  top = dpp_umax<0x141>(top);    // mirrored within 8 lanes: the other four
  // max|x| = m * 2^p, 1 <= m < 2: k = p - 6 if m <= 127 / 64 (fraction bits <= 0x7E0000), else p - 5
  const int k = (int)(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7E0000u ? 1 : 0);
  const bool bad = top >= 0x7f800000u;
  step = bad ? SCP_Q8_BAD : (unsigned)(k < 1 ? 1 : k > 248 ? 248 : k);
  const float inv = bad ? 0.f : __uint_as_float((254u - step) << 23);
  unsigned w[2] = {0u, 0u};
  if (!bad) {
#pragma unroll
    for (int i = 0; i < 8; i++) w[i >> 2] |= ((unsigned)(int)__builtin_amdgcn_fmed3f(rintf(f[i] * inv), -127.f, 127.f) & 0xffu) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

// chunk -> (row, first column): a row has ld / 8 chunks, a multiple of 8, so a group never straddles rows, and a group's 8
// lanes are in range together
struct Shape8 {
  long rows;
  int cols, ld, cpr;
  int dch;       // a thread's stride of gridDim.x * 256 chunks as rows and chunks
  long drow;
};
#define FOR_CHUNKS(s)                                                                                       \
  const unsigned i0_ = blockIdx.x * 256 + threadIdx.x; /* below 2^21 */                                     \
  long row = i0_ / (unsigned)(s).cpr;                                                                       \
  int ch = (int)(i0_ % (unsigned)(s).cpr);                                                                  \
  for (; row < (s).rows; ch += (s).dch, row += (s).drow + (ch >= (s).cpr), ch -= ch >= (s).cpr ? (s).cpr : 0)

enum { ACT_GELU = 0, ACT_SILU = 1, ACT_LEAKY = 2 };

__device__ __forceinline__ float act_value(float x, int kind, float slope) {
  if (kind == ACT_GELU) return 0.5f * x * (1.f + erff(x * 0.70710678f));
  if (kind == ACT_SILU) return x / (1.f + expf(-x));
  return x > 0.f ? x : slope * x;
}
__device__ __forceinline__ float act_slope(float x, int kind, float slope) {
  if (kind == ACT_GELU) return 0.5f * (1.f + erff(x * 0.70710678f)) + x * 0.39894228f * expf(-0.5f * x * x);
  if (kind == ACT_SILU) {
    const float s = 1.f / (1.f + expf(-x));
    return s * (1.f + x * (1.f - s));
  }
  return x > 0.f ? 1.f : slope;
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
      for (int j = 0; j < 8; j++) f[j] = act_value(f[j], kind, slope);
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
      if (GRAD) f[j] = g[j] * act_slope(f[j], kind, slope);
    }
    store8<T>(out + row * s.cols, col, s.cols, f);
  }
}

unsigned grid_of(Shape8& s) {
  const long need = (s.rows * s.cpr + 255) / 256, cap = 256 * 32, grid = need < cap ? need : cap;
  s.drow = grid * 256 / s.cpr;
  s.dch = (int)(grid * 256 % s.cpr);
  return (unsigned)grid;
}

// dst[rows][ldd] = src[rows][lds], zeros in columns cols .. ldd - 1: the 16-byte rows that the matrix kernels take
__global__ __launch_bounds__(256) void pad_bf16_kernel(const __bf16* __restrict__ src, long lds, Shape8 s, __bf16* __restrict__ dst) {
  FOR_CHUNKS(s) {
    const int col = ch * 8;
    float f[8];
    load8<__bf16>(src + row * lds, col, s.cols, f);
    store8<__bf16>(dst + row * s.ld, col, s.ld, f);
  }
}

// Partial column sums of a bf16 matrix: a workgroup takes 512 columns (8 per lane) and every gridDim.y-th group of four
// rows, one row a wave; part[blockIdx.y][cols].  Their sum in a fixed order follows in colsum_finish_kernel.
__global__ __launch_bounds__(256) void colsum_bf16_kernel(const __bf16* __restrict__ x, long ldx, long rows, int cols,
                                                          float* __restrict__ part) {
  __shared__ float buf[3][8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 512 + lane * 8;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < cols) {
    for (long r = (long)blockIdx.y * 4 + wave; r < rows; r += (long)gridDim.y * 4) {
      float f[8];
      load8<__bf16>(x + r * ldx, col, cols, f);
#pragma unroll
      for (int i = 0; i < 8; i++) acc[i] += f[i];
    }
  }
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
__global__ __launch_bounds__(256) void colsum_finish_kernel(const float* __restrict__ part, int n, int cols, float* __restrict__ out) {
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

int colsum_parts(long rows, int cols) {
  const long groups = (rows + 3) / 4, cap = 1024 / ((cols + 511) / 512);
  return (int)(groups < cap ? groups : cap < 32 ? (groups < 32 ? groups : 32) : cap);
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

extern "C" int scp_pad_bf16(const void* src, long lds, long rows, int cols, void* dst, long ldd, void* stream) {
  SCP_CHECK(rows > 0 && cols > 0 && src && dst && lds >= 0, SCP_ERR_ARG, "scp_pad_bf16: empty shape or null pointer");
  SCP_CHECK(ldd == (cols + 7) / 8 * 8 && ((uintptr_t)dst & 15) == 0, SCP_ERR_ARG,
            "scp_pad_bf16: the copy's rows are cols rounded up to 8, 16-byte aligned");
  Shape8 s;
  s.rows = rows;
  s.cols = cols;
  s.ld = (int)ldd;
  s.cpr = s.ld / 8;
  const unsigned grid = grid_of(s);
  hipLaunchKernelGGL(pad_bf16_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const __bf16*)src, lds, s, (__bf16*)dst);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}

extern "C" long scp_colsum_bf16_ws_floats(long rows, int cols) {
  return rows > 0 && cols > 0 ? (long)colsum_parts(rows, cols) * cols : 0;
}

extern "C" int scp_colsum_bf16(const void* x, long ldx, long rows, int cols, float* out, float* ws, void* stream) {
  SCP_CHECK(rows > 0 && cols > 0 && x && out && ws && ldx >= 0, SCP_ERR_ARG, "scp_colsum_bf16: empty shape or null pointer");
  const int n = colsum_parts(rows, cols);
  hipLaunchKernelGGL(colsum_bf16_kernel, dim3((cols + 511) / 512, n), dim3(256), 0, (hipStream_t)stream, (const __bf16*)x, ldx,
                     rows, cols, ws);
  SCP_LAUNCH_CHECK();
  hipLaunchKernelGGL(colsum_finish_kernel, dim3((cols + 15) / 16), dim3(256), 0, (hipStream_t)stream, ws, n, cols, out);
  SCP_LAUNCH_CHECK();
  return SCP_OK;
}
