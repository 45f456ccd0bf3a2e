// 8-bit activation checkpoints: what the kernels that read them share (the format is described in ckpt8.hip).
#pragma once
#include "common.h"

#define SCP_Q8_BAD 255u           // step byte of a group that held an infinity or a NaN
#define SCP_Q8_MAX_COLS (1 << 24)

// the step a step byte stands for: 2^(e - 127), NaN for a bad group
__device__ __forceinline__ float q8_step(unsigned e) { return __uint_as_float(e == SCP_Q8_BAD ? 0x7fc00000u : e << 23); }

// Four codes to bf16 values, for the products that read a checkpoint.  127 - code is the byte's bits but the top one inverted, an
// unsigned byte that converts in one instruction; the fma's addend 127 * step is finite for every step up to 2^121 (128 * 2^121
// is not), and its result is exact.
__device__ __forceinline__ void q8_values(unsigned codes, float step, __bf16* out) {
  const unsigned u = codes ^ 0x7f7f7f7fu;
#pragma unroll
  for (int b = 0; b < 4; b++) out[b] = (__bf16)fmaf((float)((u >> (8 * b)) & 0xffu), -step, 127.f * step);
}

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

static inline unsigned grid_of(Shape8& s) {
  const long need = (s.rows * s.cpr + 255) / 256, cap = 256 * 32, grid = need < cap ? need : cap;
  s.drow = grid * 256 / s.cpr;
  s.dch = (int)(grid * 256 % s.cpr);
  return (unsigned)grid;
}

}  // namespace
