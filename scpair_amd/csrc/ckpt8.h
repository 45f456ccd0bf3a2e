// 8-bit activation checkpoints: what the kernels that read them share (the format is described in ckpt8.hip).
#pragma once
#include "common.h"

#define SCP_Q8_BAD 255u           // step byte of a group that held an infinity or a NaN
#define SCP_Q8_MAX_COLS (1 << 24)

// the step a step byte stands for: 2^(e - 127), NaN for a bad group
__device__ __forceinline__ float q8_step(unsigned e) { return __uint_as_float(e == SCP_Q8_BAD ? 0x7fc00000u : e << 23); }
