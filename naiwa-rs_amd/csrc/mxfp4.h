// The MXFP4 tile order of include/naiwa_mxfp4.h, shared by the quantiser and the expert
// products, and the internal entry point of the latter.
#pragma once

#include "common.h"

// Steps of 128 values, groups of 4 steps and bytes of a 16-row strip of k values.
__host__ __device__ inline int naiwa_mx_steps(int64_t k) { return (int)((k + 127) / 128); }
__host__ __device__ inline int naiwa_mx_groups(int64_t k) { return (naiwa_mx_steps(k) + 3) / 4; }
__host__ __device__ inline int64_t naiwa_mx_strip_bytes(int64_t k) {
    return (int64_t)1024 * naiwa_mx_steps(k) + (int64_t)256 * naiwa_mx_groups(k);
}

// One call of the expert products over MXFP4 banks (mxfp4_experts.hip).
struct NaiwaMxCall {
    const naiwa_bank *gate, *up, *down;
    const void* x;
    int x_dtype;
    const uint32_t* ids;
    const float* w;
    int rows, width, act;
    float* out;      // may be null with res
    int accumulate;
    int skip_zero;   // entries of weight 0 are left out (decode)
    uint16_t* res;   // bf16 [rows, H]: also res = bf16(res + out), or null
};

// Refusals that need no device; NAIWA_OK for a call that naiwa_mx_run takes.
int naiwa_mx_check(const NaiwaMxCall& c);
// Scratch bytes of a call, for any number of slots and either type of x.
size_t naiwa_mx_scratch_bytes(int rows, int width, int H, int I);
// The launches of a checked call over scratch ws.
int naiwa_mx_run(const NaiwaMxCall& c, uint8_t* ws, hipStream_t st);
