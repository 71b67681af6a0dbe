// Rows of router logits in registers: how a row lies over lanes, its loads, its softmax.
// Used by the balance loss (balance.hip) and the routed weights' gradient (router_grad.hip).
#pragma once

#include "common.h"

namespace {

constexpr int kMaxE = 1024;

template <bool BF16> __device__ __forceinline__ float load(const void* p, int64_t i) {
    return BF16 ? naiwa_bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}
// 4 values from an address that is a multiple of their size.
template <bool BF16> __device__ __forceinline__ void load4(const void* p, int64_t i, float* o) {
    if (BF16) {
        const uint2 v = *(const uint2*)((const uint16_t*)p + i);
        o[0] = naiwa_bf16_to_f32(v.x & 0xffffu), o[1] = naiwa_bf16_to_f32(v.x >> 16);
        o[2] = naiwa_bf16_to_f32(v.y & 0xffffu), o[3] = naiwa_bf16_to_f32(v.y >> 16);
    } else {
        const float4 v = *(const float4*)((const float*)p + i);
        o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    }
}

// How a row lies over lanes: L of them, V experts each, 4 by 4 where X4.
template <int L_, int V_, bool X4_> struct Row {
    static constexpr int L = L_, V = V_;
    static constexpr bool X4 = X4_;
    static __device__ __forceinline__ int expert(int l, int i) { return X4 ? 4 * l + 4 * L * (i / 4) + i % 4 : l + L * i; }
};

// v over aligned groups of L lanes (16 or 64), in every lane.
template <int L, class F> __device__ __forceinline__ float lanes_all(float v, F f) {
    v = f(v, naiwa_dpp<0xB1>(v));
    v = f(v, naiwa_dpp<0x4E>(v));
    v = f(v, naiwa_dpp<0x141>(v));
    v = f(v, naiwa_dpp<0x140>(v));
#pragma unroll
    for (int m = 16; m < L; m <<= 1) v = f(v, __shfl_xor(v, m, 64));
    return v;
}

// A row's logits (-inf past E, and for a row that is not `in` the batch).
template <class R, bool BF16>
__device__ __forceinline__ void row_load(const void* logits, int64_t row, bool in, int E, int l, float (&e)[R::V]) {
#pragma unroll
    for (int i = 0; i < R::V; ++i) e[i] = -INFINITY;
    if constexpr (R::X4) {
#pragma unroll
        for (int i = 0; i < R::V; i += 4)
            if (in && R::expert(l, i) < E) load4<BF16>(logits, row + R::expert(l, i), e + i);
    } else {
#pragma unroll
        for (int i = 0; i < R::V; ++i)
            if (in && R::expert(l, i) < E) e[i] = load<BF16>(logits, row + R::expert(l, i));
    }
}
// In place: the exponentials (0 past E) relative to the largest; their sum's inverse.  A row that
// is not `live` gives zeros, whatever it holds.
template <class R> __device__ __forceinline__ float row_exp(bool live, int E, int l, float (&e)[R::V]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < R::V; ++i) m = fmaxf(m, e[i]);
    m = lanes_all<R::L>(m, [](float a, float b) { return fmaxf(a, b); });
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < R::V; ++i) {
        e[i] = live && R::expert(l, i) < E ? expf(e[i] - m) : 0.0f;
        s += e[i];
    }
    s = lanes_all<R::L>(s, [](float a, float b) { return a + b; });
    return live ? 1.0f / s : 0.0f;
}

// f(Row) for rows of E experts; x4: rows of all tensors take 4 values at once.
template <class F> void by_experts(int E, bool x4, F f) {
    if (E <= 16) f(Row<16, 1, false>());
    else if (E <= 64) x4 ? f(Row<16, 4, true>()) : f(Row<16, 4, false>());
    else if (E <= 128) x4 ? f(Row<16, 8, true>()) : f(Row<16, 8, false>());
    else if (E <= 256) x4 ? f(Row<64, 4, true>()) : f(Row<64, 4, false>());
    else x4 ? f(Row<64, 16, true>()) : f(Row<64, 16, false>());
}
bool takes4(const void* p, int dtype, int ld, int E) {
    return !(((uintptr_t)p & (dtype == NAIWA_BF16 ? 7 : 15)) | (ld & 3) | (E & 3));
}

} // namespace
