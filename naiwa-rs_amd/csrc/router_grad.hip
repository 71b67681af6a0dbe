// The gradient of the routed weights with respect to the router's logits
// (include/naiwa_tokens.h): dl_e = p_e (sum_{j: id_j = e} dw_j - sum_j p_{id_j} dw_j), p the
// softmax over all experts or over the chosen ones.  A softmax of the chosen values of a full
// softmax, renormalised, is the softmax of the chosen logits, so two of the three modes are one.
//
// 16 lanes take a row of up to 128 experts and 16 chosen (64 lanes a longer one): its values stay in registers.
// Calls that add to a gradient where only chosen experts have one touch those alone.
// 32768 rows of 128, us (f32 and bf16): over the chosen 9.0 and 8.2, added 7.3 and 5.1; over all experts 10.7 and 9.8, added 11.2
// and 10.0, of 6.9 and 3.7 (added 10.2 and 5.3) at a copy's rate; a launch takes 3.
#include "../../include/naiwa_tokens.h"
#include "common.h"
#include "router_rows.h"
#include "spans.h"

#include <algorithm>

namespace {

constexpr int kThreads = 256;

// v over aligned groups of L lanes (up to 64), in every lane.
template <class F> __device__ __forceinline__ float group_all(float v, int L, F f) {
    for (int m = 1; m < L; m <<= 1) v = f(v, __shfl_xor(v, m, 64));
    return v;
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float plus(float a, float b) { return a + b; }

struct Chosen { // what lane j of a row's lanes knows of the row's pair j (j < k)
    uint32_t id; // >= E: none
    float dw;
};
__device__ __forceinline__ Chosen chosen(const uint32_t* ids, int64_t ids_ld, const float* dw, int64_t dw_ld, int64_t t,
                                         bool live, int j, int k, int E) {
    Chosen c{0xffffffffu, 0.0f};
    if (live && j < k) c.id = ids[t * ids_ld + j];
    if (c.id < (uint32_t)E) c.dw = dw[t * dw_ld + j];
    else c.id = 0xffffffffu;
    return c;
}
// p_j (dw_j - sum p dw) of the lane's pair, with p the softmax over the chosen logits.
__device__ __forceinline__ float chosen_grad(const Chosen& c, float logit, int L) {
    const bool in = c.id != 0xffffffffu;
    const float m = group_all(in ? logit : -INFINITY, L, larger);
    const float e = in ? expf(logit - m) : 0.0f;
    const float p = e / group_all(e, L, plus);
    const float mean = group_all(in ? p * c.dw : 0.0f, L, plus);
    return in ? p * (c.dw - mean) : 0.0f;
}

template <bool BF16> __device__ __forceinline__ void store(void* p, int64_t i, float v) {
    if (BF16)
        ((uint16_t*)p)[i] = (uint16_t)naiwa_f32_to_bf16(v);
    else
        ((float*)p)[i] = v;
}

// Added to the chosen experts' gradients alone: L lanes a row, a lane a pair.
template <bool BF16>
__global__ void __launch_bounds__(kThreads)
chosen_kernel(const void* logits, int64_t ld, const uint32_t* ids, int64_t ids_ld, const float* dw, int64_t dw_ld,
              int64_t T, int E, int k, int L, const uint8_t* mask, void* dlogits, int64_t dld) {
    const int tid = threadIdx.x, j = tid & (L - 1), G = kThreads / L;
    for (int64_t t0 = (int64_t)blockIdx.x * G; t0 < T; t0 += (int64_t)gridDim.x * G) {
        const int64_t t = t0 + tid / L;
        const bool live = t < T && (!mask || mask[t]);
        const Chosen c = chosen(ids, ids_ld, dw, dw_ld, t, live, j, k, E);
        const bool in = c.id != 0xffffffffu;
        const float g = chosen_grad(c, in ? load<BF16>(logits, t * ld + c.id) : 0.0f, L);
        // an id that a row names twice gets both shares, from the first
        float sum = 0.0f;
        bool first = true;
        for (int i = 0; i < k; ++i) {
            const uint32_t id = (uint32_t)__shfl((int)c.id, i, L);
            const float other = __shfl(g, i, L);
            if (id == c.id) sum += other, first = first && i >= j;
        }
        if (in && first) {
            const int64_t at = t * dld + c.id;
            store<BF16>(dlogits, at, load<BF16>(dlogits, at) + sum);
        }
    }
}

// Whole rows.  FULL: p over all experts.
template <class R, bool BF16, bool FULL>
__global__ void __launch_bounds__(kThreads)
row_kernel(const void* logits, int64_t ld, const uint32_t* ids, int64_t ids_ld, const float* dw, int64_t dw_ld, int64_t T,
           int E, int k, const uint8_t* mask, void* dlogits, int64_t dld, int accumulate) {
    constexpr int L = R::L, V = R::V, G = kThreads / L;
    const int tid = threadIdx.x, l = tid % L;
    for (int64_t t0 = (int64_t)blockIdx.x * G; t0 < T; t0 += (int64_t)gridDim.x * G) {
        const int64_t t = t0 + tid / L;
        const bool in = t < T, live = in && (!mask || mask[t]);
        const Chosen c = chosen(ids, ids_ld, dw, dw_ld, t, live, l, k, E);
        float p[V], d[V] = {}, inv = 0.0f, g = c.dw;
        if constexpr (FULL) {
            row_load<R, BF16>(logits, t * ld, live, E, l, p);
            inv = row_exp<R>(live, E, l, p);
        } else {
            g = chosen_grad(c, c.id != 0xffffffffu ? load<BF16>(logits, t * ld + c.id) : 0.0f, L);
        }
        for (int j = 0; j < k; ++j) {
            const uint32_t id = (uint32_t)__shfl((int)c.id, j, L);
            const float v = __shfl(g, j, L);
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] += (uint32_t)R::expert(l, i) == id ? v : 0.0f;
        }
        if constexpr (FULL) {
            float mean = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] *= inv, mean = __builtin_fmaf(p[i], d[i], mean);
            mean = lanes_all<L>(mean, [](float a, float b) { return a + b; });
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = p[i] * (d[i] - mean);
        }
        if (!in || (!live && accumulate)) continue;
        constexpr int S = R::X4 ? 4 : 1;
#pragma unroll
        for (int i = 0; i < V; i += S) {
            if (R::expert(l, i) >= E) break;
            const int64_t at = t * dld + R::expert(l, i);
            float o[S] = {};
            if constexpr (R::X4) {
                if (accumulate) load4<BF16>(dlogits, at, o);
#pragma unroll
                for (int j = 0; j < S; ++j) o[j] += live ? d[i + j] : 0.0f;
                if (BF16)
                    *(uint2*)((uint16_t*)dlogits + at) = make_uint2(naiwa_f32_to_bf16(o[0]) | naiwa_f32_to_bf16(o[1]) << 16,
                                                                    naiwa_f32_to_bf16(o[2]) | naiwa_f32_to_bf16(o[3]) << 16);
                else
                    *(float4*)((float*)dlogits + at) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
                if (accumulate) o[0] = load<BF16>(dlogits, at);
                store<BF16>(dlogits, at, o[0] + (live ? d[i] : 0.0f));
            }
        }
    }
}

} // namespace

extern "C" int naiwa_router_topk_backward(const void* logits, int dtype, int ld, const uint32_t* ids, int ids_ld,
                                          const float* dw, int dw_ld, int64_t T, int E, int k, int mode,
                                          const uint8_t* mask, void* dlogits, int dld, int flags, int64_t stream) {
    if (T < 0 || k <= 0 || E <= 0 || ld < 0 || ids_ld < 0 || dw_ld < 0 || dld < 0 || (ld && ld < E) ||
        (dld && dld < E) || (ids_ld && ids_ld < k) || (dw_ld && dw_ld < k) || (flags & ~NAIWA_TOKENS_ACCUMULATE))
        return NAIWA_E_INVALID;
    if (dtype != NAIWA_F32 && dtype != NAIWA_BF16) return NAIWA_E_UNSUPPORTED;
    if (mode < NAIWA_ROUTE_SOFTMAX_TOPK_RENORM || mode > NAIWA_ROUTE_SOFTMAX_TOPK) return NAIWA_E_UNSUPPORTED;
    if (E > kMaxE || k > 32 || T > INT32_MAX / k) return NAIWA_E_UNSUPPORTED;
    if (T == 0) return NAIWA_OK;
    if (!logits || !ids || !dw || !dlogits) return NAIWA_E_INVALID;
    ld = ld ? ld : E, dld = dld ? dld : E, ids_ld = ids_ld ? ids_ld : k, dw_ld = dw_ld ? dw_ld : k;
    // in the logits' place row by row, or apart from all that is read
    const int size = dtype == NAIWA_BF16 ? 2 : 4;
    const Span to = span_of(dlogits, T, dld, E, size);
    if (!(dlogits == logits && dld == ld) && overlap(to, span_of(logits, T, ld, E, size))) return NAIWA_E_INVALID;
    if (overlap(to, span_of(ids, T, ids_ld, k, 4)) || overlap(to, span_of(dw, T, dw_ld, k, 4)) || overlap(to, span_of(mask, T)))
        return NAIWA_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    const int accumulate = flags & NAIWA_TOKENS_ACCUMULATE;
    auto blocks = [&](int L) { return (unsigned)std::min<int64_t>((T * L + kThreads - 1) / kThreads, 4096); };
    if (mode != NAIWA_ROUTE_SOFTMAX_TOPK && accumulate) {
        int L = 1;
        while (L < k) L <<= 1;
        auto go = [&](auto* kernel) {
            kernel<<<blocks(L), kThreads, 0, st>>>(logits, ld, ids, ids_ld, dw, dw_ld, T, E, k, L, mask, dlogits, dld);
        };
        dtype == NAIWA_BF16 ? go(chosen_kernel<true>) : go(chosen_kernel<false>);
        return naiwa_hip_rc(hipGetLastError());
    }
    auto row = [&](auto r) {
        typedef decltype(r) R;
        auto go = [&](auto* kernel) {
            kernel<<<blocks(R::L), kThreads, 0, st>>>(logits, ld, ids, ids_ld, dw, dw_ld, T, E, k, mask, dlogits, dld, accumulate);
        };
        if (mode == NAIWA_ROUTE_SOFTMAX_TOPK)
            dtype == NAIWA_BF16 ? go(row_kernel<R, true, true>) : go(row_kernel<R, false, true>);
        else
            dtype == NAIWA_BF16 ? go(row_kernel<R, true, false>) : go(row_kernel<R, false, false>);
    };
    const bool x4 = takes4(logits, dtype, ld, E) && takes4(dlogits, dtype, dld, E);
    if (k > 16 && E <= 256) // a row's pairs need a lane each
        x4 ? row(Row<64, 4, true>()) : row(Row<64, 4, false>());
    else
        by_experts(E, x4, row);
    return naiwa_hip_rc(hipGetLastError());
}
