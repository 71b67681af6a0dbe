// Per-expert counts, the router's balance loss and its gradient (include/naiwa_balance.h).
//
// Forward: up to kMaxBlocks blocks take runs of rows.  A wave takes one row at a time, lane
// l the experts l, l + 64, ..: the row's maximum, its exponentials and their sum stay in
// registers (one read of the logits), and the probabilities are added up per expert in
// registers.  The counts meet in an LDS histogram.  Each block leaves its partial sums in
// the scratch buffer and a second launch of one block adds them in block order and forms
// the loss; with one block the first launch does that itself.  Backward: the same row in
// registers, dlogits from it in the same pass.
//
// Bound: HBM for long batches (the logits are read once each way and the gradient
// written once); launches for short ones.
#include "../../include/naiwa_balance.h"
#include "common.h"
#include "workspace.h"

#include <algorithm>

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMaxE = 1024;
constexpr int kMaxBlocks = 256;
constexpr int kRun = 64; // rows that a wave adds up in f32

template <bool BF16> __device__ __forceinline__ float load(const void* p, int64_t i) {
    return BF16 ? naiwa_bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}

template <int W, class T, class F> __device__ __forceinline__ T wave_all(T v, F f) {
#pragma unroll
    for (int m = 1; m < W; m <<= 1) v = f(v, __shfl_xor(v, m, 64));
    return v;
}

// A row's exponentials e[i] (expert lane + 64 i; 0 past E) relative to its largest logit, and
// their sum's inverse.
template <int V, bool BF16>
__device__ __forceinline__ float row_exp(const void* logits, int64_t row, int E, int lane, float (&e)[V]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        e[i] = lane + 64 * i < E ? load<BF16>(logits, row + lane + 64 * i) : -INFINITY;
        m = fmaxf(m, e[i]);
    }
    m = wave_all<64>(m, [](float a, float b) { return fmaxf(a, b); });
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        e[i] = lane + 64 * i < E ? expf(e[i] - m) : 0.0f;
        s += e[i];
    }
    s = wave_all<64>(s, [](float a, float b) { return a + b; });
    return 1.0f / s;
}

struct Part { // one block's partial sums
    double* probs;      // [blocks][E]
    uint32_t* counts;   // [blocks][E]
    uint32_t* valid;    // [blocks]
};

// The results from `blocks` partial sums, by one block.
__device__ void finish(const Part& part, int blocks, int E, int k, uint32_t* counts, uint32_t* valid, float* probs,
                       float* loss) {
    __shared__ double red[kThreads];
    const int tid = threadIdx.x;
    uint32_t N = 0;
    for (int b = 0; b < blocks; ++b) N += part.valid[b];
    const double inv = N ? 1.0 / (double)N : 0.0;
    double mine = 0.0;
    for (int e = tid; e < E; e += kThreads) {
        uint32_t c = 0;
        double p = 0.0;
        for (int b = 0; b < blocks; ++b) {
            c += part.counts[(size_t)b * E + e];
            if (probs) p += part.probs[(size_t)b * E + e];
        }
        counts[e] = c;
        if (probs) {
            probs[e] = (float)(p * inv);
            mine += (double)c * (p * inv);
        }
    }
    if (!probs) return;
    red[tid] = mine;
    __syncthreads();
    for (int m = kThreads / 2; m; m >>= 1) {
        if (tid < m) red[tid] += red[tid + m];
        __syncthreads();
    }
    if (tid == 0) {
        *valid = N;
        *loss = (float)(red[0] * inv * ((double)E / (double)k));
    }
}

// Blocks of `rows` rows.  V = 0: counts alone.
template <int V, bool BF16>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const void* logits, int64_t ld, const uint32_t* ids, int64_t ids_ld, int64_t T, int64_t rows, int E, int k,
               const uint8_t* mask, Part part, uint32_t* counts, uint32_t* valid, float* probs, float* loss,
               uint32_t* bad) {
    __shared__ uint32_t hist[kMaxE];
    __shared__ double sums[V ? kMaxE : 1];
    __shared__ uint32_t nvalid;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, blk = blockIdx.x;
    const int64_t r0 = blk * rows, r1 = min(T, r0 + rows);
    for (int e = tid; e < E; e += kThreads) {
        hist[e] = 0;
        if (V) sums[e] = 0.0;
    }
    if (tid == 0) nvalid = 0;
    __syncthreads();
    uint32_t nbad = 0;
    for (int64_t i = tid; i < (r1 - r0) * k; i += kThreads) {
        const int64_t t = r0 + i / k;
        if (mask && !mask[t]) continue;
        const uint32_t id = ids[t * ids_ld + i % k];
        if (id < (uint32_t)E)
            atomicAdd(&hist[id], 1u);
        else
            ++nbad;
    }
    if (bad && nbad) atomicAdd(bad, nbad);
    if constexpr (V > 0) {
        double total[V] = {};
        uint32_t n = 0;
        int64_t t = r0 + wave;
        while (t < r1) {
            float acc[V] = {};
            for (int i = 0; i < kRun && t < r1; ++i, t += kWaves) {
                if (mask && !mask[t]) continue;
                float e[V];
                const float inv = row_exp<V, BF16>(logits, t * ld, E, lane, e);
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = __builtin_fmaf(e[j], inv, acc[j]);
                ++n;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) total[j] += (double)acc[j];
        }
        if (lane == 0 && n) atomicAdd(&nvalid, n);
        // the waves one after the other, so that the order of the sums is fixed
        for (int w = 0; w < kWaves; ++w) {
            if (w == wave)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (lane + 64 * j < E) sums[lane + 64 * j] += total[j];
            __syncthreads();
        }
    }
    __syncthreads();
    for (int e = tid; e < E; e += kThreads) {
        part.counts[(size_t)blk * E + e] = hist[e];
        if (V) part.probs[(size_t)blk * E + e] = sums[e];
    }
    if (tid == 0) part.valid[blk] = nvalid;
    if (gridDim.x == 1) {
        __syncthreads();
        finish(part, 1, E, k, counts, valid, probs, loss);
    }
}

__global__ void __launch_bounds__(kThreads)
finish_kernel(Part part, int blocks, int E, int k, uint32_t* counts, uint32_t* valid, float* probs, float* loss) {
    finish(part, blocks, E, k, counts, valid, probs, loss);
}

__global__ void zero_kernel(uint32_t* p) { *p = 0; }

template <int V, bool BF16>
__global__ void __launch_bounds__(kThreads)
backward_kernel(const void* logits, int64_t ld, const uint32_t* counts, const uint32_t* valid, int64_t T, int E, int k,
                const uint8_t* mask, const float* grad_loss, void* dlogits, int64_t dld, int accumulate) {
    const int lane = threadIdx.x & 63;
    const double N = (double)max(1u, *valid);
    const float coef = (float)((double)*grad_loss * (double)E / ((double)k * N * N));
    float c[V];
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = lane + 64 * i < E ? (float)counts[lane + 64 * i] : 0.0f;
    for (int64_t t = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); t < T; t += (int64_t)gridDim.x * kWaves) {
        const bool live = !mask || mask[t];
        if (!live && accumulate) continue;
        float e[V] = {}, s = 0.0f, inv = 0.0f;
        if (live) {
            inv = row_exp<V, BF16>(logits, t * ld, E, lane, e);
#pragma unroll
            for (int i = 0; i < V; ++i) s = __builtin_fmaf(e[i] * inv, c[i], s);
            s = wave_all<64>(s, [](float a, float b) { return a + b; });
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (lane + 64 * i >= E) break;
            const int64_t at = t * dld + lane + 64 * i;
            float g = live ? coef * (e[i] * inv) * (c[i] - s) : 0.0f;
            if (accumulate) g += load<BF16>(dlogits, at);
            if (BF16)
                ((uint16_t*)dlogits)[at] = (uint16_t)naiwa_f32_to_bf16(g);
            else
                ((float*)dlogits)[at] = g;
        }
    }
}

// Blocks of a batch of T tokens: a wave gets at least 4 rows.
int blocks_of(int64_t T) { return (int)std::max<int64_t>(1, std::min<int64_t>(kMaxBlocks, T / (4 * kWaves))); }

int ids_ok(const uint32_t* ids, int ids_ld, int64_t T, int k, int E) {
    if (T < 0 || k <= 0 || E <= 0 || ids_ld < 0 || (ids_ld && ids_ld < k)) return NAIWA_E_INVALID;
    if (E > kMaxE || T > INT32_MAX / k) return NAIWA_E_UNSUPPORTED;
    return T > 0 && !ids ? NAIWA_E_INVALID : NAIWA_OK;
}

int part_of(int blocks, int E, Part* p) {
    const size_t n = (size_t)blocks * E;
    int rc = 0;
    uint8_t* ws = (uint8_t*)naiwa_scratch(NAIWA_SCRATCH_BALANCE, n * 12 + (size_t)blocks * 4, &rc);
    if (!ws) return rc;
    *p = Part{(double*)ws, (uint32_t*)(ws + 8 * n), (uint32_t*)(ws + 12 * n)};
    return NAIWA_OK;
}

#define NAIWA_BALANCE_V(E, CALL)                                                                                       \
    ((E) <= 64 ? CALL(1) : (E) <= 128 ? CALL(2) : (E) <= 256 ? CALL(4) : (E) <= 512 ? CALL(8) : CALL(16))

} // namespace

extern "C" int naiwa_expert_counts(const uint32_t* ids, int ids_ld, int64_t T, int k, int E, const uint8_t* mask,
                                   uint32_t* counts, uint32_t* bad, int64_t stream) {
    if (int rc = ids_ok(ids, ids_ld, T, k, E)) return rc;
    if (!counts) return NAIWA_E_INVALID;
    const int blocks = blocks_of(T);
    Part part;
    if (int rc = part_of(blocks, E, &part)) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (bad) zero_kernel<<<1, 1, 0, st>>>(bad);
    forward_kernel<0, false><<<blocks, kThreads, 0, st>>>(nullptr, 0, ids, ids_ld ? ids_ld : k, T,
                                                          (T + blocks - 1) / blocks, E, k, mask, part, counts, nullptr,
                                                          nullptr, nullptr, bad);
    if (blocks > 1) finish_kernel<<<1, kThreads, 0, st>>>(part, blocks, E, k, counts, nullptr, nullptr, nullptr);
    return naiwa_hip_rc(hipGetLastError());
}

extern "C" int naiwa_router_balance(const void* logits, int dtype, int ld, const uint32_t* ids, int ids_ld, int64_t T,
                                    int E, int k, const uint8_t* mask, uint32_t* counts, uint32_t* valid, float* probs,
                                    float* loss, int64_t stream) {
    if (int rc = ids_ok(ids, ids_ld, T, k, E)) return rc;
    if (dtype != NAIWA_F32 && dtype != NAIWA_BF16) return NAIWA_E_UNSUPPORTED;
    if (ld < 0 || (ld && ld < E) || (T > 0 && !logits) || !counts || !valid || !probs || !loss) return NAIWA_E_INVALID;
    const int blocks = blocks_of(T);
    Part part;
    if (int rc = part_of(blocks, E, &part)) return rc;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto* kernel) {
        kernel<<<blocks, kThreads, 0, st>>>(logits, ld ? ld : E, ids, ids_ld ? ids_ld : k, T, (T + blocks - 1) / blocks,
                                            E, k, mask, part, counts, valid, probs, loss, nullptr);
    };
#define NAIWA_CALL(V) (dtype == NAIWA_BF16 ? go(forward_kernel<V, true>) : go(forward_kernel<V, false>))
    NAIWA_BALANCE_V(E, NAIWA_CALL);
#undef NAIWA_CALL
    if (blocks > 1) finish_kernel<<<1, kThreads, 0, st>>>(part, blocks, E, k, counts, valid, probs, loss);
    return naiwa_hip_rc(hipGetLastError());
}

extern "C" int naiwa_router_balance_backward(const void* logits, int dtype, int ld, const uint32_t* counts,
                                             const uint32_t* valid, int64_t T, int E, int k, const uint8_t* mask,
                                             const float* grad_loss, void* dlogits, int dld, int flags,
                                             int64_t stream) {
    if (T < 0 || k <= 0 || E <= 0 || ld < 0 || dld < 0 || (ld && ld < E) || (dld && dld < E) ||
        (flags & ~NAIWA_BALANCE_ACCUMULATE))
        return NAIWA_E_INVALID;
    if (dtype != NAIWA_F32 && dtype != NAIWA_BF16) return NAIWA_E_UNSUPPORTED;
    if (E > kMaxE || T > INT32_MAX / k) return NAIWA_E_UNSUPPORTED;
    if (T == 0) return NAIWA_OK;
    if (!logits || !counts || !valid || !grad_loss || !dlogits) return NAIWA_E_INVALID;
    const unsigned blocks = (unsigned)std::min<int64_t>((T + kWaves - 1) / kWaves, 2048);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto* kernel) {
        kernel<<<blocks, kThreads, 0, st>>>(logits, ld ? ld : E, counts, valid, T, E, k, mask, grad_loss, dlogits,
                                            dld ? dld : E, flags & NAIWA_BALANCE_ACCUMULATE);
    };
#define NAIWA_CALL(V) (dtype == NAIWA_BF16 ? go(backward_kernel<V, true>) : go(backward_kernel<V, false>))
    NAIWA_BALANCE_V(E, NAIWA_CALL);
#undef NAIWA_CALL
    return naiwa_hip_rc(hipGetLastError());
}
