// Per-expert counts, the router's balance loss and its gradient (include/naiwa_balance.h).
//
// Forward: up to kMaxBlocks blocks take runs of rows.  16 lanes take a row of up to 128
// experts (64 lanes a longer one), lane l the experts l, l + L, .. or, where rows allow 4 at
// once, 4 l .. 4 l + 3, 4 l + 4 L, ..: the row's maximum, its exponentials and their sum stay in
// registers (one read of the logits), and the probabilities are added up per expert in
// registers.  The counts meet in an LDS histogram.  Each block leaves its partial sums in the
// scratch buffer; a second launch, a block per 16 experts, adds them in a fixed order, and the
// last of its blocks to end adds up the loss.  With one block the first launch does all that.
// Backward: the same row in registers, dlogits from it in the same pass: p (c - sum p c), with the row's
// mean count taken off the counts first as an integer, so that nearly even counts lose nothing.
//
// Bound: HBM for long batches (the logits are read once each way and the gradient
// written once); launches and the latency of a row for short ones.  32768 tokens, 128 experts,
// top-8, f32: forward 7.9 + 5.1 us, backward 10.0 us (33.6 MB: 3.4 TB/s); 61 tokens 3.6 and 1.8 us.
// 64 lanes a row, and one block that joins all partial sums, took 120 us for all three.
#include "../../include/naiwa_balance.h"
#include "common.h"
#include "workspace.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMaxE = 1024;
constexpr int kMaxBlocks = 512;
constexpr int kRun = 64; // rows that a lane adds up in f32
constexpr int kFinish = 1024, kFinishE = 16;

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

struct Part {         // the blocks' partial sums
    double* probs;    // [blocks][E]
    double* loss;     // [blocks of the second launch]
    uint32_t* counts; // [blocks][E]
    uint32_t* valid;  // [blocks]
    uint32_t* ended;  // blocks of the second launch that have ended, cleared by the first launch
};

// The results of experts e0 .. e0 + kFinishE - 1 from `blocks` (at most kMaxBlocks) partial
// sums, by one block of TH threads: the lanes of 16 take an expert each and every TH / 16-th
// block, all loads at once.  Returns the sum of c_e P_e over the experts in thread 0.
template <int TH>
__device__ double finish(const Part& part, int blocks, int E, int e0, uint32_t* counts, float* probs, uint32_t* N) {
    constexpr int G = TH / kFinishE, W = TH / 64, M = kMaxBlocks / G;
    static_assert(kFinishE == 16, "an expert a lane of 16");
    __shared__ double pw[W][kFinishE];
    __shared__ uint32_t cw[W][kFinishE], nw[W];
    const int tid = threadIdx.x, i = tid % kFinishE, e = e0 + i, g = tid / kFinishE, wave = tid >> 6;
    uint32_t n = probs && tid < blocks ? part.valid[tid] : 0u, cv[M];
    static_assert(TH >= kMaxBlocks, "a block's number of tokens a thread");
    double pv[M];
#pragma unroll
    for (int j = 0; j < M; ++j) {
        const int b = g + j * G;
        const bool in = e < E && b < blocks;
        cv[j] = in ? part.counts[(size_t)b * E + e] : 0u;
        pv[j] = in && probs ? part.probs[(size_t)b * E + e] : 0.0;
    }
    uint32_t c = 0;
    double p = 0.0;
#pragma unroll
    for (int j = 0; j < M; ++j) c += cv[j], p += pv[j];
#pragma unroll
    for (int m = kFinishE; m < 64; m <<= 1) {
        c += __shfl_xor((int)c, m, 64);
        p += __shfl_xor(p, m, 64);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) n += __shfl_xor((int)n, m, 64);
    if ((tid & 63) < kFinishE) cw[wave][i] = c, pw[wave][i] = p;
    if ((tid & 63) == 0) nw[wave] = n;
    __syncthreads();
    double share = 0.0;
    if (wave == 0) { // every 16 lanes the same
        c = 0, p = 0.0, n = 0;
        for (int w = 0; w < W; ++w) c += cw[w][i], p += pw[w][i], n += nw[w];
        p = n ? p / (double)n : 0.0;
        if (tid < kFinishE && e < E) {
            counts[e] = c;
            if (probs) probs[e] = (float)p;
        }
        share = e < E && n ? (double)c * p / (double)n : 0.0;
#pragma unroll
        for (int m = 1; m < kFinishE; m <<= 1) share += __shfl_xor(share, m, 64);
        *N = n;
    }
    __syncthreads();
    return share;
}

// Blocks of `rows` rows.  V = 0: counts alone.
template <class R, bool BF16>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const void* logits, int64_t ld, const uint32_t* ids, int64_t ids_ld, int64_t T, int rows, int E, int k,
               const uint8_t* mask, Part part, uint32_t* counts, uint32_t* valid, float* probs, float* loss,
               uint32_t* bad) {
    constexpr int L = R::L, V = R::V;
    __shared__ uint32_t hist[kMaxE];
    constexpr bool kApart = L * V <= 256; // the waves' sums apart in LDS, else one after the other
    __shared__ double sums[V == 0 ? 1 : kApart ? kWaves * L * V : kMaxE];
    __shared__ uint32_t nvalid;
    const int tid = threadIdx.x, blk = blockIdx.x;
    const int64_t r0 = (int64_t)blk * rows;
    const int nrows = (int)min((int64_t)rows, T - r0);
    for (int e = tid; e < E; e += kThreads) {
        hist[e] = 0;
        if (V && !kApart) sums[e] = 0.0;
    }
    if (tid == 0) nvalid = 0;
    // the first two rows of the lane: under way while the ids are counted
    constexpr int G = kThreads / L, VV = V ? V : 1;
    const int l = tid % L;
    float ea[VV], eb[VV];
    bool la = false, lb = false;
    auto rows_at = [&](int base) {
        const int ra = base + tid / L, rb = ra + G;
        if constexpr (V > 0) {
            row_load<R, BF16>(logits, (r0 + ra) * ld, ra < nrows, E, l, ea);
            row_load<R, BF16>(logits, (r0 + rb) * ld, rb < nrows, E, l, eb);
        }
        la = ra < nrows && (!mask || mask[r0 + ra]);
        lb = rb < nrows && (!mask || mask[r0 + rb]);
    };
    if (V) rows_at(0);
    __syncthreads();
    uint32_t nbad = 0;
    for (uint32_t i = tid; (int64_t)i < (int64_t)nrows * k; i += kThreads) {
        const uint32_t r = i / (uint32_t)k;
        if (mask && !mask[r0 + r]) continue;
        const uint32_t id = ids[(r0 + r) * ids_ld + (i - r * (uint32_t)k)];
        if (id < (uint32_t)E)
            atomicAdd(&hist[id], 1u);
        else
            ++nbad;
    }
    if (bad && nbad) atomicAdd(bad, nbad);
    if constexpr (V > 0) {
        double total[V] = {};
        uint32_t n = 0;
        for (int run = 0; run < nrows; run += kRun * G) {
            float acc[V] = {};
            // two rows a round, the same rounds for every lane
            for (int base = run; base < min(nrows, run + kRun * G); base += 2 * G) {
                const float ia = row_exp<R>(la, E, l, ea), ib = row_exp<R>(lb, E, l, eb);
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = __builtin_fmaf(eb[j], ib, __builtin_fmaf(ea[j], ia, acc[j]));
                n += (la ? 1 : 0) + (lb ? 1 : 0);
                if (base + 2 * G < nrows) rows_at(base + 2 * G);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) total[j] += (double)acc[j];
        }
        if (l == 0 && n) atomicAdd(&nvalid, n);
        // a wave's rows, then the waves in their order: the order of the sums is fixed
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int m = L; m < 64; m <<= 1) total[j] += __shfl_xor(total[j], m, 64);
        const int wave = tid >> 6;
        if constexpr (kApart) {
            if ((tid & 63) < L)
#pragma unroll
                for (int j = 0; j < V; ++j) sums[wave * L * V + R::expert(l, j)] = total[j];
        } else {
            for (int w = 0; w < kWaves; ++w) {
                if (w == wave && (tid & 63) < L)
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (R::expert(l, j) < E) sums[R::expert(l, j)] += total[j];
                __syncthreads();
            }
        }
    }
    __syncthreads();
    for (int e = tid; e < E; e += kThreads) {
        part.counts[(size_t)blk * E + e] = hist[e];
        if constexpr (V > 0) {
            double p = sums[e];
            if constexpr (kApart)
                for (int w = 1; w < kWaves; ++w) p += sums[w * L * V + e];
            part.probs[(size_t)blk * E + e] = p;
        }
    }
    if (tid == 0) part.valid[blk] = nvalid;
    // (no call relies on what an earlier one left: the first one may be captured and run later)
    if (blk == 0 && tid == 0) *part.ended = 0;
    if (gridDim.x == 1) {
        double sum = 0.0;
        uint32_t N = 0;
        __syncthreads();
        for (int e0 = 0; e0 < E; e0 += kFinishE) sum += finish<kThreads>(part, 1, E, e0, counts, probs, &N);
        if (probs && tid == 0) {
            *valid = N;
            *loss = (float)(sum * ((double)E / (double)k));
        }
    }
}

__global__ void __launch_bounds__(kFinish)
finish_kernel(Part part, int blocks, int E, int k, uint32_t* counts, uint32_t* valid, float* probs, float* loss) {
    uint32_t N = 0;
    const double mine = finish<kFinish>(part, blocks, E, blockIdx.x * kFinishE, counts, probs, &N);
    if (!probs || threadIdx.x) return;
    // the block that ends last adds up the blocks' shares, in their order
    __hip_atomic_store(part.loss + blockIdx.x, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint32_t before = __hip_atomic_fetch_add(part.ended, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    if (before + 1 != gridDim.x) return;
    double sum = 0.0;
    for (unsigned b = 0; b < gridDim.x; ++b)
        sum += __hip_atomic_load(part.loss + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *valid = N;
    *loss = (float)(sum * ((double)E / (double)k));
}

template <class R, bool BF16>
__global__ void __launch_bounds__(kThreads)
backward_kernel(const void* logits, int64_t ld, const uint32_t* counts, const uint32_t* valid, int64_t T, int E, int k,
                const uint8_t* mask, const float* grad_loss, void* dlogits, int64_t dld, int accumulate) {
    constexpr int L = R::L, V = R::V, G = kThreads / L;
    const int tid = threadIdx.x, l = tid % L;
    const double N = (double)max(1u, *valid);
    const float coef = (float)((double)*grad_loss * (double)E / ((double)k * N * N));
    int c[V];
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = R::expert(l, i) < E ? (int)counts[R::expert(l, i)] : 0;
    for (int64_t t0 = (int64_t)blockIdx.x * G; t0 < T; t0 += (int64_t)gridDim.x * G) {
        const int64_t t = t0 + tid / L;
        const bool in = t < T;
        float e[V], d[V], mean = 0.0f, s = 0.0f;
        row_load<R, BF16>(logits, t * ld, in, E, l, e);
        const bool live = in && (!mask || mask[t]);
        const float inv = row_exp<R>(live, E, l, e);
        // The row's mean count, rounded to an integer, comes off the counts as an integer first (the
        // gradient does not change when all counts do): what follows errs relative to the counts' spread
        // about it, not to the counts, which in a well balanced batch are a thousand times that.  Counts
        // are under 2^31 (T k is).
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] *= inv, mean = __builtin_fmaf(e[i], (float)c[i], mean);
        mean = lanes_all<L>(mean, [](float a, float b) { return a + b; });
        const int m = (int)rintf(fminf(mean, 2147483520.0f)); // (a NaN stays in e)
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = (float)(c[i] - m), s = __builtin_fmaf(e[i], d[i], s);
        s = lanes_all<L>(s, [](float a, float b) { return a + b; });
        if (!in || (!live && accumulate)) continue;
        constexpr int S = R::X4 ? 4 : 1;
#pragma unroll
        for (int i = 0; i < V; i += S) {
            if (R::expert(l, i) >= E) break;
            const int64_t at = t * dld + R::expert(l, i);
            float g[S], old[S] = {};
            if (accumulate) {
                if constexpr (R::X4)
                    load4<BF16>(dlogits, at, old);
                else
                    old[0] = load<BF16>(dlogits, at);
            }
#pragma unroll
            for (int j = 0; j < S; ++j) g[j] = old[j] + (live ? coef * e[i + j] * (d[i + j] - s) : 0.0f);
            if constexpr (R::X4 && BF16)
                *(uint2*)((uint16_t*)dlogits + at) = make_uint2(naiwa_f32_to_bf16(g[0]) | naiwa_f32_to_bf16(g[1]) << 16,
                                                                naiwa_f32_to_bf16(g[2]) | naiwa_f32_to_bf16(g[3]) << 16);
            else if constexpr (R::X4)
                *(float4*)((float*)dlogits + at) = make_float4(g[0], g[1], g[2], g[3]);
            else if (BF16)
                ((uint16_t*)dlogits)[at] = (uint16_t)naiwa_f32_to_bf16(g[0]);
            else
                ((float*)dlogits)[at] = g[0];
        }
    }
}

// Blocks of a batch of T tokens: at least 64 rows a block.
int blocks_of(int64_t T) { return (int)std::max<int64_t>(1, std::min<int64_t>(kMaxBlocks, T / 64)); }

int ids_ok(const uint32_t* ids, int ids_ld, int64_t T, int k, int E) {
    if (T < 0 || k <= 0 || E <= 0 || ids_ld < 0 || (ids_ld && ids_ld < k)) return NAIWA_E_INVALID;
    if (E > kMaxE || T > INT32_MAX / k) return NAIWA_E_UNSUPPORTED;
    return T > 0 && !ids ? NAIWA_E_INVALID : NAIWA_OK;
}

__global__ void zero_kernel(uint32_t* p) { *p = 0; }

// The scratch of a call; nothing in it outlives the call.
int part_of(int blocks, int E, hipStream_t st, Part* p) {
    const size_t n = (size_t)blocks * E;
    int rc = 0;
    uint8_t* ws = (uint8_t*)naiwa_scratch(NAIWA_SCRATCH_BALANCE, 1024 + n * 12 + (size_t)blocks * 4, &rc, st);
    if (!ws) return rc;
    *p = Part{(double*)(ws + 1024), (double*)ws, (uint32_t*)(ws + 1024 + 8 * n), (uint32_t*)(ws + 1024 + 12 * n),
              (uint32_t*)(ws + 1020)};
    return NAIWA_OK;
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

extern "C" int naiwa_expert_counts(const uint32_t* ids, int ids_ld, int64_t T, int k, int E, const uint8_t* mask,
                                   uint32_t* counts, uint32_t* bad, int64_t stream) {
    if (int rc = ids_ok(ids, ids_ld, T, k, E)) return rc;
    if (!counts) return NAIWA_E_INVALID;
    const int blocks = blocks_of(T);
    hipStream_t st = (hipStream_t)stream;
    Part part;
    if (int rc = part_of(blocks, E, st, &part)) return rc;
    if (bad) zero_kernel<<<1, 1, 0, st>>>(bad);
    forward_kernel<Row<64, 0, false>, false><<<blocks, kThreads, 0, st>>>(nullptr, 0, ids, ids_ld ? ids_ld : k, T,
                                                          (int)((T + blocks - 1) / blocks), E, k, mask, part, counts, nullptr,
                                                          nullptr, nullptr, bad);
    if (blocks > 1) finish_kernel<<<(E + kFinishE - 1) / kFinishE, kFinish, 0, st>>>(part, blocks, E, k, counts, nullptr, nullptr, nullptr);
    return naiwa_hip_rc(hipGetLastError());
}

extern "C" int naiwa_router_balance(const void* logits, int dtype, int ld, const uint32_t* ids, int ids_ld, int64_t T,
                                    int E, int k, const uint8_t* mask, uint32_t* counts, uint32_t* valid, float* probs,
                                    float* loss, int64_t stream) {
    if (int rc = ids_ok(ids, ids_ld, T, k, E)) return rc;
    if (dtype != NAIWA_F32 && dtype != NAIWA_BF16) return NAIWA_E_UNSUPPORTED;
    if (ld < 0 || (ld && ld < E) || (T > 0 && !logits) || !counts || !valid || !probs || !loss) return NAIWA_E_INVALID;
    const int blocks = blocks_of(T);
    hipStream_t st = (hipStream_t)stream;
    Part part;
    if (int rc = part_of(blocks, E, st, &part)) return rc;
    auto go = [&](auto* kernel) {
        kernel<<<blocks, kThreads, 0, st>>>(logits, ld ? ld : E, ids, ids_ld ? ids_ld : k, T,
                                            (int)((T + blocks - 1) / blocks), E, k, mask, part, counts, valid, probs, loss, nullptr);
    };
    by_experts(E, takes4(logits, dtype, ld, E), [&](auto r) {
        dtype == NAIWA_BF16 ? go(forward_kernel<decltype(r), true>) : go(forward_kernel<decltype(r), false>);
    });
    if (blocks > 1) finish_kernel<<<(E + kFinishE - 1) / kFinishE, kFinish, 0, st>>>(part, blocks, E, k, counts, valid, probs, loss);
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
    if (dlogits == logits && (dld ? dld : E) != (ld ? ld : E)) return NAIWA_E_INVALID; // rows over other rows
    const int at_once = E <= 128 ? kThreads / 16 : kWaves; // rows of a block
    const unsigned blocks = (unsigned)std::min<int64_t>((T + at_once - 1) / at_once, 1024);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto* kernel) {
        kernel<<<blocks, kThreads, 0, st>>>(logits, ld ? ld : E, counts, valid, T, E, k, mask, grad_loss, dlogits,
                                            dld ? dld : E, flags & NAIWA_BALANCE_ACCUMULATE);
    };
    by_experts(E, takes4(logits, dtype, ld, E) && takes4(dlogits, dtype, dld, E), [&](auto r) {
        dtype == NAIWA_BF16 ? go(backward_kernel<decltype(r), true>) : go(backward_kernel<decltype(r), false>);
    });
    return naiwa_hip_rc(hipGetLastError());
}
