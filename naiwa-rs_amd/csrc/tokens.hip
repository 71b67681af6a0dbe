// Tokens sorted by expert and back (include/naiwa_tokens.h).
//
// The sort is a stable counting sort: every block counts a run of pairs per expert, a second
// launch adds the counts up over the blocks, a third places the pairs; one block does it all
// for up to kOne pairs.  Inside a block each wave owns a contiguous part of the run and ranks 64 pairs at
// a time with ballots, so that flat order is kept without atomics that could reorder it.
//
// The rows move once: to the experts a token's row is read once and written to its k rows; back, the k
// rows are read once and added up in registers; the gradient takes a pair at a time, so that its dot product stays
// in one group of lanes.  Rows of any length and alignment move in 16-byte pieces (the hardware
// takes unaligned ones) with single values behind the last whole piece.
#include "../../include/naiwa_tokens.h"
#include "common.h"
#include "spans.h"
#include "workspace.h"

#include <algorithm>
#include <type_traits>

namespace {

// ---- sort -------------------------------------------------------------------------------

constexpr int kSortE = 4096;
constexpr int kOne = 4096;        // pairs that one block sorts in one launch
constexpr int kSortBlocks = 512;  // most blocks of the three launches
constexpr int kRunLeast = 512;    // fewest pairs of their blocks (131,072 pairs of 128 experts: 18.8 us with 2048, 12.6 with 512)

struct Pairs {
    const uint32_t* ids;
    int64_t ids_ld, n;
    int k, E;
    const uint8_t* mask;
};
// Pair p's expert, E if it has none; *bad: the token is valid and the id is not.
__device__ __forceinline__ uint32_t expert_of(const Pairs& a, int64_t p, bool* bad) {
    const uint32_t t = (uint32_t)p / (uint32_t)a.k, j = (uint32_t)p - t * (uint32_t)a.k;
    *bad = false;
    if (a.mask && !a.mask[t]) return (uint32_t)a.E;
    const uint32_t id = a.ids[(int64_t)t * a.ids_ld + j];
    *bad = id >= (uint32_t)a.E;
    return *bad ? (uint32_t)a.E : id;
}

// Exclusive prefix sums of v[0 .. E) in LDS, by the block; *total their sum (in every thread).
template <int TH> __device__ void scan(uint32_t* v, int E, uint32_t* waves, uint32_t* total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (E + TH - 1) / TH, e0 = min(E, tid * per), e1 = min(E, e0 + per);
    uint32_t sum = 0;
    for (int e = e0; e < e1; ++e) sum += v[e];
    uint32_t in = sum;
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t x = (uint32_t)__shfl_up((int)in, m, 64);
        if (lane >= m) in += x;
    }
    if (lane == 63) waves[wave] = in;
    __syncthreads();
    uint32_t at = in - sum, all = 0;
    for (int w = 0; w < TH / 64; ++w) {
        if (w < wave) at += waves[w];
        all += waves[w];
    }
    for (int e = e0; e < e1; ++e) {
        const uint32_t c = v[e];
        v[e] = at;
        at += c;
    }
    *total = all;
    __syncthreads();
}

// Pairs p0 .. p1 of a wave, placed: pos[e] is the row of the wave's next pair of expert e.
__device__ __forceinline__ void place(const Pairs& a, int64_t p0, int64_t p1, uint32_t* pos, uint32_t* perm, uint32_t* inv) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = (1ull << lane) - 1ull;
    for (int64_t b = p0; b < p1; b += 64) {
        const int64_t p = b + lane;
        bool bad;
        const uint32_t e = p < p1 ? expert_of(a, p, &bad) : (uint32_t)a.E;
        const bool in = e < (uint32_t)a.E;
        uint64_t same = __ballot(in); // the lanes with this lane's expert: one ballot a bit
        for (int bit = 0; (a.E - 1) >> bit; ++bit) {
            const uint64_t ones = __ballot((e >> bit) & 1u);
            same &= ((e >> bit) & 1u) ? ones : ~ones;
        }
        const uint32_t rank = (uint32_t)__popcll(same & below);
        uint32_t row = NAIWA_NO_ROW;
        if (in) row = __hip_atomic_load(pos + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT) + rank;
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) // (the wave's own counter; its LDS operations keep their order)
            __hip_atomic_store(pos + e, row + (uint32_t)__popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
        __builtin_amdgcn_wave_barrier();
        if (p < p1) inv[p] = row;
        if (in) perm[row] = (uint32_t)p;
    }
}

// hist[w][e]: the pairs of expert e in wave w's part p0 .. p1.  Returns the lane's bad ids.
__device__ __forceinline__ uint32_t count(const Pairs& a, int64_t p0, int64_t p1, uint32_t* hist) {
    uint32_t nbad = 0;
    for (int64_t p = p0 + (threadIdx.x & 63); p < p1; p += 64) {
        bool bad;
        const uint32_t e = expert_of(a, p, &bad);
        if (e < (uint32_t)a.E) atomicAdd(hist + e, 1u);
        nbad += bad;
    }
    return nbad;
}

// Up to kOne pairs in one launch of one block of W waves.
template <int W>
__global__ void __launch_bounds__(64 * W)
sort_one_kernel(Pairs a, uint32_t* perm, uint32_t* inv, uint32_t* offsets, uint32_t* bad) {
    extern __shared__ uint32_t lds[]; // start[E], hist[W][E]
    __shared__ uint32_t waves[W], nbad;
    uint32_t *start = lds, *hist = lds + a.E;
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int i = tid; i < W * a.E; i += 64 * W) hist[i] = 0;
    if (tid == 0) nbad = 0;
    __syncthreads();
    const int64_t part = ((a.n + W - 1) / W + 63) & ~63ll;
    const int64_t p0 = min(a.n, wave * part), p1 = min(a.n, p0 + part);
    const uint32_t b = count(a, p0, p1, hist + wave * a.E);
    if (b) atomicAdd(&nbad, b);
    __syncthreads();
    for (int e = tid; e < a.E; e += 64 * W) {
        uint32_t sum = 0;
        for (int w = 0; w < W; ++w) {
            const uint32_t c = hist[w * a.E + e];
            hist[w * a.E + e] = sum;
            sum += c;
        }
        start[e] = sum;
    }
    __syncthreads();
    uint32_t total;
    scan<64 * W>(start, a.E, waves, &total);
    for (int e = tid; e < a.E; e += 64 * W) {
        offsets[e] = start[e];
        for (int w = 0; w < W; ++w) hist[w * a.E + e] += start[e];
    }
    if (tid == 0) {
        offsets[a.E] = total;
        if (bad) *bad = nbad;
    }
    __syncthreads();
    place(a, p0, p1, hist + wave * a.E, perm, inv);
}

// counts[b][e] of the blocks' runs, badof[b] their ids that are none.  W waves a block.
template <int W>
__global__ void __launch_bounds__(64 * W)
sort_count_kernel(Pairs a, int64_t run, uint32_t* counts, uint32_t* badof) {
    extern __shared__ uint32_t lds[]; // hist[E]
    __shared__ uint32_t nbad;
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int i = tid; i < a.E; i += 64 * W) lds[i] = 0;
    if (tid == 0) nbad = 0;
    __syncthreads();
    const int64_t r0 = blockIdx.x * run, part = run / W;
    const int64_t p0 = min(a.n, r0 + wave * part), p1 = min(a.n, p0 + part);
    const uint32_t b = count(a, p0, p1, lds);
    if (b) atomicAdd(&nbad, b);
    __syncthreads();
    for (int e = tid; e < a.E; e += 64 * W) counts[(size_t)blockIdx.x * a.E + e] = lds[e];
    if (tid == 0) badof[blockIdx.x] = nbad;
}

// counts[b][e] -> the pairs of expert e in blocks below b; totals[e].  A wave an expert.
constexpr int kSumW = 4;
__global__ void __launch_bounds__(64 * kSumW)
sort_sum_kernel(int blocks, int E, uint32_t* counts, uint32_t* totals, const uint32_t* badof, uint32_t* bad) {
    const int lane = threadIdx.x & 63, e = blockIdx.x * kSumW + (threadIdx.x >> 6);
    if (e == 0 && bad) {
        uint32_t s = 0;
        for (int b = lane; b < blocks; b += 64) s += badof[b];
        for (int m = 1; m < 64; m <<= 1) s += (uint32_t)__shfl_xor((int)s, m, 64);
        if (lane == 0) *bad = s;
    }
    if (e >= E) return;
    uint32_t below = 0;
    for (int b0 = 0; b0 < blocks; b0 += 64) {
        const int b = b0 + lane;
        const uint32_t c = b < blocks ? counts[(size_t)b * E + e] : 0u;
        uint32_t in = c;
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t x = (uint32_t)__shfl_up((int)in, m, 64);
            if (lane >= m) in += x;
        }
        if (b < blocks) counts[(size_t)b * E + e] = below + in - c;
        below += (uint32_t)__shfl((int)in, 63, 64);
    }
    if (lane == 0) totals[e] = below;
}

template <int W>
__global__ void __launch_bounds__(64 * W)
sort_place_kernel(Pairs a, int64_t run, const uint32_t* counts, const uint32_t* totals, uint32_t* perm, uint32_t* inv,
                  uint32_t* offsets) {
    extern __shared__ uint32_t lds[]; // start[E], hist[W][E]
    __shared__ uint32_t waves[W];
    uint32_t *start = lds, *hist = lds + a.E;
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int e = tid; e < a.E; e += 64 * W) start[e] = totals[e];
    for (int i = tid; i < W * a.E; i += 64 * W) hist[i] = 0;
    __syncthreads();
    const int64_t r0 = blockIdx.x * run, part = run / W;
    const int64_t p0 = min(a.n, r0 + wave * part), p1 = min(a.n, p0 + part);
    count(a, p0, p1, hist + wave * a.E);
    __syncthreads();
    uint32_t total;
    scan<64 * W>(start, a.E, waves, &total);
    for (int e = tid; e < a.E; e += 64 * W) {
        uint32_t at = start[e] + counts[(size_t)blockIdx.x * a.E + e];
        if (blockIdx.x == 0) offsets[e] = start[e];
        for (int w = 0; w < W; ++w) {
            const uint32_t c = hist[w * a.E + e];
            hist[w * a.E + e] = at;
            at += c;
        }
    }
    if (blockIdx.x == 0 && tid == 0) offsets[a.E] = total;
    __syncthreads();
    place(a, p0, p1, hist + wave * a.E, perm, inv);
}

__global__ void sort_none_kernel(uint32_t* offsets, int E, uint32_t* bad) {
    for (int e = threadIdx.x; e <= E; e += blockDim.x) offsets[e] = 0;
    if (bad && threadIdx.x == 0) *bad = 0;
}

// ---- rows -------------------------------------------------------------------------------

constexpr int kThreads = 256;

// S values of one type, as f32 and back; N of them at once, from any address of the type.
struct F32 {
    typedef float T;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
struct BF16 {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(T v) { return naiwa_bf16_to_f32(v); }
    static __device__ __forceinline__ T put(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
struct F16 {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(T v) { return naiwa_f16_to_f32(v); }
    static __device__ __forceinline__ T put(float v) { return (uint16_t)naiwa_f32_to_f16(v); }
};
// 16 bytes of an expert's row, which a launch reads or writes once.  PAST: past the caches, for calls whose rows they would not
// hold (kPast): 16384 tokens of top-8, 2048 bf16 each, 537 MB, take 107 and 95 us to the experts, 140 and 126 back, 214 and
// 200 for the gradient; 2048 tokens, 67 MB, 18 and 27 us back, 23 and 29 for the gradient.
constexpr int64_t kPast = (int64_t)256 << 20;
constexpr int64_t kMaxLd = 1 << 28; // row lengths: all offsets fit 63 bits
typedef uint32_t piece16 __attribute__((ext_vector_type(4), aligned(2)));
template <bool PAST> __device__ __forceinline__ void put16(void* p, uint4 v) {
    const piece16 w = __builtin_bit_cast(piece16, v);
    if (PAST) __builtin_nontemporal_store(w, (piece16*)p);
    else *(piece16*)p = w;
}
template <bool PAST> __device__ __forceinline__ uint4 get16(const void* p) {
    return __builtin_bit_cast(uint4, PAST ? __builtin_nontemporal_load((const piece16*)p) : *(const piece16*)p);
}

template <class D, int N> __device__ __forceinline__ void loads(const typename D::T* p, float (&o)[N]) {
    typename D::T v[N];
    __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = D::get(v[i]);
}
template <class D, int N> __device__ __forceinline__ void stores(typename D::T* p, const float (&o)[N]) {
    typename D::T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = D::put(o[i]);
    __builtin_memcpy(p, v, sizeof(v));
}

// L lanes take an item (a token or a pair): f(item, lane of L) for every item of the grid's share.  With a wave an item, the
// item is a scalar, and so is what is read of its pairs.
template <bool WAVE, class F> __device__ __forceinline__ void by_item(int64_t items, int L, F f) {
    const int G = WAVE ? kThreads / 64 : kThreads / L, l = WAVE ? threadIdx.x & 63 : threadIdx.x & (L - 1);
    const int mine = WAVE ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / L;
    for (int64_t i0 = (int64_t)blockIdx.x * G; i0 < items; i0 += (int64_t)gridDim.x * G)
        if (i0 + mine < items) f(i0 + mine, l);
}
// A row's pieces of N values, kAhead a lane at a time: f(c0, whole) takes those at c0, c0 + L N, .. (whole: all of them lie in
// the row).
constexpr int kAhead = 4;
template <int N, class F> __device__ __forceinline__ void by_pieces(int H, int L, int l, F f) {
    for (int c = l * N; c < H; c += kAhead * L * N) f(c, c + (kAhead - 1) * L * N + N <= H);
}

constexpr int kMaxH = 1 << 24;

// U: a value of the rows' size (its bits are what moves).
template <class U, bool WAVE, bool PAST>
__global__ void __launch_bounds__(kThreads)
to_experts_kernel(const U* x, int64_t ld, const uint32_t* inv, int64_t T, int k, int H, U* rows, int64_t rows_ld, int L) {
    constexpr int N = 16 / sizeof(U);
    if (WAVE) L = 64;
    const uint32_t n = (uint32_t)(T * k);
    by_item<WAVE>(T, L, [&](int64_t t, int l) {
        const U* from = x + t * ld;
        by_pieces<N>(H, L, l, [&](int c0, bool all) {
            uint4 v[kAhead] = {};
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (all || c0 + u * L * N + N <= H) __builtin_memcpy(&v[u], from + c0 + u * L * N, 16);
            for (int j = 0; j < k; ++j) {
                const uint32_t r = inv[t * k + j];
                if (r >= n) continue;
                U* to = rows + (int64_t)r * rows_ld;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int c = c0 + u * L * N;
                    if (all || c + N <= H)
                        put16<PAST>(to + c, v[u]);
                    else
                        for (int i = c; i < H; ++i) to[i] = from[i];
                }
            }
        });
    });
}

// Y: the rows' type, O: out's.  A lane takes one piece of a token's row (`parts` waves a row); eight rows' pieces are read before
// the first is added.
template <class Y, class O, bool WAVE, bool PAST>
__global__ void __launch_bounds__(kThreads)
from_experts_kernel(const typename Y::T* y, int64_t ld, const uint32_t* inv, const float* w, int64_t w_ld, int64_t T, int k,
                    int H, typename O::T* out, int64_t out_ld, int accumulate, int L, uint32_t parts) {
    constexpr int N = 16 / sizeof(typename Y::T), kRows = 8;
    if (WAVE) L = 64;
    const uint32_t n = (uint32_t)(T * k);
    by_item<WAVE>(T * parts, L, [&](int64_t item, int l) {
        const int64_t t = WAVE ? item / parts : item;
        typename O::T* to = out + t * out_ld;
        const int c = ((WAVE ? (int)(item - t * parts) * 64 : 0) + l) * N;
        if (c < H) {
            if (c + N <= H) {
                float s[N] = {};
                if (accumulate) loads<O, N>(to + c, s);
                for (int j0 = 0; j0 < k; j0 += kRows) {
                    float f[kRows];
                    typename Y::T v[kRows][N];
#pragma unroll
                    for (int u = 0; u < kRows; ++u) {
                        const int j = min(j0 + u, k - 1);
                        const uint32_t r = inv[t * k + j];
                        const bool in = j0 + u < k && r < n;
                        f[u] = !in ? 0.0f : w ? w[t * w_ld + j] : 1.0f;
                        if (in) {
                            const uint4 z = get16<PAST>(y + (int64_t)r * ld + c);
                            __builtin_memcpy(v[u], &z, 16);
                        } else {
#pragma unroll
                            for (int i = 0; i < N; ++i) v[u][i] = Y::put(-0.0f); // 0 times it changes no sum, -0 neither
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kRows; ++u)
#pragma unroll
                        for (int i = 0; i < N; ++i) s[i] = __builtin_fmaf(f[u], Y::get(v[u][i]), s[i]);
                }
                stores<O, N>(to + c, s);
                return;
            }
            for (int x = c; x < H; ++x) { // the one lane whose piece passes the end
                float s = accumulate ? O::get(to[x]) : 0.0f;
                for (int j = 0; j < k; ++j) {
                    const uint32_t r = inv[t * k + j];
                    if (r < n) s = __builtin_fmaf(w ? w[t * w_ld + j] : 1.0f, Y::get(y[(int64_t)r * ld + x]), s);
                }
                to[x] = O::put(s);
            }
        }
    });
}

template <class Y, class O, bool WAVE, bool PAST>
__global__ void __launch_bounds__(kThreads)
from_experts_backward_kernel(const typename O::T* dout, int64_t dout_ld, const typename Y::T* y, int64_t ld,
                             const uint32_t* inv, const float* w, int64_t w_ld, int64_t T, int k, int H,
                             typename Y::T* dy, int64_t dy_ld, float* dw, int64_t dw_ld, int L) {
    constexpr int N = 16 / sizeof(typename Y::T);
    if (WAVE) L = 64;
    const uint32_t n = (uint32_t)(T * k);
    by_item<WAVE>(T * k, L, [&](int64_t p, int l) {
        const uint32_t t = (uint32_t)p / (uint32_t)k, j = (uint32_t)p - t * (uint32_t)k, r = inv[p];
        float dot = 0.0f;
        if (r < n) {
            const float f = w ? w[t * w_ld + j] : 1.0f;
            const typename O::T* from = dout + t * dout_ld;
            const typename Y::T* row = y + (int64_t)r * ld;
            typename Y::T* to = dy + (int64_t)r * dy_ld;
            by_pieces<N>(H, L, l, [&](int c0, bool all) {
                float d[kAhead][N];
                typename Y::T v[kAhead][N];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int c = c0 + u * L * N;
                    if (!all && c + N > H) continue;
                    loads<O, N>(from + c, d[u]);
                    if (dw) {
                        const uint4 z = get16<PAST>(row + c);
                        __builtin_memcpy(v[u], &z, 16);
                    }
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int c = c0 + u * L * N;
                    if (all || c + N <= H) {
                        if (dw)
#pragma unroll
                            for (int i = 0; i < N; ++i) dot = __builtin_fmaf(d[u][i], Y::get(v[u][i]), dot);
                        if (dy) {
#pragma unroll
                            for (int i = 0; i < N; ++i) v[u][i] = Y::put(d[u][i] * f);
                            uint4 z;
                            __builtin_memcpy(&z, v[u], 16);
                            put16<PAST>(to + c, z);
                        }
                    } else {
                        for (int x = c; x < H; ++x) {
                            const float d1 = O::get(from[x]);
                            if (dw) dot = __builtin_fmaf(d1, Y::get(row[x]), dot);
                            if (dy) to[x] = Y::put(d1 * f);
                        }
                    }
                }
            });
        }
        if (dw) { // (all lanes of the item are here: its bounds are the same for them)
            for (int m = 1; m < L; m <<= 1) dot += __shfl_xor(dot, m, 64);
            if (l == 0) dw[t * dw_ld + j] = dot;
        }
    });
}

int lanes_of(int H, int N) { // lanes of an item whose row has H values, N a piece
    const int pieces = (H + N - 1) / N;
    int L = 1;
    while (L < 64 && L < pieces) L <<= 1;
    return L;
}
unsigned blocks_of(int64_t items, int L) {
    return (unsigned)std::min<int64_t>((items * L + kThreads - 1) / kThreads, (int64_t)1 << 20);
}

// f(whether a wave takes an item, whether its rows' `bytes` go past the caches).
template <class F> void by_wave(int L, int64_t bytes, F f) {
    if (L < 64) f(std::false_type(), std::false_type());
    else if (bytes < kPast) f(std::true_type(), std::false_type());
    else f(std::true_type(), std::true_type());
}

int size_of(int dtype) { return dtype == NAIWA_F32 ? 4 : 2; }
bool row_type(int dtype) { return dtype == NAIWA_F32 || dtype == NAIWA_BF16 || dtype == NAIWA_F16; }

int sizes_ok(int64_t T, int k, int H) {
    if (T < 0 || k <= 0 || H <= 0) return NAIWA_E_INVALID;
    return T > INT32_MAX / k || H > kMaxH ? NAIWA_E_UNSUPPORTED : NAIWA_OK;
}

// f(types of y and out) for rows of dtype and out of out_dtype.
template <class F> int by_types(int dtype, int out_dtype, F f) {
    if (dtype == NAIWA_F32) f(F32(), F32());
    else if (dtype == NAIWA_BF16) out_dtype == NAIWA_F32 ? f(BF16(), F32()) : f(BF16(), BF16());
    else out_dtype == NAIWA_F32 ? f(F16(), F32()) : f(F16(), F16());
    return naiwa_hip_rc(hipGetLastError());
}

} // namespace

extern "C" int naiwa_expert_sort(const uint32_t* ids, int ids_ld, int64_t T, int k, int E, const uint8_t* mask,
                                 uint32_t* perm, uint32_t* inv, uint32_t* offsets, uint32_t* bad, int64_t stream) {
    if (T < 0 || k <= 0 || E <= 0 || ids_ld < 0 || (ids_ld && ids_ld < k) || !offsets) return NAIWA_E_INVALID;
    if (E > kSortE || T > INT32_MAX / k) return NAIWA_E_UNSUPPORTED;
    hipStream_t st = (hipStream_t)stream;
    if (T == 0) {
        sort_none_kernel<<<1, 256, 0, st>>>(offsets, E, bad);
        return naiwa_hip_rc(hipGetLastError());
    }
    if (!ids || !perm || !inv) return NAIWA_E_INVALID;
    const Pairs a{ids, ids_ld ? ids_ld : k, T * k, k, E, mask};
    const Span ins[] = {span_of(ids, T, a.ids_ld, k, 4), span_of(mask, T)};
    const Span outs[] = {span_of(perm, a.n * 4), span_of(inv, a.n * 4), span_of(offsets, (E + 1) * 4), span_of(bad, 4)};
    for (int i = 0; i < 4; ++i) {
        for (const Span& in : ins)
            if (overlap(outs[i], in)) return NAIWA_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (overlap(outs[i], outs[j])) return NAIWA_E_INVALID;
    }
    if (a.n <= kOne) {
        if (E <= 512)
            sort_one_kernel<16><<<1, 1024, 17 * 4 * E, st>>>(a, perm, inv, offsets, bad);
        else
            sort_one_kernel<2><<<1, 128, 3 * 4 * E, st>>>(a, perm, inv, offsets, bad);
        return naiwa_hip_rc(hipGetLastError());
    }
    // runs of whole rounds of 64 pairs a wave
    const int64_t unit = 64 * 4, least = (a.n + kSortBlocks - 1) / kSortBlocks;
    const int64_t run = std::max<int64_t>(kRunLeast, (least + unit - 1) / unit * unit);
    const int blocks = (int)((a.n + run - 1) / run);
    int rc = 0;
    uint32_t* ws = (uint32_t*)naiwa_scratch_of_stream(NAIWA_SCRATCH_SORT, ((size_t)blocks * E + E + blocks) * 4, &rc, st);
    if (!ws) return rc;
    uint32_t *totals = ws + (size_t)blocks * E, *badof = totals + E;
    auto go = [&](auto waves) { // fewer waves where their counts would pass 64 KB of LDS
        constexpr int W = decltype(waves)::value;
        sort_count_kernel<W><<<blocks, 64 * W, 4 * E, st>>>(a, run, ws, badof);
        sort_sum_kernel<<<(E + kSumW - 1) / kSumW, 64 * kSumW, 0, st>>>(blocks, E, ws, totals, badof, bad);
        sort_place_kernel<W><<<blocks, 64 * W, (1 + W) * 4 * E, st>>>(a, run, ws, totals, perm, inv, offsets);
    };
    E <= 2048 ? go(std::integral_constant<int, 4>()) : go(std::integral_constant<int, 2>());
    return naiwa_hip_rc(hipGetLastError());
}

extern "C" int naiwa_tokens_to_experts(const void* x, int dtype, int64_t ld, const uint32_t* inv, int64_t T, int k, int H,
                                       void* rows, int64_t rows_ld, int64_t stream) {
    if (int rc = sizes_ok(T, k, H)) return rc;
    if (ld < 0 || rows_ld < 0 || (ld && ld < H) || (rows_ld && rows_ld < H)) return NAIWA_E_INVALID;
    if (!row_type(dtype) || std::max(ld, rows_ld) > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (T == 0) return NAIWA_OK;
    if (!x || !inv || !rows) return NAIWA_E_INVALID;
    const int s = size_of(dtype);
    ld = ld ? ld : H, rows_ld = rows_ld ? rows_ld : H;
    const Span to = span_of(rows, T * k, rows_ld, H, s);
    if (overlap(to, span_of(x, T, ld, H, s)) || overlap(to, span_of(inv, T * k * 4))) return NAIWA_E_INVALID;
    const int L = lanes_of(H, 16 / s);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto u, auto wave, auto past) {
        typedef decltype(u) U;
        to_experts_kernel<U, decltype(wave)::value, decltype(past)::value><<<blocks_of(T, L), kThreads, 0, st>>>((const U*)x, ld, inv, T, k, H, (U*)rows, rows_ld, L);
    };
    by_wave(L, T * k * H * s, [&](auto wave, auto past) { s == 4 ? go(uint32_t(), wave, past) : go(uint16_t(), wave, past); });
    return naiwa_hip_rc(hipGetLastError());
}

extern "C" int naiwa_tokens_from_experts(const void* y, int dtype, int64_t ld, const uint32_t* inv, const float* w,
                                         int w_ld, int64_t T, int k, int H, void* out, int out_dtype, int64_t out_ld,
                                         int flags, int64_t stream) {
    if (int rc = sizes_ok(T, k, H)) return rc;
    if (ld < 0 || out_ld < 0 || w_ld < 0 || (ld && ld < H) || (out_ld && out_ld < H) || (w_ld && w_ld < k) ||
        (flags & ~NAIWA_TOKENS_ACCUMULATE))
        return NAIWA_E_INVALID;
    if (!row_type(dtype) || (out_dtype != NAIWA_F32 && out_dtype != dtype) || std::max(ld, out_ld) > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (T == 0) return NAIWA_OK;
    if (!y || !inv || !out) return NAIWA_E_INVALID;
    ld = ld ? ld : H, out_ld = out_ld ? out_ld : H, w_ld = w_ld ? w_ld : k;
    const Span sums = span_of(out, T, out_ld, H, size_of(out_dtype));
    if (overlap(sums, span_of(y, T * k, ld, H, size_of(dtype))) || overlap(sums, span_of(inv, T * k * 4)) ||
        overlap(sums, span_of(w, T, w_ld, k, 4)))
        return NAIWA_E_INVALID;
    const int N = 16 / size_of(dtype), L = lanes_of(H, N);
    const uint32_t parts = L == 64 ? (H + 64 * N - 1) / (64 * N) : 1;
    return by_types(dtype, out_dtype, [&](auto ty, auto to) {
        typedef decltype(ty) Y;
        typedef decltype(to) O;
        by_wave(L, T * k * H * size_of(dtype), [&](auto wave, auto past) {
            from_experts_kernel<Y, O, decltype(wave)::value, decltype(past)::value><<<blocks_of(T * parts, L), kThreads, 0, (hipStream_t)stream>>>(
                (const typename Y::T*)y, ld, inv, w, w_ld, T, k, H, (typename O::T*)out, out_ld, flags & NAIWA_TOKENS_ACCUMULATE, L, parts);
        });
    });
}

extern "C" int naiwa_tokens_from_experts_backward(const void* dout, int dout_dtype, int64_t dout_ld, const void* y,
                                                  int dtype, int64_t ld, const uint32_t* inv, const float* w, int w_ld,
                                                  int64_t T, int k, int H, void* dy, int64_t dy_ld, float* dw, int dw_ld,
                                                  int64_t stream) {
    if (int rc = sizes_ok(T, k, H)) return rc;
    if (dout_ld < 0 || ld < 0 || dy_ld < 0 || w_ld < 0 || dw_ld < 0 || (dout_ld && dout_ld < H) || (ld && ld < H) ||
        (dy_ld && dy_ld < H) || (w_ld && w_ld < k) || (dw_ld && dw_ld < k))
        return NAIWA_E_INVALID;
    if (!row_type(dtype) || (dout_dtype != NAIWA_F32 && dout_dtype != dtype) || std::max({dout_ld, ld, dy_ld}) > kMaxLd)
        return NAIWA_E_UNSUPPORTED;
    if (T == 0 || (!dy && !dw)) return NAIWA_OK;
    if (!dout || !inv || (dw && !y)) return NAIWA_E_INVALID;
    const int s = size_of(dtype);
    dout_ld = dout_ld ? dout_ld : H, ld = ld ? ld : H, dy_ld = dy_ld ? dy_ld : H;
    w_ld = w_ld ? w_ld : k, dw_ld = dw_ld ? dw_ld : k;
    const Span rows = span_of(dw ? y : nullptr, T * k, ld, H, s), drows = span_of(dy, T * k, dy_ld, H, s);
    const Span sums = span_of(dout, T, dout_ld, H, size_of(dout_dtype)), dots = span_of(dw, T, dw_ld, k, 4);
    for (const Span& out : {drows, dots})
        for (const Span& in : {sums, span_of(inv, T * k * 4), span_of(w, T, w_ld, k, 4)})
            if (overlap(out, in)) return NAIWA_E_INVALID;
    if (overlap(dots, rows) || overlap(dots, drows)) return NAIWA_E_INVALID;
    // in y's place row by row, or nowhere near it
    if (!(dy == y && dy_ld == ld) && overlap(drows, rows)) return NAIWA_E_INVALID;
    const int L = lanes_of(H, 16 / s);
    return by_types(dtype, dout_dtype, [&](auto ty, auto to) {
        typedef decltype(ty) Y;
        typedef decltype(to) O;
        by_wave(L, T * k * H * s, [&](auto wave, auto past) {
            from_experts_backward_kernel<Y, O, decltype(wave)::value, decltype(past)::value><<<blocks_of(T * k, L), kThreads, 0, (hipStream_t)stream>>>(
                (const typename O::T*)dout, dout_ld, (const typename Y::T*)y, ld, inv, w, w_ld, T, k, H, (typename Y::T*)dy, dy_ld,
                dw, dw_ld, L);
        });
    });
}
