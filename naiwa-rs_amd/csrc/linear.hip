// naiwa_linear and naiwa_act_backward (include/naiwa_linear.h): rows times weights, everything behind the
// product in the same pass.  The tiles are linear_tiles.h's: I is the weights (for a gated product half
// a tile of each matrix), J the rows, so that a lane ends with 4 consecutive features of a row.
#include "linear_tiles.h"

namespace {

struct ForwardArgs {
    const uint16_t *w, *u, *x; // u: NULL without a gate
    int64_t w_ld, w_stride, u_ld, u_stride, x_ld;
    const float *b, *c;
    const uint32_t* offsets;
    uint32_t rows;
    int experts, n, k, act;
    const void* residual;
    void* out;
    uint16_t *pre, *pre_up;
    int64_t residual_ld, out_ld, pre_ld;
    bool out_f32, past;
};

// What follows the product, for features n0 + i .. n0 + i + 3 of row m0 + j.
template <bool F16> struct ForwardOut {
    struct More {
        lin_u32x4 residual;
        __device__ __forceinline__ void here() { in_registers(residual); }
    };
    const ForwardArgs& a;
    int e, n0;
    int64_t m0;
    lin_f32x4 b, c;
    __device__ __forceinline__ void column(int i) {
        const int n = n0 + i, left = a.n - n;
        b = a.b ? load_4(a.b + (int64_t)e * a.n + n, left) : lin_f32x4{};
        c = a.u && a.c ? load_4(a.c + (int64_t)e * a.n + n, left) : lin_f32x4{};
    }
    __device__ __forceinline__ bool reads() const { return a.residual; }
    __device__ __forceinline__ More more(int j, int i) const {
        return {a.residual ? raw_4(cell(a.residual, m0, a.residual_ld, n0, j, i, a.out_f32), a.n - n0 - i, a.out_f32) : lin_u32x4{}};
    }
    __device__ __forceinline__ void store(int j, int i, lin_f32x4 p, lin_f32x4 q, const More& more) const {
        const int left = a.n - n0 - i;
        p += b;
        if (a.pre) store_4<F16>(cell(a.pre, m0, a.pre_ld, n0, j, i, false), left, false, p, a.past);
        lin_f32x4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = lin_act(a.act, p[x]);
        if (a.u) {
            q += c;
            if (a.pre_up) store_4<F16>(cell(a.pre_up, m0, a.pre_ld, n0, j, i, false), left, false, q, a.past);
            v *= q;
        }
        if (a.residual) v += wide_4<F16>(more.residual, a.out_f32);
        store_4<F16>(cell(a.out, m0, a.out_ld, n0, j, i, a.out_f32), left, a.out_f32, v, a.past);
    }
    // One piece alone.
    __device__ __forceinline__ void one(int j, int i, lin_f32x4 p, lin_f32x4 q) {
        column(i);
        store(j, i, p, q, more(j, i));
    }
};

// A tile of out, or a part of its sums.  Streams of weights bound it up to some 48 rows an expert (8 gated experts of 14336 x 4096,
// 4 rows each: 1.88 GB in 310 to 322 us, 6 TB/s), the tiles' rows out of L2 beyond (4096 x 4096 x 14336 340 to 375 us; 128 gated
// experts of 768 x 2048 with 243 rows 330 to 350, their 256-row tiles 0.7 filled and 4.2 rounds taking as long as 5).
template <class S>
__global__ void __launch_bounds__(S::TH, 2)
linear_kernel(ForwardArgs a, uint32_t nI, Parts parts) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
    constexpr int kN = S::PAIR ? S::TI / 2 : S::TI; // features of a tile
    const Segments seg(a.offsets, a.rows, a.experts, S::TJ);
    uint32_t it, jt, m0;
    if (!tile_of_block(blockIdx.x, nI, seg.tiles, &it, &jt)) return;
    int e, nj;
    seg.find(jt, S::TJ, &e, &m0, &nj);
    const int n0 = it * kN, ni = min(kN, a.n - n0), z = blockIdx.y;
    const TileView iv[2] = {{a.w + e * a.w_stride + (int64_t)n0 * a.w_ld, a.w_ld, ni},
                            {a.u + e * a.u_stride + (int64_t)n0 * a.u_ld, a.u_ld, ni}};
    const TileView jv[1] = {{a.x + (int64_t)m0 * a.x_ld, a.x_ld, nj}};
    lin_f32x4 acc[S::FI][S::FJ] = {};
    const int64_t steps = (a.k + S::kStep - 1) / S::kStep;
    const int s0 = (int)(steps * z / parts.splits), s1 = (int)(steps * (z + 1) / parts.splits);
    tile_product<S, false>(iv, jv, a.k, s0, s1, turn_of_block(blockIdx.x, s1 - s0, false), lds, acc, [](auto&) {});
    if (parts.splits == 1) {
        each_piece<S>(lds, acc, ni, nj, ForwardOut<S::F16>{a, e, n0, m0});
    } else {
        const int64_t at = (int64_t)m0 * a.n + n0;
        each_piece<S>(lds, acc, ni, nj, PartOut<S::PAIR>{parts.at(z, 0) + at, S::PAIR ? parts.at(z, 1) + at : nullptr, a.n, ni});
    }
}

// Behind linear_kernel's parts: 4 features of a row at a time.
template <bool F16, int G>
__global__ void __launch_bounds__(256)
linear_finish_kernel(ForwardArgs a, Parts parts) {
    const uint32_t quads = (a.n + 3) / 4;
    each_sum<G>(parts, (uint64_t)quads * a.rows, [&](uint64_t i, bool in, bool first, auto sum) {
        const uint32_t m = (uint32_t)(i / quads), n = (uint32_t)(i - (uint64_t)m * quads) * 4;
        const int e = in ? expert_of_row(a.offsets, a.experts, a.rows, m) : -1;
        const int64_t at = (int64_t)m * a.n + n;
        const lin_f32x4 p = sum(0, at, a.n - n, e >= 0), q = a.u ? sum(1, at, a.n - n, e >= 0) : p;
        if (first && e >= 0) ForwardOut<F16>{a, e, (int)n, m}.one(0, 0, p, q);
    });
}

// Few rows an expert: every block takes 32 features (16 of each matrix of a PAIR) and up to 16 FJ rows, its 8 waves every
// eighth 64 values of the contraction, straight from memory into the MFMA operands, at any address: a lane takes 16
// contiguous values as two products' (8 lanes x 16 bytes side by side, 64 bytes a row, fetched half lines).  The waves' sums meet in LDS.
constexpr int kFewWaves = 8, kFewAhead = 2;
template <bool F16, bool PAIR, int FJ>
__global__ void __launch_bounds__(64 * kFewWaves)
linear_few_kernel(ForwardArgs a, uint32_t nI) {
    __shared__ lin_f32x4 sums[kFewWaves][2 * FJ][64];
    constexpr int kN = PAIR ? 16 : 32;
    const Segments seg(a.offsets, a.rows, a.experts, 16 * FJ);
    // (the row tiles of a weight strip one after the other, on one XCD)
    const uint64_t total = (uint64_t)nI * seg.tiles, per = (total + 7) / 8, t = blockIdx.x % 8 * per + blockIdx.x / 8;
    if (blockIdx.x / 8 >= per || t >= total) return;
    int e, nj;
    uint32_t m0;
    seg.find((uint32_t)(t / nI), 16 * FJ, &e, &m0, &nj);
    const int n0 = (int)(t % nI) * kN, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, c0 = 16 * (lane >> 4);
    // rows that do not exist are read as the last one that does; their products are not stored
    const uint16_t* wp[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        const int n = min(n0 + (PAIR ? 0 : 16 * f) + r, a.n - 1);
        wp[f] = PAIR && f ? a.u + e * a.u_stride + n * a.u_ld + c0 : a.w + e * a.w_stride + n * a.w_ld + c0;
    }
    const uint16_t* xp[FJ];
#pragma unroll
    for (int f = 0; f < FJ; ++f) xp[f] = a.x + (m0 + min(16 * f + r, nj - 1)) * a.x_ld + c0;
    lin_f32x4 acc[2][FJ] = {};
    auto get = [&](const uint16_t* p, int c) {
        lin_s16x8 v = {};
        if (c + c0 + 8 <= a.k) {
            __builtin_memcpy(&v, p + c, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + c0 + j < a.k) v[j] = (short)p[c + j];
        }
        return v;
    };
    auto product = [&](const lin_s16x8 (&w)[2], const lin_s16x8 (&x)[FJ]) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) acc[i][j] = lin_mfma<F16>(w[i], x[j], acc[i][j]);
    };
    constexpr int kStride = 64 * kFewWaves;
    int c = 64 * wave;
    for (; c + kStride * (kFewAhead - 1) + 64 <= a.k; c += kStride * kFewAhead) {
        lin_s16x8 w[2 * kFewAhead][2], x[2 * kFewAhead][FJ];
#pragma unroll
        for (int u = 0; u < 2 * kFewAhead; ++u) {
            const int at = c + u / 2 * kStride + u % 2 * 8;
#pragma unroll
            for (int i = 0; i < 2; ++i) __builtin_memcpy(&w[u][i], wp[i] + at, 16);
#pragma unroll
            for (int j = 0; j < FJ; ++j) __builtin_memcpy(&x[u][j], xp[j] + at, 16);
        }
#pragma unroll
        for (int u = 0; u < 2 * kFewAhead; ++u) product(w[u], x[u]);
    }
    for (; c < a.k; c += kStride) {
        lin_s16x8 w[2][2], x[2][FJ];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 2; ++i) w[u][i] = get(wp[i], c + 8 * u);
#pragma unroll
            for (int j = 0; j < FJ; ++j) x[u][j] = get(xp[j], c + 8 * u);
        }
        product(w[0], x[0]), product(w[1], x[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) sums[wave][i * FJ + j][lane] = acc[i][j];
    __syncthreads();
    // a wave a fragment of rows, and of features where they are one matrix's
    constexpr int kParts = PAIR ? FJ : 2 * FJ;
    for (int f = wave; f < kParts; f += kFewWaves) {
        lin_f32x4 p = {}, q = {};
        for (int w = 0; w < kFewWaves; ++w) {
            p += sums[w][f][lane];
            if (PAIR) q += sums[w][FJ + f][lane];
        }
        const int j = 16 * (f % FJ) + r, n = n0 + 16 * (f / FJ) + 4 * (lane >> 4);
        if (j < nj && n < a.n) ForwardOut<F16>{a, e, n, m0}.one(j, 0, p, q);
    }
}

template <class S> int launch(const ForwardArgs& a, hipStream_t st) {
    constexpr int kN = S::PAIR ? S::TI / 2 : S::TI, kPlanes = S::PAIR ? 2 : 1;
    const int64_t nI = (a.n + kN - 1) / kN, nJ = lin_j_tiles(a.rows, a.experts, a.offsets, S::TJ);
    const int64_t plane = (int64_t)a.rows * a.n;
    const int splits = lin_splits(nI * nJ, (a.k + S::kStep - 1) / S::kStep, plane * kPlanes);
    const int64_t blocks = (nI * nJ + 7) / 8 * 8;
    if (blocks * splits * S::TH >= (int64_t)1 << 32) return NAIWA_E_UNSUPPORTED; // a launch's threads
    Parts parts;
    if (int rc = lin_parts(splits, kPlanes, plane, st, &parts)) return rc;
    linear_kernel<S><<<dim3((unsigned)blocks, splits), S::TH, 0, st>>>(a, (uint32_t)nI, parts);
    if (splits > 1) {
        const int64_t quads = (int64_t)(a.n + 3) / 4 * a.rows;
        if (splits <= 8) linear_finish_kernel<S::F16, 1><<<lin_finish_blocks(quads, 1), 256, 0, st>>>(a, parts);
        else linear_finish_kernel<S::F16, 16><<<lin_finish_blocks(quads, 16), 256, 0, st>>>(a, parts);
    }
    return naiwa_hip_rc(hipGetLastError());
}
template <bool F16, bool PAIR, int FJ> int launch_few(const ForwardArgs& a, hipStream_t st) {
    constexpr int kN = PAIR ? 16 : 32;
    const int64_t nI = (a.n + kN - 1) / kN, nJ = lin_j_tiles(a.rows, a.experts, a.offsets, 16 * FJ);
    const int64_t blocks = (nI * nJ + 7) / 8 * 8;
    if (blocks * 64 * kFewWaves >= (int64_t)1 << 32) return NAIWA_E_UNSUPPORTED;
    linear_few_kernel<F16, PAIR, FJ><<<(unsigned)blocks, 64 * kFewWaves, 0, st>>>(a, (uint32_t)nI);
    return naiwa_hip_rc(hipGetLastError());
}

// Which kernel a call takes (experts 0: dense; odd: rows at addresses that are no multiples of 4 bytes, which 16-byte reads are slow at).
enum { kFew16 = kKinds, kFew32, kFew64 };
int lin_forward_kind(int64_t rows, int experts, int64_t n, int64_t k, bool pair, bool odd) {
    const bool grouped = experts > 0;
    const int64_t avg = grouped ? rows / experts : rows, bytes = 2 * std::max(experts, 1) * n * k * (pair ? 2 : 1);
    const int64_t strips = (n + (pair ? 15 : 31)) / (pair ? 16 : 32);
    // Straight from memory while a strip's rows are one tile's or what more read again is in the caches, and a block a CU takes it.
    // A block reads its whole sum, so long ones are the tiles' parts.  Both take as long at 4096 values, odd rows at 1500 (straight
    // from memory and tiles, us: 1 row x 16 x 4096 7.7 and 8.4, 8192 12.9 and 8.1, 262144 344 and 44; 16 rows x 1003 x 4096 13.2 and
    // 13.3, 8192 23.6 and 9.9; 1 row x 200 x 1001 7.9 and 10.0, 2501 16.6 and 10.1, 4097 28.4 and 10.3).
    const int64_t longest = odd ? 1536 : 4096;
    if (bytes <= (16 << 20)) {
        for (int f = 0; f < 3; ++f)
            if (k <= longest && strips * lin_j_alike(rows, experts, grouped, 16 << f) <= 256) return kFew16 + f;
    } else if (avg <= 2 && strips * std::min<int64_t>(std::max(experts, 1), rows) >= 256) {
        // Every CU has blocks, so long sums do not matter here, but odd rows do where there are many (8192 x 1001 gated 12.9 and
        // 14.7, 14336 x 1001 gated 22.9 and 19.1, 64 experts of 1000 x 1001 42 and 26, 14336 x 4097 53 and 27; 4096 21 and 22).
        if (!odd || (k <= longest && bytes <= (32 << 20))) return kFew16;
    }
    // (Empty places cost little here, where a tile's rows are read whole: 16 experts of 7600 x 1568 with 73 rows take 213 us in
    // 256 x 256 tiles, 239 in 128 x 128.)
    return lin_kind(k, avg, (n * (pair ? 2 : 1) + 255) / 256 * lin_j_alike(rows, experts, grouped, 256), true);
}

template <bool F16, bool PAIR> int forward(const ForwardArgs& a, bool direct, bool odd, hipStream_t st) {
    const int kind = lin_forward_kind(a.rows, a.offsets ? a.experts : 0, a.n, a.k, PAIR, odd);
    if (kind == kFew16) return launch_few<F16, PAIR, 1>(a, st);
    if (kind == kFew32) return launch_few<F16, PAIR, 2>(a, st);
    if (kind == kFew64) return launch_few<F16, PAIR, 4>(a, st);
    if (!direct && lin_narrow(a.rows / (a.offsets ? a.experts : 1)))
        return launch<Shape<128, 64, 2, 2, 32, 2, kRows, kRows, F16, false, PAIR>>(a, st);
    if (!direct) return launch<Shape<128, 128, 2, 2, 32, 2, kRows, kRows, F16, false, PAIR>>(a, st);
    switch (kind) {
    case kThin: return launch<Shape<128, 32, 4, 1, 64, 4, kRows, kRows, F16, true, PAIR>>(a, st);
    case kShort: return launch<Shape<128, 128, 2, 2, 32, 2, kRows, kRows, F16, true, PAIR>>(a, st);
    case kMid: return launch<Shape<128, 128, 2, 2, 32, 4, kRows, kRows, F16, true, PAIR>>(a, st);
    default: return launch<Shape<256, 256, 2, 4, 64, 2, kRows, kRows, F16, true, PAIR>>(a, st);
    }
}

// ---- the activation's gradient alone

struct ActF32 {
    typedef float T;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
template <bool F16> struct Act16 {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(T v) { return lin_get<F16>(v); }
    static __device__ __forceinline__ T put(float v) { return lin_put<F16>(v); }
};

// One thread takes N values at a time (those behind a row's last whole piece one by one).  Memory bounds it: 24576 x 1408 gated
// bf16 take 58 us, 6.0 TB/s, in f32 125, 5.5; not gated 33 and 73; 61 x 2048 are a launch of 3.4.
template <class D>
__global__ void __launch_bounds__(256)
act_backward_kernel(const typename D::T* dout, const typename D::T* pre, const typename D::T* pre_up, int64_t rows, int n,
                    int64_t ld, int act, typename D::T* dpre, typename D::T* dpre_up) {
    typedef typename D::T T;
    constexpr int N = 16 / sizeof(T);
    const int pieces = (n + N - 1) / N;
    const int64_t all = rows * pieces;
    auto one = [&](float d, float p, float q, float* dp, float* dq) {
        float a, slope;
        lin_act_slope(act, p, &a, &slope);
        *dp = d * slope * q, *dq = d * a;
    };
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / pieces;
        const int c = (int)(i - r * pieces) * N;
        const int64_t at = r * ld + c;
        if (c + N <= n) {
            T d[N], p[N], q[N], x[N], y[N];
            __builtin_memcpy(d, dout + at, 16);
            __builtin_memcpy(p, pre + at, 16);
            if (pre_up) __builtin_memcpy(q, pre_up + at, 16);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float dp, dq;
                one(D::get(d[j]), D::get(p[j]), pre_up ? D::get(q[j]) : 1.0f, &dp, &dq);
                x[j] = D::put(dp), y[j] = D::put(dq);
            }
            __builtin_memcpy(dpre + at, x, 16);
            if (pre_up) __builtin_memcpy(dpre_up + at, y, 16);
        } else {
            for (int j = 0; j < n - c; ++j) {
                float dp, dq;
                one(D::get(dout[at + j]), D::get(pre[at + j]), pre_up ? D::get(pre_up[at + j]) : 1.0f, &dp, &dq);
                dpre[at + j] = D::put(dp);
                if (pre_up) dpre_up[at + j] = D::put(dq);
            }
        }
    }
}

} // namespace

extern "C" int naiwa_linear(const naiwa_weights* w, const naiwa_weights* up, const void* x, int64_t x_ld,
                            const uint32_t* offsets, int64_t rows, int act, const void* residual, int64_t residual_ld,
                            void* out, int out_dtype, int64_t out_ld, void* pre, void* pre_up, int64_t pre_ld,
                            int64_t stream) {
    if (int rc = lin_pair_ok(w, up)) return rc;
    const int n = w->n, k = w->k;
    if (rows < 0 || x_ld < 0 || residual_ld < 0 || out_ld < 0 || pre_ld < 0 || (x_ld && x_ld < k) ||
        (residual_ld && residual_ld < n) || (out_ld && out_ld < n) || (pre_ld && pre_ld < n) || (!offsets && w->experts != 1) ||
        (pre_up && !up))
        return NAIWA_E_INVALID;
    x_ld = x_ld ? x_ld : k, residual_ld = residual_ld ? residual_ld : n, out_ld = out_ld ? out_ld : n, pre_ld = pre_ld ? pre_ld : n;
    if (!lin_act_ok(act) || (out_dtype != NAIWA_F32 && out_dtype != w->dtype)) return NAIWA_E_UNSUPPORTED;
    if (rows > INT32_MAX || std::max({x_ld, residual_ld, out_ld, pre_ld}) > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (rows == 0) return NAIWA_OK;
    if (!x || !out) return NAIWA_E_INVALID;
    const ForwardArgs a{(const uint16_t*)w->w, up ? (const uint16_t*)up->w : nullptr, (const uint16_t*)x,
                        lin_ld(w), lin_stride(w), up ? lin_ld(up) : 0, up ? lin_stride(up) : 0, x_ld,
                        w->bias, up ? up->bias : nullptr, offsets, (uint32_t)rows, w->experts, n, k, act,
                        residual, out, (uint16_t*)pre, (uint16_t*)pre_up, residual_ld, out_ld, pre_ld, out_dtype == NAIWA_F32,
                        rows * n * lin_size(out_dtype) >= kLinPast};
    // an output is written where nothing else is read or written
    const int so = lin_size(out_dtype);
    const int64_t b_bytes = (int64_t)w->experts * n * 4;
    const Span ins[] = {span_of(x, rows, x_ld, k, 2), lin_span(w), lin_span(up), span_of(a.b, b_bytes), span_of(a.c, b_bytes),
                        lin_span(offsets, w->experts)};
    const Span outs[] = {span_of(out, rows, out_ld, n, so), span_of(pre, rows, pre_ld, n, 2), span_of(pre_up, rows, pre_ld, n, 2)};
    const Span added = span_of(residual, rows, residual_ld, n, so);
    for (int i = 0; i < 3; ++i) {
        for (const Span& in : ins)
            if (overlap(outs[i], in)) return NAIWA_E_INVALID;
        if (!(i == 0 && residual == out && residual_ld == out_ld) && overlap(outs[i], added)) return NAIWA_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (overlap(outs[i], outs[j])) return NAIWA_E_INVALID;
    }
    const bool direct = !(k & 7) && lin_aligned(a.w, a.w_ld, a.w_stride) && lin_aligned(a.x, x_ld, 0) &&
                        (!up || lin_aligned(a.u, a.u_ld, a.u_stride));
    const bool odd = lin_odd(a.w, a.w_ld, a.w_stride) || lin_odd(a.x, x_ld, 0) || (up && lin_odd(a.u, a.u_ld, a.u_stride));
    hipStream_t st = (hipStream_t)stream;
    if (w->dtype == NAIWA_BF16) return up ? forward<false, true>(a, direct, odd, st) : forward<false, false>(a, direct, odd, st);
    return up ? forward<true, true>(a, direct, odd, st) : forward<true, false>(a, direct, odd, st);
}

extern "C" int naiwa_act_backward(const void* dout, const void* pre, const void* pre_up, int dtype, int64_t rows, int n,
                                  int64_t ld, int act, void* dpre, void* dpre_up, int64_t stream) {
    if (rows < 0 || n <= 0 || ld < 0 || (ld && ld < n)) return NAIWA_E_INVALID;
    if (!lin_act_ok(act) || (dtype != NAIWA_F32 && dtype != NAIWA_BF16 && dtype != NAIWA_F16)) return NAIWA_E_UNSUPPORTED;
    ld = ld ? ld : n;
    if (rows > INT32_MAX || ld > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (rows == 0) return NAIWA_OK;
    if (!dout || !pre || !dpre || (!pre_up) != (!dpre_up)) return NAIWA_E_INVALID;
    // in place element by element, or apart
    auto span = [&](const void* p) { return span_of(p, rows, ld, n, lin_size(dtype)); };
    for (const void* o : {(const void*)dpre, (const void*)dpre_up})
        for (const void* i : {dout, pre, pre_up})
            if (o != i && overlap(span(o), span(i))) return NAIWA_E_INVALID;
    if (overlap(span(dpre), span(dpre_up))) return NAIWA_E_INVALID;
    const int pieces = dtype == NAIWA_F32 ? (n + 3) / 4 : (n + 7) / 8;
    const unsigned blocks = (unsigned)std::min<int64_t>((rows * pieces + 255) / 256, 1 << 16);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto d) {
        typedef decltype(d) D;
        typedef typename D::T T;
        act_backward_kernel<D><<<blocks, 256, 0, st>>>((const T*)dout, (const T*)pre, (const T*)pre_up, rows, n, ld, act, (T*)dpre,
                                                       (T*)dpre_up);
    };
    if (dtype == NAIWA_F32) go(ActF32());
    else if (dtype == NAIWA_BF16) go(Act16<false>());
    else go(Act16<true>());
    return naiwa_hip_rc(hipGetLastError());
}

// Which kernel a call with aligned rows takes (experts 0: one matrix for all rows), for tests: kThin ... kBig of linear_tiles.h,
// behind them those that read rows straight from memory, 16, 32 or 64 at a time.  how: 1 a gated product, 2 odd rows (of which only
// the latter kinds are told apart), or both.
extern "C" int naiwa_linear_kind(int64_t rows, int experts, int n, int k, int how) {
    return lin_forward_kind(rows, experts, n, k, how & 1, how & 2);
}
