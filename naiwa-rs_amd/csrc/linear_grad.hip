// naiwa_linear_input_grad and naiwa_linear_weight_grad (include/naiwa_linear.h) on linear_tiles.h's tiles.
//
// Input: dx[m][k] = sum_n dy[m][n] W[n][k]; J is dy, I the weights with the contraction as row index.  Two
// matrices (a gate and its up) are one contraction of twice the length.
// Weights: dw[n][k] = sum_m dy[m][n] x[m][k]; the contraction is the row index of both operands, and a block's
// sum runs over its expert's rows.  The bias gradient is one more product per fragment of dy, with ones.
#include "linear_tiles.h"

namespace {

struct InputArgs {
    const uint16_t *w, *u, *dy, *dy_up;
    int64_t w_ld, w_stride, u_ld, u_stride, dy_ld;
    const uint32_t* offsets;
    uint32_t rows;
    int experts, n, k, act;
    const uint16_t *pre, *pre_up;
    void *dx, *dx_up;
    int64_t pre_ld, dx_ld;
    bool dx_f32, accumulate, past;
};

// What follows the product, for values k0 + i .. k0 + i + 3 of row m0 + j.
template <bool F16> struct InputOut {
    struct More {
        lin_u32x4 p, q; // pre and pre_up, or dx's old values in p
        __device__ __forceinline__ void here() { in_registers(p), in_registers(q); }
    };
    const InputArgs& a;
    int k0;
    int64_t m0;
    __device__ __forceinline__ void column(int) {}
    __device__ __forceinline__ bool reads() const { return a.pre || a.accumulate; }
    __device__ __forceinline__ More more(int j, int i) const {
        const int left = a.k - k0 - i;
        More m = {};
        if (a.pre) {
            m.p = raw_4(cell(a.pre, m0, a.pre_ld, k0, j, i, false), left, false);
            if (a.pre_up) m.q = raw_4(cell(a.pre_up, m0, a.pre_ld, k0, j, i, false), left, false);
        } else if (a.accumulate) {
            m.p = raw_4(cell(a.dx, m0, a.dx_ld, k0, j, i, a.dx_f32), left, a.dx_f32);
        }
        return m;
    }
    __device__ __forceinline__ void store(int j, int i, lin_f32x4 g, lin_f32x4, const More& m) const {
        const int left = a.k - k0 - i;
        if (a.pre) {
            const lin_f32x4 p = wide_4<F16>(m.p, false), q = a.pre_up ? wide_4<F16>(m.q, false) : lin_f32x4{1.0f, 1.0f, 1.0f, 1.0f};
            lin_f32x4 up;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float v, slope;
                lin_act_slope(a.act, p[x], &v, &slope);
                up[x] = g[x] * v;
                g[x] = g[x] * slope * q[x];
            }
            if (a.pre_up) store_4<F16>(cell(a.dx_up, m0, a.dx_ld, k0, j, i, a.dx_f32), left, a.dx_f32, up, a.past);
        } else if (a.accumulate) {
            g += wide_4<F16>(m.p, a.dx_f32);
        }
        store_4<F16>(cell(a.dx, m0, a.dx_ld, k0, j, i, a.dx_f32), left, a.dx_f32, g, a.past);
    }
};

// dx = dy W (+ dy_up U, the sum going on through both).  64 experts of 1408 x 2048 x 2 with 384 rows each take 325 to 355 us, the
// products alone at a large library product's rate 210: the rows fill three quarters of the 256-row tiles, 4.06 rounds of blocks
// take as long as 5, and a step takes 1.6 us as in the forward (the tiles' rows coming out of L2).
// One matrix of 4096 x 14336 and 4096 rows takes 381 (1.26 PFLOP/s), 14336 x 4096 339.  What follows the product, 64 experts of
// 2048 x 1408 with 384 rows: 193 alone, 242 with pre, 276 with pre and pre_up (208 MB more to read and write, 40 at a copy's rate).
template <class S, bool DUAL>
__global__ void __launch_bounds__(S::TH, 2)
input_grad_kernel(InputArgs a, uint32_t nI, Parts parts) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
    const Segments seg(a.offsets, a.rows, a.experts, S::TJ);
    uint32_t it, jt, m0;
    if (!tile_of_block(blockIdx.x, nI, seg.tiles, &it, &jt)) return;
    int e, nj;
    seg.find(jt, S::TJ, &e, &m0, &nj);
    const int k0 = it * S::TI, ni = min(S::TI, a.k - k0), z = blockIdx.y;
    const TileView iv[2] = {{a.w + e * a.w_stride + k0, a.w_ld, ni, k0}, {a.u + e * a.u_stride + k0, a.u_ld, ni, k0}};
    const TileView jv[2] = {{a.dy + (int64_t)m0 * a.dy_ld, a.dy_ld, nj}, {a.dy_up + (int64_t)m0 * a.dy_ld, a.dy_ld, nj}};
    lin_f32x4 acc[S::FI][S::FJ] = {};
    const int64_t steps = (int64_t)((a.n + S::kStep - 1) / S::kStep) * (DUAL ? 2 : 1);
    const int s0 = (int)(steps * z / parts.splits), s1 = (int)(steps * (z + 1) / parts.splits);
    tile_product<S, DUAL>(iv, jv, a.n, s0, s1, turn_of_block(blockIdx.x, s1 - s0, false), lds, acc, [](auto&) {});
    if (parts.splits == 1) each_piece<S>(lds, acc, ni, nj, InputOut<S::F16>{a, k0, m0});
    else each_piece<S>(lds, acc, ni, nj, PartOut<false>{parts.at(z, 0) + (int64_t)m0 * a.k + k0, nullptr, a.k, ni});
}

// Behind its parts: 4 values of a row at a time.
template <bool F16, int G>
__global__ void __launch_bounds__(256)
input_finish_kernel(InputArgs a, Parts parts) {
    const uint32_t quads = (a.k + 3) / 4;
    each_sum<G>(parts, (uint64_t)quads * a.rows, [&](uint64_t i, bool in, bool first, auto sum) {
        const uint32_t m = (uint32_t)(i / quads), k = (uint32_t)(i - (uint64_t)m * quads) * 4;
        in = in && expert_of_row(a.offsets, a.experts, a.rows, m) >= 0;
        const lin_f32x4 g = sum(0, (int64_t)m * a.k + k, a.k - k, in);
        const InputOut<F16> out{a, (int)k, m};
        if (first && in) out.store(0, 0, g, {}, out.more(0, 0));
    });
}

struct WeightArgs {
    const uint16_t *dy, *x;
    int64_t dy_ld, x_ld;
    const uint32_t* offsets;
    uint32_t rows;
    int n, k;
    void* dw;
    int64_t ld, stride;
    float* dbias;
    bool dw_f32, accumulate, past;
};

// What follows the sum, for values k0 + i .. k0 + i + 3 of weight row n0 + j.
template <bool F16> struct WeightOut {
    struct More {
        lin_u32x4 old;
        __device__ __forceinline__ void here() { in_registers(old); }
    };
    const WeightArgs& a;
    int e, n0, k0;
    __device__ __forceinline__ char* at(int j, int i) const { return cell(a.dw, n0, a.ld, e * a.stride + k0, j, i, a.dw_f32); }
    __device__ __forceinline__ void column(int) {}
    __device__ __forceinline__ bool reads() const { return a.accumulate; }
    __device__ __forceinline__ More more(int j, int i) const {
        return {a.accumulate ? raw_4(at(j, i), a.k - k0 - i, a.dw_f32) : lin_u32x4{}};
    }
    __device__ __forceinline__ void store(int j, int i, lin_f32x4 v, lin_f32x4, const More& m) const {
        if (a.accumulate) v += wide_4<F16>(m.old, a.dw_f32);
        store_4<F16>(at(j, i), a.k - k0 - i, a.dw_f32, v, a.past);
    }
};
__device__ __forceinline__ void bias_store(const WeightArgs& a, int e, int n, float v) {
    float* to = a.dbias + (int64_t)e * a.n + n;
    *to = v + (a.accumulate ? *to : 0.0f);
}
__device__ __forceinline__ void segment_of(const WeightArgs& a, int e, uint32_t* m0, uint32_t* m1) {
    *m0 = a.offsets ? offset_at(a.offsets, e, a.rows) : 0;
    *m1 = a.offsets ? max(*m0, offset_at(a.offsets, e + 1, a.rows)) : a.rows;
}

// dw = dy' x of a segment: sums as short as the segment, and results that are often the largest thing a call touches.  64 experts
// of 1408 x 2048 with 384 rows each take 243 to 270 us: 143 for 738 MB of f32 at a copy's rate and 105 for the products, which a
// CU's one block does one after the other; added to what is there 382.
// parts: plane 0 [experts][n][k]; the bias's parts lie behind all planes, [splits][experts][n].
template <class S>
__global__ void __launch_bounds__(S::TH, 2)
weight_grad_kernel(WeightArgs a, uint32_t nI, uint32_t nJ, Parts parts) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
    uint32_t it, jt, m0, m1;
    if (!tile_of_block(blockIdx.x, nI, nJ, &it, &jt)) return;
    const int e = blockIdx.y, z = blockIdx.z; // (all XCDs share an expert: with an expert each, uneven ones took 1.4 times as long)
    segment_of(a, e, &m0, &m1);
    const int k0 = it * S::TI, ni = min(S::TI, a.k - k0), n0 = jt * S::TJ, nj = min(S::TJ, a.n - n0);
    const TileView iv[2] = {{a.x + m0 * a.x_ld + k0, a.x_ld, ni, k0}, {}}, jv[1] = {{a.dy + m0 * a.dy_ld + n0, a.dy_ld, nj, n0}};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    lin_f32x4 acc[S::FI][S::FJ] = {}, sum[S::FJ] = {};
    const bool bias = a.dbias && it == 0 && S::i_first(wave) == 0; // whose share the bias gradient is
    const short one = S::F16 ? (short)0x3c00 : (short)0x3f80;
    const lin_s16x8 ones = {one, one, one, one, one, one, one, one};
    const int64_t steps = (m1 - m0 + S::kStep - 1) / S::kStep;
    const int s0 = (int)(steps * z / parts.splits), s1 = (int)(steps * (z + 1) / parts.splits);
    tile_product<S, false>(iv, jv, m1 - m0, s0, s1, turn_of_block(blockIdx.x, s1 - s0, true), lds, acc, [&](auto& b) {
        if (bias)
#pragma unroll
            for (int f = 0; f < S::FJ; ++f) sum[f] = lin_mfma<S::F16>(ones, b[f], sum[f]);
    });
    if (a.accumulate && m0 == m1) return;
    if (bias && lane < 16) {
#pragma unroll
        for (int fj = 0; fj < S::FJ; ++fj) {
            const int j = S::j_first(wave) + 16 * fj + lane;
            if (j >= nj) continue;
            if (parts.splits == 1) bias_store(a, e, n0 + j, sum[fj][0]);
            else parts.at(parts.splits, 0)[((int64_t)z * gridDim.y + e) * a.n + n0 + j] = sum[fj][0];
        }
    }
    if (parts.splits == 1) {
        each_piece<S>(lds, acc, ni, nj, WeightOut<S::F16>{a, e, n0, k0});
    } else {
        each_piece<S>(lds, acc, ni, nj, PartOut<false>{parts.at(z, 0) + ((int64_t)e * a.n + n0) * a.k + k0, nullptr, a.k, ni});
    }
}

// Behind its parts: 4 values of a weight's row at a time, and a block's share of the biases behind them.
template <bool F16, int G>
__global__ void __launch_bounds__(256)
weight_finish_kernel(WeightArgs a, int experts, Parts parts) {
    const uint32_t quads = (a.k + 3) / 4;
    auto live = [&](uint32_t e) { // an accumulating call leaves experts without rows alone
        uint32_t m0, m1;
        segment_of(a, e, &m0, &m1);
        return !(a.accumulate && m0 == m1);
    };
    each_sum<G>(parts, (uint64_t)quads * a.n * experts, [&](uint64_t i, bool in, bool first, auto sum) {
        const uint64_t row = i / quads;
        const uint32_t k = (uint32_t)(i - row * quads) * 4, e = (uint32_t)(row / a.n), n = (uint32_t)(row - (uint64_t)e * a.n);
        in = in && live(e);
        const lin_f32x4 v = sum(0, (int64_t)row * a.k + k, a.k - k, in);
        const WeightOut<F16> out{a, (int)e, (int)n, (int)k};
        if (first && in) out.store(0, 0, v, {}, out.more(0, 0));
    });
    if (!a.dbias) return;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)a.n * experts; i += (uint64_t)gridDim.x * 256) {
        const uint32_t e = (uint32_t)(i / a.n), n = (uint32_t)(i - (uint64_t)e * a.n);
        if (!live(e)) continue;
        float v = 0.0f;
        for (int z = 0; z < parts.splits; ++z) v += parts.at(parts.splits, 0)[((int64_t)z * experts + e) * a.n + n];
        bias_store(a, e, n, v);
    }
}

template <class S> int launch_input(const InputArgs& a, hipStream_t st) {
    const int64_t nI = (a.k + S::TI - 1) / S::TI, nJ = lin_j_tiles(a.rows, a.experts, a.offsets, S::TJ);
    const int64_t plane = (int64_t)a.rows * a.k;
    const int splits = lin_splits(nI * nJ, (int64_t)(a.n + S::kStep - 1) / S::kStep * (a.u ? 2 : 1), plane);
    const int64_t blocks = (nI * nJ + 7) / 8 * 8;
    if (blocks * splits * S::TH >= (int64_t)1 << 32) return NAIWA_E_UNSUPPORTED; // a launch's threads
    Parts parts;
    if (int rc = lin_parts(splits, 1, plane, st, &parts)) return rc;
    const dim3 grid((unsigned)blocks, splits);
    if (a.u) input_grad_kernel<S, true><<<grid, S::TH, 0, st>>>(a, (uint32_t)nI, parts);
    else input_grad_kernel<S, false><<<grid, S::TH, 0, st>>>(a, (uint32_t)nI, parts);
    if (splits > 1) {
        const int64_t quads = (int64_t)(a.k + 3) / 4 * a.rows;
        if (splits <= 8) input_finish_kernel<S::F16, 1><<<lin_finish_blocks(quads, 1), 256, 0, st>>>(a, parts);
        else input_finish_kernel<S::F16, 16><<<lin_finish_blocks(quads, 16), 256, 0, st>>>(a, parts);
    }
    return naiwa_hip_rc(hipGetLastError());
}
// Whether 256 x 256 tiles have at most `most` times the places that 128 x 128 ones have.
bool lin_packed(int64_t i, int64_t j256, int64_t j128, double most) {
    return (double)((i + 255) / 256 * j256 * 4) <= most * (double)((i + 127) / 128 * j128);
}
int lin_input_kind(int64_t rows, int experts, int64_t n, int64_t k, bool dual) {
    const bool grouped = experts > 0;
    const int64_t j256 = lin_j_alike(rows, experts, grouped, 256), j128 = lin_j_alike(rows, experts, grouped, 128);
    // (64 experts of 1240 x 88 with 918 rows, two matrices: 139 us in 256 x 256 tiles, 60 in 128 x 128; of 2248 x 176: 257 and 385.)
    return lin_kind(n * (dual ? 2 : 1), rows / std::max(experts, 1), (k + 255) / 256 * j256, lin_packed(k, j256, j128, 1.5));
}
template <bool F16> int input_grad(const InputArgs& a, bool direct, hipStream_t st) {
    if (!direct && lin_narrow(a.rows / (a.offsets ? a.experts : 1)))
        return launch_input<Shape<128, 64, 2, 2, 32, 2, kCols, kRows, F16, false>>(a, st);
    if (!direct) return launch_input<Shape<128, 128, 2, 2, 32, 2, kCols, kRows, F16, false>>(a, st);
    switch (lin_input_kind(a.rows, a.offsets ? a.experts : 0, a.n, a.k, a.u != nullptr)) {
    case kThin: return launch_input<Shape<128, 32, 4, 1, 64, 4, kCols, kRows, F16, true>>(a, st);
    case kShort: return launch_input<Shape<128, 128, 2, 2, 32, 2, kCols, kRows, F16, true>>(a, st);
    case kMid: return launch_input<Shape<128, 128, 2, 2, 32, 4, kCols, kRows, F16, true>>(a, st);
    default: return launch_input<Shape<256, 256, 2, 4, 64, 2, kCols, kRows, F16, true>>(a, st);
    }
}

template <class S> int launch_weight(const WeightArgs& a, int experts, hipStream_t st) {
    const int64_t nI = (a.k + S::TI - 1) / S::TI, nJ = (a.n + S::TJ - 1) / S::TJ;
    const int64_t plane = (int64_t)experts * a.n * a.k, bias = a.dbias ? (int64_t)experts * a.n : 0;
    const int splits = lin_splits(nI * nJ * experts, a.rows / experts / S::kStep, plane + bias);
    const int64_t blocks = (nI * nJ + 7) / 8 * 8;
    if (blocks * experts * splits * S::TH >= (int64_t)1 << 32) return NAIWA_E_UNSUPPORTED;
    Parts parts;
    if (int rc = lin_parts(splits, 1, plane + bias, st, &parts)) return rc;
    parts.plane = plane; // (the bias's parts behind the planes)
    weight_grad_kernel<S><<<dim3((unsigned)blocks, experts, splits), S::TH, 0, st>>>(a, (uint32_t)nI, (uint32_t)nJ, parts);
    if (splits > 1) {
        const int64_t quads = (int64_t)(a.k + 3) / 4 * a.n * experts;
        if (splits <= 8) weight_finish_kernel<S::F16, 1><<<lin_finish_blocks(quads, 1), 256, 0, st>>>(a, experts, parts);
        else weight_finish_kernel<S::F16, 16><<<lin_finish_blocks(quads, 16), 256, 0, st>>>(a, experts, parts);
    }
    return naiwa_hip_rc(hipGetLastError());
}
int lin_weight_kind(int64_t rows, int experts, int64_t n, int64_t k) {
    const int64_t j256 = (n + 255) / 256, tiles = experts * ((k + 255) / 256) * j256, avg = rows / experts;
    // Sums are as long as a segment is, and all of dw is written, so empty places count, and few tiles are split more ways by the
    // smaller ones (ring of 2, of 4 and 256 x 256, us: 64 experts of 1408 x 2048 with 16 rows each 157, 202 and 169; 128 of
    // 768 x 2800 with 209 450, 484 and 432; 64 of 184 x 8112 with 602 357, 350 and 257; of 56 x 2384 with 720 79, 78 and 134; of
    // 184 x 912 with 1166 114, 104 and 142; 9335 rows, 208 x 6952 63, 56 and 87; 10085, 3200 x 2288 220, 188 and 148).
    const bool many = tiles >= 384 || std::min(n, k) >= 1024;
    if (avg > 64 && many && tiles * (avg / 64 + 1) >= kManySteps && lin_packed(k, j256, (n + 127) / 128, 1.25)) return kBig;
    return avg <= 384 ? kShort : kMid;
}
template <bool F16> int weight_grad(const WeightArgs& a, int experts, bool direct, hipStream_t st) {
    // (128 x 64 and 128 x 128, us: 2048 rows, 2049 x 2047 64 and 72, 4097, 4099 x 4101 296 and 300, 64 experts of 1407 x 2049 with 64 rows
    // 207 and 264, with 384 406 and 376; 60 rows, 153 x 1088 with its input gradient 37 and 46.)
    if (!direct) return launch_weight<Shape<128, 64, 2, 2, 32, 2, kCols, kCols, F16, false>>(a, experts, st);
    switch (lin_weight_kind(a.rows, experts, a.n, a.k)) {
    case kShort: return launch_weight<Shape<128, 128, 2, 2, 32, 2, kCols, kCols, F16, true>>(a, experts, st);
    case kMid: return launch_weight<Shape<128, 128, 2, 2, 32, 4, kCols, kCols, F16, true>>(a, experts, st);
    default: return launch_weight<Shape<256, 256, 2, 4, 64, 2, kCols, kCols, F16, true>>(a, experts, st);
    }
}

} // namespace

extern "C" int naiwa_linear_input_grad(const naiwa_weights* w, const naiwa_weights* up, const void* dy, const void* dy_up,
                                       int64_t dy_ld, const uint32_t* offsets, int64_t rows, int act, const void* pre,
                                       const void* pre_up, int64_t pre_ld, void* dx, void* dx_up, int dx_dtype,
                                       int64_t dx_ld, int flags, int64_t stream) {
    if (int rc = lin_pair_ok(w, up)) return rc;
    const int n = w->n, k = w->k;
    if (rows < 0 || dy_ld < 0 || pre_ld < 0 || dx_ld < 0 || (dy_ld && dy_ld < n) || (pre_ld && pre_ld < k) ||
        (dx_ld && dx_ld < k) || (!offsets && w->experts != 1) || (flags & ~NAIWA_LINEAR_ACCUMULATE) || !up != !dy_up ||
        (pre_up && !pre) || !pre_up != !dx_up || (pre && flags))
        return NAIWA_E_INVALID;
    dy_ld = dy_ld ? dy_ld : n, pre_ld = pre_ld ? pre_ld : k, dx_ld = dx_ld ? dx_ld : k;
    if (!lin_act_ok(act)) return NAIWA_E_UNSUPPORTED;
    if (dx_dtype != NAIWA_F32 && dx_dtype != w->dtype) return NAIWA_E_UNSUPPORTED;
    if (rows > INT32_MAX || std::max({dy_ld, pre_ld, dx_ld}) > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (rows == 0) return NAIWA_OK;
    if (!dy || !dx) return NAIWA_E_INVALID;
    const InputArgs a{(const uint16_t*)w->w, up ? (const uint16_t*)up->w : nullptr, (const uint16_t*)dy, (const uint16_t*)dy_up,
                      lin_ld(w), lin_stride(w), up ? lin_ld(up) : 0, up ? lin_stride(up) : 0, dy_ld, offsets, (uint32_t)rows,
                      w->experts, n, k, act, (const uint16_t*)pre, (const uint16_t*)pre_up, dx, dx_up, pre_ld, dx_ld,
                      dx_dtype == NAIWA_F32, (flags & NAIWA_LINEAR_ACCUMULATE) != 0,
                      !flags && rows * k * lin_size(dx_dtype) >= kLinPast};
    const Span ins[] = {span_of(dy, rows, dy_ld, n, 2), span_of(dy_up, rows, dy_ld, n, 2), lin_span(w), lin_span(up),
                        span_of(pre, rows, pre_ld, k, 2), span_of(pre_up, rows, pre_ld, k, 2), lin_span(offsets, w->experts)};
    const Span outs[] = {span_of(dx, rows, dx_ld, k, lin_size(dx_dtype)), span_of(dx_up, rows, dx_ld, k, lin_size(dx_dtype))};
    for (const Span& o : outs)
        for (const Span& in : ins)
            if (overlap(o, in)) return NAIWA_E_INVALID;
    if (overlap(outs[0], outs[1])) return NAIWA_E_INVALID;
    const bool direct = !((n | k) & 7) && lin_aligned(a.w, a.w_ld, a.w_stride) && lin_aligned(dy, dy_ld, 0) &&
                        (!up || (lin_aligned(a.u, a.u_ld, a.u_stride) && lin_aligned(dy_up, dy_ld, 0)));
    hipStream_t st = (hipStream_t)stream;
    return w->dtype == NAIWA_BF16 ? input_grad<false>(a, direct, st) : input_grad<true>(a, direct, st);
}

extern "C" int naiwa_linear_weight_grad(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int dtype,
                                        const uint32_t* offsets, int experts, int64_t rows, int n, int k, void* dw,
                                        int dw_dtype, int64_t ld, int64_t stride, float* dbias, int flags, int64_t stream) {
    if (int rc = lin_sizes_ok(experts, n, k, ld, stride)) return rc;
    if (rows < 0 || dy_ld < 0 || x_ld < 0 || (dy_ld && dy_ld < n) || (x_ld && x_ld < k) || (!offsets && experts != 1) ||
        (flags & ~NAIWA_LINEAR_ACCUMULATE) || !dw)
        return NAIWA_E_INVALID;
    dy_ld = dy_ld ? dy_ld : n, x_ld = x_ld ? x_ld : k, ld = ld ? ld : k, stride = stride ? stride : n * ld;
    if ((dtype != NAIWA_BF16 && dtype != NAIWA_F16) || (dw_dtype != NAIWA_F32 && dw_dtype != dtype)) return NAIWA_E_UNSUPPORTED;
    if (rows > INT32_MAX || dy_ld > kMaxLd || x_ld > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (rows && (!dy || !x)) return NAIWA_E_INVALID;
    const WeightArgs a{(const uint16_t*)dy, (const uint16_t*)x, dy_ld, x_ld, offsets, (uint32_t)rows, n, k, dw, ld, stride, dbias,
                       dw_dtype == NAIWA_F32, (flags & NAIWA_LINEAR_ACCUMULATE) != 0,
                       !flags && (int64_t)experts * n * k * lin_size(dw_dtype) >= kLinPast};
    const Span ins[] = {span_of(dy, rows, dy_ld, n, 2), span_of(x, rows, x_ld, k, 2), lin_span(offsets, experts)};
    const Span to = span_of(dw, ((experts - 1) * stride + (n - 1) * ld + k) * lin_size(dw_dtype));
    const Span bias = span_of(dbias, (int64_t)experts * n * 4);
    for (const Span& in : ins)
        if (overlap(to, in) || overlap(bias, in)) return NAIWA_E_INVALID;
    if (overlap(to, bias)) return NAIWA_E_INVALID;
    const bool direct = !((n | k) & 7) && lin_aligned(dy, dy_ld, 0) && lin_aligned(x, x_ld, 0);
    hipStream_t st = (hipStream_t)stream;
    return dtype == NAIWA_BF16 ? weight_grad<false>(a, experts, direct, st) : weight_grad<true>(a, experts, direct, st);
}

// Which kernel a call with aligned rows takes (experts 0: one matrix for all rows), for tests.
extern "C" int naiwa_linear_input_grad_kind(int64_t rows, int experts, int n, int k, int dual) {
    return lin_input_kind(rows, experts, n, k, dual != 0);
}
extern "C" int naiwa_linear_weight_grad_kind(int64_t rows, int experts, int n, int k) {
    return lin_weight_kind(rows, experts, n, k);
}
