// naiwa_linear and naiwa_act_backward (include/naiwa_linear.h): rows times weights, everything behind the
// product in the same pass.  The tiles are linear_tiles.h's: I is the weights (for a gated product half
// a tile of each matrix), J the rows, so that a lane ends with 4 consecutive features of a row.
#include "linear_tiles.h"

#include <algorithm>

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
    bool out_f32;
};

// 4 features of a row, n .. n + 3 (`left` of them exist), behind the product.
template <bool F16> __device__ __forceinline__ void forward_store(const ForwardArgs& a, int e, uint32_t m, int n, lin_f32x4 p, lin_f32x4 q) {
    const int left = a.n - n;
    if (a.b) p += load_4<F16>(a.b, (int64_t)e * a.n + n, left, true);
    if (a.pre) store_4<F16>(a.pre, m * a.pre_ld + n, left, false, p);
    lin_f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lin_act(a.act, p[i]);
    if (a.u) {
        if (a.c) q += load_4<F16>(a.c, (int64_t)e * a.n + n, left, true);
        if (a.pre_up) store_4<F16>(a.pre_up, m * a.pre_ld + n, left, false, q);
        v *= q;
    }
    if (a.residual) v += load_4<F16>(a.residual, m * a.residual_ld + n, left, a.out_f32);
    store_4<F16>(a.out, m * a.out_ld + n, left, a.out_f32, v);
}

template <class S>
__global__ void __launch_bounds__(S::TH, S::kWavesEU)
linear_kernel(ForwardArgs a, uint32_t nI) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
    constexpr int kN = S::PAIR ? S::TI / 2 : S::TI; // features of a tile
    const Segments seg(a.offsets, a.rows, a.experts, S::TJ);
    uint32_t it, jt, m0;
    if (!tile_of_block(blockIdx.x, nI, seg.tiles, &it, &jt)) return;
    int e, nj;
    seg.find(jt, S::TJ, &e, &m0, &nj);
    const int n0 = it * kN, ni = min(kN, a.n - n0);
    const TileView iv[2] = {{a.w + e * a.w_stride + (int64_t)n0 * a.w_ld, a.w_ld, ni},
                            {a.u + e * a.u_stride + (int64_t)n0 * a.u_ld, a.u_ld, ni}};
    const TileView jv[1] = {{a.x + (int64_t)m0 * a.x_ld, a.x_ld, nj}};
    lin_f32x4 acc[S::FI][S::FJ] = {};
    tile_product<S>(iv, jv, a.k, 0, (a.k + kStep - 1) / kStep, lds, acc, [](auto&) {});
    each_piece<S>(lds, acc, [&](int j, int i, lin_f32x4 p, lin_f32x4 q) {
        if (j < nj && i < ni) forward_store<S::F16>(a, e, m0 + j, n0 + i, p, q);
    });
}

template <class S> int launch(const ForwardArgs& a, hipStream_t st) {
    constexpr int kN = S::PAIR ? S::TI / 2 : S::TI;
    const int64_t nI = (a.n + kN - 1) / kN;
    const int64_t nJ = (int64_t)a.rows / S::TJ + (a.offsets ? std::min<int64_t>(a.experts, a.rows) : a.rows % S::TJ != 0);
    const int64_t blocks = (nI * nJ + 7) / 8 * 8;
    if (blocks * S::TH >= (int64_t)1 << 32) return NAIWA_E_UNSUPPORTED; // a launch's threads
    linear_kernel<S><<<(unsigned)blocks, S::TH, 0, st>>>(a, (uint32_t)nI);
    return naiwa_hip_rc(hipGetLastError());
}

template <bool F16, bool PAIR> int forward(const ForwardArgs& a, bool direct, hipStream_t st) {
    return direct ? launch<Shape<256, 256, 2, 4, 4, kRows, kRows, F16, true, PAIR>>(a, st)
                  : launch<Shape<128, 128, 2, 2, 4, kRows, kRows, F16, false, PAIR>>(a, st);
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

// One thread takes N values at a time (those behind a row's last whole piece one by one).
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
    if (rows > INT32_MAX || x_ld > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (rows == 0) return NAIWA_OK;
    if (!x || !out) return NAIWA_E_INVALID;
    const ForwardArgs a{(const uint16_t*)w->w, up ? (const uint16_t*)up->w : nullptr, (const uint16_t*)x,
                        lin_ld(w), lin_stride(w), up ? lin_ld(up) : 0, up ? lin_stride(up) : 0, x_ld,
                        w->bias, up ? up->bias : nullptr, offsets, (uint32_t)rows, w->experts, n, k, act,
                        residual, out, (uint16_t*)pre, (uint16_t*)pre_up, residual_ld, out_ld, pre_ld, out_dtype == NAIWA_F32};
    // an output is written where nothing else is read or written
    const int64_t w_bytes = lin_bytes(w), u_bytes = up ? lin_bytes(up) : 0;
    const int64_t b_bytes = (int64_t)w->experts * n * 4;
    const int so = lin_size(out_dtype);
    struct Out {
        const void* p;
        int64_t bytes;
    } outs[3] = {{out, lin_span(rows, out_ld, n, so)}, {pre, lin_span(rows, pre_ld, n, 2)}, {pre_up, lin_span(rows, pre_ld, n, 2)}};
    for (int i = 0; i < 3; ++i) {
        const Out& o = outs[i];
        if (lin_overlap(o.p, o.bytes, x, lin_span(rows, x_ld, k, 2)) || lin_overlap(o.p, o.bytes, a.w, w_bytes) ||
            lin_overlap(o.p, o.bytes, a.u, u_bytes) || lin_overlap(o.p, o.bytes, a.b, b_bytes) ||
            lin_overlap(o.p, o.bytes, a.c, b_bytes))
            return NAIWA_E_INVALID;
        if (!(i == 0 && residual == out && residual_ld == out_ld) &&
            lin_overlap(o.p, o.bytes, residual, lin_span(rows, residual_ld, n, so)))
            return NAIWA_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (lin_overlap(o.p, o.bytes, outs[j].p, outs[j].bytes)) return NAIWA_E_INVALID;
    }
    const bool direct = !(k & 7) && lin_aligned(a.w, a.w_ld, a.w_stride) && lin_aligned(a.x, x_ld, 0) &&
                        (!up || lin_aligned(a.u, a.u_ld, a.u_stride));
    hipStream_t st = (hipStream_t)stream;
    if (w->dtype == NAIWA_BF16) return up ? forward<false, true>(a, direct, st) : forward<false, false>(a, direct, st);
    return up ? forward<true, true>(a, direct, st) : forward<true, false>(a, direct, st);
}

extern "C" int naiwa_act_backward(const void* dout, const void* pre, const void* pre_up, int dtype, int64_t rows, int n,
                                  int64_t ld, int act, void* dpre, void* dpre_up, int64_t stream) {
    if (rows < 0 || n <= 0 || ld < 0 || (ld && ld < n)) return NAIWA_E_INVALID;
    if (!lin_act_ok(act) || (dtype != NAIWA_F32 && dtype != NAIWA_BF16 && dtype != NAIWA_F16)) return NAIWA_E_UNSUPPORTED;
    if (rows > INT32_MAX || ld > kMaxLd) return NAIWA_E_UNSUPPORTED;
    if (rows == 0) return NAIWA_OK;
    if (!dout || !pre || !dpre || (!pre_up) != (!dpre_up)) return NAIWA_E_INVALID;
    ld = ld ? ld : n;
    const int64_t bytes = lin_span(rows, ld, n, lin_size(dtype));
    // in place element by element, or apart
    const void* ins[3] = {dout, pre, pre_up};
    for (const void* o : {(const void*)dpre, (const void*)dpre_up})
        for (const void* i : ins)
            if (o != i && lin_overlap(o, bytes, i, bytes)) return NAIWA_E_INVALID;
    if (lin_overlap(dpre, bytes, dpre_up, bytes)) return NAIWA_E_INVALID;
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
