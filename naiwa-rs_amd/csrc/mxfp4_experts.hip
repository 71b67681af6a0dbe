// The SwiGLU experts over MXFP4 banks on the matrix cores: naiwa_moe_decode and
// naiwa_moe_prefill calls whose banks are NAIWA_MXFP4_T.
//
//   out[t] = sum_j w[t,j] * down_s( act(gate_s x_t) * up_s x_t ),  s = ids[t,j]
//
// The weights go into v_mfma_scale_f32_16x16x128_f8f6f4 as they lie in memory: its A
// operand is FP4 with one scale byte per 32 values, lane 16 b + m holding block b of row
// m, which is the tile order.  Nothing is dequantised.  The instruction's B operand is at
// most 8 bits wide, so an activation enters as a sum of E2M3 planes (6 bits: 4 significant
// ones, values up to 7.5 in steps of 1/8): with a block of 32 scaled so that its largest
// magnitude lies in [2, 4), plane 0 is the value rounded to E2M3 (off by at most 1/8), plane
// 1 the rest times 2^5 (at most 4) rounded again, and so on; plane p has the scale
// 2^(s - 127 - 5 p).  With M the block's largest magnitude, P planes hold a value to within
// 2^(1 - 5 P) M:
//   4 planes (f32 x, h, and any x of a decode step): 2^-19 M; a bf16 value of at least
//     2^-12 M exactly;
//   3 planes (x of a prompt chunk, bf16): 2^-14 M; a value of at least 2^-7 M exactly.
// FP4 x E2M3 runs at twice the rate of FP4 x FP8 and of bf16 per step (5.4 against 3.4
// PFLOP/s measured), and its sums are exact up to the f32 accumulator's rounding; with e4m3
// the matrix cores drop products under about 2^-15 of a step's largest (5e-5 of a sum of
// codes of all magnitudes).  A block with a NaN or an infinity gets the scale byte 255,
// which makes its products NaN.
//
// Launches, stream-ordered:
//   1. the (token, expert) pairs sorted by slot;
//   2. x laid out in planes, one row per token;
//   3. gate/up: a block per (slot segment, 32 features): 16 tokens a pass, the steps of K
//      dealt to its waves, whose partial sums meet in LDS; h = act(g) u in planes;
//   4. down: a block per (slot segment, 64 rows, K part); unweighted dots per pair;
//   5. combine: out[t] = the weighted sum over t's pairs in ascending slot order.
// No atomics: every run adds the same terms in the same order, and a pair's terms do not
// depend on the other pairs of the call.
#include "mxfp4.h"
#include "segments.h"

#include <algorithm>

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v32f __attribute__((ext_vector_type(32)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v6u __attribute__((ext_vector_type(6)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kMaxWidth = 64; // pairs a token that the combine orders

struct Bank {
    const uint8_t* base;
    int64_t stride;
    int64_t strip; // bytes of 16 rows
};

// Rows of activations in P planes of E2M3: row i at base + i * row.  A step of 128 values (4
// blocks) is 96 P bytes: the first 16 of a block's 24 bytes per plane at head_at, the other 8
// at tail_at, in the order that the tiles' copies to LDS take (mxfp4_tiles.h).  Scales: row i
// at scales + i * groups * 16, byte 16 (kb / 16) + 4 (kb % 4) + kb / 4 % 4 for block kb (a
// lane's dword holds its block's scale in 4 steps).
struct Planes {
    uint8_t* base;
    uint8_t* scales;
    int64_t row;
    int groups;
};
__host__ __device__ inline int64_t plane_row(int planes, int k) { return (int64_t)naiwa_mx_steps(k) * 96 * planes; }
__device__ __forceinline__ int scale_at(int kb) { return 16 * (kb >> 4) + 4 * (kb & 3) + ((kb >> 2) & 3); }

// Bytes of plane p of block b (of its step's 4).
__host__ __device__ constexpr int head_at(int P, int b, int p) { return 32 * P * (b & 1) + 16 * ((b >> 1) * P + p); }
__host__ __device__ constexpr int tail_at(int P, int b, int p) { return 64 * P + 16 * ((b >> 1) * P + p) + 8 * (b & 1); }

// The scale byte of a block whose largest magnitude has the bits m: that magnitude in
// [2, 4) times 2^(s - 127).  At least 16, so that the planes' scales stay normal.
__device__ __forceinline__ int scale_byte(uint32_t m) {
    const int e = (int)(m >> 23);
    return e == 255 ? 255 : max(16, e - 1);
}

// N values (a multiple of 2, up to a block) as planes: N codes of 6 bits, value 0 lowest, in
// the low bits of 6 words per plane.
template <int P, int N> __device__ __forceinline__ void to_planes(const float (&f)[N], int s, v6u (&o)[P]) {
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = s == 255 ? 0.0f : f[i];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const float scale = __uint_as_float((uint32_t)((s == 255 ? 127 : s) - 5 * p) << 23);
        v16f even = {}, odd = {}; // the conversion takes even and odd values apart
#pragma unroll
        for (int i = 0; i < N / 2; ++i) even[i] = y[2 * i], odd[i] = y[2 * i + 1];
        v6u c = __builtin_bit_cast(v6u, __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, scale));
        // The conversions run in several passes, and the compiler may give the result registers
        // of an operand, which then are overwritten before they are read (seen: the codes of the
        // last plane, off by whole binades).  The operands stay in use past the result.
        asm volatile("" : "+v"(c) : "v"(even), "v"(odd), "v"(scale));
        o[p] = c;
        if (p + 1 < P) {
            v32f back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(c, scale);
            asm volatile("" : "+v"(back) : "v"(c), "v"(scale));
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] -= back[i];
        }
    }
}

// The largest magnitude as bits: a NaN is larger than every number.
template <int N> __device__ __forceinline__ uint32_t abs_max(const float (&f)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
}

__global__ void __launch_bounds__(NAIWA_SEG_THREADS)
segments_kernel(const uint32_t* ids, const float* w, int n, int slots, uint32_t* perm, uint32_t* offsets, int* bad) {
    __shared__ NaiwaSegSmem sm;
    naiwa_segment(sm, ids, w, n, slots, perm, offsets, nullptr, nullptr, nullptr, bad);
}

__device__ __forceinline__ v8i fp4_operand(v4u v) {
    v8i o = {};
    o[0] = (int)v.x, o[1] = (int)v.y, o[2] = (int)v.z, o[3] = (int)v.w;
    return o;
}

#include "mxfp4_tiles.h"

// x [rows, H] in P planes, a block of 32 values a thread; the blocks that pad H to whole
// steps are zeros.  Bound: HBM.  With tiles, the last block of the launch cuts the sorted pairs
// into them: the two do not depend on each other.
template <int P, bool BF16>
__global__ void __launch_bounds__(kThreads)
planes_kernel(const void* x, int64_t rows, int H, Planes out, const uint32_t* offsets, int slots, Tiles tl) {
    if (tl.n && blockIdx.x == gridDim.x - 1) {
        tiles_block(offsets, slots, tl);
        return;
    }
    const int blocks = 4 * naiwa_mx_steps(H);
    const int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (b >= rows * blocks) return;
    const int64_t t = b / blocks;
    const int kb = (int)(b % blocks);
    float f[32] = {};
    if (32 * kb < H) {
        if constexpr (BF16) {
            const v4u* src = (const v4u*)((const uint16_t*)x + t * H + 32 * kb);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const v4u v = src[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f[8 * i + 2 * j] = naiwa_bf16_to_f32(v[j] & 0xffffu);
                    f[8 * i + 2 * j + 1] = naiwa_bf16_to_f32(v[j] >> 16);
                }
            }
        } else {
            const v4f* src = (const v4f*)((const float*)x + t * H + 32 * kb);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const v4f v = src[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[4 * i + j] = v[j];
            }
        }
    }
    const int s = scale_byte(abs_max(f));
    v6u o[P];
    to_planes<P>(f, s, o);
    uint8_t* dst = out.base + t * out.row + (int64_t)(kb >> 2) * 96 * P;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        *(v4u*)(dst + head_at(P, kb & 3, p)) = v4u{o[p][0], o[p][1], o[p][2], o[p][3]};
        *(v2u*)(dst + tail_at(P, kb & 3, p)) = v2u{o[p][4], o[p][5]};
    }
    out.scales[t * out.groups * 16 + scale_at(kb)] = (uint8_t)s;
}

// The E2M3 operand: plane p of block b of the step at `at`.
template <int P> __device__ __forceinline__ v8i e2m3_operand(const uint8_t* at, int b, int p) {
    const v4u h = *(const v4u*)(at + head_at(P, b, p));
    const v2u t = *(const v2u*)(at + tail_at(P, b, p));
    v8i o = {};
    o[0] = (int)h.x, o[1] = (int)h.y, o[2] = (int)h.z, o[3] = (int)h.w, o[4] = (int)t.x, o[5] = (int)t.y;
    return o;
}

// acc += strip rows x planes over steps [t0, t1): S strips of 16 rows, one token row of
// planes a lane.  wp[i]: strip i's first byte plus 16 lane; xp: the lane's token row;
// xs: the row's scales.
template <int S, int P>
__device__ __forceinline__ void strips_dot(const uint8_t* const (&wp)[S], const uint8_t* xp, const uint8_t* xs, int steps,
                                           int t0, int t1, int lane, v4f (&acc)[S]) {
    const int kb = lane >> 4;
    for (int t = t0; t < t1; ++t) {
        const int g = t >> 2, j = t & 3, in_group = min(4, steps - 4 * g);
        const int64_t at = (int64_t)1024 * t + 256 * g;
        const int64_t sc = (int64_t)1024 * (4 * g + in_group) + 256 * g - 12 * lane; // 4 lane, from wp's 16 lane
        v8i b[P];
#pragma unroll
        for (int p = 0; p < P; ++p) b[p] = e2m3_operand<P>(xp + (int64_t)(96 * P) * t, kb, p);
        const uint32_t bs = *(const uint32_t*)(xs + 16 * g + 4 * kb) >> (8 * j) & 255u;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const v8i a = fp4_operand(*(const v4u*)(wp[i] + at));
            const uint32_t as = *(const uint32_t*)(wp[i] + sc) >> (8 * j) & 255u;
#pragma unroll
            for (int p = 0; p < P; ++p)
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b[p], acc[i], 4, 2, 0, (int)as, 0,
                                                                         (int)(bs - 5 * p));
        }
    }
}

// Gate/up of one slot segment and 32 features.  Lane l holds D[4 (l / 16) + i][l % 16]:
// feature 4 (l / 16) + i of a strip, token l % 16.
template <int P>
__global__ void __launch_bounds__(kThreads)
gateup_kernel(Bank gate, Bank up, Planes x, int H, int I, int width, const uint32_t* offsets, const uint32_t* perm,
              int act, Planes h) {
    __shared__ v4f red[kWaves][4][64];
    __shared__ uint32_t mx[2][16];
    __shared__ __align__(16) uint8_t codes[16][96]; // a token's 4 planes of the block's 32 features
    const int s = blockIdx.x, fb = blockIdx.y;
    const int b = (int)offsets[s], e = (int)offsets[s + 1];
    if (b == e) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int steps = naiwa_mx_steps(H);
    const int t0 = steps * wave / kWaves, t1 = steps * (wave + 1) / kWaves;
    const int64_t go = (int64_t)s * gate.stride + 2 * fb * gate.strip + 16 * lane;
    const int64_t uo = (int64_t)s * up.stride + 2 * fb * up.strip + 16 * lane;
    // the features past I that pad h to whole steps: zeros
    const bool pad = 32 * fb >= I;
    for (int c0 = b; c0 < e; c0 += 16) {
        v4f acc[4] = {};
        const int pos = min(c0 + (lane & 15), e - 1);
        if (!pad) {
            const uint8_t* const wp[4] = {gate.base + go, gate.base + go + gate.strip, up.base + uo,
                                          up.base + uo + up.strip};
            const int64_t row = perm[pos] / (uint32_t)width;
            strips_dot<4, P>(wp, x.base + row * x.row, x.scales + row * x.groups * 16, steps, t0,
                             t1, lane, acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][i][lane] = acc[i];
        __syncthreads();
        const int half = wave & 1; // waves 0 and 1: strips 0 and 1 of the 32 features
        float f[4] = {};
        if (wave < 2) {
            v4f g = red[0][half][lane], u = red[0][2 + half][lane];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) {
                g += red[w][half][lane];
                u += red[w][2 + half][lane];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = pad ? 0.0f : naiwa_act(act, g[i]) * u[i];
            uint32_t m = abs_max(f);
            m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
            m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
            if (lane < 16) mx[half][lane] = m;
        }
        __syncthreads();
        if (wave < 2 && c0 + (lane & 15) < e) {
            const int sb = scale_byte(max(mx[0][lane & 15], mx[1][lane & 15]));
            v6u o[4];
            to_planes<4>(f, sb, o);
            // 4 codes are 3 bytes: features 4 q .. 4 q + 3 at byte 3 q, q = 4 half + lane / 16
            uint8_t* dst = codes[lane & 15] + 12 * half + 3 * (lane >> 4);
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int j = 0; j < 3; ++j) dst[24 * p + j] = (uint8_t)(o[p][0] >> (8 * j));
            if (half == 0 && lane < 16) h.scales[(int64_t)(c0 + lane) * h.groups * 16 + scale_at(fb)] = (uint8_t)sb;
        }
        __syncthreads();
        if (const int tok = tid >> 3, p = (tid >> 1) & 3; c0 + tok < e && tok < 16) {
            uint8_t* dst = h.base + (int64_t)(c0 + tok) * h.row + (int64_t)(fb >> 2) * 384;
            const v2u* src = (const v2u*)(codes[tok] + 24 * p);
            if (tid & 1)
                *(v2u*)(dst + tail_at(4, fb & 3, p)) = src[2];
            else
                *(v4u*)(dst + head_at(4, fb & 3, p)) = v4u{src[0].x, src[0].y, src[1].x, src[1].y};
        }
    }
}

// Down of one slot segment, 64 rows and one K part: y[part][pair][H] unweighted.
__global__ void __launch_bounds__(kThreads)
down_kernel(Bank down, Planes h, int H, int I, int64_t n, int parts, const uint32_t* offsets, const uint32_t* perm,
            float* y) {
    __shared__ v4f red[kWaves][4][64];
    const int s = blockIdx.x, rb = blockIdx.y, part = blockIdx.z;
    const int b = (int)offsets[s], e = (int)offsets[s + 1];
    if (b == e) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int steps = naiwa_mx_steps(I), all = parts * kWaves, mine = part * kWaves + wave;
    const int t0 = (int)((int64_t)steps * mine / all), t1 = (int)((int64_t)steps * (mine + 1) / all);
    const uint8_t* base = down.base + (int64_t)s * down.stride + 4 * rb * down.strip + 16 * lane;
    const int strips = min(4, H / 16 - 4 * rb);
    // strips past H read the last one again
    const uint8_t* wp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) wp[i] = base + min(i, strips - 1) * down.strip;
    for (int c0 = b; c0 < e; c0 += 16) {
        v4f acc[4] = {};
        const int64_t pos = min(c0 + (lane & 15), e - 1);
        const uint8_t* const wc[4] = {wp[0], wp[1], wp[2], wp[3]};
        strips_dot<4, 4>(wc, h.base + pos * h.row, h.scales + pos * h.groups * 16, steps, t0, t1,
                         lane, acc);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][i][lane] = acc[i];
        __syncthreads();
        v4f v = red[0][wave][lane]; // wave i adds strip i
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += red[w][wave][lane];
        if (wave < strips && c0 + (lane & 15) < e)
            *(v4f*)(y + ((int64_t)part * n + perm[pos]) * H + 64 * rb + 16 * wave + 4 * (lane >> 4)) = v;
    }
}

// out[t] (+)= the weighted dots of t's pairs in ascending slot order, a pair's K parts in
// part order; res: also res = bf16(res + out).
__global__ void __launch_bounds__(kThreads)
combine_kernel(const float* y, int64_t n, int parts, const uint32_t* ids, const float* w, int width, int slots, int H,
               int skip_zero, int accumulate, float* out, uint16_t* res) {
    __shared__ int list[kMaxWidth];
    __shared__ float wl[kMaxWidth];
    __shared__ int count;
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x;
    if (tid < 64) {
        const uint32_t id = tid < width ? ids[t * width + tid] : 0xffffffffu;
        const float wt = tid < width ? w[t * width + tid] : 0.0f;
        const bool in = id < (uint32_t)slots && !(skip_zero && wt == 0.0f);
        int rank = 0;
        for (int j = 0; j < width; ++j) {
            const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)(in ? id : 0xffffffffu), j);
            rank += o < id || (o == id && j < tid) ? 1 : 0;
        }
        const int c = __popcll(__ballot(in));
        if (in) {
            list[rank] = tid;
            wl[rank] = wt;
        }
        if (tid == 0) count = c;
    }
    __syncthreads();
    const int c = count;
    for (int r = 4 * (blockIdx.y * kThreads + tid); r < H; r += 4 * kThreads * gridDim.y) {
        const int64_t o = t * H + r;
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
        if (accumulate) acc = *(const v4f*)(out + o);
        for (int i = 0; i < c; ++i) {
            const float* yp = y + (t * width + list[i]) * H + r;
            v4f v = *(const v4f*)yp;
            for (int p = 1; p < parts; ++p) v += *(const v4f*)(yp + (int64_t)p * n * H);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(wl[i], v[j], acc[j]);
        }
        if (res) {
            const uint2 x = *(const uint2*)(res + o);
            uint2 z;
            z.x = naiwa_f32_to_bf16(naiwa_bf16_to_f32(x.x & 0xffffu) + acc[0]) |
                  naiwa_f32_to_bf16(naiwa_bf16_to_f32(x.x >> 16) + acc[1]) << 16;
            z.y = naiwa_f32_to_bf16(naiwa_bf16_to_f32(x.y & 0xffffu) + acc[2]) |
                  naiwa_f32_to_bf16(naiwa_bf16_to_f32(x.y >> 16) + acc[3]) << 16;
            *(uint2*)(res + o) = z;
        }
        if (out) *(v4f*)(out + o) = acc;
    }
}

bool bank_ok(const naiwa_bank* b) {
    if (!b || !b->base || b->slots <= 0 || b->n <= 0 || b->k <= 0) return false;
    const int64_t bytes = naiwa_projection_bytes(NAIWA_MXFP4_T, b->n, b->k);
    return bytes > 0 && b->slot_stride >= bytes && !(((uintptr_t)b->base | (uintptr_t)b->slot_stride) & 15);
}

// K parts of the down projection.
int down_parts(int64_t n, int H, int I) {
    (void)n, (void)H, (void)I;
    return 1;
}

struct Layout {
    size_t offsets, perm, bad, tiles, x, xs, h, hs, y, total;
    int64_t max_tiles;
    int parts;
    Layout(int64_t rows, int width, int H, int I) {
        auto a256 = [](size_t b) { return (b + 255) & ~size_t(255); };
        const size_t n = (size_t)rows * width;
        parts = down_parts(rows * width, H, I);
        offsets = 0;
        perm = a256(offsets + (size_t)(NAIWA_SEG_MAX_KEYS + 1) * 4);
        bad = a256(perm + n * 4);
        tiles = a256(bad + 4);
        max_tiles = (int64_t)n / kTile + std::min<int64_t>((int64_t)n, NAIWA_SEG_MAX_KEYS);
        x = a256(tiles + (size_t)(3 * max_tiles + 1) * 4);
        xs = a256(x + (size_t)rows * plane_row(4, H));
        h = a256(xs + (size_t)rows * naiwa_mx_groups(H) * 16);
        hs = a256(h + n * plane_row(4, I));
        y = a256(hs + n * naiwa_mx_groups(I) * 16);
        total = a256(y + (size_t)parts * n * H * 4);
    }
};


} // namespace

// Whether a call takes tiles of up to 64 pairs (mxfp4_tiles.h) rather than passes of 16.
extern "C" int naiwa_mx_tiled(int64_t n, int slots) { return n > (int64_t)16 * slots; }

int naiwa_mx_check(const NaiwaMxCall& c) {
    if (!c.gate || !c.up || !c.down) return NAIWA_E_INVALID;
    if (c.gate->dtype != NAIWA_MXFP4_T || c.up->dtype != NAIWA_MXFP4_T || c.down->dtype != NAIWA_MXFP4_T)
        return NAIWA_E_UNSUPPORTED;
    if (c.rows < 0 || c.width < 0 || (int64_t)c.rows * c.width > 65536) return NAIWA_E_INVALID;
    if (!bank_ok(c.gate) || !bank_ok(c.up) || !bank_ok(c.down)) return NAIWA_E_INVALID;
    const int H = c.gate->k, I = c.gate->n;
    if (c.up->k != H || c.up->n != I || c.down->k != I || c.down->n != H) return NAIWA_E_INVALID;
    if (c.gate->slots != c.up->slots || c.gate->slots != c.down->slots) return NAIWA_E_INVALID;
    if (H % 32 || I % 32) return NAIWA_E_INVALID;
    if (c.gate->slots > NAIWA_SEG_MAX_KEYS || c.width > kMaxWidth) return NAIWA_E_UNSUPPORTED;
    if (c.x_dtype != NAIWA_BF16 && c.x_dtype != NAIWA_F32) return NAIWA_E_UNSUPPORTED;
    if (c.act != NAIWA_ACT_SILU && c.act != NAIWA_ACT_GELU_PYTORCH_TANH) return NAIWA_E_UNSUPPORTED;
    if (c.rows > 0 && (!c.x || !(c.out || c.res) || (c.width > 0 && (!c.ids || !c.w)))) return NAIWA_E_INVALID;
    if (((uintptr_t)c.x | (uintptr_t)c.out) & 15) return NAIWA_E_INVALID;
    return NAIWA_OK;
}

size_t naiwa_mx_scratch_bytes(int rows, int width, int H, int I) {
    return rows == 0 || width == 0 ? 0 : Layout(rows, width, H, I).total;
}

int naiwa_mx_run(const NaiwaMxCall& c, uint8_t* ws, hipStream_t st) {
    if (c.rows == 0) return NAIWA_OK;
    const int H = c.gate->k, I = c.gate->n, slots = c.gate->slots, n = c.rows * c.width;
    const unsigned cs = (unsigned)((H + 4 * kThreads - 1) / (4 * kThreads));
    if (n == 0) {
        combine_kernel<<<dim3(c.rows, cs), kThreads, 0, st>>>(nullptr, 0, 1, c.ids, c.w, 0, slots, H, c.skip_zero,
                                                             c.accumulate, c.out, c.res);
        return naiwa_hip_rc(hipGetLastError());
    }
    const int P = c.skip_zero ? 4 : 3; // a prompt chunk's x in 3 planes
    const Layout L(c.rows, c.width, H, I);
    uint32_t* offsets = (uint32_t*)(ws + L.offsets);
    uint32_t* perm = (uint32_t*)(ws + L.perm);
    float* y = (float*)(ws + L.y);
    const Planes xp{ws + L.x, ws + L.xs, plane_row(P, H), naiwa_mx_groups(H)};
    const Planes hp{ws + L.h, ws + L.hs, plane_row(4, I), naiwa_mx_groups(I)};
    const Bank g{(const uint8_t*)c.gate->base, c.gate->slot_stride, naiwa_mx_strip_bytes(H)};
    const Bank u{(const uint8_t*)c.up->base, c.up->slot_stride, naiwa_mx_strip_bytes(H)};
    const Bank d{(const uint8_t*)c.down->base, c.down->slot_stride, naiwa_mx_strip_bytes(I)};
    const int64_t xb = (int64_t)c.rows * 4 * naiwa_mx_steps(H);
    const unsigned pb = (unsigned)((xb + kThreads - 1) / kThreads);
    const bool tiled = naiwa_mx_tiled(n, slots) && (uint64_t)c.rows * xp.row <= UINT32_MAX; // the copies' offsets have 32 bits
    Tiles tl{nullptr, nullptr, nullptr, nullptr};
    if (tiled) {
        tl.start = (int*)(ws + L.tiles);
        tl.count = tl.start + L.max_tiles;
        tl.slot = tl.count + L.max_tiles;
        tl.n = tl.slot + L.max_tiles;
        // pairs of weight 0 are sorted in with the others and left out by the combine
        if (int rc = naiwa_moe_gather(c.ids, n, slots, perm, offsets, (int*)(ws + L.bad), (int64_t)st)) return rc;
    } else {
        segments_kernel<<<1, NAIWA_SEG_THREADS, 0, st>>>(c.ids, c.skip_zero ? c.w : nullptr, n, slots, perm, offsets,
                                                         (int*)(ws + L.bad));
    }
    const unsigned px = pb + (tiled ? 1 : 0);
    if (P == 3)
        planes_kernel<3, true><<<px, kThreads, 0, st>>>(c.x, c.rows, H, xp, offsets, slots, tl);
    else if (c.x_dtype == NAIWA_BF16)
        planes_kernel<4, true><<<px, kThreads, 0, st>>>(c.x, c.rows, H, xp, offsets, slots, tl);
    else
        planes_kernel<4, false><<<px, kThreads, 0, st>>>(c.x, c.rows, H, xp, offsets, slots, tl);
    if (tiled) {
        constexpr int NA = 4;
        const int64_t most = n / kTile + std::min(n, slots);
        const unsigned t8 = (unsigned)((most + 7) / 8 * 8);
        const int xcd = n <= (int64_t)128 * slots ? 1 : 0;
        const unsigned b1 = t8 * ((4 * naiwa_mx_steps(I) + 2 * NA - 1) / (2 * NA)), b2 = t8 * ((H / 32 + 4 * NA - 1) / (4 * NA));
        if (P == 3)
            tile_gateup_kernel<NA, 3><<<b1, kThreads, 2 * sizeof(Stage<3>), st>>>(g, u, xp, H, I, c.width, perm, tl, c.act,
                                                                                  xcd, hp);
        else
            tile_gateup_kernel<NA, 4><<<b1, kThreads, 2 * sizeof(Stage<4>), st>>>(g, u, xp, H, I, c.width, perm, tl, c.act,
                                                                                  xcd, hp);
        tile_down_kernel<NA><<<b2, kThreads, 2 * sizeof(Stage<4>), st>>>(d, hp, H, I, perm, tl, xcd, y);
    } else {
        const dim3 gg(slots, 4 * naiwa_mx_steps(I)), gd(slots, (H + 63) / 64, L.parts);
        if (P == 3)
            gateup_kernel<3><<<gg, kThreads, 0, st>>>(g, u, xp, H, I, c.width, offsets, perm, c.act, hp);
        else
            gateup_kernel<4><<<gg, kThreads, 0, st>>>(g, u, xp, H, I, c.width, offsets, perm, c.act, hp);
        down_kernel<<<gd, kThreads, 0, st>>>(d, hp, H, I, n, L.parts, offsets, perm, y);
    }
    combine_kernel<<<dim3(c.rows, cs), kThreads, 0, st>>>(y, n, L.parts, c.ids, c.w, c.width, slots, H, c.skip_zero,
                                                          c.accumulate, c.out, c.res);
    return naiwa_hip_rc(hipGetLastError());
}
