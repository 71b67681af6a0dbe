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
//   3 planes (x of a prompt chunk, bf16): 2^-14 M; a value of at least 2^-7 M exactly;
//   4 planes (h of a prompt chunk, bf16 x of a decode step): 2^-19 M; a bf16 value of at least
//     2^-12 M exactly;
//   5 planes (h and f32 x of a decode step, which HBM bounds): 2^-24 M, an f32's own rounding.
// FP4 x E2M3 runs at twice the rate of FP4 x FP8 and of bf16 per step (5.4 against 3.4
// PFLOP/s measured), and its sums are exact up to the f32 accumulator's rounding; with e4m3
// the matrix cores drop products under about 2^-15 of a step's largest (5e-5 of a sum of
// codes of all magnitudes).  A block with a NaN or an infinity gets the scale byte 255,
// which makes its products NaN.
//
// Launches, stream-ordered:
//   1. x laid out in planes, one row per token, and in a block beside it the (token, expert)
//      pairs sorted by slot (calls of many pairs: sorted by a launch of their own);
//   2. gate/up: a block per (slot segment, 32 features): 16 tokens a pass, the steps of K
//      dealt to its waves, whose partial sums meet in LDS; h = act(g) u in planes;
//   3. down: a block per (slot segment, 64 rows, K part); unweighted dots per pair;
//   4. combine: out[t] = the weighted sum over t's pairs in ascending slot order.
// One token: 2. takes x itself and a block per pair, 3. and 4. are one launch (down_one_kernel).
// Many tokens an expert: 2. and 3. by tiles of 64 pairs (mxfp4_tiles.h).
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
// [2, 4) times 2^(s - 127).  At least 24, so that the planes' scales stay normal.
__device__ __forceinline__ int scale_byte(uint32_t m) {
    const int e = (int)(m >> 23);
    return e == 255 ? 255 : max(24, e - 1);
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

// The pairs of a call by slot: sorted (perm) with a list of the slots that have pairs (key,
// begin, their number) or, with key null, every slot's range (begin: slots + 1 offsets); or, with
// ids, every pair as it is, a segment of its own.
struct Segments {
    const uint32_t *key, *begin, *perm;
    const int* count;
    const uint32_t* ids;
    const float* w; // null: pairs of weight 0 count
    int slots;
    // Segment i of a grid with one for each: false if there is none.
    __device__ __forceinline__ bool at(int i, int* slot, int* b, int* e) const {
        if (ids) {
            *slot = __builtin_amdgcn_readfirstlane((int)ids[i]);
            *b = i;
            *e = i + 1;
            return (uint32_t)*slot < (uint32_t)slots && !(w && w[i] == 0.0f);
        }
        // the loads go out together; past the list they read what nobody uses
        const int c = key ? *count : i + 1, k = key ? (int)key[i] : i, b0 = (int)begin[i], e0 = (int)begin[i + 1];
        *slot = __builtin_amdgcn_readfirstlane(k);
        *b = __builtin_amdgcn_readfirstlane(b0);
        *e = __builtin_amdgcn_readfirstlane(e0);
        return i < __builtin_amdgcn_readfirstlane(c) && *b < *e;
    }
    __device__ __forceinline__ uint32_t pair(int64_t pos) const { return ids ? (uint32_t)pos : perm[pos]; }
};

// Operands in the 8 registers that the product's builtin takes; FP4 uses 4 of them, E2M3 6.
__device__ __forceinline__ v8i fp4_operand(v4u v) {
    return __builtin_bit_cast(v8i, __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1));
}
__device__ __forceinline__ v8i e2m3_operand(v6u v) {
    return __builtin_bit_cast(v8i, __builtin_shufflevector(v, v, 0, 1, 2, 3, 4, 5, -1, -1));
}

// Block kb of a row of x (zeros past H).
template <bool BF16> __device__ __forceinline__ void load_block(const void* x, int64_t row, int H, int kb, float (&f)[32]) {
    if (32 * kb >= H) {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = 0.0f;
    } else if constexpr (BF16) {
        const v4u* src = (const v4u*)((const uint16_t*)x + row + 32 * kb);
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
        const v4f* src = (const v4f*)((const float*)x + row + 32 * kb);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const v4f v = src[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[4 * i + j] = v[j];
        }
    }
}

// A block's planes to a row of them.
template <int P> __device__ __forceinline__ void put_block(uint8_t* row, uint8_t* scales, int kb, const v6u (&o)[P], int s) {
    uint8_t* dst = row + (int64_t)(kb >> 2) * 96 * P;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        *(v4u*)(dst + head_at(P, kb & 3, p)) = v4u{o[p][0], o[p][1], o[p][2], o[p][3]};
        *(v2u*)(dst + tail_at(P, kb & 3, p)) = v2u{o[p][4], o[p][5]};
    }
    scales[scale_at(kb)] = (uint8_t)s;
}

#include "mxfp4_tiles.h"

// What a launch's last block does beside the planes, which do not depend on it.
enum { kPlanesOnly, kWithTiles, kWithSegments };
struct Beside {
    const uint32_t* offsets; // kWithTiles
    Tiles tiles;
    const uint32_t* ids; // kWithSegments
    const float* w;
    int n;
    uint32_t *perm, *key, *begin;
    int *count, *bad;
    int slots;
};

// x [rows, H] in P planes, a block of 32 values a thread; the blocks that pad H to whole
// steps are zeros.  Bound: HBM, and latency where rows are few.
template <int P, bool BF16, int MODE>
__global__ void __launch_bounds__(kThreads) planes_kernel(const void* x, int64_t rows, int H, Planes out, Beside with) {
    if (MODE != kPlanesOnly && blockIdx.x == gridDim.x - 1) {
        if constexpr (MODE == kWithTiles) {
            tiles_block(with.offsets, with.slots, with.tiles);
        } else if constexpr (MODE == kWithSegments) {
            __shared__ NaiwaSegSmem sm;
            naiwa_segment(sm, with.ids, with.w, with.n, with.slots, with.perm, nullptr, with.count, with.key, with.begin,
                          with.bad);
        }
        return;
    }
    const int blocks = 4 * naiwa_mx_steps(H);
    const int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (b >= rows * blocks) return;
    const int64_t t = b / blocks;
    const int kb = (int)(b % blocks);
    float f[32];
    load_block<BF16>(x, t * H, H, kb, f);
    const int s = scale_byte(abs_max(f));
    v6u o[P];
    to_planes<P>(f, s, o);
    put_block<P>(out.base + t * out.row, out.scales + t * out.groups * 16, kb, o, s);
}

// Plane p of block b of the step at `at`.
template <int P> __device__ __forceinline__ v6u load_plane(const uint8_t* at, int b, int p) {
    const v4u h = *(const v4u*)(at + head_at(P, b, p));
    const v2u t = *(const v2u*)(at + tail_at(P, b, p));
    return v6u{h.x, h.y, h.z, h.w, t.x, t.y};
}

// acc += strip rows x planes over steps [t0, t1): S strips of 16 rows, one token row of
// planes a lane.  wp[i]: strip i's first byte; xp: the lane's token row; xs: the row's scales.  Weights are loaded three steps ahead and planes one, so that a wave keeps
// 3 S KB of weights in flight.
template <int S, int P>
__device__ __forceinline__ void strips_dot(const uint8_t* const (&wp)[S], const uint8_t* xp, const uint8_t* xs, int steps,
                                           int t0, int t1, int lane, v4f (&acc)[S]) {
    if (t0 >= t1) return;
    const int kb = lane >> 4;
    struct A {
        v4u v[S];
        uint32_t s[S];
    } a[4];
    struct B {
        v6u v[P];
        uint32_t s;
    } b[2];
    auto load_a = [&](int t, A& o) {
        t = min(t, t1 - 1);
        const int g = t >> 2;
        const int64_t at = (int64_t)1024 * t + 256 * g;
        const int64_t sc = (int64_t)1024 * min(4 * g + 4, steps) + 256 * g;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            o.v[i] = *(const v4u*)(wp[i] + at + 16u * lane);
            o.s[i] = *(const uint32_t*)(wp[i] + sc + 4u * lane) >> (8 * (t & 3));
        }
    };
    auto load_b = [&](int t, B& o) {
        t = min(t, t1 - 1);
#pragma unroll
        for (int p = 0; p < P; ++p) o.v[p] = load_plane<P>(xp + (int64_t)(96 * P) * t, kb, p);
        o.s = *(const uint32_t*)(xs + 16 * (t >> 2) + 4 * kb) >> (8 * (t & 3)) & 255u;
    };
#pragma unroll
    for (int j = 0; j < 3; ++j) load_a(t0 + j, a[j]);
    load_b(t0, b[0]);
    for (int t = t0; t < t1; t += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (t + j >= t1) break;
            load_b(t + j + 1, b[(j + 1) & 1]);
            load_a(t + j + 3, a[(j + 3) & 3]);
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        fp4_operand(a[j].v[i]), e2m3_operand(b[j & 1].v[p]), acc[i], 4, 2, 0, (int)a[j].s[i], 0, (int)(b[j & 1].s - 5 * p));
        }
    }
    // the sums stay where every lane computes them
#pragma unroll
    for (int i = 0; i < S; ++i) asm volatile("" : "+v"(acc[i]));
}

// The same for one token whose planes are in LDS (xp, xs: the row, the same for every lane):
// rounds of U steps, all their weights in flight; `before` runs once the first round's are.
template <int S, int P, class F>
__device__ __forceinline__ void strips_dot_one(const uint8_t* const (&wp)[S], const uint8_t* xp, const uint8_t* xs, int steps,
                                               int t0, int t1, int lane, v4f (&acc)[S], F before) {
    constexpr int U = 16 / S < 8 ? 16 / S : 8;
    const int kb = lane >> 4;
    v4u a[U][S];
    uint32_t as[U][S];
    auto load = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int tt = min(t + u, t1 - 1), g = tt >> 2;
            const int64_t at = (int64_t)1024 * tt + 256 * g;
            const int64_t sc = (int64_t)1024 * min(4 * g + 4, steps) + 256 * g;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                a[u][i] = *(const v4u*)(wp[i] + at + 16u * lane);
                as[u][i] = *(const uint32_t*)(wp[i] + sc + 4u * lane) >> (8 * (tt & 3));
            }
        }
    };
    if (t0 < t1) load(t0);
    before();
    // what `before` wrote to LDS is read by other lanes of the wave
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int t = t0; t < t1; t += U) {
        if (t > t0) load(t);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u >= t1) break;
            const uint32_t bs = *(const uint32_t*)(xs + 16 * ((t + u) >> 2) + 4 * kb) >> (8 * ((t + u) & 3)) & 255u;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const v8i b = e2m3_operand(load_plane<P>(xp + (int64_t)(96 * P) * (t + u), kb, p));
#pragma unroll
                for (int i = 0; i < S; ++i)
                    acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(a[u][i]), b, acc[i], 4, 2, 0,
                                                                             (int)as[u][i], 0, (int)(bs - 5 * p));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) asm volatile("" : "+v"(acc[i]));
}

// A wave's steps of `steps` dealt to `all` waves.
__device__ __forceinline__ void deal(int steps, int mine, int all, int* t0, int* t1) {
    *t0 = (int)((int64_t)steps * mine / all);
    *t1 = (int)((int64_t)steps * (mine + 1) / all);
}

// The sums of a block's NW waves over 4 strips of 16 rows and 16 tokens.  Lane l of a wave holds
// D[4 (l / 16) + i][l % 16]: row 4 (l / 16) + i of a strip, token l % 16; a group of 4 rows is
// padded by a token, so that reads down the rows of a token spread over the banks.
template <int NW> struct Sums {
    v4f v[NW][4][4][17];
    __device__ __forceinline__ void put(int wave, int lane, const v4f (&acc)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[wave][i][lane >> 4][lane & 15] = acc[i];
    }
    __device__ __forceinline__ float row(int strip, int r, int tok) const {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) o += v[w][strip][r >> 2][tok][r & 3];
        return o;
    }
    __device__ __forceinline__ v4f rows4(int strip, int lane) const {
        v4f o = v[0][strip][lane >> 4][lane & 15];
#pragma unroll
        for (int w = 1; w < NW; ++w) o += v[w][strip][lane >> 4][lane & 15];
        return o;
    }
};

// h of 32 features (strips 0, 1 of the sums: gate, 2, 3: up) and one token, a feature a lane of
// 32, to row `row` of the planes as block fb.  Bits of E2M3 by hand: |y| <= 4 is a multiple of 1/8
// under 2 and of 1/4 from there on, so adding 1.5 2^20 or 1.5 2^21 rounds it to nearest even, and
// the low bits of that sum are the code (less 8 in the upper binade).
template <int PH, int NW>
__device__ __forceinline__ void put_h(const Sums<NW>& sums, int tok, bool pad, int act, int fb, int64_t row, const Planes& h) {
    const int f = threadIdx.x & 31;
    const float g = sums.row(f >> 4, f & 15, tok), u = sums.row(2 + (f >> 4), f & 15, tok);
    const float v = pad ? 0.0f : naiwa_act(act, g) * u;
    uint32_t m = __float_as_uint(v) & 0x7fffffffu;
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, false));
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    const int s = scale_byte(m);
    float y = s == 255 ? 0.0f : v * __uint_as_float((uint32_t)(254 - s) << 23);
    uint32_t word[PH]; // a lane's word of each plane: see below
#pragma unroll
    for (int p = 0; p < PH; ++p) {
        const float a = fabsf(y);
        const bool big = a >= 2.0f;
        const float c = big ? 0x1.8p21f : 0x1.8p20f, t = a + c;
        uint32_t code = __float_as_uint(t) - __float_as_uint(c) + (big ? 8u : 0u);
        code |= (__float_as_uint(y) >> 26) & 32u;
        y = __uint_as_float(__float_as_uint((a - (t - c)) * 32.0f) ^ (__float_as_uint(y) & 0x80000000u));
        // 4 lanes' codes are 24 bits, 16 lanes' 3 words: the first 3 quads make one each with their
        // neighbour's bits
        uint32_t q = code << (6 * (f & 3));
        q |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)q, 0xB1, 0xF, 0xF, false);
        q |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)q, 0x4E, 0xF, 0xF, false);
        const uint32_t next = (uint32_t)__shfl_down((int)q, 4, 64);
        const int j = (f >> 2) & 3;
        word[p] = (q >> (8 * j)) | (next << (24 - 8 * j));
    }
    uint8_t* dst = h.base + row * h.row + (int64_t)(fb >> 2) * 96 * PH;
    const int j = (f >> 2) & 3, d = 3 * (f >> 4) + j; // the block's word d of 6
    auto store = [&](int p, uint32_t v) {
        *(uint32_t*)(dst + (d < 4 ? head_at(PH, fb & 3, p) + 4 * d : tail_at(PH, fb & 3, p) + 4 * (d - 4))) = v;
    };
    // lane f % 4 of a quad stores plane f % 4
    uint32_t mine = word[0];
#pragma unroll
    for (int p = 1; p < 4; ++p) mine = (f & 3) == p ? word[p] : mine;
    if (j < 3) store(f & 3, mine);
    if (PH == 5 && j < 3 && (f & 3) == 0) store(4, word[PH - 1]);
    if (f == 0) h.scales[row * h.groups * 16 + scale_at(fb)] = (uint8_t)s;
}

// Gate/up of one slot segment and 32 features; blocks past I (h padded to whole steps) write zeros.
template <int PX, int PH>
__global__ void __launch_bounds__(kThreads, 2)
gateup_kernel(Bank gate, Bank up, Planes x, int H, int I, int width, Segments seg, int act, Planes h) {
    __shared__ Sums<kWaves> sums;
    const int fb = blockIdx.y;
    int s, b, e, t0, t1;
    if (!seg.at(blockIdx.x, &s, &b, &e)) return;
    const int lane = threadIdx.x & 63, steps = naiwa_mx_steps(H);
    deal(steps, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kWaves, &t0, &t1);
    const bool pad = 32 * fb >= I;
    const uint8_t* g = gate.base + (int64_t)s * gate.stride + 2 * fb * gate.strip;
    const uint8_t* u = up.base + (int64_t)s * up.stride + 2 * fb * up.strip;
    for (int c0 = b; c0 < e; c0 += 16) {
        v4f acc[4] = {};
        if (!pad) {
            const uint8_t* const wp[4] = {g, g + gate.strip, u, u + up.strip};
            const int64_t row = seg.pair(min(c0 + (lane & 15), e - 1)) / (uint32_t)width;
            strips_dot<4, PX>(wp, x.base + row * x.row, x.scales + row * x.groups * 16, steps, t0, t1, lane, acc);
        }
        sums.put(threadIdx.x >> 6, lane, acc);
        __syncthreads();
        for (int t = threadIdx.x >> 5; t < min(16, e - c0); t += kThreads / 32) put_h<PH>(sums, t, pad, act, fb, c0 + t, h);
        __syncthreads();
    }
}

// The same for one token: a block per (pair, 32 features), no segments; each wave lays out
// its own steps of x in LDS while its first weights are on the way.  Pair j is row j of h.
// Dynamic LDS: the planes of x (96 PX bytes a step) and their scales (16 a group).
template <int PX, int PH, bool BF16>
__global__ void __launch_bounds__(kThreads, 2)
gateup_one_kernel(Bank gate, Bank up, const void* x, int H, int I, const uint32_t* ids, const float* w, int slots,
                  int skip_zero, int act, Planes h) {
    extern __shared__ __align__(16) uint8_t xl[];
    __shared__ Sums<kWaves> sums;
    const int j = blockIdx.x, fb = blockIdx.y;
    const uint32_t s = (uint32_t)uniform((int)ids[j]);
    if (s >= (uint32_t)slots || (skip_zero && w[j] == 0.0f)) return;
    const int lane = threadIdx.x & 63, steps = naiwa_mx_steps(H);
    int t0, t1;
    deal(steps, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kWaves, &t0, &t1);
    const bool pad = 32 * fb >= I;
    v4f acc[4] = {};
    if (!pad) {
        const uint8_t* g = gate.base + (int64_t)s * gate.stride + 2 * fb * gate.strip;
        const uint8_t* u = up.base + (int64_t)s * up.stride + 2 * fb * up.strip;
        const uint8_t* const wp[4] = {g, g + gate.strip, u, u + up.strip};
        uint8_t* scales = xl + (size_t)steps * 96 * PX;
        auto stage = [&] {
            for (int kb = 4 * t0 + lane; kb < 4 * t1; kb += 64) {
                float f[32];
                load_block<BF16>(x, 0, H, kb, f);
                const int sb = scale_byte(abs_max(f));
                v6u o[PX];
                to_planes<PX>(f, sb, o);
                put_block<PX>(xl, scales, kb, o, sb);
            }
        };
        strips_dot_one<4, PX>(wp, xl, scales, steps, t0, t1, lane, acc, stage);
    }
    sums.put(threadIdx.x >> 6, lane, acc);
    __syncthreads();
    if (threadIdx.x < 32) put_h<PH>(sums, 0, pad, act, fb, j, h);
}

// Down of one slot segment, 64 rows and one K part: y[part][pair][H] unweighted.
template <int PH>
__global__ void __launch_bounds__(kThreads, 2)
down_kernel(Bank down, Planes h, int H, int I, int64_t n, int parts, Segments seg, float* y) {
    __shared__ v4f red[kWaves][4][64];
    const int rb = blockIdx.y, part = blockIdx.z;
    int s, b, e, t0, t1;
    if (!seg.at(blockIdx.x, &s, &b, &e)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = naiwa_mx_steps(I), strips = min(4, H / 16 - 4 * rb);
    deal(steps, part * kWaves + wave, parts * kWaves, &t0, &t1);
    const uint8_t* base = down.base + (int64_t)s * down.stride + 4 * rb * down.strip;
    for (int c0 = b; c0 < e; c0 += 16) {
        v4f acc[4] = {};
        const int64_t pos = min(c0 + (lane & 15), e - 1);
        // strips past H read the last one again
        const uint8_t* const wp[4] = {base, base + down.strip, base + min(2, strips - 1) * down.strip,
                                      base + min(3, strips - 1) * down.strip};
        strips_dot<4, PH>(wp, h.base + pos * h.row, h.scales + pos * h.groups * 16, steps, t0, t1, lane, acc);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][i][lane] = acc[i];
        __syncthreads();
        v4f v = red[0][wave][lane]; // wave i adds strip i
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += red[w][wave][lane];
        if (wave < strips && c0 + (lane & 15) < e)
            *(v4f*)(y + ((int64_t)part * n + seg.pair(pos)) * H + 64 * rb + 16 * wave + 4 * (lane >> 4)) = v;
    }
}

// ---------------------------------------------------------------------------
// Streams: the same products with the activations held in registers
// ---------------------------------------------------------------------------
// A block of 8 waves takes up to 16 tokens of a slot segment (several blocks share a longer
// one) and a run of feature blocks (or of 64 rows).  The
// steps of K (at most 8 NS of them) are dealt to the waves, and a wave keeps its NS steps of
// up to 16 tokens' planes in registers and streams the run's weights past them: the weights
// of the next feature block are under way from the moment the present ones are used, through
// the exchange of the waves' sums in LDS and the epilogue, which the waves take in turn.
constexpr int kStreamWaves = 8, kStreamThreads = 64 * kStreamWaves;

// One wave's share of 4 strips: NS steps of weights and of planes.
template <int NS, int P> struct Streamed {
    v6u b[NS][P];
    uint32_t bs;
    v4u a[NS][4];
    uint32_t as[4];

    // The scale bytes of steps t0 .. t0 + NS - 1 from the words of their groups, `next` bytes
    // apart: NS = 3 alone has runs that go past a group.
    static __device__ __forceinline__ uint32_t scales_of(const uint8_t* p, int64_t next, bool past, int t0) {
        const uint32_t lo = *(const uint32_t*)p;
        if constexpr (NS != 3) return lo >> (8 * (t0 & 3));
        return __builtin_amdgcn_alignbyte(past ? *(const uint32_t*)(p + next) : 0u, lo, (uint32_t)(t0 & 3));
    }
    // Steps t0 .. t0 + NS - 1, those below `end`.
    __device__ __forceinline__ void load_b(const uint8_t* row, const uint8_t* scales, int t0, int end, int lane) {
        const int kb = lane >> 4;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int t = min(t0 + i, end - 1);
#pragma unroll
            for (int p = 0; p < P; ++p) b[i][p] = load_plane<P>(row + (int64_t)(96 * P) * t, kb, p);
        }
        bs = scales_of(scales + 16 * (t0 >> 2) + 4 * kb, 16, end > 4 * (t0 >> 2) + 4, t0);
    }
    __device__ __forceinline__ void load_a(const uint8_t* const (&wp)[4], int i, int t0, int end, int lane) {
        const int t = min(t0 + i, end - 1);
        const int64_t at = (int64_t)1024 * t + 256 * (t >> 2);
#pragma unroll
        for (int s = 0; s < 4; ++s) a[i][s] = *(const v4u*)(wp[s] + at + 16u * lane);
    }
    __device__ __forceinline__ void load_as(const uint8_t* const (&wp)[4], int t0, int steps, int lane) {
        const int g = t0 >> 2;
        const int64_t sc = (int64_t)1024 * min(4 * g + 4, steps) + 256 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s)
            as[s] = scales_of(wp[s] + sc + 4u * lane, 1024 * (min(4 * g + 8, steps) - (4 * g + 4)) + 256, steps > 4 * g + 4, t0);
    }
    __device__ __forceinline__ void dot(int i, v4f (&acc)[4]) const {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int p = 0; p < P; ++p)
                acc[s] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    fp4_operand(a[i][s]), e2m3_operand(b[i][p]), acc[s], 4, 2, 0, (int)(as[s] >> (8 * i)), 0,
                    (int)((bs >> (8 * i) & 255u) - 5 * p));
    }
};

// The run of item x of `items` dealt to `splits` blocks.
__device__ __forceinline__ void run_of(int items, int split, int splits, int* i0, int* i1) {
    *i0 = (int)((int64_t)items * split / splits);
    *i1 = (int)((int64_t)items * (split + 1) / splits);
}

// Gate/up of a slot segment and a run of blocks of 32 features.
template <int NS, int PX, int PH>
__global__ void __launch_bounds__(kStreamThreads, NS == 1 ? 4 : 2)
gateup_stream_kernel(Bank gate, Bank up, Planes x, int H, int I, int width, Segments seg, int act, Planes h) {
    __shared__ Sums<kStreamWaves> sums;
    int s, b, e, f0, f1;
    if (!seg.at(blockIdx.x, &s, &b, &e)) return;
    run_of(4 * naiwa_mx_steps(I), blockIdx.y, gridDim.y, &f0, &f1);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tok = lane & 15;
    const int steps = naiwa_mx_steps(H), t0 = wave * NS;
    const uint8_t* g0 = gate.base + (int64_t)s * gate.stride;
    const uint8_t* u0 = up.base + (int64_t)s * up.stride;
    Streamed<NS, PX> w;
    for (int c0 = b + 16 * blockIdx.z; c0 < e; c0 += 16 * gridDim.z) {
        const int ntok = min(16, e - c0);
        auto strips = [&](int fb, const uint8_t*(&wp)[4]) {
            fb = min(fb, I / 32 - 1); // past I: the last one again
            wp[0] = g0 + 2 * fb * gate.strip;
            wp[1] = wp[0] + gate.strip;
            wp[2] = u0 + 2 * fb * up.strip;
            wp[3] = wp[2] + up.strip;
        };
        if (t0 < steps) {
            const uint8_t* wp[4];
            strips(f0, wp);
#pragma unroll
            for (int i = 0; i < NS; ++i) w.load_a(wp, i, t0, steps, lane);
            w.load_as(wp, t0, steps, lane);
            const int64_t row = seg.perm[c0 + min(tok, ntok - 1)] / (uint32_t)width;
            w.load_b(x.base + row * x.row, x.scales + row * x.groups * 16, t0, steps, lane);
        }
        for (int fb = f0; fb < f1; ++fb) {
            v4f acc[4] = {};
            if (t0 < steps) {
                const uint8_t* wp[4];
                strips(fb + 1 < f1 ? fb + 1 : fb, wp);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    if (t0 + i < steps) w.dot(i, acc);
                    w.load_a(wp, i, t0, steps, lane);
                }
                w.load_as(wp, t0, steps, lane);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(acc[i]));
            sums.put(wave, lane, acc);
            lds_barrier();
            if (const int t = threadIdx.x >> 5; t < ntok) put_h<PH>(sums, t, 32 * fb >= I, act, fb, c0 + t, h);
            lds_barrier();
        }
    }
}

// Down of a slot segment, a run of blocks of 64 rows and a K part of `part_steps` steps.
template <int NS, int PH>
__global__ void __launch_bounds__(kStreamThreads, NS == 1 ? 4 : 2)
down_stream_kernel(Bank down, Planes h, int H, int I, int64_t n, int part_steps, int passes, Segments seg, float* y) {
    __shared__ Sums<kStreamWaves> sums;
    int s, b, e, r0, r1;
    if (!seg.at(blockIdx.x, &s, &b, &e)) return;
    const int blocks = (H + 63) / 64, part = blockIdx.z / passes;
    run_of(blocks, blockIdx.y, gridDim.y, &r0, &r1);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tok = lane & 15;
    const int steps = naiwa_mx_steps(I), t0 = part * part_steps + wave * NS, end = min(steps, (part + 1) * part_steps);
    const uint8_t* base = down.base + (int64_t)s * down.stride;
    Streamed<NS, PH> w;
    for (int c0 = b + 16 * (blockIdx.z % passes); c0 < e; c0 += 16 * passes) {
        const int ntok = min(16, e - c0);
        auto strips = [&](int rb, const uint8_t*(&wp)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) wp[i] = base + min(4 * rb + i, H / 16 - 1) * down.strip; // past H: the last one again
        };
        const int64_t pos = c0 + min(tok, ntok - 1);
        if (t0 < end) {
            const uint8_t* wp[4];
            strips(r0, wp);
#pragma unroll
            for (int i = 0; i < NS; ++i) w.load_a(wp, i, t0, end, lane);
            w.load_as(wp, t0, steps, lane);
            w.load_b(h.base + pos * h.row, h.scales + pos * h.groups * 16, t0, end, lane);
        }
        const int64_t pair = seg.pair(pos);
        for (int rb = r0; rb < r1; ++rb) {
            v4f acc[4] = {};
            if (t0 < end) {
                const uint8_t* wp[4];
                strips(rb + 1 < r1 ? rb + 1 : rb, wp);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    if (t0 + i < end) w.dot(i, acc);
                    w.load_a(wp, i, t0, end, lane);
                }
                w.load_as(wp, t0, steps, lane);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(acc[i]));
            sums.put(wave, lane, acc);
            lds_barrier();
            // waves 0-3 and 4-7 in turn: a strip a wave
            const int strip = wave & 3;
            if ((wave >> 2) == ((rb - r0) & 1) && 4 * rb + strip < H / 16 && tok < ntok)
                *(v4f*)(y + ((int64_t)part * n + pair) * H + 64 * rb + 16 * strip + 4 * (lane >> 4)) = sums.rows4(strip, lane);
            lds_barrier();
        }
    }
}

// A token's pairs that count, in ascending slot order (pair j before j' of the same slot, j < j').
struct Order {
    int list[kMaxWidth];
    float w[kMaxWidth];
    int count;
    // By the first wave of a block; a barrier has to follow.
    __device__ __forceinline__ void make(const uint32_t* ids, const float* wt, int width, int slots, int skip_zero) {
        const int lane = threadIdx.x;
        if (lane >= 64) return;
        const uint32_t id = lane < width ? ids[lane] : 0xffffffffu;
        const float v = lane < width ? wt[lane] : 0.0f;
        const bool in = id < (uint32_t)slots && !(skip_zero && v == 0.0f);
        int rank = 0;
        for (int j = 0; j < width; ++j) {
            const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)(in ? id : 0xffffffffu), j);
            rank += o < id || (o == id && j < lane) ? 1 : 0;
        }
        const int c = __popcll(__ballot(in));
        if (in) list[rank] = lane, w[rank] = v;
        if (lane == 0) count = c;
    }
};

// x = bf16(x + y) of 4 values.
__device__ __forceinline__ void residual4(uint16_t* x, const v4f& y) {
    const uint2 v = *(const uint2*)x;
    uint2 z;
    z.x = naiwa_f32_to_bf16(naiwa_bf16_to_f32(v.x & 0xffffu) + y[0]) |
          naiwa_f32_to_bf16(naiwa_bf16_to_f32(v.x >> 16) + y[1]) << 16;
    z.y = naiwa_f32_to_bf16(naiwa_bf16_to_f32(v.y & 0xffffu) + y[2]) |
          naiwa_f32_to_bf16(naiwa_bf16_to_f32(v.y >> 16) + y[3]) << 16;
    *(uint2*)x = z;
}

// Down and combine of one token: a block of 8 waves per 16 rows.  A pair's steps go to the
// `split` waves of one of 8 / split groups, the groups take the pairs in turn; the sums meet in
// LDS and 4 lanes of the first wave add them up, pairs in ascending slot order.  Dynamic LDS:
// h's planes and scales of every pair, copied by all waves.
constexpr int kOneWaves = 8;
template <int PH>
__global__ void __launch_bounds__(64 * kOneWaves)
down_one_kernel(Bank down, Planes h, int H, int I, const uint32_t* ids, const float* w, int width, int slots, int skip_zero,
                int split, int accumulate, float* out, uint16_t* res) {
    extern __shared__ __align__(16) uint8_t hl[];
    __shared__ Order order;
    __shared__ v4f red[kMaxWidth][kOneWaves][4]; // [pair][wave of the group][row / 4]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rb = blockIdx.x, steps = naiwa_mx_steps(I), groups = kOneWaves / split, in = wave % split;
    int t0, t1;
    deal(steps, in, split, &t0, &t1);
    order.make(ids, w, width, slots, skip_zero);
    const int row16 = (int)(h.row / 16);
    for (int i = tid; i < width * (row16 + h.groups); i += 64 * kOneWaves) {
        const int j = i / (row16 + h.groups), c = i % (row16 + h.groups);
        // pairs that do not count have rows that nobody wrote: copied, never used
        *(v4u*)(hl + (size_t)16 * i) = c < row16 ? *(const v4u*)(h.base + j * h.row + 16 * c)
                                                 : *(const v4u*)(h.scales + ((int64_t)j * h.groups + c - row16) * 16);
    }
    __syncthreads();
    const int count = order.count;
    for (int q = wave / split; q < count; q += groups) {
        const int j = uniform(order.list[q]), s = uniform((int)ids[j]);
        const uint8_t* const wp[1] = {down.base + (int64_t)s * down.stride + rb * down.strip};
        const uint8_t* hr = hl + (size_t)16 * j * (row16 + h.groups);
        v4f acc[1] = {};
        strips_dot_one<1, PH>(wp, hr, hr + 16 * row16, steps, t0, t1, lane, acc, [] {});
        if ((lane & 15) == 0) red[q][in][lane >> 4] = acc[0];
    }
    __syncthreads();
    if (tid >= 4) return;
    const int64_t o = 16 * rb + 4 * tid;
    v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
    if (accumulate) y = *(const v4f*)(out + o);
    for (int q = 0; q < count; ++q) {
        v4f v = red[q][0][tid];
        for (int i = 1; i < split; ++i) v += red[q][i][tid];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(order.w[q], v[i], y[i]);
    }
    if (res) residual4(res + o, y);
    if (out) *(v4f*)(out + o) = y;
}

// out[t] (+)= the weighted dots of t's pairs in ascending slot order, a pair's K parts in
// part order; res: also res = bf16(res + out).
__global__ void __launch_bounds__(kThreads)
combine_kernel(const float* y, int64_t n, int parts, const uint32_t* ids, const float* w, int width, int slots, int H,
               int skip_zero, int accumulate, float* out, uint16_t* res) {
    __shared__ Order order;
    const int64_t t = blockIdx.x;
    order.make(ids + t * width, w + t * width, width, slots, skip_zero);
    __syncthreads();
    const int c = order.count;
    constexpr int Q = 8; // pairs whose loads go out together
    for (int r = 4 * (blockIdx.y * kThreads + threadIdx.x); r < H; r += 4 * kThreads * gridDim.y) {
        const int64_t o = t * H + r;
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
        if (accumulate) acc = *(const v4f*)(out + o);
        for (int q0 = 0; q0 < c; q0 += Q) {
            v4f v[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (q0 + q < c) v[q] = *(const v4f*)(y + (t * width + order.list[q0 + q]) * H + r);
            for (int p = 1; p < parts; ++p)
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    if (q0 + q < c) v[q] += *(const v4f*)(y + (p * n + t * width + order.list[q0 + q]) * H + r);
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (q0 + q < c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(order.w[q0 + q], v[q][j], acc[j]);
        }
        if (res) residual4(res + o, acc);
        if (out) *(v4f*)(out + o) = acc;
    }
}

bool bank_ok(const naiwa_bank* b) {
    if (!b || !b->base || b->slots <= 0 || b->n <= 0 || b->k <= 0) return false;
    const int64_t bytes = naiwa_projection_bytes(NAIWA_MXFP4_T, b->n, b->k);
    return bytes > 0 && b->slot_stride >= bytes && !(((uintptr_t)b->base | (uintptr_t)b->slot_stride) & 15);
}

// K parts of the down projection of a call of at most `segs` segments: blocks for two a CU, as
// long as each of a part's waves has 4 steps.
int down_parts(int segs, int H, int I) {
    const int blocks = segs * ((H + 63) / 64), most = naiwa_mx_steps(I) / (4 * kWaves);
    return std::max(1, std::min({8, most, 512 / std::max(1, blocks)}));
}

// Blocks that share a segment's `items` feature or row blocks, of a call of `segs` segments: about
// one block a CU in all where a wave has 3 or 4 steps, so that runs are long, and two where it has
// fewer.  Gate/up and down kernels, 256 and 512 blocks: 16 rows of 8 experts top-2, H 4096, I
// 14336 (4 and 3 steps) 98.7 and 106, 70 and 87 us; 96 rows of 128 experts top-8, H 2048, I 768 (2
// and 1) 79.6 and 70.6, 45.8 and 38.1; 5 rows of 64 top-6, H 2048, I 1408 (2 and 2) 29.7 and 26.4,
// 18.8 and 16.8.
int stream_splits(int segs, int items, int ns) {
    return std::max(1, std::min(items, ((ns > 2 ? 256 : 512) + segs - 1) / segs));
}
// K parts of a streamed down projection: at most 3 steps a wave (4 spill with 5 planes).
int stream_parts(int I) { return (naiwa_mx_steps(I) + 3 * kStreamWaves - 1) / (3 * kStreamWaves); }

constexpr int kPlanesMost = 5;

struct Layout {
    size_t count, begin, key, perm, tiles, x, xs, h, hs, y, total;
    int64_t max_tiles;
    Layout(int64_t rows, int width, int H, int I) {
        auto a256 = [](size_t b) { return (b + 255) & ~size_t(255); };
        const size_t n = (size_t)rows * width;
        size_t dots = n; // a pair's rows, a K part each where it has them
        if (rows == 1) dots = 8 * n;
        if (fits((int64_t)n, stream_parts(I), H)) dots = std::max(dots, n * stream_parts(I));
        count = 0;
        begin = 256;
        key = a256(begin + (size_t)(NAIWA_SEG_MAX_KEYS + 1) * 4);
        perm = a256(key + n * 4);
        tiles = a256(perm + n * 4);
        max_tiles = (int64_t)n / kTile + std::min<int64_t>((int64_t)n, NAIWA_SEG_MAX_KEYS);
        x = a256(tiles + (size_t)(3 * max_tiles + 1) * 4);
        xs = a256(x + (size_t)rows * plane_row(kPlanesMost, H));
        h = a256(xs + (size_t)rows * naiwa_mx_groups(H) * 16);
        hs = a256(h + n * plane_row(kPlanesMost, I));
        y = a256(hs + n * naiwa_mx_groups(I) * 16);
        total = a256(y + dots * H * 4);
    }
    // Whether n pairs get `parts` parts each: 64 MB of dots at most, which stay in the caches.
    static bool fits(int64_t n, int parts, int H) { return parts == 1 || n * parts * H * 4 <= (64 << 20); }
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

namespace {

struct Run { // one call's pieces
    const NaiwaMxCall& c;
    Layout L;
    uint8_t* ws;
    hipStream_t st;
    int H, I, slots, n;
    Bank g, u, d;
    Segments seg;
    Tiles tl;

    Planes x(int P) const { return Planes{ws + L.x, ws + L.xs, plane_row(P, H), naiwa_mx_groups(H)}; }
    Planes h(int P) const { return Planes{ws + L.h, ws + L.hs, plane_row(P, I), naiwa_mx_groups(I)}; }
    float* y() const { return (float*)(ws + L.y); }

    template <int PX, bool BF16> void planes(int mode) const {
        const int64_t xb = (int64_t)c.rows * 4 * naiwa_mx_steps(H);
        const unsigned pb = (unsigned)((xb + kThreads - 1) / kThreads);
        const Beside with{seg.begin, tl, c.ids, c.skip_zero ? c.w : nullptr, n, (uint32_t*)seg.perm, (uint32_t*)seg.key,
                          (uint32_t*)seg.begin, (int*)(ws + L.count), (int*)(ws + L.count) + 1, slots};
        if (mode == kWithTiles)
            planes_kernel<PX, BF16, kWithTiles><<<pb + 1, kThreads, 0, st>>>(c.x, c.rows, H, x(PX), with);
        else if (mode == kWithSegments)
            planes_kernel<PX, BF16, kWithSegments><<<pb + 1, kThreads, 0, st>>>(c.x, c.rows, H, x(PX), with);
        else
            planes_kernel<PX, BF16, kPlanesOnly><<<pb, kThreads, 0, st>>>(c.x, c.rows, H, x(PX), with);
    }
    void combine(int parts) const {
        const unsigned cs = (unsigned)((H + 4 * kThreads - 1) / (4 * kThreads));
        combine_kernel<<<dim3(c.rows, cs), kThreads, 0, st>>>(y(), n, parts, c.ids, c.w, c.width, slots, H, c.skip_zero,
                                                             c.accumulate, c.out, c.res);
    }

    // One token.  False, with nothing launched, where x does not fit in LDS.
    template <int PX, int PH, bool BF16> bool one() {
        const size_t xl = (size_t)plane_row(PX, H) + (size_t)naiwa_mx_groups(H) * 16;
        const size_t hl = ((size_t)plane_row(PH, I) + (size_t)naiwa_mx_groups(I) * 16) * c.width;
        constexpr size_t kLds = 32 * 1024;
        if (xl > kLds) return false;
        gateup_one_kernel<PX, PH, BF16><<<dim3(c.width, 4 * naiwa_mx_steps(I)), kThreads, xl, st>>>(
            g, u, c.x, H, I, c.ids, c.w, slots, c.skip_zero, c.act, h(PH));
        if (hl <= kLds) {
            int split = 1;
            while (2 * split * c.width <= kOneWaves && 8 * split <= naiwa_mx_steps(I)) split *= 2;
            down_one_kernel<PH><<<H / 16, 64 * kOneWaves, hl, st>>>(d, h(PH), H, I, c.ids, c.w, c.width, slots, c.skip_zero,
                                                                    split, c.accumulate, c.out, c.res);
            return true;
        }
        seg.ids = c.ids;
        seg.w = c.skip_zero ? c.w : nullptr;
        const int parts = down_parts(n, H, I);
        down_kernel<PH><<<dim3(n, (H + 63) / 64, parts), kThreads, 0, st>>>(d, h(PH), H, I, n, parts, seg, y());
        combine(parts);
        return true;
    }

    template <int PX, int PH, bool BF16> int go() {
        if (c.rows == 1 && one<PX, PH, BF16>()) return naiwa_hip_rc(hipGetLastError());
        // the copies of x to LDS have 32-bit offsets
        const bool tiled = naiwa_mx_tiled(n, slots) && (uint64_t)c.rows * plane_row(PX, H) <= UINT32_MAX;
        const bool sorted = !tiled && n <= 1024; // in the planes' launch; more pairs take a launch of their own
        if (!sorted) {
            // pairs of weight 0 are sorted in with the others and left out by the combine
            seg.key = nullptr;
            if (int rc = naiwa_moe_gather(c.ids, n, slots, (uint32_t*)seg.perm, (uint32_t*)seg.begin,
                                          (int*)(ws + L.count) + 1, (int64_t)st))
                return rc;
        }
        planes<PX, BF16>(tiled ? kWithTiles : sorted ? kWithSegments : kPlanesOnly);
        if (tiled) {
            constexpr int NA = 2;
            const int64_t most = n / kTile + std::min(n, slots);
            const unsigned t8 = (unsigned)((most + 7) / 8 * 8);
            const int xcd = n <= (int64_t)128 * slots ? 1 : 0;
            const unsigned b1 = t8 * ((4 * naiwa_mx_steps(I) + 2 * NA - 1) / (2 * NA));
            const unsigned b2 = t8 * ((H / 32 + 4 * NA - 1) / (4 * NA));
            tile_gateup_kernel<NA, PX, PH><<<b1, kThreads, 2 * sizeof(Stage<PX>), st>>>(g, u, x(PX), H, I, c.width, seg.perm,
                                                                                       tl, c.act, xcd, h(PH));
            tile_down_kernel<NA, PH><<<b2, kThreads, 2 * sizeof(Stage<PH>), st>>>(d, h(PH), H, I, seg.perm, tl, xcd, y());
            combine(1);
            return naiwa_hip_rc(hipGetLastError());
        }
        const int segs = std::min(n, slots), gs = sorted ? segs : slots;
        const int sx = naiwa_mx_steps(H), sh = naiwa_mx_steps(I), nfb = 4 * sh;
        const Planes xp = x(PX), hp = h(PH);
        // blocks for the passes of 16 tokens of a segment: one more than the average segment's
        const int passes = n <= 16 ? 1 : std::min(4, n / segs / 16 + 2);
        if (sx <= 4 * kStreamWaves) {
            const int ns = sx <= kStreamWaves ? 1 : sx <= 2 * kStreamWaves ? 2 : 4;
            auto launch = [&](auto* kernel) {
                kernel<<<dim3(gs, stream_splits(segs, nfb, ns), passes), kStreamThreads, 0, st>>>(g, u, xp, H, I, c.width, seg,
                                                                                                  c.act, hp);
            };
            ns == 1 ? launch(gateup_stream_kernel<1, PX, PH>)
                    : ns == 2 ? launch(gateup_stream_kernel<2, PX, PH>) : launch(gateup_stream_kernel<4, PX, PH>);
        } else {
            gateup_kernel<PX, PH><<<dim3(gs, nfb), kThreads, 0, st>>>(g, u, xp, H, I, c.width, seg, c.act, hp);
        }
        int parts = stream_parts(I);
        if (Layout::fits(n, parts, H)) {
            const int ns = ((sh + parts - 1) / parts + kStreamWaves - 1) / kStreamWaves;
            auto launch = [&](auto* kernel) {
                const dim3 grid(gs, stream_splits(segs * parts, (H + 63) / 64, ns), parts * passes);
                kernel<<<grid, kStreamThreads, 0, st>>>(d, hp, H, I, n, ns * kStreamWaves, passes, seg, y());
            };
            ns == 1 ? launch(down_stream_kernel<1, PH>)
                    : ns == 2 ? launch(down_stream_kernel<2, PH>) : launch(down_stream_kernel<3, PH>);
        } else {
            parts = 1;
            down_kernel<PH><<<dim3(gs, (H + 63) / 64, parts), kThreads, 0, st>>>(d, hp, H, I, n, parts, seg, y());
        }
        combine(parts);
        return naiwa_hip_rc(hipGetLastError());
    }
};

} // namespace

int naiwa_mx_run(const NaiwaMxCall& c, uint8_t* ws, hipStream_t st) {
    if (c.rows == 0) return NAIWA_OK;
    const int H = c.gate->k, I = c.gate->n, slots = c.gate->slots, n = c.rows * c.width;
    const Layout L(c.rows, c.width, H, I);
    int* tiles = (int*)(ws + L.tiles);
    Run r{c, L, ws, st, H, I, slots, n,
          Bank{(const uint8_t*)c.gate->base, c.gate->slot_stride, naiwa_mx_strip_bytes(H)},
          Bank{(const uint8_t*)c.up->base, c.up->slot_stride, naiwa_mx_strip_bytes(H)},
          Bank{(const uint8_t*)c.down->base, c.down->slot_stride, naiwa_mx_strip_bytes(I)},
          Segments{(uint32_t*)(ws + L.key), (uint32_t*)(ws + L.begin), (uint32_t*)(ws + L.perm), (int*)(ws + L.count), nullptr, nullptr, slots},
          Tiles{tiles, tiles + L.max_tiles, tiles + 2 * L.max_tiles, tiles + 3 * L.max_tiles}};
    if (n == 0) {
        r.combine(1);
        return naiwa_hip_rc(hipGetLastError());
    }
    if (!c.skip_zero) return r.go<3, 4, true>(); // a prompt chunk
    return c.x_dtype == NAIWA_BF16 ? r.go<4, 5, true>() : r.go<5, 5, false>();
}
