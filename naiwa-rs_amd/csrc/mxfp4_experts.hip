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
//   4 planes (bf16 x): 2^-19 M, a bf16 value of at least 2^-12 M exactly;
//   5 planes (f32 x, h): 2^-24 M, the rounding of an f32 as large as M.
// (Under M of 2^-102 the planes' scales stop: 2^-121 and 2^-126.)  What an outlier hides in its block is
// lost to rows of weights that do not see the outlier: 2^-19 2^8 of the rest at one of 2^8 times it.
// A plane less in each (3 and 4) takes 4096 tokens at Mixtral-8x7B sizes from 3.1 to 2.65 ms, with
// results off by 6e-6 instead of 4e-7, for which f32 sums have no use.
// FP4 x E2M3 runs at twice the rate of FP4 x FP8 (6 to 7 against 3.6 to 4.3 PFLOP/s from registers,
// random codes), and its sums are exact up to the f32 accumulator's rounding; with e4m3
// the matrix cores drop products under about 2^-15 of a step's largest (5e-5 of a sum of
// codes of all magnitudes).  A block with a NaN or an infinity gets the scale byte 255,
// which makes its products NaN.
//
// Launches, stream-ordered:
//   1. x laid out in planes, one row per token, and in a block beside it the (token, expert)
//      pairs sorted by slot (calls of many pairs: sorted by a launch of their own) and cut into
//      tiles of up to 64 pairs of one slot;
//   2. gate/up: a block per (tile, 128 features); h = act(g) u in planes;
//   3. down: a block per (tile, 256 rows, K part); unweighted dots per pair;
//   4. combine: out[t] = the weighted sum over t's pairs in ascending slot order.
// (2. and 3.: mxfp4_tiles.h.)  One token, and few whose experts are small, take two launches:
// gate/up lays x out itself, a block per (pair, 32 features), and down combines
// (gateup_pair_kernel, down_pair_kernel).
// No atomics: every run adds the same terms in the same order, and in calls of as many pairs the
// order of a pair's terms does not depend on the other pairs.
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
        // last plane, off by whole binades).  The operands' use past the result keeps them in place
        // with this compiler, which it need not (it may copy them): test_asm_mxfp4.py looks for
        // shared registers in what is compiled.
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

// What the last block of the planes' launch does beside them, which do not depend on it.
struct Beside {
    const uint32_t* ids; // the pairs, to be sorted first
    const float* w;      // pairs of weight 0 are left out, or null
    int n, slots;
    uint32_t *perm, *offsets; // sorted pairs and every slot's range
    int* bad;
    Tiles tiles;
};

// x [rows, H] in P planes, a block of 32 values a thread; the blocks that pad H to whole
// steps are zeros.  The launch's last block cuts the sorted pairs into tiles, SORT: after it
// sorted them.  Bound: HBM, and latency where rows are few: 4096 rows of H 4096 26 us (34 MB in,
// 50 MB out), 16 rows and their 32 pairs 5.6 us.
template <int P, bool BF16, bool SORT>
__global__ void __launch_bounds__(kThreads) planes_kernel(const void* x, int64_t rows, int H, Planes out, Beside with) {
    if (blockIdx.x == gridDim.x - 1) {
        if constexpr (SORT) {
            __shared__ NaiwaSegSmem sm;
            naiwa_segment(sm, with.ids, with.w, with.n, with.slots, with.perm, with.offsets, nullptr, nullptr, nullptr,
                          with.bad);
            __syncthreads();
        }
        tiles_block(with.offsets, with.slots, with.tiles);
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

// acc += strip rows x planes over steps [t0, t1), S strips of 16 rows (wp[i]: strip i's first
// byte), of one token whose planes are in LDS (xp, xs: the row, the same for every lane): rounds of
// U steps, all their weights in flight; `before` runs once the first round's are.
template <int S, int P, class F>
__device__ __forceinline__ void strips_dot(const uint8_t* const (&wp)[S], const uint8_t* xp, const uint8_t* xs, int steps,
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

// The sums of a block's NW waves over 4 strips of 16 rows, of one token: the columns of D are alike,
// and lane 16 q holds rows 4 q .. 4 q + 3 of column 0.
template <int NW> struct Sums {
    v4f v[NW][4][4];
    __device__ __forceinline__ void put(int wave, int lane, const v4f (&acc)[4]) {
        if (lane & 15) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[wave][i][lane >> 4] = acc[i];
    }
    __device__ __forceinline__ float row(int strip, int r) const {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) o += v[w][strip][r >> 2][r & 3];
        return o;
    }
};

// h of 32 features (strips 0, 1 of the sums: gate, 2, 3: up), a feature a lane of 32, to row `row`
// of the planes as block fb.  Bits of E2M3 by hand: |y| <= 4 is a multiple of 1/8 under 2 and of 1/4
// from there on, so adding 1.5 2^20 or 1.5 2^21 rounds it to nearest even, and the low bits of that
// sum are the code (less 8 in the upper binade).
template <int PH, int NW>
__device__ __forceinline__ void put_h(const Sums<NW>& sums, bool pad, int act, int fb, int64_t row, const Planes& h) {
    const int f = threadIdx.x & 31;
    const float g = sums.row(f >> 4, f & 15), u = sums.row(2 + (f >> 4), f & 15);
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

// Gate/up by pair, for few tokens: a block per (pair, 32 features); each wave lays out its own
// steps of the token's x in LDS while its first weights are on the way.  Pair j is row j of h;
// blocks past I (h padded to whole steps) write zeros.  Of one token, the first block lists the
// pairs that count as tiles of one pair, for tile_down_kernel, and clears the list's other entries: at
// most 64 in all (naiwa_mx_tiles).  Dynamic LDS: the planes of x, their scales (16 bytes a group).
// Bound: latency (the launch, x to planes behind the first weights' way, four waves' sums): 8 of 128
// Qwen3-30B experts 6.6 us (13.4 MB), 2 of 8 of 1024 x 2048 6.3 us (4.5 MB).
template <int PX, int PH, bool BF16>
__global__ void __launch_bounds__(kThreads, 2)
gateup_pair_kernel(Bank gate, Bank up, const void* x, int H, int I, const uint32_t* ids, const float* w, int width, int slots,
                  int skip_zero, int act, Planes h, uint32_t* perm, Tiles tl) {
    extern __shared__ __align__(16) uint8_t xl[];
    __shared__ Sums<kWaves> sums;
    const int j = blockIdx.x, fb = blockIdx.y;
    if (gridDim.x == (unsigned)width && j == 0 && fb == 0 && threadIdx.x < 64) {
        const int i = threadIdx.x;
        const uint32_t id = i < width ? ids[i] : 0xffffffffu;
        const bool in = id < (uint32_t)slots && !(skip_zero && w[i] == 0.0f);
        const uint64_t m = __ballot(in);
        const int at = __popcll(m & ((1ull << i) - 1));
        if (in) perm[i] = (uint32_t)i, tl.t[at] = make_int4(i, 1, (int)id, 0);
        if (i >= __popcll(m) && i < 8 * tl.run) tl.t[i] = make_int4(0, 0, 0, 0);
    }
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
                load_block<BF16>(x, (int64_t)(j / width) * H, H, kb, f);
                const int sb = scale_byte(abs_max(f));
                v6u o[PX];
                to_planes<PX>(f, sb, o);
                put_block<PX>(xl, scales, kb, o, sb);
            }
        };
        strips_dot<4, PX>(wp, xl, scales, steps, t0, t1, lane, acc, stage);
    }
    sums.put(threadIdx.x >> 6, lane, acc);
    __syncthreads();
    if (threadIdx.x < 32) put_h<PH>(sums, pad, act, fb, j, h);
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

// Down and combine by pair: a block of 8 waves per 16 rows and token.  A pair's steps go to the
// `split` waves of one of 8 / split groups, the groups take the pairs in turn; the sums meet in
// LDS and 4 lanes of the first wave add them up, pairs in ascending slot order.  Dynamic LDS:
// h's planes and scales of the token's pairs, copied by all waves.  Bound: latency, as gate/up: Qwen3-30B
// sizes 6.5 us (6.7 MB), 8 experts of 1024 x 2048 4.8 us.
constexpr int kPairWaves = 8;
template <int PH>
__global__ void __launch_bounds__(64 * kPairWaves)
down_pair_kernel(Bank down, Planes h, int H, int I, const uint32_t* ids, const float* w, int width, int slots, int skip_zero,
                int split, int accumulate, float* out, uint16_t* res) {
    extern __shared__ __align__(16) uint8_t hl[];
    __shared__ Order order;
    __shared__ v4f red[kMaxWidth][kPairWaves][4]; // [pair][wave of the group][row / 4]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rb = blockIdx.x, steps = naiwa_mx_steps(I), groups = kPairWaves / split, in = wave % split;
    const int64_t first = (int64_t)blockIdx.y * width; // the token's first pair
    ids += first, w += first, h.base += first * h.row, h.scales += first * h.groups * 16;
    int t0, t1;
    deal(steps, in, split, &t0, &t1);
    order.make(ids, w, width, slots, skip_zero);
    const int row16 = (int)(h.row / 16);
    for (int i = tid; i < width * (row16 + h.groups); i += 64 * kPairWaves) {
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
        strips_dot<1, PH>(wp, hr, hr + 16 * row16, steps, t0, t1, lane, acc, [] {});
        if ((lane & 15) == 0) red[q][in][lane >> 4] = acc[0];
    }
    __syncthreads();
    if (tid >= 4) return;
    const int64_t o = (int64_t)blockIdx.y * H + 16 * rb + 4 * tid;
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
// part order; res: also res = bf16(res + out).  Bound: HBM (4096 tokens at Mixtral-8x7B sizes 35 us,
// 201 MB: 5.7 TB/s), and the launch for few rows (4 to 5 us).
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

constexpr int kPlanesMost = 5;

constexpr int kNA = 2; // tiles of 32 weight rows a wave of the tile kernels
// Columns of blocks of a tile: 4 waves of kNA / 2 features blocks (gate and up) or kNA row blocks.
int gateup_cols(int I) { return (4 * naiwa_mx_steps(I) + 2 * kNA - 1) / (2 * kNA); }
int down_cols(int H) { return (H / 32 + 4 * kNA - 1) / (4 * kNA); }

// K parts of a down projection of `blocks` blocks, in groups of 4 steps: blocks for two a CU as
// long as a part has two groups, and 64 MB of dots at most, which stay in the caches.  16 rows of
// 8 experts top-2, H 4096, I 14336 (128 blocks) 4 parts and 1: 170 and 215 us a call.
int down_parts(int64_t n, int64_t blocks, int H, int I) {
    int parts = (int)std::max<int64_t>(1, std::min<int64_t>({4, naiwa_mx_groups(I) / 2, 512 / blocks}));
    while (parts > 1 && n * parts * H * 4 > (64 << 20)) --parts;
    return parts;
}

// The most tiles of n pairs over `slots` slots, a multiple of 8.
int64_t tiles_most(int64_t n, int slots) { return (n / kTile + std::min<int64_t>(n, slots) + 7) / 8 * 8; }

// Entries of a call's tile list.  One token's tiles hold a pair each (or, sorted, a slot's pairs, of
// which there are at most kTile): n of them at most.  gateup_pair_kernel lists them by a lane an entry.
static_assert(kMaxWidth <= 64 && kMaxWidth % 8 == 0 && kMaxWidth <= kTile, "a lane an entry of one token's tile list");
extern "C" int naiwa_mx_tiles(int rows, int64_t n, int slots) {
    return (int)(rows == 1 ? (n + 7) / 8 * 8 : tiles_most(n, slots));
}

struct Layout {
    size_t offsets, bad, perm, tiles, x, xs, h, hs, y, total;
    Layout(int64_t rows, int width, int H, int I) {
        auto a256 = [](size_t b) { return (b + 255) & ~size_t(255); };
        const size_t n = (size_t)rows * width;
        offsets = 0;
        bad = a256(offsets + (size_t)(NAIWA_SEG_MAX_KEYS + 1) * 4);
        perm = bad + 256;
        tiles = a256(perm + n * 4);
        x = a256(tiles + (size_t)tiles_most((int64_t)n, NAIWA_SEG_MAX_KEYS) * sizeof(int4));
        xs = a256(x + (size_t)rows * plane_row(kPlanesMost, H));
        h = a256(xs + (size_t)rows * naiwa_mx_groups(H) * 16);
        hs = a256(h + n * plane_row(kPlanesMost, I));
        y = a256(hs + n * naiwa_mx_groups(I) * 16);
        total = a256(y + (size_t)down_parts((int64_t)n, 1, H, I) * n * H * 4); // the most parts
    }
};

// Rows of a pass: the copies of x to LDS have 32-bit offsets.
int rows_per_pass(int rows, int H) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(rows, UINT32_MAX / plane_row(kPlanesMost, H)));
}

} // namespace

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
    // A grid of 2^32 threads along x wraps without an error; along y 65536 blocks are HIP's limit.
    const int rows = rows_per_pass(c.rows, H);
    const int64_t tiles = naiwa_mx_tiles(rows, (int64_t)rows * c.width, c.gate->slots);
    if (tiles * std::max(gateup_cols(I), down_cols(H)) * kThreads > UINT32_MAX) return NAIWA_E_UNSUPPORTED;
    if (4 * (int64_t)naiwa_mx_steps(I) > 65536) return NAIWA_E_UNSUPPORTED;
    return NAIWA_OK;
}

// Whether every pair reads its weights for itself (2 launches) instead of in tiles (4 or 5).  One
// token has an expert once, so always; few tokens while reading some twice costs less than the
// launches: 112 MB of weights at most, and no expert more than twice on average.  In microseconds a
// call, by pair and in tiles: Qwen3-30B 2 tokens (41 MB) 18.7 and 27.5, 4 (82) 27.1 and 30.1, 6 (123)
// 37.8 and 35.6; DeepSeek-V2-Lite 4 (112) 34.4 and 37.6, 6 (168) 47.4 and 44.1; 8 experts of H 1024, I
// 2048 top-2, 8 (54) 22.5 and 25.1, 16 (107, every expert four times) 36.1 and 25.4; Mixtral-8x7B 2
// (374) 88.0 and 86.1, 3 (562) 125 and 103.
extern "C" bool naiwa_mx_by_pair(int rows, int64_t n, int slots, int H, int I) {
    const int64_t expert = 2 * (I / 16) * naiwa_mx_strip_bytes(H) + (H / 16) * naiwa_mx_strip_bytes(I);
    return rows == 1 || (n <= 2 * (int64_t)slots && n * expert <= 112000000);
}

namespace {

// Whether tiles of ncol columns of blocks are dealt to the XCDs in runs (tile_col): where an
// XCD's 64 blocks at a time take several tiles with all their columns, neighbouring tiles of an
// expert share weights in its L2; with more columns, an XCD's share of every tile's columns
// does.  In microseconds, runs and not, prompt chunks: gate/up 6 columns (Qwen3-30B, 1999 tokens)
// 250 and 274, 11 (DeepSeek-V2-Lite, 2048) 289 and 321, 16 (8 experts of 1024 x 2048, 512) 46.9 and
// 45.8, 112 (Mixtral-8x7B, 4096) 3180 and 2822; down 8 columns (Qwen3) 250 and 255, 16 (Mixtral)
// 2822 and 2814.
int xcd_order(int ncol) { return ncol < 16; }

struct Run { // one pass's pieces
    const NaiwaMxCall& c;
    Layout L;
    uint8_t* ws;
    hipStream_t st;
    int H, I, slots, n;
    Bank g, u, d;
    uint32_t *offsets, *perm;
    Tiles tl;

    Planes x(int P) const { return Planes{ws + L.x, ws + L.xs, plane_row(P, H), naiwa_mx_groups(H)}; }
    Planes h(int P) const { return Planes{ws + L.h, ws + L.hs, plane_row(P, I), naiwa_mx_groups(I)}; }
    float* y() const { return (float*)(ws + L.y); }

    void combine(int parts) const {
        const unsigned cs = (unsigned)((H + 4 * kThreads - 1) / (4 * kThreads));
        combine_kernel<<<dim3(c.rows, cs), kThreads, 0, st>>>(y(), n, parts, c.ids, c.w, c.width, slots, H, c.skip_zero,
                                                             c.accumulate, c.out, c.res);
    }
    // Down of the tiles, and the combine.
    template <int PH> void down() const {
        const int ncol = down_cols(H);
        const unsigned blocks = (unsigned)(8 * tl.run * ncol);
        const int groups = naiwa_mx_groups(I), part = (groups + down_parts(n, blocks, H, I) - 1) / down_parts(n, blocks, H, I);
        const int parts = (groups + part - 1) / part;
        tile_down_kernel<kNA, PH><<<dim3(blocks, parts), kThreads, kStageBytes<PH>, st>>>(d, h(PH), H, I, n, part, perm, tl,
                                                                                          xcd_order(ncol), y());
        combine(parts);
    }

    // By pair.  False, with nothing launched, where x (or h of one of several tokens) does not fit in LDS.
    template <int PX, int PH, bool BF16> bool pairs() const {
        const size_t xl = (size_t)plane_row(PX, H) + (size_t)naiwa_mx_groups(H) * 16;
        const size_t hl = ((size_t)plane_row(PH, I) + (size_t)naiwa_mx_groups(I) * 16) * c.width;
        // With down's own 33 KB, what a CU has.  One token of H 16384, 4 experts of 1024 top-2, 31 us here
        // and 74 as a tile; of 8 Mixtral-8x7B experts (h of 2 x 14336) 51 and 63.
        constexpr size_t kLds = 120 * 1024;
        if (xl > kLds || (c.rows > 1 && hl > kLds)) return false;
        gateup_pair_kernel<PX, PH, BF16><<<dim3(n, 4 * naiwa_mx_steps(I)), kThreads, xl, st>>>(
            g, u, c.x, H, I, c.ids, c.w, c.width, slots, c.skip_zero, c.act, h(PH), perm, tl);
        if (hl > kLds) {
            down<PH>();
            return true;
        }
        int split = 1;
        while (2 * split * c.width <= kPairWaves && 8 * split <= naiwa_mx_steps(I)) split *= 2;
        down_pair_kernel<PH><<<dim3(H / 16, c.rows), 64 * kPairWaves, hl, st>>>(d, h(PH), H, I, c.ids, c.w, c.width, slots, c.skip_zero, split,
                                                                c.accumulate, c.out, c.res);
        return true;
    }

    template <int PX, int PH, bool BF16> int go() const {
        if (naiwa_mx_by_pair(c.rows, n, slots, H, I) && pairs<PX, PH, BF16>()) return naiwa_hip_rc(hipGetLastError());
        // The pairs are sorted in the planes' launch; many pairs, whose sorting takes its one block
        // longer than the planes take, in a launch of their own.  A call at Qwen3-30B sizes, in the
        // launch and apart: 128 pairs 52.5 and 54.1 us, 512 77.0 and 78.2, 768 81.3 and 80.4, 2048 115
        // and 105.
        const bool sort = n <= 512;
        const Beside with{c.ids, c.skip_zero ? c.w : nullptr, n, slots, perm, offsets, (int*)(ws + L.bad), tl};
        const unsigned pb = (unsigned)(((int64_t)c.rows * 4 * naiwa_mx_steps(H) + kThreads - 1) / kThreads) + 1;
        if (sort) {
            planes_kernel<PX, BF16, true><<<pb, kThreads, 0, st>>>(c.x, c.rows, H, x(PX), with);
        } else {
            // pairs of weight 0 are sorted in with the others and left out by the combine
            if (int rc = naiwa_moe_gather(c.ids, n, slots, perm, offsets, (int*)(ws + L.bad), (int64_t)st)) return rc;
            planes_kernel<PX, BF16, false><<<pb, kThreads, 0, st>>>(c.x, c.rows, H, x(PX), with);
        }
        const int ncol = gateup_cols(I);
        const unsigned blocks = (unsigned)(8 * tl.run * ncol);
        tile_gateup_kernel<kNA, PX, PH><<<blocks, kThreads, kStageBytes<PX>, st>>>(g, u, x(PX), H, I, c.width, perm, tl, c.act,
                                                                                  xcd_order(ncol), h(PH));
        down<PH>();
        return naiwa_hip_rc(hipGetLastError());
    }
};

// One pass over scratch ws.
int run_pass(const NaiwaMxCall& c, uint8_t* ws, hipStream_t st) {
    const int H = c.gate->k, I = c.gate->n, n = c.rows * c.width;
    const Layout L(c.rows, c.width, H, I);
    const Run r{c, L, ws, st, H, I, c.gate->slots, n,
                Bank{(const uint8_t*)c.gate->base, c.gate->slot_stride, naiwa_mx_strip_bytes(H)},
                Bank{(const uint8_t*)c.up->base, c.up->slot_stride, naiwa_mx_strip_bytes(H)},
                Bank{(const uint8_t*)c.down->base, c.down->slot_stride, naiwa_mx_strip_bytes(I)},
                (uint32_t*)(ws + L.offsets), (uint32_t*)(ws + L.perm),
                Tiles{(int4*)(ws + L.tiles), naiwa_mx_tiles(c.rows, n, c.gate->slots) / 8}};
    if (n == 0) {
        r.combine(1);
        return naiwa_hip_rc(hipGetLastError());
    }
    return c.x_dtype == NAIWA_BF16 ? r.go<4, 5, true>() : r.go<5, 5, false>();
}

} // namespace

size_t naiwa_mx_scratch_bytes(int rows, int width, int H, int I) {
    return rows == 0 || width == 0 ? 0 : Layout(rows_per_pass(rows, H), width, H, I).total;
}

int naiwa_mx_run(const NaiwaMxCall& c, uint8_t* ws, hipStream_t st) {
    const int64_t H = c.gate->k, pass = rows_per_pass(c.rows, c.gate->k);
    for (int64_t r0 = 0; r0 < c.rows; r0 += pass) {
        NaiwaMxCall p = c;
        p.rows = (int)std::min<int64_t>(pass, c.rows - r0);
        p.x = (const uint8_t*)c.x + r0 * H * (c.x_dtype == NAIWA_BF16 ? 2 : 4);
        p.ids = c.ids + r0 * c.width;
        p.w = c.w + r0 * c.width;
        if (c.out) p.out = c.out + r0 * H;
        if (c.res) p.res = c.res + r0 * H;
        if (int rc = run_pass(p, ws, st)) return rc;
    }
    return NAIWA_OK;
}
