// The tile product behind include/naiwa_linear.h: D[i][j] = sum_c I[i][c] J[j][c] on the
// matrix cores, for operands whose contraction index c is contiguous in memory (rows of x, W or dy) or
// is the row index (W in the input gradient, dy and x in the weights').
//
// A block computes a TI x TJ tile, its waves NWI x NWJ parts of it in 16x16 MFMAs (16x16x32).  D's lane
// holds 4 consecutive i of one j, so i is the index that is contiguous in the output: the
// weights' features forward, the input's in both gradients.
//
// Tiles of 64 contraction steps lie in LDS twice over: one is read while the next lands in the
// other, copied from memory without passing registers (16 bytes a lane).  Buffer ranges make what lies behind a
// segment's last row zero, lanes behind the last of c ask for an address out of range.  Both layouts keep
// 16-byte pieces whole and permute them so that no two lanes of a read share a bank:
//   contiguous: row r of 64 values, piece q at r * 128 + 16 (q ^ (r & 7)); 16-byte reads;
//   row index:  row c of T values, the pair of pieces f (16 values) at 32 (f ^ s(c)), s(c) = c & 3 | (c >> 3 & 1)
//               << 2, read by the transposing LDS read (4 rows x 16 values a group of 16 lanes).
// Operands that are not multiples of 16 bytes pass through registers, value by value at their ends.
#pragma once

#include "../../include/naiwa_linear.h"
#include "common.h"

#include <type_traits>

namespace {

typedef uint32_t lin_u32x4 __attribute__((ext_vector_type(4)));
typedef float lin_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 lin_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lin_f16x8 __attribute__((ext_vector_type(8)));
typedef short lin_s16x4 __attribute__((ext_vector_type(4)));
typedef short lin_s16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;           // contraction steps of a tile in LDS
constexpr uint32_t kFar = 1u << 31; // an offset past every range

enum { kRows = 0, kCols = 1 }; // the contraction index is contiguous, or the row index

// An operand's tile: what a block reads of it.
struct TileView {
    const uint16_t* base; // the tile's first value at contraction index 0
    int64_t ld;           // values between rows
    int valid;            // the tile's rows (kRows) or columns (kCols) that exist
};

__device__ __forceinline__ uint32_t lds_at(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Lane i of the wave copies 16 bytes from the range's offset `off` to lds + 16 i; zeros past the range.
// As inline assembly, so that the compiler's wait counts leave copies in flight alone.
__device__ __forceinline__ void copy16(lin_u32x4 range, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(range), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ lin_u32x4 range_of(const void* p, int64_t bytes) {
    const uint64_t a = (uint64_t)p;
    const int n = bytes < 0 ? 0 : bytes < 0x7fffffff ? (int)bytes : 0x7fffffff;
    return lin_u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)),
                     (uint32_t)__builtin_amdgcn_readfirstlane(n), 0x00020000u};
}
// The wave's copies but the newest N have landed, for all waves of the block.
template <int N> __device__ __forceinline__ void copies_landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

// One operand of T rows (or columns), loaded by NW waves.  PAIR (kRows): the second half of its rows are
// those of a second view.
template <int T, int LAYOUT, int NW, bool PAIR> struct Tile {
    static_assert(!PAIR || (LAYOUT == kRows && NW % 2 == 0), "whole waves a half");
    static constexpr int kBytes = T * kStep * 2;
    static constexpr int kCopies = kBytes / 1024 / NW; // a wave's, 1 KB each
    static constexpr int kPieces = kBytes / 16 / (NW * 64);
    static constexpr int kRowPieces = LAYOUT == kRows ? kStep / 8 : T / 8; // pieces of a row in LDS
    static_assert(kCopies * 1024 * NW == kBytes, "whole copies");

    static __device__ __forceinline__ int swizzle(int row) { // of a piece's place in its row
        if (LAYOUT == kRows) return row & 7;
        return ((row & 3) | ((row >> 1) & 4)) << 1 & (kRowPieces - 1);
    }

    // ---- by copies
    // The copies of contraction steps c0 .. c0 + 63 of C.
    static __device__ __forceinline__ void copy(const TileView* views, int64_t c0, int64_t C, uint32_t lds, int wave, int lane) {
        TileView v = PAIR && wave >= NW / 2 ? views[1] : views[0];
        if (PAIR && wave >= NW / 2) v.base -= T / 2 * v.ld, v.valid += T / 2; // (rows from T / 2 on)
        const uint32_t ld2 = (uint32_t)v.ld * 2;
        if constexpr (LAYOUT == kRows) {
            const lin_u32x4 r = range_of(v.base + c0, ((v.valid - 1) * v.ld + (C - c0)) * 2);
            const int piece = (lane & 7) ^ (lane >> 3);
            const uint32_t off = 8 * piece < C - c0 ? (uint32_t)(lane >> 3) * ld2 + 16 * piece : kFar;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int row = 8 * (wave * kCopies + i);
                copy16(r, off + (uint32_t)row * ld2, lds + (wave * kCopies + i) * 1024);
            }
        } else {
            const lin_u32x4 r = range_of(v.base + c0 * v.ld, ((C - c0 - 1) * v.ld + v.valid) * 2);
            constexpr int kPer = 64 / kRowPieces; // rows of a copy
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int row = (wave * kCopies + i) * kPer + lane / kRowPieces;
                const int piece = (lane % kRowPieces) ^ swizzle(row);
                copy16(r, (uint32_t)row * ld2 + 16 * piece, lds + (wave * kCopies + i) * 1024);
            }
        }
    }

    // ---- through registers
    struct Held {
        lin_u32x4 v[kPieces];
    };
    static __device__ __forceinline__ void load(const TileView* views, int64_t c0, int64_t C, int tid, Held& h) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = tid + i * NW * 64, at = p % kRowPieces * 8;
            int row = p / kRowPieces;
            const bool second = PAIR && row >= T / 2;
            const TileView v = second ? views[1] : views[0];
            if (second) row -= T / 2;
            // LDS row `row`, values at .. at + 7 of it, of which `n` exist
            const int64_t left = LAYOUT == kRows ? C - c0 - at : v.valid - at;
            const bool in = LAYOUT == kRows ? row < v.valid : row < C - c0;
            const uint16_t* s = LAYOUT == kRows ? v.base + row * v.ld + c0 + at : v.base + (c0 + row) * v.ld + at;
            lin_u32x4 w = {};
            if (in && left >= 8) {
                __builtin_memcpy(&w, s, 16);
            } else if (in) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) w[j / 2] |= (uint32_t)s[j] << (16 * (j % 2));
            }
            h.v[i] = w;
        }
    }
    static __device__ __forceinline__ void store(const Held& h, uint8_t* lds, int tid) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = tid + i * NW * 64, row = p / kRowPieces, piece = (p % kRowPieces) ^ swizzle(row);
            *(lin_u32x4*)(lds + row * (kRowPieces * 16) + piece * 16) = h.v[i];
        }
    }

    // ---- fragments: F of 16 rows (columns) from the wave's first, `first`, of 32 contraction steps (half kk)
    template <int F> struct Reader {
        uint32_t at[LAYOUT == kRows ? 2 : F];
        // frag f is rows first + 16 f + lane % 16, c = 32 kk + 8 (lane / 16) + 0 .. 7
        __device__ __forceinline__ Reader(int first, int lane) {
            if constexpr (LAYOUT == kRows) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    at[kk] = (uint32_t)(first + (lane & 15)) * 128 + ((((lane >> 4) + 4 * kk) ^ (lane & 7)) << 4);
            } else {
                const int row = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
                for (int f = 0; f < F; ++f)
                    at[f] = (uint32_t)row * (T * 2) + (((first / 16 + f) * 2 ^ swizzle(row)) << 4) + 8 * (lane & 3);
            }
        }
        // buf: the tile's LDS address
        __device__ __forceinline__ lin_s16x8 get(uint32_t buf, int f, int kk) const {
            typedef __attribute__((address_space(3))) const lin_s16x8* P8;
            typedef __attribute__((address_space(3))) lin_s16x4* P4;
            if constexpr (LAYOUT == kRows) {
                return *(P8)(buf + at[kk] + f * 2048);
            } else {
                const uint32_t a = buf + at[f] + kk * (32 * T * 2);
                const lin_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)a);
                const lin_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(a + 4 * T * 2));
                return lin_s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            }
        }
    };
};

template <bool F16> __device__ __forceinline__ lin_f32x4 lin_mfma(lin_s16x8 a, lin_s16x8 b, lin_f32x4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lin_f16x8, a), __builtin_bit_cast(lin_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lin_bf16x8, a), __builtin_bit_cast(lin_bf16x8, b), c, 0, 0, 0);
}

// A block's shape.  PAIR: the I tile's halves are two matrices' rows of the same features (a gate
// and its up), and a wave's first and second half of fragments belong to them.
template <int TI_, int TJ_, int NWI_, int NWJ_, int LI_, int LJ_, bool F16_, bool DIRECT_, bool PAIR_ = false> struct Shape {
    static constexpr int TI = TI_, TJ = TJ_, NWI = NWI_, NWJ = NWJ_, NW = NWI * NWJ, TH = NW * 64;
    static constexpr int FI = TI / NWI / 16, FJ = TJ / NWJ / 16;
    static constexpr bool F16 = F16_, DIRECT = DIRECT_, PAIR = PAIR_;
    typedef Tile<TI, LI_, NW, PAIR_> I;
    typedef Tile<TJ, LJ_, NW, false> J;
    static constexpr int kBuf = I::kBytes + J::kBytes;
    static constexpr int kLds = 2 * kBuf;
    // The wave's first I row (fragments of a PAIR: f < FI / 2 from here, the others TI / 2 on).
    static __device__ __forceinline__ int i_first(int wave) { return wave % NWI * (TI / NWI) / (PAIR ? 2 : 1); }
    static __device__ __forceinline__ int j_first(int wave) { return wave / NWI * (TJ / NWJ); }
};

// acc[fi][fj] += the tile's product over `sources` contraction ranges of C each: iv[0] and jv[0], then iv[1] and
// jv[1].  (A PAIR has one range, and iv[0], iv[1] are the matrices of its halves.)  each(b) is called with every
// half step's J fragments.
template <class S, class Each>
__device__ __forceinline__ void tile_product(const TileView* iv, const TileView* jv, int sources, int64_t C, uint8_t* lds,
                                             lin_f32x4 (&acc)[S::FI][S::FJ], Each each) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per = (int)((C + kStep - 1) / kStep), steps = per * sources;
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_at(lds));
    typedef typename S::I I;
    typedef typename S::J J;
    const typename I::template Reader<S::PAIR ? S::FI / 2 : S::FI> ri(S::i_first(wave), lane);
    const typename J::template Reader<S::FJ> rj(S::j_first(wave), lane);
    typename I::Held hi;
    typename J::Held hj;
    auto fetch = [&](int step, int buf) {
        const int s = step >= per ? 1 : 0; // (of a PAIR always 0)
        const int64_t c0 = (int64_t)(step - s * per) * kStep;
        if constexpr (S::DIRECT) {
            I::copy(S::PAIR || !s ? iv : iv + 1, c0, C, at + buf * S::kBuf, wave, lane);
            J::copy(s ? jv + 1 : jv, c0, C, at + buf * S::kBuf + I::kBytes, wave, lane);
        } else {
            I::load(S::PAIR || !s ? iv : iv + 1, c0, C, tid, hi);
            J::load(s ? jv + 1 : jv, c0, C, tid, hj);
        }
    };
    auto keep = [&](int buf) {
        if constexpr (!S::DIRECT) {
            I::store(hi, lds + buf * S::kBuf, tid);
            J::store(hj, lds + buf * S::kBuf + I::kBytes, tid);
        }
    };
    if (steps == 0) return;
    fetch(0, 0);
    keep(0);
    copies_landed<0>();
    for (int step = 0; step < steps; ++step) {
        const int buf = step & 1;
        if (step + 1 < steps) fetch(step + 1, buf ^ 1);
        const uint32_t ib = at + buf * S::kBuf, jb = ib + I::kBytes;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            lin_s16x8 a[S::FI], b[S::FJ];
#pragma unroll
            for (int f = 0; f < S::FI; ++f) {
                if (S::PAIR && f >= S::FI / 2)
                    a[f] = ri.get(ib + S::TI / 2 * 128, f - S::FI / 2, kk); // (a PAIR's I is kRows)
                else
                    a[f] = ri.get(ib, f, kk);
            }
#pragma unroll
            for (int f = 0; f < S::FJ; ++f) b[f] = rj.get(jb, f, kk);
            each(b);
#pragma unroll
            for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
                for (int fj = 0; fj < S::FJ; ++fj) acc[fi][fj] = lin_mfma<S::F16>(a[fi], b[fj], acc[fi][fj]);
        }
        if (step + 1 < steps) {
            keep(buf ^ 1);
            copies_landed<0>();
        }
    }
}

// ---- segments ---------------------------------------------------------------------------

// Row r of offsets, never past `rows`.
__device__ __forceinline__ uint32_t offset_at(const uint32_t* offsets, int e, uint32_t rows) { return min(offsets[e], rows); }

// The J tiles (of TJ rows) of all segments in order; every lane of a wave calls it.
struct Segments {
    uint32_t tiles, first; // all; below this lane's experts
    const uint32_t* offsets;
    uint32_t rows;
    int experts, per;
    __device__ __forceinline__ uint32_t count(int e) const {
        const uint32_t a = offset_at(offsets, e, rows), b = offset_at(offsets, e + 1, rows);
        return b > a ? b - a : 0;
    }
    __device__ __forceinline__ Segments(const uint32_t* o, uint32_t rows_, int experts_, int TJ)
        : first(0), offsets(o), rows(rows_), experts(experts_) {
        if (!offsets) {
            tiles = (rows + TJ - 1) / TJ;
            return;
        }
        const int lane = threadIdx.x & 63;
        per = (experts + 63) / 64;
        uint32_t mine = 0;
        for (int e = lane * per; e < min(experts, (lane + 1) * per); ++e) mine += (count(e) + TJ - 1) / TJ;
        uint32_t in = mine;
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t x = (uint32_t)__shfl_up((int)in, m, 64);
            if (lane >= m) in += x;
        }
        first = in - mine;
        tiles = (uint32_t)__builtin_amdgcn_readlane((int)in, 63);
    }
    // Tile t < tiles: its expert, first row, and rows (up to TJ).
    __device__ __forceinline__ void find(uint32_t t, int TJ, int* e, uint32_t* start, int* n) const {
        if (!offsets) {
            *e = 0, *start = t * TJ, *n = (int)min((uint32_t)TJ, rows - t * TJ);
            return;
        }
        const int lane = threadIdx.x & 63;
        uint32_t at = first, begin = 0, left = 0;
        int mine = -1;
        for (int x = lane * per; x < min(experts, (lane + 1) * per); ++x) {
            const uint32_t c = count(x), nt = (c + TJ - 1) / TJ;
            if (t >= at && t < at + nt) {
                mine = x;
                begin = offset_at(offsets, x, rows) + (t - at) * TJ;
                left = c - (t - at) * TJ;
            }
            at += nt;
        }
        const int who = __builtin_ctzll(__ballot(mine >= 0) | (1ull << 63)); // (t < tiles: some lane's)
        *e = __builtin_amdgcn_readlane(mine, who);
        *start = (uint32_t)__builtin_amdgcn_readlane((int)begin, who);
        *n = (int)min((uint32_t)TJ, (uint32_t)__builtin_amdgcn_readlane((int)left, who));
    }
};

// Block b's tile of nI x nJ: consecutive blocks go to the 8 XCDs in turn, each of which takes a contiguous
// part of the tiles, eight J tiles wide, so that what runs at a time on one XCD shares rows in its L2.
__device__ __forceinline__ bool tile_of_block(uint32_t b, uint32_t nI, uint32_t nJ, uint32_t* it, uint32_t* jt) {
    const uint64_t total = (uint64_t)nI * nJ;
    const uint64_t per = (total + 7) / 8, t = (b % 8) * per + b / 8;
    if (b / 8 >= per || t >= total) return false;
    constexpr uint32_t kWide = 8;
    const uint32_t g = (uint32_t)(t / (kWide * (uint64_t)nI)), j0 = g * kWide, wide = min(kWide, nJ - j0);
    const uint32_t r = (uint32_t)(t - (uint64_t)g * kWide * nI);
    *jt = j0 + r % wide;
    *it = r / wide;
    return true;
}

// ---- values -----------------------------------------------------------------------------

template <bool F16> __device__ __forceinline__ float lin_get(uint16_t v) { return F16 ? naiwa_f16_to_f32(v) : naiwa_bf16_to_f32(v); }
template <bool F16> __device__ __forceinline__ uint16_t lin_put(float v) {
    return F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v);
}
// Up to 4 values from p (n of them), f32 or 16 bits, from any address of their type.
template <bool F16> __device__ __forceinline__ lin_f32x4 load_4(const void* p, int64_t at, int n, bool f32) {
    lin_f32x4 o = {};
    if (f32) {
        const float* s = (const float*)p + at;
        if (n >= 4) {
            __builtin_memcpy(&o, s, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) o[i] = s[i];
        }
    } else {
        const uint16_t* s = (const uint16_t*)p + at;
        uint16_t v[4] = {};
        if (n >= 4) {
            __builtin_memcpy(v, s, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) v[i] = s[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = lin_get<F16>(v[i]);
    }
    return o;
}
template <bool F16> __device__ __forceinline__ void store_4(void* p, int64_t at, int n, bool f32, lin_f32x4 o) {
    if (f32) {
        float* s = (float*)p + at;
        if (n >= 4) {
            __builtin_memcpy(s, &o, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) s[i] = o[i];
        }
    } else {
        uint16_t* s = (uint16_t*)p + at;
        uint16_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lin_put<F16>(o[i]);
        if (n >= 4) {
            __builtin_memcpy(s, v, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) s[i] = v[i];
        }
    }
}

__device__ __forceinline__ float lin_act(int act, float v) { return act == NAIWA_ACT_NONE ? v : naiwa_act(act, v); }
// act and its slope.
__device__ __forceinline__ void lin_act_slope(int act, float v, float* a, float* slope) {
    if (act == NAIWA_ACT_NONE) {
        *a = v, *slope = 1.0f;
    } else if (act == NAIWA_ACT_SILU) {
        const float s = 1.0f / (1.0f + __expf(-v));
        *a = v * s, *slope = s * (1.0f + v * (1.0f - s));
    } else {
        const float k0 = 0.7978845608028654f, k1 = 0.044715f, t = tanhf(k0 * (v + k1 * v * v * v));
        *a = 0.5f * v * (1.0f + t);
        const float dt = 1.0f - t * t; // (0 far out, where v * v may be infinite)
        *slope = 0.5f * (1.0f + t) + (dt > 0.0f ? 0.5f * v * dt * (k0 * (1.0f + 3.0f * k1 * v * v)) : dt);
    }
}

// ---- host -------------------------------------------------------------------------------

constexpr int64_t kMaxLd = 1 << 21;
constexpr int kMaxExperts = 4096;

static inline bool lin_aligned(const void* p, int64_t ld, int64_t stride) {
    return !(((uintptr_t)p & 15) | (ld & 7) | (stride & 7));
}
static inline bool lin_overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && a_bytes > 0 && b_bytes > 0 && x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}
static inline int64_t lin_span(int64_t rows, int64_t ld, int64_t n, int size) { return rows > 0 ? ((rows - 1) * ld + n) * size : 0; }
static inline int lin_size(int dtype) { return dtype == NAIWA_F32 ? 4 : 2; }
static inline bool lin_act_ok(int act) {
    return act == NAIWA_ACT_NONE || act == NAIWA_ACT_SILU || act == NAIWA_ACT_GELU_PYTORCH_TANH;
}
// Rows of length ld at least as long as their values, experts `stride` apart at least as far as their rows.
static inline int lin_sizes_ok(int64_t experts, int64_t n, int64_t k, int64_t ld, int64_t stride) {
    if (experts <= 0 || n <= 0 || k <= 0 || ld < 0 || stride < 0 || (ld && ld < k)) return NAIWA_E_INVALID;
    ld = ld ? ld : k;
    if (ld > kMaxLd || experts > kMaxExperts || stride > (int64_t)1 << 48) return NAIWA_E_UNSUPPORTED;
    return stride && experts > 1 && stride < (n - 1) * ld + k ? NAIWA_E_INVALID : NAIWA_OK;
}
static inline int lin_weights_ok(const naiwa_weights* w) {
    if (!w || !w->w) return NAIWA_E_INVALID;
    if (w->dtype != NAIWA_BF16 && w->dtype != NAIWA_F16) return NAIWA_E_UNSUPPORTED;
    return lin_sizes_ok(w->experts, w->n, w->k, w->ld, w->stride);
}
// W, and U beside it, of one size and type.
static inline int lin_pair_ok(const naiwa_weights* w, const naiwa_weights* up) {
    if (int rc = lin_weights_ok(w)) return rc;
    if (!up) return NAIWA_OK;
    if (int rc = lin_weights_ok(up)) return rc;
    return up->experts != w->experts || up->n != w->n || up->k != w->k || up->dtype != w->dtype ? NAIWA_E_INVALID : NAIWA_OK;
}
static inline int64_t lin_ld(const naiwa_weights* w) { return w->ld ? w->ld : w->k; }
static inline int64_t lin_stride(const naiwa_weights* w) { return w->stride ? w->stride : w->n * lin_ld(w); }
static inline int64_t lin_bytes(const naiwa_weights* w) {
    return ((w->experts - 1) * lin_stride(w) + (w->n - 1) * lin_ld(w) + w->k) * 2;
}

} // namespace
