// The tile product behind include/naiwa_linear.h: D[i][j] = sum_c I[i][c] J[j][c] on the
// matrix cores, for operands whose contraction index c is contiguous in memory (rows of x, W or dy) or
// is the row index (W in the input gradient, dy and x in the weights').
//
// A block computes a TI x TJ tile, its waves NWI x NWJ parts of it in 16x16 MFMAs (16x16x32).  D's lane
// holds 4 consecutive i of one j, so i is the index that is contiguous in the output: the
// weights' features forward, the input's in both gradients.
//
// Steps of the contraction lie in LDS several times over: while one is read, others land, copied from memory
// without passing registers (16 bytes a lane).  Buffer ranges make what lies behind a segment's last row zero, lanes
// behind the last of c ask for an address out of range, and so do steps behind the last (the counted
// waits stay the same to the end).  The kinds of block:
//   8 waves, 256 x 256, steps of 64, all of a CU's LDS.  The waves are two groups, one wave of each on a SIMD, that
//     take turns in reading and multiplying (setprio and a barrier a phase).  4096 x 4096 x 14336 takes 340 to 375 us,
//     1.3 to 1.4 PFLOP/s.  What bounds it is how fast rows come out of L2 (with the copies left out it took 233 us, without the
//     products as long as with them): hence whole 128-byte lines, three buffers of I and two of J, and copies spread
//     over the phases.  Leaving out the products and copies of a tile's empty rows gained nothing.
//   4 waves, 128 x 128, steps of 32 in a ring of 4 (64 KB, two blocks a CU) or 2 (three, by registers): in step t a wave multiplies
//     what it read of step t, reads step t + 1 and starts the copies of step t + 4 (t + 2), interleaved; one barrier a step.
//     Or 128 x 32, steps of 64 in a ring of 4 (80 KB, two blocks a CU), for few rows.
//   4 waves, 128 x 128 or 128 x 64, steps of 32 in a ring of 2, for rows that are not aligned (two or three blocks a CU).
// The XCDs begin at different steps and go round (turn_of_block): reading the same columns at a time they meet at
// the same memory channels (4096 x 4096 x 14336 403 -> 389 us, the weights' gradient of 64 experts 332 -> 286).
// Both layouts keep 16-byte pieces whole and permute them so that no two lanes of a read share a bank (the LDS takes
// lanes 0-3, 12-15, 20-27 of a 16-byte read at a time, then 4-11, 16-19, 28-31, and so on):
//   contiguous: row r, piece q at place q ^ (r & 6) of its row of 64 values, of one of 32 at q ^ g with g = 0, 2, 3, 1 for
//     rows in fours;
//   row index: row c of T values, the pair of pieces f (16 values) at 32 (f ^ s(c)), s(c) = c & 3 | (c >> 3 & 1)
//     << 2, read by the transposing LDS read (4 rows x 16 values a group of 16 lanes).
// Operands that are not multiples of 16 bytes pass through registers two steps ahead, whole pieces moved back into their row at its end.
// At the end the accumulators go through LDS once more, so that what follows the product works on rows:
// whole lines of memory, and code that is there once.
#pragma once

#include "../../include/naiwa_linear.h"
#include "common.h"
#include "spans.h"
#include "workspace.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef uint32_t lin_u32x4 __attribute__((ext_vector_type(4)));
typedef float lin_f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t lin_u16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 lin_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lin_f16x8 __attribute__((ext_vector_type(8)));
typedef short lin_s16x4 __attribute__((ext_vector_type(4)));
typedef short lin_s16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kFar = 1u << 31; // an offset past every range

enum { kRows = 0, kCols = 1 }; // the contraction index is contiguous, or the row index

// An operand's tile: what a block reads of it.
struct TileView {
    const uint16_t* base; // the tile's first value at contraction index 0
    int64_t ld;           // values between rows
    int valid;            // the tile's rows (kRows) or columns (kCols) that exist
    int first;            // columns that lie before them (kCols)
};
__device__ __forceinline__ TileView pick(bool second, const TileView& a, const TileView& b) {
    return {second ? b.base : a.base, second ? b.ld : a.ld, second ? b.valid : a.valid, second ? b.first : a.first};
}

__device__ __forceinline__ uint32_t lds_at(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Lane i of the wave copies 16 bytes from the range's offset `off` to lds + 16 i; zeros past the range.
// As inline assembly, so that the compiler's wait counts leave copies in flight alone.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // (that m0 is reserved: nothing else here uses it)
__device__ __forceinline__ void copy16(lin_u32x4 range, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(range), "s"(lds)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
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
template <int T, int LAYOUT, int NW, bool PAIR, int STEP> struct Tile {
    static_assert(!PAIR || (LAYOUT == kRows && NW % 2 == 0), "whole waves a half");
    static constexpr int kBytes = T * STEP * 2;
    static constexpr int kLanes = kBytes / NW / 16 < 64 ? kBytes / NW / 16 : 64; // that take part in a copy
    static constexpr int kCopies = kBytes / NW / 16 / kLanes;                    // a wave's
    static constexpr int kPieces = kBytes / 16 / (NW * 64);                      // a thread's, through registers
    static constexpr int kRowPieces = LAYOUT == kRows ? STEP / 8 : T / 8;       // pieces of a row in LDS
    static constexpr int kPer = kLanes / kRowPieces;                             // rows of a copy
    static_assert(kCopies * kLanes * 16 * NW == kBytes && kPer > 0, "whole copies of whole rows");

    static __device__ __forceinline__ int swizzle(int row) { // of a piece's place in its row
        if (LAYOUT == kRows) return STEP == 64 ? row & 6 : ((row >> 1) & 2) ^ ((row >> 3) & 1) * 3;
        return ((row & 3) | ((row >> 1) & 4)) << 1 & (kRowPieces - 1);
    }

    // ---- by copies: begin(), then one(i) for a wave's copies
    struct Copier {
        uint32_t off[kCopies]; // of the lane's pieces, from the step's first value
        uint32_t lds;          // of the wave's part of the first buffer
        int piece;             // of its row (kRows: the same in all of a wave's copies)
        bool in;
        __device__ __forceinline__ Copier(uint32_t at, int wave, int lane) : in(lane < kLanes) {
            lds = __builtin_amdgcn_readfirstlane(at + wave * (kBytes / NW));
        }
        // At the wave's view: rows so far apart.
        __device__ __forceinline__ void aim(const TileView& v, int wave, int lane) {
            const bool second = PAIR && wave >= NW / 2;
            const uint32_t ld2 = (uint32_t)v.ld * 2;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int r = (wave * kCopies + i) * kPer + lane / kRowPieces; // (rows of a PAIR's second half from its view's own first)
                piece = (lane % kRowPieces) ^ swizzle(r);
                off[i] = (uint32_t)(second ? r - T / 2 : r) * ld2 + 16 * piece;
            }
        }
        lin_u32x4 range;
        bool far;
        // The step of contraction values c0 .. c0 + 31 of C (none if c0 >= C).
        __device__ __forceinline__ void begin(const TileView& v, int64_t c0, int64_t C) {
            const int64_t left = C - c0;
            if constexpr (LAYOUT == kRows) {
                range = range_of(v.base + c0, left > 0 && v.valid > 0 ? ((v.valid - 1) * v.ld + left) * 2 : 0);
                far = 8 * piece >= left;
            } else {
                range = range_of(v.base + c0 * v.ld, left > 0 ? ((left - 1) * v.ld + v.valid) * 2 : 0);
                far = false;
            }
        }
        __device__ __forceinline__ void one(int i, uint32_t buffer) const {
            if (kLanes == 64 || in) copy16(range, LAYOUT == kRows && far ? kFar : off[i], lds + buffer + i * (kLanes * 16));
        }
    };

    // ---- through registers: aim() at a view, then load() a step's pieces and store() them
    struct Held {
        lin_u32x4 v[kPieces];
    };
    struct Loader {
        int off[kPieces];   // bytes from the step's first value to the lane's piece, moved back into its row where it passes the end
        int moved[kPieces]; // by so many values
        int tid;
        __device__ __forceinline__ Loader(int t) : tid(t) {}
        static __device__ __forceinline__ bool second(int i) { return PAIR && i * (NW * 64) / kRowPieces >= T / 2; } // (uniform)
        __device__ __forceinline__ int row_of(int i) const { return (tid + i * (NW * 64)) / kRowPieces - (second(i) ? T / 2 : 0); }
        __device__ __forceinline__ int at_of(int i) const { return (tid + i * (NW * 64)) % kRowPieces * 8; }
        __device__ __forceinline__ void aim(const TileView* views) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const TileView v = second(i) ? views[1] : views[0];
                const int at = at_of(i), to = LAYOUT == kRows || v.first + v.valid < 8 ? at : min(at, v.valid - 8);
                // (rows that do not exist are read as the last that does: what comes of them is not stored)
                const int row = LAYOUT == kRows ? min(row_of(i), v.valid - 1) : row_of(i);
                off[i] = row * ((int)v.ld * 2) + to * 2;
                moved[i] = at - to;
            }
        }
        // v's values from `by` on, zeros behind.
        static __device__ __forceinline__ lin_u32x4 from(lin_u32x4 v, int by) {
            if (by & 4) v = lin_u32x4{v[2], v[3], 0, 0};
            if (by & 2) v = lin_u32x4{v[1], v[2], v[3], 0};
            if (by & 1) v = lin_u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
            return by < 8 ? v : lin_u32x4{};
        }
        // The step of contraction values c0 .. of C (none if c0 >= C).
        __device__ __forceinline__ void load(const TileView* views, int64_t c0, int64_t C, Held& h) const {
            const int64_t left = C - c0;
            // a row of fewer than 8 values holds no piece to move: value by value
            const bool tiny = LAYOUT == kRows ? C < 8 : views[0].first + views[0].valid < 8;
            if (left >= STEP && !tiny) { // (uniform)
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const TileView& v = second(i) ? views[1] : views[0];
                    const uint8_t* s = (const uint8_t*)(LAYOUT == kRows ? v.base + c0 : v.base + c0 * v.ld);
                    __builtin_memcpy(&h.v[i], s + off[i], 16);
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const TileView& v = second(i) ? views[1] : views[0];
                const int row = row_of(i), at = at_of(i);
                const bool in = LAYOUT == kRows ? row < v.valid && at < left : row < left && at < v.valid;
                lin_u32x4 w = {};
                if (in && tiny) {
                    const uint16_t* s = LAYOUT == kRows ? v.base + row * v.ld + c0 + at : v.base + (c0 + row) * v.ld + at;
                    const int n = (int)min((int64_t)8, LAYOUT == kRows ? left - at : (int64_t)v.valid - at);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < n) w[j / 2] |= (uint32_t)s[j] << (16 * (j % 2));
                } else if (in) {
                    const uint8_t* s = (const uint8_t*)(LAYOUT == kRows ? v.base + c0 : v.base + c0 * v.ld);
                    const int back = LAYOUT == kRows ? max(0, at + 8 - (int)left) : 0;
                    __builtin_memcpy(&w, s + off[i] - 2 * back, 16);
                    w = from(w, back);
                }
                h.v[i] = w;
            }
        }
        __device__ __forceinline__ void store(const Held& h, uint8_t* lds) const {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int p = tid + i * (NW * 64), row = p / kRowPieces, piece = (p % kRowPieces) ^ swizzle(row);
                lin_u32x4 w = h.v[i];
                if (LAYOUT == kCols && moved[i]) w = from(w, moved[i]);
                *(lin_u32x4*)(lds + row * (kRowPieces * 16) + piece * 16) = w;
            }
        }
    };

    // ---- fragments: F of 16 rows (columns) from `first` on
    template <int F> struct Reader {
        uint32_t at[LAYOUT == kRows ? STEP / 32 : F];
        // frag f is rows first + 16 f + lane % 16, c = 32 h + 8 (lane / 16) + 0 .. 7
        __device__ __forceinline__ Reader(int first, int lane) {
            if constexpr (LAYOUT == kRows) {
#pragma unroll
                for (int h = 0; h < STEP / 32; ++h)
                    at[h] = (uint32_t)(first + (lane & 15)) * (STEP * 2) + ((((lane >> 4) + 4 * h) ^ swizzle(lane & 15)) << 4);
            } else {
                const int row = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
                for (int f = 0; f < F; ++f)
                    at[f] = (uint32_t)row * (T * 2) + (((first / 16 + f) * 2 ^ swizzle(row)) << 4) + 8 * (lane & 3);
            }
        }
        // buf: the step's LDS address
        __device__ __forceinline__ lin_s16x8 get(uint32_t buf, int f, int h) const {
            typedef __attribute__((address_space(3))) const lin_s16x8* P8;
            typedef __attribute__((address_space(3))) lin_s16x4* P4;
            if constexpr (LAYOUT == kRows) {
                return *(P8)(uintptr_t)(buf + at[h] + f * (STEP * 32));
            } else {
                const uint32_t a = buf + at[f] + h * (32 * T * 2);
                const lin_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(uintptr_t)a);
                const lin_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(uintptr_t)(a + 4 * T * 2));
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

// A block's shape.  PAIR: the I tile's halves are two matrices' rows of the same features (a gate and its up), and a wave's
// first and second half of fragments belong to them.
template <int TI_, int TJ_, int NWI_, int NWJ_, int STEP_, int RING_, int LI_, int LJ_, bool F16_, bool DIRECT_, bool PAIR_ = false>
struct Shape {
    static constexpr int TI = TI_, TJ = TJ_, NWI = NWI_, NWJ = NWJ_, NW = NWI * NWJ, TH = NW * 64;
    static constexpr int FI = TI / NWI / 16, FJ = TJ / NWJ / 16;
    static constexpr bool F16 = F16_, DIRECT = DIRECT_, PAIR = PAIR_;
    static constexpr int kStep = STEP_, kRing = RING_; // contraction values of a step, steps in LDS
    typedef Tile<TI, LI_, NW, PAIR_, kStep> I;
    typedef Tile<TJ, LJ_, NW, false, kStep> J;
    static constexpr int kBuf = I::kBytes + J::kBytes;
    static constexpr int kLds = NW == 8 ? 3 * I::kBytes + 2 * J::kBytes : kRing * kBuf;
    static constexpr int kWaveI = TI / NWI, kWaveJ = TJ / NWJ;
    // The wave's first I row (fragments of a PAIR: f < FI / 2 from here, the others TI / 2 on).
    static __device__ __forceinline__ int i_first(int wave) { return wave % NWI * kWaveI / (PAIR ? 2 : 1); }
    static __device__ __forceinline__ int j_first(int wave) { return wave / NWI * kWaveJ; }
};

// acc[fi][fj] += the tile's product over steps s0 .. s1 - 1 of one contraction range of C, or two (DUAL): iv[0] and jv[0],
// then iv[1] and jv[1], beginning `turn` steps behind s0 and going round.  (A PAIR has one range, and iv[0], iv[1] are the
// matrices of its halves.)  each(b) is called with every step's J fragments.
template <class S, bool DUAL, class Each>
__device__ __forceinline__ void tile_product(const TileView* iv, const TileView* jv, int64_t C, int s0, int s1, int turn, uint8_t* lds,
                                             lin_f32x4 (&acc)[S::FI][S::FJ], Each each) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int kStep = S::kStep;
    const int per = (int)((C + kStep - 1) / kStep);
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_at(lds));
    typedef typename S::I I;
    typedef typename S::J J;
    constexpr int kCopies = I::kCopies + J::kCopies;
    const typename I::template Reader<S::PAIR ? S::FI / 2 : S::FI> ri(S::i_first(wave), lane);
    const typename J::template Reader<S::FJ> rj(S::j_first(wave), lane);
    typename I::Copier ci(at, wave, lane);
    typename J::Copier cj(at + (S::NW == 8 ? 3 : 1) * I::kBytes, wave, lane);
    typename I::Held hi[2];
    typename J::Held hj[2];
    if (s1 > s0) turn %= s1 - s0;
    // Step `step`'s first contraction value (C behind the last), and whether it is of the second range.
    auto source = [&](int step, int64_t* c0) {
        const int u = step + turn < s1 ? step + turn : step + turn - (s1 - s0);
        const bool second = DUAL && u >= per;
        *c0 = step < s1 ? (int64_t)(second ? u - per : u) * kStep : C;
        return second;
    };
    bool at_i = false, at_j = false; // which range the copies are aimed at
    auto begin_i = [&](int step) {
        int64_t c0;
        const bool second = source(step, &c0);
        const TileView v = pick(S::PAIR ? wave >= S::NW / 2 : second, iv[0], iv[1]);
        if (step == s0 || (DUAL && second != at_i)) ci.aim(v, wave, lane), at_i = second;
        ci.begin(v, c0, C);
    };
    auto begin_j = [&](int step) {
        int64_t c0;
        const bool second = source(step, &c0);
        const TileView v = DUAL ? pick(second, jv[0], jv[1]) : jv[0];
        if (step == s0 || (DUAL && second != at_j)) cj.aim(v, wave, lane), at_j = second;
        cj.begin(v, c0, C);
    };
    auto begin = [&](int step) { begin_i(step), begin_j(step); };
    auto copy = [&](int i, uint32_t buffer) { i < I::kCopies ? ci.one(i, buffer) : cj.one(i - I::kCopies, buffer); };
    typename I::Loader li(tid);
    typename J::Loader lj(tid);
    auto load = [&](int step, int p) {
        int64_t c0;
        const bool second = source(step, &c0);
        const TileView i[2] = {S::PAIR ? iv[0] : pick(second, iv[0], iv[1]), iv[1]}, j = DUAL ? pick(second, jv[0], jv[1]) : jv[0];
        if (step == s0 || (DUAL && second != at_i)) li.aim(i), lj.aim(&j), at_i = second;
        li.load(i, c0, C, hi[p]);
        lj.load(&j, c0, C, hj[p]);
    };
    auto store = [&](uint32_t buffer, int p) {
        li.store(hi[p], lds + buffer);
        lj.store(hj[p], lds + buffer + I::kBytes);
    };
    auto read_i = [&](uint32_t buffer, int f, int h = 0) {
        if (S::PAIR && f >= S::FI / 2) return ri.get(at + buffer + S::TI / 2 * (kStep * 2), f - S::FI / 2, h); // (a PAIR's I is kRows)
        return ri.get(at + buffer, f, h);
    };
    auto read_j = [&](uint32_t buffer, int f, int h = 0) { return rj.get(at + buffer + I::kBytes, f, h); };

    if constexpr (S::NW == 8) {
        static_assert(S::DIRECT, "");
        // Two groups of 4 waves, one wave of each on a SIMD, a phase apart: while one reads half a step, the other
        // multiplies one.  J's fragments of both halves are read with the first, so that the copies of J's step t + 2 can
        // begin in the second half of step t and have six phases to land; I's begin in the first, with a third buffer.
        const bool second = wave >= 4;
        begin(s0);
#pragma unroll
        for (int c = 0; c < I::kCopies; ++c) ci.one(c, 0);
#pragma unroll
        for (int c = 0; c < J::kCopies; ++c) cj.one(c, 0);
        begin(s0 + 1);
#pragma unroll
        for (int c = 0; c < I::kCopies; ++c) ci.one(c, I::kBytes);
#pragma unroll
        for (int c = 0; c < J::kCopies; ++c) cj.one(c, J::kBytes);
        copies_landed<kCopies>();
        if (second) asm volatile("s_barrier" ::: "memory");
        uint32_t mi = 0, mj = 0, then = 2 * I::kBytes;
        lin_s16x8 a[S::FI], b[2][S::FJ];
        for (int t = s0; t < s1; ++t) {
            begin(t + 2);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int f = 0; f < S::FI; ++f) a[f] = read_i(mi, f, h);
                if (h == 0) {
#pragma unroll
                    for (int f = 0; f < 2 * S::FJ; ++f) b[f / S::FJ][f % S::FJ] = rj.get(at + 3 * I::kBytes + mj, f % S::FJ, f / S::FJ);
#pragma unroll
                    for (int c = 0; c < I::kCopies; ++c) ci.one(c, then);
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                } else {
#pragma unroll
                    for (int c = 0; c < J::kCopies; ++c) cj.one(c, mj);
                    copies_landed<kCopies>(); // (of the next step)
                }
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
                each(b[h]);
#pragma unroll
                for (int fi = 0; fi < S::FI; ++fi)
#pragma unroll
                    for (int fj = 0; fj < S::FJ; ++fj) acc[fi][fj] = lin_mfma<S::F16>(a[fi], b[h][fj], acc[fi][fj]);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_barrier" ::: "memory");
            }
            mi = mi == 2 * I::kBytes ? 0 : mi + I::kBytes;
            then = then == 2 * I::kBytes ? 0 : then + I::kBytes;
            mj = J::kBytes - mj;
        }
        if (!second) asm volatile("s_barrier" ::: "memory");
        return;
    }
    constexpr int kRing = S::kRing, kHalves = kStep / 32;
    lin_s16x8 a[2][kHalves][S::FI], b[2][kHalves][S::FJ];
    if constexpr (S::DIRECT) {
#pragma unroll
        for (int i = 0; i < kRing; ++i) {
            begin(s0 + i);
#pragma unroll
            for (int c = 0; c < kCopies; ++c) copy(c, i * S::kBuf);
        }
        copies_landed<(kRing - 1) * kCopies>();
    } else {
        static_assert(S::DIRECT || kRing == 2, "two steps in LDS, two more in registers");
        load(s0, 0), load(s0 + 1, 1);
        store(0, 0), store(S::kBuf, 1);
        load(s0 + 2, 0), load(s0 + 3, 1);
        __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
#pragma unroll
        for (int f = 0; f < S::FI; ++f) a[0][h][f] = read_i(0, f, h);
#pragma unroll
        for (int f = 0; f < S::FJ; ++f) b[0][h][f] = read_j(0, f, h);
    }
    uint32_t mine = 0; // the buffer of step t
    auto step = [&](int t, auto parity) {
        constexpr int p = decltype(parity)::value;
        const uint32_t next = mine + S::kBuf == S::kLds ? 0 : mine + S::kBuf;
        if constexpr (S::DIRECT) {
            copies_landed<(kRing - 2) * kCopies>();
            begin(t + kRing);
        } else {
            __syncthreads();
            store(mine, p); // (every wave has read step t)
            load(t + 4, p);
        }
        // Parts of the step in order: some reads of the next, some copies, a row of products.
        constexpr int kReads = S::FI + S::FJ, kParts = S::FI;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            each(b[p][h]);
#pragma unroll
            for (int fi = 0; fi < kParts; ++fi) {
#pragma unroll
                for (int r = 0; r < kReads; ++r)
                    if (r * kParts / kReads == fi) {
                        if (r < S::FI) a[p ^ 1][h][r] = read_i(next, r, h);
                        else b[p ^ 1][h][r - S::FI] = read_j(next, r - S::FI, h);
                    }
                if constexpr (S::DIRECT)
#pragma unroll
                    for (int c = 0; c < kCopies; ++c)
                        if (c * kParts * kHalves / kCopies == h * kParts + fi) copy(c, mine);
#pragma unroll
                for (int fj = 0; fj < S::FJ; ++fj) acc[fi][fj] = lin_mfma<S::F16>(a[p][h][fi], b[p][h][fj], acc[fi][fj]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        mine = next;
    };
    for (int t = s0; t < s1; t += 2) { // (an odd number's last step multiplies zeros)
        step(t, std::integral_constant<int, 0>());
        step(t + 1, std::integral_constant<int, 1>());
    }
}

// What follows the product, for 4 values at a time: i .. i + 3 of row j of the tile (of a PAIR i runs over one matrix's).  An
// Out has
//   column(i): what is the same for all rows of a lane;
//   More, more(j, i): what is read for 4 values of a row, if reads(); its here() waits for it;
//   store(j, i, v, q, more): v, and of a PAIR the second matrix's q.
// Several rows' reads go out before the first is stored: their latency passes once.  Every wave of the block calls it.
template <class S, class Out>
__device__ __forceinline__ void each_piece(uint8_t* lds, const lin_f32x4 (&acc)[S::FI][S::FJ], int ni, int nj, Out out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int kPieces = S::kWaveI / 4;                               // of a row in LDS
    constexpr int kFit = S::kLds / S::NW / (S::kWaveI * 16 * 4);         // J fragments at a time
    constexpr int kAt = kFit >= S::FJ ? S::FJ : kFit >= 2 ? 2 : 1;
    static_assert(kFit > 0 && S::FJ % kAt == 0, "whole fragments");
    constexpr int kTake = S::PAIR ? kPieces / 2 : kPieces;               // lanes of a row
    static_assert(64 % kTake == 0, "whole rows");
    constexpr int kRowsAt = 64 / kTake, kMost = S::NW == 8 ? 8 : 4, kAhead = kAt * 16 / kRowsAt < kMost ? kAt * 16 / kRowsAt : kMost;
    static_assert(kAt * 16 % (kRowsAt * kAhead) == 0, "whole turns");
    uint8_t* mine = lds + wave * (kAt * 16 * S::kWaveI * 4);
    auto at = [&](int row, int piece) { return (lin_f32x4*)(mine + row * (kPieces * 16) + ((piece ^ (row & 15 & (kPieces - 1))) << 4)); };
    const int piece = lane % kTake, i = S::i_first(wave) + 4 * piece;
    if (i < ni) out.column(i);
    copies_landed<0>(); // of steps behind the last too
    // Without reads apart: a wait for reads in a loop is one for the stores of the turn before, and would be made in both.
    auto rows = [&](int h, auto reads) {
        constexpr bool kReads = decltype(reads)::value;
#pragma unroll 1
        for (int r = 0; r < kAt * 16; r += kRowsAt * kAhead) {
            const int row = r + lane / kTake, j = S::j_first(wave) + 16 * h + row;
            lin_f32x4 v[kAhead], q[kAhead];
            typename Out::More m[kAhead] = {};
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                v[u] = *at(row + u * kRowsAt, piece), q[u] = S::PAIR ? *at(row + u * kRowsAt, piece + kTake) : v[u];
                if (kReads && j + u * kRowsAt < nj && i < ni) m[u] = out.more(j + u * kRowsAt, i);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (kReads) m[u].here(); // (one wait for all: behind the first store it would wait for that as well)
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (j + u * kRowsAt < nj && i < ni) out.store(j + u * kRowsAt, i, v[u], q[u], m[u]);
        }
    };
#pragma unroll
    for (int h = 0; h < S::FJ; h += kAt) {
        if (S::j_first(wave) + 16 * h >= nj) break; // (the wave's other rows lie behind)
#pragma unroll
        for (int fj = 0; fj < kAt; ++fj)
#pragma unroll
            for (int fi = 0; fi < S::FI; ++fi) *at(16 * fj + (lane & 15), 4 * fi + (lane >> 4)) = acc[fi][h + fj];
        __builtin_amdgcn_wave_barrier();
        if (out.reads()) rows(h, std::true_type());
        else rows(h, std::false_type());
        __builtin_amdgcn_wave_barrier();
    }
}
struct NoMore {
    __device__ __forceinline__ void here() {}
};
__device__ __forceinline__ void in_registers(lin_u32x4& v) { asm volatile("" : "+v"(v)); }
// f32 sums of a tile, to a part.
template <bool PAIR> struct PartOut {
    typedef NoMore More;
    float *p, *q;   // at the tile's first value
    int64_t width;  // of a row
    int ni;
    __device__ __forceinline__ void column(int) {}
    static constexpr bool reads() { return false; }
    __device__ __forceinline__ More more(int, int) const { return {}; }
    __device__ __forceinline__ void store(int j, int i, lin_f32x4 v, lin_f32x4 u, More) const;
};

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

// Where a block begins a contraction of so many steps, its XCD's blocks alike or each a step on.
__device__ __forceinline__ int turn_of_block(uint32_t b, int steps, bool apart) {
    return (int)((b % 8) * (uint32_t)steps / 8 + (apart ? b / 8 % 8 : 0));
}

// ---- values -----------------------------------------------------------------------------

template <bool F16> __device__ __forceinline__ float lin_get(uint16_t v) { return F16 ? naiwa_f16_to_f32(v) : naiwa_bf16_to_f32(v); }
template <bool F16> __device__ __forceinline__ uint16_t lin_put(float v) {
    return F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v);
}
// Where value (row + j, col + i) of p lies, rows ld values apart, j < 256: one 32-bit product a lane where row and col are the block's.
__device__ __forceinline__ char* cell(const void* p, int64_t row, int64_t ld, int64_t col, int j, int i, bool f32) {
    const int shift = f32 ? 2 : 1;
    return (char*)p + ((row * ld + col) << shift) + (((uint32_t)j * (uint32_t)ld + (uint32_t)i) << shift);
}
// Up to 4 values from p (n of them), f32 or 16 bits, from any address of their type, as they lie in memory: what is waited for is
// the first use.
__device__ __forceinline__ lin_u32x4 raw_4(const void* p, int n, bool f32) {
    lin_u32x4 o = {};
    if (f32) {
        const uint32_t* s = (const uint32_t*)p;
        if (n >= 4) {
            __builtin_memcpy(&o, s, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) o[i] = s[i];
        }
    } else {
        const uint16_t* s = (const uint16_t*)p;
        if (n >= 4) {
            __builtin_memcpy(&o, s, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) o[i / 2] |= (uint32_t)s[i] << 16 * (i % 2);
        }
    }
    return o;
}
template <bool F16> __device__ __forceinline__ lin_f32x4 wide_4(lin_u32x4 v, bool f32) {
    if (f32) return __builtin_bit_cast(lin_f32x4, v);
    lin_f32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = lin_get<F16>((uint16_t)(v[i / 2] >> 16 * (i % 2)));
    return o;
}
__device__ __forceinline__ lin_f32x4 load_4(const float* p, int n) { return __builtin_bit_cast(lin_f32x4, raw_4(p, n, true)); }
// To an address that is a multiple of ALIGN bytes.  (The empty statements keep the two stores from becoming one.)
template <int ALIGN, class V> __device__ __forceinline__ void put(bool past, void* to, V v) {
    typedef V U __attribute__((aligned(ALIGN)));
    if (past) {
        asm volatile("");
        __builtin_nontemporal_store(v, (U*)to);
        asm volatile("");
    } else {
        *(U*)to = v;
    }
}
template <bool F16> __device__ __forceinline__ void store_4(void* p, int n, bool f32, lin_f32x4 o, bool past = false) {
    if (f32) {
        float* s = (float*)p;
        if (n >= 4) {
            put<4>(past, s, o);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) s[i] = o[i];
        }
    } else {
        typedef __bf16 B __attribute__((ext_vector_type(4)));
        typedef _Float16 H __attribute__((ext_vector_type(4)));
        uint16_t* s = (uint16_t*)p;
        const lin_u16x4 v = F16 ? __builtin_bit_cast(lin_u16x4, __builtin_convertvector(o, H))
                                : __builtin_bit_cast(lin_u16x4, __builtin_convertvector(o, B));
        if (n >= 4) {
            put<2>(past, s, v);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) s[i] = v[i];
        }
    }
}

template <bool PAIR> __device__ __forceinline__ void PartOut<PAIR>::store(int j, int i, lin_f32x4 v, lin_f32x4 u, More) const {
    store_4<false>(cell(p, 0, width, 0, j, i, true), ni - i, true, v);
    if (PAIR) store_4<false>(cell(q, 0, width, 0, j, i, true), ni - i, true, u);
}

// 1 / (1 + exp(-v)): SiLU is v times it, GELU's tanh form v times that of twice tanh's argument (1 + tanh x = 2 / (1 + exp(-2 x))).
// exp as a power of 2 errs by 1.22 |v| + 2 units of 2^-24, the sum by 1, the reciprocal by 2 (and is 0 below 2^-126): in
// the negative tail too, where 1 + tanh x in f32 would have no digits left.
__device__ __forceinline__ float lin_sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }
__device__ __forceinline__ float gelu_twice(float v) { return 1.5957691216057308f * (v + 0.044715f * v * v * v); }

__device__ __forceinline__ float lin_act(int act, float v) {
    if (act == NAIWA_ACT_NONE) return v;
    return v * lin_sigmoid(act == NAIWA_ACT_SILU ? v : gelu_twice(v));
}
// act and its slope.
__device__ __forceinline__ void lin_act_slope(int act, float v, float* a, float* slope) {
    if (act == NAIWA_ACT_NONE) {
        *a = v, *slope = 1.0f;
        return;
    }
    const bool silu = act == NAIWA_ACT_SILU;
    const float s = lin_sigmoid(silu ? v : gelu_twice(v)), d = s * (1.0f - s); // (d is 0 far out, where v * v may be infinite)
    *a = v * s;
    *slope = s + (d > 0.0f ? v * d * (silu ? 1.0f : 1.5957691216057308f * (1.0f + 0.134145f * v * v)) : d);
}

// ---- sums in parts ----------------------------------------------------------------------

// Where a call has few tiles and long sums, `splits` blocks take a tile, each a part of its steps, and leave f32 sums in
// scratch: part z's of plane p (a PAIR has two) [rows][width].  A second launch adds the parts up in their order.
struct Parts {
    float* p;
    int splits, planes;
    int64_t plane; // values of one
    __device__ __forceinline__ float* at(int z, int q) const { return p + ((int64_t)z * planes + q) * plane; }
};

// Blocks of 256 threads that add up the parts of 4 values at a time: f(index, sum) for every index < all, sum(q, i, n) being the
// sum over the parts of plane q's values i .. i + 3 (n of them exist).  G threads share an index, each every G-th part.
template <int G, class F> __device__ __forceinline__ void each_sum(const Parts& parts, uint64_t all, F f) {
    constexpr int Q = 256 / G;
    __shared__ lin_f32x4 sums[G == 1 ? 1 : G][G == 1 ? 1 : Q];
    const int t = threadIdx.x % Q, g = threadIdx.x / Q;
    for (uint64_t b = (uint64_t)blockIdx.x * Q; b < all; b += (uint64_t)gridDim.x * Q) {
        // (with G > 1 all threads come to every sum, and the first of an index goes on with it)
        f(b + t, b + t < all, g == 0, [&](int q, int64_t i, int n, bool in) {
            lin_f32x4 v = {};
            if (in)
                for (int z = g; z < parts.splits; z += G) v += load_4(parts.at(z, q) + i, n);
            if constexpr (G > 1) {
                __syncthreads();
                sums[g][t] = v;
                __syncthreads();
                v = {};
                if (g == 0)
                    for (int x = 0; x < G; ++x) v += sums[x][t];
            }
            return v;
        });
    }
}

// The expert whose rows hold m (at most `rows` rows): -1 if none.
__device__ __forceinline__ int expert_of_row(const uint32_t* offsets, int experts, uint32_t rows, uint32_t m) {
    if (!offsets) return 0;
    int lo = 0, hi = experts; // the last e with offsets[e] <= m
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (offset_at(offsets, mid, rows) <= m) lo = mid;
        else hi = mid - 1;
    }
    return lo < experts && offset_at(offsets, lo, rows) <= m && m < offset_at(offsets, lo + 1, rows) ? lo : -1;
}

// ---- host -------------------------------------------------------------------------------

constexpr int64_t kMaxLd = 1 << 21;
// Results of so many bytes are written past the caches, which cannot hold them (past and through, us: weight gradients in f32 of 64
// experts of 1408 x 2048 286 and 317, 128 of 768 x 1408 113 and 147; 524288 rows x 576 x 64 in bf16 352 and 378), unless they are added
// to what was there and so read first (474 and 467).
constexpr int64_t kLinPast = 256 << 20;
constexpr int kMaxExperts = 4096;

static inline bool lin_aligned(const void* p, int64_t ld, int64_t stride) {
    return !(((uintptr_t)p & 15) | (ld & 7) | (stride & 7));
}
// Rows at addresses that are no multiples of 4 bytes.
static inline bool lin_odd(const void* p, int64_t ld, int64_t stride) { return ((uintptr_t)p & 3) | (ld & 1) | (stride & 1); }
static inline int lin_size(int dtype) { return dtype == NAIWA_F32 ? 4 : 2; }
// How many blocks take a tile of `steps` steps in a call of `tiles` tiles whose sums are `values` f32 values: a block a CU, of 8
// steps at least, or of long sums two, and at most 64 MB of parts.  (One block a tile, 16 rows x 88 x 728 and 1 x 128 x 3424
// took 28 and 38 us, a step's latency each.  Two blocks a CU instead of one: the input gradient of 16 rows x 4096 x 14336 33 and
// 27 us, 1024 rows x 2048 x 2048, of 64 steps in all, 25 and 28.)
static inline int lin_splits(int64_t tiles, int64_t steps, int64_t values) {
    tiles = std::max<int64_t>(tiles, 1);
    const int64_t one = std::min(256 / tiles, steps / 8), two = std::min(512 / tiles, steps / 24);
    const int64_t s = std::min<int64_t>({std::max(one, two), 256, (16 << 20) / std::max<int64_t>(values, 1)});
    return s < 2 ? 1 : (int)s;
}
static inline int lin_parts(int splits, int planes, int64_t plane, hipStream_t st, Parts* p) {
    *p = Parts{nullptr, splits, planes, plane};
    if (splits == 1) return NAIWA_OK;
    int rc = 0;
    p->p = (float*)naiwa_scratch_of_stream(NAIWA_SCRATCH_LINEAR, (size_t)splits * planes * plane * 4, &rc, st);
    return p->p ? NAIWA_OK : rc;
}
// Blocks of 256 threads that finish so many quads of sums, `group` threads each.
static inline unsigned lin_finish_blocks(int64_t quads, int group) {
    return (unsigned)std::min<int64_t>((quads * group + 255) / 256, 1 << 16);
}
constexpr int64_t kManySteps = 2500; // steps of 64 of 256 x 256 tiles, 10 a CU
// Which blocks a call takes: 4 waves on 128 x 32 (steps of 64), on 128 x 128 with a ring of 2 or of 4, 8 waves on 256 x 256.
enum { kThin, kShort, kMid, kBig, kKinds };
// For a contraction of so many values, segments of `rows` rows on average and `tiles` 256 x 256 tiles; `packed`: few enough of
// the tiles' places are empty.  Segments lie on the device, so their average speaks for all of them: the figures here are of
// segments of unequal popularity (logits N(0, 0.5) apart).  With all 2048 rows of 64 experts of 1408 x 2048 one expert's, their
// forward and input gradient take 34 and 32 in thin tiles, one matrix's 32 in 128 x 128.  All times in us.
// - 32 rows or fewer: thin blocks hold less of nothing, so that a step copies and multiplies 160 rows and not 256, and have 64
//   values of a weight's row a step in flight and not 32, two a CU like 128 x 128 (thin and 128 x 128: gated, 64
//   experts of 1408 x 2048 with 16 rows each 136 and 150, 8 of 14336 x 4096 329 and 363, one of 14336 x 4096 22 and 26; 48 rows 180
//   and 173, 458 and 413; input gradients of 60 experts of 1000 x 1000 with 16 rows 24 and 29).
// - A short sum hardly goes round a ring of 4, and a ring of 2 leaves room for three blocks and not two, whose epilogues overlap (ring of 2,
//   of 4, and 256 x 256: 16384 rows x 4096 x 64 62, 87 and 89, 7827 x 1392 x 392 28, 34 and 30, 16 experts of 576 x 1704 with 850 rows
//   67, 75 and 55, input gradients of 64 experts of 368 x 608 with 1946 rows 134, 145 and 153, 1551 x 672 x 2520 20, 21 and 28).
// - 256 x 256 where tiles are many or their sums long (128 and 256 wide: 1043 rows x 2920 x 584 gated 23 and 27, 555 rows of 16
//   experts of 96 x 5488 60 and 46, 1024 rows x 2048 x 2048 25 and 31, 4096 48 and 52, 512 rows x 4096 x 14336 91 and 70, 2048
//   277 and 188; gated, 64 experts of 1408 x 2048 with 96 rows 201 and 189, 512 590 and 444).
static inline int lin_kind(int64_t contraction, int64_t rows, int64_t tiles, bool packed) {
    const int64_t steps = (contraction + 63) / 64;
    if (rows <= 32 && contraction >= 256) return kThin;
    if (steps <= 9) return kShort;
    return packed && tiles * steps >= kManySteps ? kBig : kMid;
}
// Rows that are not aligned pass registers, which leave a CU two blocks of 128 x 128, three of 128 x 64: the narrow ones with 64
// rows a segment or fewer (narrow and wide, us: 64 experts of 1407 x 2049 with 64 rows each 131 and 150, 128 203 and 168, input
// gradients 113 and 148, 169 and 164).
static inline bool lin_narrow(int64_t rows) { return rows <= 64; }
// J tiles of `tile` rows that segments of `rows` rows have in all, if they are alike.
static inline int64_t lin_j_alike(int64_t rows, int experts, bool grouped, int tile) {
    return grouped ? std::max<int64_t>(std::min<int64_t>(experts, rows), rows / tile) : (rows + tile - 1) / tile;
}
// J tiles of `tile` rows that segments of `rows` rows may have.
static inline int64_t lin_j_tiles(int64_t rows, int experts, bool grouped, int tile) {
    return grouped ? rows / tile + std::min<int64_t>(experts, rows) : (rows + tile - 1) / tile;
}
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
static inline Span lin_span(const uint32_t* offsets, int experts) { return span_of(offsets, ((int64_t)experts + 1) * 4); }
// From the first weight to the last.
static inline Span lin_span(const naiwa_weights* w) {
    return w ? span_of(w->w, ((w->experts - 1) * lin_stride(w) + (w->n - 1) * lin_ld(w) + w->k) * 2) : Span{};
}

} // namespace
