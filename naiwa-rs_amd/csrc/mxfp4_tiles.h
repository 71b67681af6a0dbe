// The MXFP4 experts of more than one token: tiles of up to 64 sorted pairs of one slot
// against strips of weights, on v_mfma_scale_f32_32x32x64_f8f6f4 (included by
// mxfp4_experts.hip).
//
// A block of 4 waves takes one tile; a wave takes NA tiles of 32 weight rows (half of them
// gate and half up rows, or down rows) and both halves of the tile's tokens.  A operand:
// FP4, lane l holds block l / 32 of a 64-value step of row l % 32, 16 bytes straight from the
// tile order in memory to registers.  B operand: one E2M3 plane, lane l block l / 32 of token
// l % 32, from LDS.  Accumulator v of lane l is D[8 (v / 4) + 4 (l / 32) + v % 4][l % 32]: row,
// token.
//
// The planes' rows (of x by token, of h by sorted pair) go to LDS by DMA in chunks of 128
// values: of 64 rows two chunks deep, of 32 (a tile of at most 32 pairs, which HBM bounds)
// four.  A row's chunk is 3 classes of 2 P pieces of 16 bytes: the first 16 bytes of every plane of blocks 0 and 2 (class 0) and of blocks 1 and 3 (class 1), step by
// step; and the last 8 bytes of a plane of both blocks of a step (class 2).  In LDS a class is
// groups of 4 pieces (and 2 for the rest), [token][piece], the piece number xored with bits of
// the token so that 16 neighbouring tokens' reads of one piece fall on distinct banks, while
// 4 neighbouring lanes of a copy read 64 contiguous bytes.
//
// Bound.  Few tokens an expert: HBM, the weights are read once, at the rates that stand at the
// kernels (reads alone are not held to a copy's 5.1 TB/s).  Many: the scaled products and the
// power they draw; 4096 tokens at Mixtral sizes run 1.8 + 1.2 ms, 4.3 and 3.9 PFLOP/s of FP4 x
// E2M3, where the same products from registers alone reach 6 to 7 with random codes and 9.9 with
// zeros, the chip's full rate: its power is the limit.  Without the weights' loads gate/up takes
// 17 % less, without the copies 14 %, without the LDS reads no less.
// Between (about 50 tokens of small experts): the memory's and the products' times, which two blocks
// a CU overlap in part, and 1.7 rounds of blocks with 10 us of first loads and epilogue each.
// Set aside: 128 weight rows a wave (one block a CU), 18 to 25 % slower; three blocks a CU (the
// compiler spills), 20 % slower; planes of 24 contiguous bytes, three pieces read for two planes
// (register moves), 3 to 6 % slower; three chunks of 64 rows in LDS, no faster.
#pragma once

#include <type_traits>

// lane i of the wave copies 16 bytes from base + off to lds + 16 i.  Issued as inline assembly
// so that the compiler does not make every later LDS read wait for every copy in flight; each
// read of copied data follows an explicit vmcnt wait of the issuing wave and a barrier.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(size_t)(__attribute__((address_space(3))) const void*)p);
}
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
// All but the last N copies and loads of this wave have landed, and every wave is here.
template <int N> __device__ __forceinline__ void landed_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A value that every lane has, in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

constexpr int kTile = 64; // pairs a tile

struct Tiles {
    int4* t; // {first sorted position, pairs (at most kTile, 0: no tile), slot}, 8 runs of `run`
    int run;
};

// The sorted pairs cut into tiles of up to 64 pairs of one slot, by one block of kThreads: dealt to
// the runs in order, as evenly as they go.
__device__ inline void tiles_block(const uint32_t* offsets, int slots, Tiles t) {
    __shared__ int part[kThreads];
    const int tid = threadIdx.x, per = (slots + kThreads - 1) / kThreads;
    const int s0 = min(slots, tid * per), s1 = min(slots, s0 + per);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += (int)((offsets[s + 1] - offsets[s] + kTile - 1) / kTile);
    part[tid] = mine;
    for (int i = tid; i < 8 * t.run; i += kThreads) t.t[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    for (int m = 1; m < kThreads; m <<= 1) {
        const int v = tid >= m ? part[tid - m] : 0;
        __syncthreads();
        part[tid] += v;
        __syncthreads();
    }
    int at = part[tid] - mine;
    const int all = part[kThreads - 1];
    for (int s = s0; s < s1; ++s) {
        const int b = (int)offsets[s], n = (int)(offsets[s + 1] - offsets[s]);
        // the fewest tiles, of about equal numbers of 32-pair halves
        const int subs = (n + 31) / 32, nt = (n + kTile - 1) / kTile;
        for (int j = 0; j < nt; ++j, ++at) {
            const int m0 = 32 * (subs * j / nt), m1 = min(n, 32 * (subs * (j + 1) / nt));
            const int x = (8 * (at + 1) - 1) / all; // run x holds tiles all x / 8 .. all (x + 1) / 8 - 1
            t.t[x * t.run + at - all * x / 8] = make_int4(b + m0, m1 - m0, s, 0);
        }
    }
}

// The tile and column of block b of a grid of 8 * run * ncol.  xcd: blocks are dealt to the 8 XCDs
// round-robin (block b to XCD b % 8), and each XCD takes a run of tiles, all columns of one after
// the other; otherwise column by column within a tile.
__device__ __forceinline__ int4 tile_col(int b, Tiles t, int ncol, int xcd, int* col) {
    const int r = xcd ? b >> 3 : b;
    *col = r % ncol;
    const int4 v = t.t[(xcd ? (b & 7) * t.run : 0) + r / ncol];
    return make_int4(uniform(v.x), uniform(v.y), uniform(v.z), 0);
}

// One chunk of 32 NH rows in P planes.
template <int P, int NH> struct Stage {
    static constexpr int kRows = 32 * NH;
    static constexpr int kFour = 2 * P / 4, kTwo = 2 * P % 4 / 2; // groups of 4 pieces and of 2, per class
    static constexpr int kClass = kRows * 32 * P;
    __align__(16) uint8_t v[3 * kClass];
};
// LDS of a tile kernel: the same for either.
template <int P> constexpr size_t kStageBytes = 2 * sizeof(Stage<P, 2>);
static_assert(2 * sizeof(Stage<5, 2>) == 4 * sizeof(Stage<5, 1>), "two chunks of 64 rows or four of 32");

// The wave's copies of chunk t to `st`.  NH = 2: both groups of 4 pieces for tokens 16 wave ..
// + 15; NH = 1: one of them, for tokens 16 (wave & 1) .. + 15.  Groups of 2 for 32 tokens: NH =
// 2, of classes 0 and 2 by waves 0 and 1, of class 1 by waves 2 and 3, twice; NH = 1, of class 0,
// 1, 2, 2 by wave 0 .. 3.  Every wave has as many copies, so that no branch divides them.
// off4, off2: the byte offsets of the lane's rows, its piece's included.
template <int P, int NH>
__device__ __forceinline__ void stage(uint8_t* st, const uint8_t* base, uint32_t off4, uint32_t off2, int t, int wave) {
    using S = Stage<P, NH>;
    static_assert(S::kFour == 2);
    const uint32_t lds = lds_addr(st), at = (uint32_t)t * (96 * P);
#pragma unroll
    for (int c = 0; c < 3; ++c) {
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const int g = NH == 2 ? i : wave >> 1;
            dma16(base, off4 + at + 32 * P * c + 64 * g,
                  lds + S::kClass * c + 64 * S::kRows * g + 1024 * (NH == 2 ? wave : wave & 1));
        }
    }
    if (S::kTwo) {
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const int c = NH == 1 ? min(wave, 2) : wave < 2 ? 2 * i : 1;
            dma16(base, off2 + at + 32 * P * c + 64 * S::kFour,
                  lds + S::kClass * c + 64 * S::kRows * S::kFour + (NH == 2 ? 1024 * (wave & 1) : 0));
        }
    }
}

// A lane's place in a Stage: piece i of a class for token `tok`.
template <int P, int NH> __device__ __forceinline__ int piece_at(int tok, int i) {
    using S = Stage<P, NH>;
    return i < 4 * S::kFour ? 64 * S::kRows * (i / 4) + 64 * tok + 16 * ((i & 3) ^ ((tok >> 2) & 3))
                            : 64 * S::kRows * S::kFour + 32 * tok + 16 * ((i - 4 * S::kFour) ^ ((tok >> 3) & 1));
}

// Plane k % P of the lane's block of step k / P, token `tok`.
template <int P, int NH> __device__ __forceinline__ v6u staged_plane(const uint8_t* v, int par, int tok, int k) {
    const v4u head = *(const v4u*)(v + Stage<P, NH>::kClass * par + piece_at<P, NH>(tok, k));
    const v2u tail = *(const v2u*)(v + Stage<P, NH>::kClass * 2 + piece_at<P, NH>(tok, k) + 8 * par);
    return v6u{head.x, head.y, head.z, head.w, tail.x, tail.y};
}

// acc[i][s] += weight tile i x token half s < NH over all of K.  wp[i]: the tile's first strip, the
// same for every lane; strip: bytes to its second.  to_row(row(token)): the token's row of x (row
// may load; it is waited for when the first weights are on the way).  A chunk's operands (step,
// half, plane) are read from LDS one ahead of the products.
// Loads and copies end in the order of their issue.  Before chunk t its copies have to have
// landed; the wave issued since then at least the weights of chunk t + 1 (NH = 2), or those of
// chunk t and the copies and weights of chunks t + 1 and t + 2 (NH = 1): kUnder may be under way.
// The first weights are issued before the first copies, so fewer follow those: `first` of them.
// The loop issues them without branches, of the last chunk again where there are no more, since
// the compiler waits for every load where paths with different loads meet; the last group
// (which may be the first) issues what there is and waits for everything from its second chunk on.  The empty asm makes
// the compiler wait for the weights before the next loads are issued: it does not know of
// the copies, and a later wait of its own would count them among the weights.
template <int NA, int P, int NH, class R, class T>
__device__ __forceinline__ void tile_dot(uint8_t* st, const uint8_t* base, const Planes& x, R row, T to_row,
                                         const uint8_t* const (&wp)[NA], uint32_t strip, const uint8_t* xs, int steps,
                                         int lane, int wave, v16f (&acc)[NA][2]) {
    // D chunks of the rows and DA of the weights are in LDS and registers or on the way
    constexpr int D = NH == 1 ? 4 : 2, DA = NH == 1 ? 4 : 3, kCopies = P == 5 ? 4 : 3;
    constexpr int kUnder = NH == 1 ? 2 * NA + 2 * (kCopies + 2 * NA) : 2 * NA;
    constexpr uint32_t kStage = sizeof(Stage<P, NH>);
    const int par = lane >> 5, tok = lane & 31;
    // the tokens whose rows the lane copies, and those of its scales
    const int tok4 = 16 * (NH == 2 ? wave : wave & 1) + (lane >> 2), tok2 = 32 * (NH == 2 ? wave & 1 : 0) + (lane >> 1);
    const uint32_t r4 = row(tok4), r2 = row(tok2);
    uint32_t rx[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) rx[h] = row(32 * h + tok);
    // the lane's 16 bytes of weights and 4 of scales: row lane % 16 of a strip, block par
    const uint32_t lw = ((lane >> 4) & 1) * strip + 256 * par + 16 * (lane & 15);
    const uint32_t ls = ((lane >> 4) & 1) * strip + 64 * par + 4 * (lane & 15);
    v4u a[4][2][NA]; // [chunk mod 4][step of the chunk][tile]
    auto load_a = [&](int t, v4u(&o)[2][NA]) {
        t = min(t, steps - 1);
        const int64_t at = (int64_t)1024 * t + 256 * (t >> 2);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < NA; ++i) o[s][i] = *(const v4u*)(wp[i] + at + lw + 512 * s);
    };
    // the lane's scale bytes of a group of 4 chunks: a byte a chunk, blocks par and 2 + par
    struct Scales {
        uint32_t a[NA][2], b[NH][2];
    };
    const int groups = (steps + 3) / 4;
    auto scales_a = [&](int g, Scales& o) {
        const int64_t sc = (int64_t)1024 * min(4 * g + 4, steps) + 256 * g;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < NA; ++i) o.a[i][s] = *(const uint32_t*)(wp[i] + sc + ls + 128 * s);
    };
    Scales sc, next;
#pragma unroll
    for (int t = 0; t < DA - 1; ++t) load_a(t, a[t]);
    scales_a(0, sc);
    __builtin_amdgcn_sched_barrier(0); // the weights first, then what waits for the rows' numbers
    const uint32_t off4 = to_row(r4) * (uint32_t)x.row + 16 * ((lane & 3) ^ ((tok4 >> 2) & 3));
    const uint32_t off2 = to_row(r2) * (uint32_t)x.row + 16 * ((lane & 1) ^ ((tok2 >> 3) & 1));
    uint32_t xo[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) xo[h] = to_row(rx[h]) * (uint32_t)x.groups * 16 + 4 * par;
    auto copy = [&](int t, int buffer) {
        stage<P, NH>(st + kStage * buffer, base, off4, off2, min(t, steps - 1), wave);
    };
    auto scales_b = [&](int g, Scales& o) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int h = 0; h < NH; ++h) o.b[h][s] = *(const uint32_t*)(xs + 16 * g + xo[h] + 8 * s);
    };
#pragma unroll
    for (int t = 0; t < D - 1; ++t) copy(t, t);
    scales_b(0, sc);
    const int last = (steps - 1) / 4; // the last group, of 1 to 4 chunks
    auto chunk = [&](auto j, auto in_last, int g) {
        constexpr int J = decltype(j)::value;
        constexpr bool kLast = decltype(in_last)::value;
        const int t = 4 * g + J;
        constexpr int first = NH == 1 ? 2 * kCopies + 2 * NA * J : 0;
        if (kLast)
            landed_barrier<J ? 0 : first>();
        else if (g == 0 && J < (NH == 1 ? 3 : 1))
            landed_barrier<first>();
        else
            landed_barrier<kUnder>();
#pragma unroll
        for (int i = 0; i < NA; ++i) asm volatile("" : "+v"(a[J][0][i]), "+v"(a[J][1][i]));
        if constexpr (J == 0 && !kLast) {
            scales_a(min(g + 1, groups - 1), next);
            scales_b(min(g + 1, groups - 1), next);
        }
        if constexpr (J == 3 && !kLast) {
#pragma unroll
            for (int i = 0; i < NA; ++i) asm volatile("" : "+v"(next.a[i][0]), "+v"(next.a[i][1]));
#pragma unroll
            for (int h = 0; h < NH; ++h) asm volatile("" : "+v"(next.b[h][0]), "+v"(next.b[h][1]));
        }
        if (!kLast || t + D - 1 < steps) copy(t + D - 1, (J + D - 1) % D);
        if (!kLast || t + DA - 1 < steps) load_a(t + DA - 1, a[(J + DA - 1) % 4]);
        __builtin_amdgcn_sched_barrier(0); // the loads first
        const uint8_t* v = st + kStage * (J % D);
        v6u b[2];
        b[0] = staged_plane<P, NH>(v, par, tok, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int o = 0; o < 2 * NH * P; ++o) {
            const int s = o / (NH * P), h = o / P % NH, p = o % P;
            if (o + 1 < 2 * NH * P) {
                const int n = o + 1, k = n / (NH * P) * P + n % P;
                b[n & 1] = staged_plane<P, NH>(v, par, 32 * (n / P % NH) + tok, k);
            }
#pragma unroll
            for (int i = 0; i < NA; ++i)
                acc[i][h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                    fp4_operand(a[J][s][i]), e2m3_operand(b[o & 1]), acc[i][h], 4, 2, J, (int)sc.a[i][s], J,
                    (int)(sc.b[h][s] - 0x05050505u * p));
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, NA, 0);
        }
    };
    const std::integral_constant<int, 0> c0;
    const std::integral_constant<int, 1> c1;
    const std::integral_constant<int, 2> c2;
    const std::integral_constant<int, 3> c3;
    for (int g = 0; g < last; ++g) {
        chunk(c0, std::false_type{}, g);
        chunk(c1, std::false_type{}, g);
        chunk(c2, std::false_type{}, g);
        chunk(c3, std::false_type{}, g);
        sc = next;
    }
    const int rest = steps - 4 * last;
    chunk(c0, std::true_type{}, last);
    if (rest > 1) chunk(c1, std::true_type{}, last);
    if (rest > 2) chunk(c2, std::true_type{}, last);
    if (rest > 3) chunk(c3, std::true_type{}, last);
    if (rest == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // copies of no use: LDS ends with the block
    // the results stay where every lane computes them
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int h = 0; h < NH; ++h) asm volatile("" : "+v"(acc[i][h]));
}

// Gate/up of a tile: a wave's NA / 2 blocks of 32 features, gate and up; h in PH planes.
// 16 tokens at Mixtral-8x7B sizes 94 us (5.3 TB/s), 96 at Qwen3-30B sizes 40 us (5.3 TB/s), 4096 at
// Mixtral sizes 1.79 ms (1.07 PFLOP/s in 4 planes).
template <int NA, int P, int PH>
__global__ void __launch_bounds__(kThreads, 2)
tile_gateup_kernel(Bank gate, Bank up, Planes x, int H, int I, int width, const uint32_t* perm, Tiles tl, int act, int xcd,
                   Planes h) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int NF = NA / 2; // feature blocks a wave
    const int blocks = 4 * naiwa_mx_steps(I), ncol = (blocks + 4 * NF - 1) / (4 * NF);
    int col;
    const int4 tile = tile_col(blockIdx.x, tl, ncol, xcd, &col);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int start = tile.x, cnt = tile.y, slot = tile.z;
    if (cnt == 0) return;
    auto pair = [&](int tok) -> uint32_t { return perm[start + min(tok, cnt - 1)]; };
    auto token = [&](uint32_t p) -> uint32_t { return p / (uint32_t)width; };
    const int fb0 = (4 * col + wave) * NF; // the wave's first feature block
    const uint8_t* wp[NA];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const int fb = min(fb0 + f, I / 32 - 1); // blocks past I read the last one again
        wp[f] = gate.base + (int64_t)slot * gate.stride + 2 * fb * gate.strip;
        wp[NF + f] = up.base + (int64_t)slot * up.stride + 2 * fb * up.strip;
    }
    v16f acc[NA][2] = {};
    const int steps = naiwa_mx_steps(H);
    const uint32_t strip = (uint32_t)gate.strip;
    if (cnt > 32)
        tile_dot<NA, P, 2>(smem, x.base, x, pair, token, wp, strip, x.scales, steps, lane, wave, acc);
    else
        tile_dot<NA, P, 1>(smem, x.base, x, pair, token, wp, strip, x.scales, steps, lane, wave, acc);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        const int fb = fb0 + f;
        if (fb >= blocks) break;
        // both halves of the tile's tokens: afterwards a lane holds the 32 features of token `lane`
        float v[32];
        auto fold = [&](auto f_act) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int s = 0; s < 2; ++s) acc[f][s][i] = f_act(acc[f][s][i]) * acc[NF + f][s][i];
        };
        if (act == NAIWA_ACT_GELU_PYTORCH_TANH) // one branch, not one a value
            fold([](float g) { return naiwa_gelu_tanh(g); });
        else
            fold([](float g) { return naiwa_silu(g); });
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float a = acc[f][0][i], b = acc[f][1][i];
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
            v[8 * (i / 4) + i % 4] = __uint_as_float(sw[0]);
            v[8 * (i / 4) + 4 + i % 4] = __uint_as_float(sw[1]);
        }
        if (32 * fb >= I)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.0f;
        const int sb = scale_byte(abs_max(v));
        v6u o[PH];
        to_planes<PH>(v, sb, o);
        if (lane < cnt)
            put_block<PH>(h.base + (int64_t)(start + lane) * h.row, h.scales + (int64_t)(start + lane) * h.groups * 16, fb, o, sb);
    }
}

// Down of a tile and a K part of part_groups groups of 4 steps: NA tiles of 32 rows a wave;
// y[part][pair][H] unweighted.  16 tokens at Mixtral-8x7B sizes 48 us (5.2 TB/s), 4096 1.23 ms
// (0.78 PFLOP/s in 5 planes).
template <int NA, int P>
__global__ void __launch_bounds__(kThreads, 2)
tile_down_kernel(Bank down, Planes h, int H, int I, int64_t n, int part_groups, const uint32_t* perm, Tiles tl, int xcd,
                 float* y) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int blocks = H / 32, ncol = (blocks + 4 * NA - 1) / (4 * NA);
    int col;
    const int4 tile = tile_col(blockIdx.x, tl, ncol, xcd, &col);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int start = tile.x, cnt = tile.y, slot = tile.z;
    if (cnt == 0) return;
    auto row = [&](int tok) -> uint32_t { return (uint32_t)min(tok, cnt - 1); };
    auto same = [](uint32_t r) { return r; };
    const int rb0 = (4 * col + wave) * NA, g0 = blockIdx.y * part_groups;
    const int steps = min(naiwa_mx_steps(I) - 4 * g0, 4 * part_groups);
    const uint8_t* wp[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i)
        wp[i] = down.base + (int64_t)slot * down.stride + 2 * min(rb0 + i, blocks - 1) * down.strip + (int64_t)4352 * g0;
    const uint8_t* hs = h.scales + (int64_t)start * h.groups * 16 + 16 * g0;
    v16f acc[NA][2] = {};
    const uint8_t* rows = h.base + (int64_t)start * h.row + (int64_t)4 * g0 * 96 * P;
    const uint32_t strip = (uint32_t)down.strip;
    if (cnt > 32)
        tile_dot<NA, P, 2>(smem, rows, h, row, same, wp, strip, hs, steps, lane, wave, acc);
    else
        tile_dot<NA, P, 1>(smem, rows, h, row, same, wp, strip, hs, steps, lane, wave, acc);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int tok = 32 * s + (lane & 31);
        if (tok >= cnt) break;
        float* dst = y + (blockIdx.y * n + perm[start + tok]) * H + 4 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (rb0 + i < blocks)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(v4f*)(dst + 32 * (rb0 + i) + 8 * q) =
                        v4f{acc[i][s][4 * q], acc[i][s][4 * q + 1], acc[i][s][4 * q + 2], acc[i][s][4 * q + 3]};
    }
}
