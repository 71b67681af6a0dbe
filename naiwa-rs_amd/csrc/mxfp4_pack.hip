// MXFP4 quantisation to tile order and back (include/naiwa_mxfp4.h).
//
// A block of 256 threads takes 16 rows x 512 values: one strip's group of 4 steps.
// Four neighbouring lanes share a 32-value block, 8 values each, so a wave covers 4 rows
// x 128 values of a step and reads 256 contiguous bytes of each 16-bit row; the block's
// largest magnitude meets over the four lanes in two DPP moves.  The codes are one
// hardware conversion per two values (round to nearest even, saturating at 6) after an
// exact multiplication by the inverse scale.  The 256 scale bytes of the group meet in
// LDS.  Bound: HBM, every value is read once and written once: 128 bf16 projections of 768 x
// 2048 116 us to MXFP4 (403 MB in, 107 MB out: 4.4 TB/s) and 75 us back (6.8 TB/s); one
// projection 3.5 us either way, the launch.
#include "../../include/naiwa_mxfp4.h"
#include "mxfp4.h"

#include <string.h>

namespace {

constexpr int kThreads = 256;
// Blocks of a launch: HIP takes fewer than 2^32 threads along a dimension.
constexpr int64_t kLaunch = 1 << 23;

// 8 values of a row from p as f32; T: float, or uint16_t holding bf16 (DT NAIWA_BF16) or f16.
template <int DT>
__device__ __forceinline__ void load8(const void* p, float (&f)[8]) {
    if constexpr (DT == NAIWA_F32) {
        const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
        const uint4 v = *(const uint4*)p;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = DT == NAIWA_BF16 ? naiwa_bf16_to_f32(w[i] & 0xffffu) : naiwa_f16_to_f32(w[i] & 0xffffu);
            f[2 * i + 1] = DT == NAIWA_BF16 ? naiwa_bf16_to_f32(w[i] >> 16) : naiwa_f16_to_f32(w[i] >> 16);
        }
    }
}

// Group number b of a launch: projection, strip, group of steps.
struct Where {
    int64_t strips, groups, first;
    __device__ __forceinline__ void split(int64_t b, int64_t& proj, int64_t& strip, int& group) const {
        b += first;
        group = (int)(b % groups);
        strip = b / groups % strips;
        proj = b / groups / strips;
    }
};

template <int DT>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const uint8_t* src, Where wh, int k, int64_t ld, int64_t src_stride, uint8_t* dst, int64_t dst_stride) {
    __shared__ __align__(16) uint8_t sc[256];
    constexpr int S = DT == NAIWA_F32 ? 4 : 2;
    int64_t proj, strip;
    int group;
    wh.split(blockIdx.x, proj, strip, group);
    const int tid = threadIdx.x, lane = tid & 63, q = lane & 3, kb = (lane >> 2) & 3, r = 4 * (tid >> 6) + (lane >> 4);
    const int steps = min(4, naiwa_mx_steps(k) - 4 * group);
    const uint8_t* row = src + (proj * src_stride + (16 * strip + r) * ld) * S;
    uint8_t* out = dst + proj * dst_stride + strip * naiwa_mx_strip_bytes(k) + (int64_t)group * 4352;
    float f[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = 512 * group + 128 * j + 32 * kb + 8 * q;
        if (at < k)
            load8<DT>(row + (int64_t)at * S, f[j]);
        else
            for (int i = 0; i < 8; ++i) f[j][i] = 0.0f;
    }
    uint32_t bytes = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // magnitudes compared as integers: a NaN is larger than every number
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[j][i]) & 0x7fffffffu);
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
        const int e = (int)(m >> 23);
        const bool bad = e == 255;
        const int s = bad ? 255 : max(0, e - 2);
        // 2^(127 - s): a normal number, 2^-125 at the largest finite exponent
        const float inv = __uint_as_float((uint32_t)(bad ? 127 : 254 - s) << 23);
        uint32_t codes = 0;
        if (!bad) {
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[j][0] * inv, f[j][1] * inv, 1.0f, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[j][2] * inv, f[j][3] * inv, 1.0f, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[j][4] * inv, f[j][5] * inv, 1.0f, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[j][6] * inv, f[j][7] * inv, 1.0f, 3);
        }
        if (j < steps) *(uint32_t*)(out + 1024 * j + 16 * (16 * kb + r) + 4 * q) = codes;
        const bool in = j < steps && 512 * group + 128 * j + 32 * kb < k;
        bytes |= (in ? (uint32_t)s : 0u) << (8 * j);
    }
    if (q == 0) *(uint32_t*)(sc + 4 * (16 * kb + r)) = bytes;
    __syncthreads();
    if (tid < 16) *(uint4*)(out + 1024 * steps + 16 * tid) = *(const uint4*)(sc + 16 * tid);
}

// The same split; a thread turns 4 bytes of codes into 8 values.
template <int DT>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t* src, Where wh, int k, int64_t src_stride, uint8_t* dst, int64_t ld,
                  int64_t dst_stride) {
    constexpr int S = DT == NAIWA_F32 ? 4 : 2;
    int64_t proj, strip;
    int group;
    wh.split(blockIdx.x, proj, strip, group);
    const int tid = threadIdx.x, lane = tid & 63, q = lane & 3, kb = (lane >> 2) & 3, r = 4 * (tid >> 6) + (lane >> 4);
    const int steps = min(4, naiwa_mx_steps(k) - 4 * group);
    const uint8_t* in = src + proj * src_stride + strip * naiwa_mx_strip_bytes(k) + (int64_t)group * 4352;
    uint8_t* row = dst + (proj * dst_stride + (16 * strip + r) * ld) * S;
    const uint32_t bytes = *(const uint32_t*)(in + 1024 * steps + 4 * (16 * kb + r));
    uint32_t codes[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        codes[j] = j < steps ? *(const uint32_t*)(in + 1024 * j + 16 * (16 * kb + r) + 4 * q) : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = 512 * group + 128 * j + 32 * kb + 8 * q;
        if (at >= k) break;
        const int s = (int)((bytes >> (8 * j)) & 255u);
        typedef float float2v __attribute__((ext_vector_type(2)));
        float f[8];
        float2v v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], 1.0f, 0);
        f[0] = v[0], f[1] = v[1];
        v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], 1.0f, 1);
        f[2] = v[0], f[3] = v[1];
        v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], 1.0f, 2);
        f[4] = v[0], f[5] = v[1];
        v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], 1.0f, 3);
        f[6] = v[0], f[7] = v[1];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            f[i] = s == 255 ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(f[i], s - 127);
        if constexpr (DT == NAIWA_F32) {
            ((float4*)(row + (int64_t)at * S))[0] = make_float4(f[0], f[1], f[2], f[3]);
            ((float4*)(row + (int64_t)at * S))[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = naiwa_f32_to_bf16(f[2 * i]) | (naiwa_f32_to_bf16(f[2 * i + 1]) << 16);
            *(uint4*)(row + (int64_t)at * S) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// Checks shared by both directions, with the defaults of the strides put in.  rows: the
// unpacked side.
int check(const void* rows, int64_t batch, int64_t n, int64_t k, int64_t& ld, int64_t& rows_stride,
          const void* packed, int64_t& packed_stride) {
    if (batch < 0 || n < 0 || k < 0 || n % 16 || k % 32 || ld < 0 || rows_stride < 0 || packed_stride < 0)
        return NAIWA_E_INVALID;
    if (batch == 0 || n == 0 || k == 0) return NAIWA_OK;
    if (n > INT32_MAX || k > INT32_MAX) return NAIWA_E_UNSUPPORTED;
    const int64_t bytes = naiwa_projection_bytes(NAIWA_MXFP4_T, n, k);
    if (!ld) ld = k;
    if (ld < k || ld > INT64_MAX / 64 / n) return NAIWA_E_INVALID;
    if (!rows_stride) rows_stride = n * ld;
    if (!packed_stride) packed_stride = bytes;
    if (!rows || !packed || (batch > 1 && (rows_stride < (n - 1) * ld + k || packed_stride < bytes)))
        return NAIWA_E_INVALID;
    if (((uintptr_t)packed | (uintptr_t)packed_stride) & 15) return NAIWA_E_INVALID;
    if (((uintptr_t)rows & 15) || (ld | rows_stride) % 8) return NAIWA_E_INVALID;
    if (batch > INT32_MAX || (n / 16) * naiwa_mx_groups(k) > INT32_MAX / batch) return NAIWA_E_UNSUPPORTED;
    return NAIWA_OK;
}

// f(blocks, where) for the groups of a call, at most kLaunch of them at a time.
template <class F> int launches(int64_t batch, int64_t n, int64_t k, F f) {
    Where wh{n / 16, naiwa_mx_groups(k), 0};
    const int64_t all = batch * wh.strips * wh.groups;
    for (; wh.first < all; wh.first += kLaunch) f((unsigned)(all - wh.first < kLaunch ? all - wh.first : kLaunch), wh);
    return naiwa_hip_rc(hipGetLastError());
}

} // namespace

extern "C" int naiwa_mxfp4_quantize(const void* src, int src_dtype, int64_t batch, int64_t n, int64_t k, int64_t ld,
                                    int64_t src_stride, void* dst, int64_t dst_stride, int64_t stream) {
    if (src_dtype != NAIWA_F32 && src_dtype != NAIWA_BF16 && src_dtype != NAIWA_F16) return NAIWA_E_UNSUPPORTED;
    if (int rc = check(src, batch, n, k, ld, src_stride, dst, dst_stride)) return rc;
    if (batch == 0 || n == 0 || k == 0) return NAIWA_OK;
    return launches(batch, n, k, [&](unsigned blocks, const Where& wh) {
        hipStream_t st = (hipStream_t)stream;
        const uint8_t* s = (const uint8_t*)src;
        uint8_t* d = (uint8_t*)dst;
        if (src_dtype == NAIWA_F32)
            quantize_kernel<NAIWA_F32><<<blocks, kThreads, 0, st>>>(s, wh, (int)k, ld, src_stride, d, dst_stride);
        else if (src_dtype == NAIWA_BF16)
            quantize_kernel<NAIWA_BF16><<<blocks, kThreads, 0, st>>>(s, wh, (int)k, ld, src_stride, d, dst_stride);
        else
            quantize_kernel<NAIWA_F16><<<blocks, kThreads, 0, st>>>(s, wh, (int)k, ld, src_stride, d, dst_stride);
    });
}

extern "C" int naiwa_mxfp4_dequantize(const void* src, int64_t batch, int64_t n, int64_t k, int64_t src_stride,
                                      void* dst, int dst_dtype, int64_t ld, int64_t dst_stride, int64_t stream) {
    if (dst_dtype != NAIWA_F32 && dst_dtype != NAIWA_BF16) return NAIWA_E_UNSUPPORTED;
    if (int rc = check(dst, batch, n, k, ld, dst_stride, src, src_stride)) return rc;
    if (batch == 0 || n == 0 || k == 0) return NAIWA_OK;
    return launches(batch, n, k, [&](unsigned blocks, const Where& wh) {
        hipStream_t st = (hipStream_t)stream;
        const uint8_t* s = (const uint8_t*)src;
        uint8_t* d = (uint8_t*)dst;
        if (dst_dtype == NAIWA_F32)
            dequantize_kernel<NAIWA_F32><<<blocks, kThreads, 0, st>>>(s, wh, (int)k, src_stride, d, ld, dst_stride);
        else
            dequantize_kernel<NAIWA_BF16><<<blocks, kThreads, 0, st>>>(s, wh, (int)k, src_stride, d, ld, dst_stride);
    });
}

extern "C" int naiwa_mxfp4_from_ggml(const void* src, int64_t n, int64_t k, void* dst) {
    if (n < 0 || k < 0 || n % 16 || k % 32) return NAIWA_E_INVALID;
    if (n == 0 || k == 0) return NAIWA_OK;
    if (!src || !dst) return NAIWA_E_INVALID;
    const int64_t bytes = naiwa_mx_strip_bytes(k), blocks = k / 32, steps = naiwa_mx_steps(k);
    const uint8_t* s = (const uint8_t*)src;
    memset(dst, 0, (size_t)(n / 16 * bytes));
    for (int64_t row = 0; row < n; ++row) {
        uint8_t* strip = (uint8_t*)dst + row / 16 * bytes;
        const int64_t r = row % 16;
        for (int64_t b = 0; b < blocks; ++b, s += 17) {
            const int64_t step = b / 4, group = step / 4, lane = 16 * (b % 4) + r;
            uint8_t* at = strip + 1024 * step + 256 * group + 16 * lane;
            const int64_t last = 4 * group + 4 < steps ? 4 * group + 4 : steps; // the group's scales follow its last step
            strip[1024 * last + 256 * group + 4 * lane + step % 4] = s[0];
            for (int i = 0; i < 8; ++i) {
                const uint8_t a = s[1 + 2 * i], c = s[2 + 2 * i];
                at[i] = (uint8_t)((a & 15) | (c << 4));
                at[8 + i] = (uint8_t)((a >> 4) | (c & 0xf0));
            }
        }
    }
    return NAIWA_OK;
}
