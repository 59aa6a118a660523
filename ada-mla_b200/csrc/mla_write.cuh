// mla_write.cuh -- latent rows into the cache: RMS norm of the 512 latent columns,
// rotary embedding of the 64 rope columns, one rounding to the cache's type.
//
//   y = x * rsqrt(mean(x^2) + eps) * w        (columns 0..511; skipped without w)
//   (a, b) -> (a cos - b sin, a sin + b cos)  (column pairs of 512..575; skipped
//                                              without positions)
//   cache[slot] = [y, rope], or e4m3([y, rope] / s) with s = max|row| / 448 kept in
//   kv_scales[slot] (1 for a row of zeros).
//
// A warp per row: lane l holds latent columns 8l.. and 256 + 8l.. (or 4-column
// pieces of fp32 input) and rope pair l, so a row is read once in 16-byte loads, its
// sum of squares and its largest value are warp sums in registers, and the row is
// written once.  All arithmetic is fp32.  Bound by memory: 576 * (in + out) bytes
// a row.
#pragma once

#include "mla_common.cuh"

namespace mla {
namespace write {

constexpr int kWarps = 8;  // rows per block
constexpr int kLat = kDV;
constexpr int kRope = kDK - kDV;

struct WriteParams {
    const void *latent;
    long long stride;  // elements from one row to the next
    const long long *slots;
    const int32_t *positions;  // null: no rotation
    const void *weight;        // [512] in the input's type; null: no norm
    const float *cos_sin;      // [max_pos, 64]: cos of the 32 angles, then their sin
    int max_pos;
    int interleaved;  // pairs (2i, 2i + 1); else (i, i + 32)
    float eps;
    int num_tokens;
    void *cache;
    long long cache_rows;
    float *kv_scales;  // e4m3
};

template <typename T> __device__ __forceinline__ float2 two_f32(uint32_t u);
template <> __device__ __forceinline__ float2 two_f32<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <> __device__ __forceinline__ float2 two_f32<__nv_bfloat16>(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u));
}

// Eight consecutive elements at `src`: 16-byte loads, or single ones where the row
// does not start on 16 bytes.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T *src, float (&v)[8]) {
    if constexpr (!kVec) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)src[k];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float4 u = __ldg(reinterpret_cast<const float4 *>(src) + k);
            v[4 * k] = u.x; v[4 * k + 1] = u.y; v[4 * k + 2] = u.z; v[4 * k + 3] = u.w;
        }
    } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(src));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = two_f32<T>(w[k]);
            v[2 * k] = f.x;
            v[2 * k + 1] = f.y;
        }
    }
}

// Two consecutive elements at an even offset of a vector row.
__device__ __forceinline__ void load2(const float *src, float &a, float &b) {
    const float2 f = __ldg(reinterpret_cast<const float2 *>(src));
    a = f.x;
    b = f.y;
}
template <typename T>
__device__ __forceinline__ void load2(const T *src, float &a, float &b) {
    const float2 f = two_f32<T>(__ldg(reinterpret_cast<const uint32_t *>(src)));
    a = f.x;
    b = f.y;
}

__device__ __forceinline__ uint32_t pack2_to(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2_to(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2_e4m3(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

template <typename InT, typename OutT, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) cache_write_kernel(const WriteParams p) {
    constexpr bool kFp8 = sizeof(OutT) == 1;
    const int lane = threadIdx.x & 31;
    const long long t = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= p.num_tokens) return;
    // every load that depends on no other goes out first: slot and position, the row
    const long long slot = __ldg(p.slots + t);
    const int pos = p.positions != nullptr ? __ldg(p.positions + t) : 0;
    const InT *row = static_cast<const InT *>(p.latent) + t * p.stride;
    float v[2][8];
    load8<InT, kVec>(row + 8 * lane, v[0]);
    load8<InT, kVec>(row + 256 + 8 * lane, v[1]);
    // this lane's rope pair
    const int ia = p.interleaved ? 2 * lane : lane, ib = p.interleaved ? 2 * lane + 1 : lane + 32;
    float a, b;
    if (kVec && p.interleaved) {
        load2(row + kLat + ia, a, b);
    } else {
        a = (float)row[kLat + ia];
        b = (float)row[kLat + ib];
    }
    if (slot < 0 || slot >= p.cache_rows) return;  // a token without a page: nothing is written
    if (p.positions != nullptr && (pos < 0 || pos >= p.max_pos)) return;  // no angle for it: likewise
    if (p.positions != nullptr) {
        const float c = __ldg(p.cos_sin + (long long)pos * kRope + lane);
        const float s = __ldg(p.cos_sin + (long long)pos * kRope + 32 + lane);
        const float ra = a * c - b * s, rb = a * s + b * c;
        a = ra;
        b = rb;
    }
    if (p.weight != nullptr) {
        float sq = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 8; ++k) sq = fmaf(v[h][k], v[h][k], sq);
        sq = warp_sum(sq);
        const float inv = rsqrtf(sq * (1.f / kLat) + p.eps);
        const InT *w = static_cast<const InT *>(p.weight);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float g[8];
            load8<InT, kVec>(w + 256 * h + 8 * lane, g);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[h][k] = v[h][k] * inv * g[k];
        }
    }
    if constexpr (kFp8) {
        float mx = fmaxf(fabsf(a), fabsf(b));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(v[h][k]));
        mx = warp_max(mx);
        // a positive normal scale, as the decode asks for, also for rows of zeros or
        // of the smallest numbers
        const float scale = mx > 0.f ? fmaxf(mx / 448.f, 1.17549435e-38f) : 1.f;
        const float r = 1.f / scale;
        uint8_t *dst = static_cast<uint8_t *>(p.cache) + slot * kDK;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t o[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                o[k] = pack2_e4m3(v[h][4 * k] * r, v[h][4 * k + 1] * r) |
                       (pack2_e4m3(v[h][4 * k + 2] * r, v[h][4 * k + 3] * r) << 16);
            *reinterpret_cast<uint2 *>(dst + 256 * h + 8 * lane) = make_uint2(o[0], o[1]);
        }
        const uint32_t ab = pack2_e4m3(a * r, b * r);
        if (p.interleaved) {
            *reinterpret_cast<unsigned short *>(dst + kLat + ia) = (unsigned short)ab;
        } else {
            dst[kLat + ia] = (uint8_t)ab;
            dst[kLat + ib] = (uint8_t)(ab >> 8);
        }
        if (lane == 0) p.kv_scales[slot] = scale;
    } else {
        OutT *dst = static_cast<OutT *>(p.cache) + slot * kDK;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<uint4 *>(dst + 256 * h + 8 * lane) =
                make_uint4(pack2_to(v[h][0], v[h][1], OutT()), pack2_to(v[h][2], v[h][3], OutT()),
                           pack2_to(v[h][4], v[h][5], OutT()), pack2_to(v[h][6], v[h][7], OutT()));
        const uint32_t ab = pack2_to(a, b, OutT());
        if (p.interleaved) {
            *reinterpret_cast<uint32_t *>(dst + kLat + ia) = ab;
        } else {
            reinterpret_cast<unsigned short *>(dst)[kLat + ia] = (unsigned short)ab;
            reinterpret_cast<unsigned short *>(dst)[kLat + ib] = (unsigned short)(ab >> 16);
        }
    }
}

}  // namespace write
}  // namespace mla
