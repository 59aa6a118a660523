// mla_write.cuh -- latent rows into the cache: RMS norm of the 512 latent columns,
// rotary embedding of the 64 rope columns, one rounding to the cache's type.
//
//   y = x * rsqrt(mean(x^2) + eps) * w        (columns 0..511; skipped without w)
//   (a, b) -> (a cos - b sin, a sin + b cos)  (column pairs of 512..575; skipped
//                                              without positions)
//   cache[slot] = [y, rope], or e4m3([y, rope] / s) with s = max|row| / 448 kept in
//   kv_scales[slot] (1 for a row of zeros).
//
// The values are multiplied by 1 / s: one on the boundary between two e4m3 numbers may go to
// the other than a division would give (divided, 131072 rows take 71.7 us).
//
// A warp per row: lane l holds latent columns 8l.. and 256 + 8l.. and rope pair l, so
// a row is read once in 16-byte loads, its sum of squares and its largest value are warp
// reductions in registers, and the row is written once.  All arithmetic is fp32.  Bound
// by memory: 576 * (in + out) bytes a row.  Each warp walks rows with the next one's
// loads in flight (its position one further ahead, so that its angles are too) and
// keeps its norm weights: a warp for one row alone left the memory 40 % idle.  32769 rows
// bf16 to bf16: 16.5 us, 4.7 TB/s; 131072 rows to e4m3: 49.5 us, 4.7 TB/s; 256 rows: 5.6 us,
// the call.
#pragma once

#include <type_traits>

#include "mla_common.cuh"

namespace mla {
namespace write {

constexpr int kWarps = 8;        // warps per block
// Resident blocks per SM, which the rows are dealt to: 4 (64 registers) or, for e4m3, 3
// (80).  32769 rows to bf16: 16.5 us with 4, 18.4 with 3, 21.7 with 5; 131072 rows to
// e4m3: 52.5, 49.5, 66.7.
template <typename OutT> constexpr int kBlocksPerSm = sizeof(OutT) == 1 ? 3 : 4;
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

// This lane's part of a row as it was loaded: latent columns 8 lane .. and 256 + 8
// lane .., and its rope pair.  16-byte loads, or single ones where rows do not start on
// 16 bytes.
template <typename T, bool kVec>
struct Raw {
    static constexpr int kN = kVec ? (int)sizeof(T) : 16;  // 16-byte vectors (8 elements: sizeof(T) / 2), or elements
    using V = std::conditional_t<kVec, uint4, T>;
    V x[kN];
    T a, b;

    __device__ __forceinline__ void load(const T *row, int lane, int ia, int ib) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int k = 0; k < kN / 2; ++k)
                x[h * (kN / 2) + k] = __ldg(reinterpret_cast<const V *>(row + 256 * h + 8 * lane) + k);
        }
        a = row[kLat + ia];
        b = row[kLat + ib];
    }

    __device__ __forceinline__ void values(float (&v)[2][8]) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (!kVec) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[h][k] = (float)x[h * 8 + k];
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint4 u = x[h * 2 + k];
                    v[h][4 * k] = __uint_as_float(u.x);
                    v[h][4 * k + 1] = __uint_as_float(u.y);
                    v[h][4 * k + 2] = __uint_as_float(u.z);
                    v[h][4 * k + 3] = __uint_as_float(u.w);
                }
            } else {
                const uint32_t w[4] = {x[h].x, x[h].y, x[h].z, x[h].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = two_f32<T>(w[k]);
                    v[h][2 * k] = f.x;
                    v[h][2 * k + 1] = f.y;
                }
            }
        }
    }
};

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
__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm<OutT>) cache_write_kernel(const WriteParams p) {
    constexpr bool kFp8 = sizeof(OutT) == 1;
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * kWarps;
    int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= p.num_tokens) return;
    const int ia = p.interleaved ? 2 * lane : lane, ib = p.interleaved ? 2 * lane + 1 : lane + 32;
    const bool rope = p.positions != nullptr, norm = p.weight != nullptr;
    const InT *base = static_cast<const InT *>(p.latent);
    auto position = [&](int i) -> int { return rope && i < p.num_tokens ? __ldg(p.positions + i) : 0; };
    auto angle = [&](int pos, float &c, float &s) {  // (no angle: the row is skipped below)
        const bool ok = rope && pos >= 0 && pos < p.max_pos;
        c = ok ? __ldg(p.cos_sin + (long long)pos * kRope + lane) : 0.f;
        s = ok ? __ldg(p.cos_sin + (long long)pos * kRope + 32 + lane) : 0.f;
    };
    Raw<InT, kVec> raw, raw_next;
    long long slot = __ldg(p.slots + t), slot_next = -1;
    int pos = position(t), pos_next = position(t + warps);
    raw.load(base + t * p.stride, lane, ia, ib);
    float g[2][8];
    if (norm) {
        Raw<InT, kVec> w;
        const InT *wp = static_cast<const InT *>(p.weight);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < w.kN / 2; ++k)
                w.x[h * (w.kN / 2) + k] = __ldg(reinterpret_cast<const typename Raw<InT, kVec>::V *>(wp + 256 * h + 8 * lane) + k);
        w.values(g);
    }
    float cos_t, sin_t, cos_n = 0.f, sin_n = 0.f;
    angle(pos, cos_t, sin_t);
    for (; t < p.num_tokens; t += warps) {
        const int tn = t + warps;
        if (tn < p.num_tokens) {  // the next row's loads, and the position after it
            slot_next = __ldg(p.slots + tn);
            raw_next.load(base + tn * p.stride, lane, ia, ib);
            angle(pos_next, cos_n, sin_n);
        }
        const int pos_after = position(tn + warps);
        // a token without a page, or a position without an angle: nothing is written
        if (slot >= 0 && slot < p.cache_rows && (!rope || (pos >= 0 && pos < p.max_pos))) {
            float v[2][8];
            raw.values(v);
            float a = (float)raw.a, b = (float)raw.b;
            if (rope) {
                const float ra = a * cos_t - b * sin_t, rb = a * sin_t + b * cos_t;
                a = ra;
                b = rb;
            }
            if (norm) {
                float sq = 0.f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 8; ++k) sq = fmaf(v[h][k], v[h][k], sq);
                sq = warp_sum(sq);
                const float inv = rsqrtf(sq * (1.f / kLat) + p.eps);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[h][k] = v[h][k] * inv * g[h][k];
            }
            if constexpr (kFp8) {
                float mx = fmaxf(fabsf(a), fabsf(b));
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(v[h][k]));
                // (the largest of non-negative floats: their bits order like whole numbers)
                mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
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
        raw = raw_next;
        slot = slot_next;
        pos = pos_next;
        pos_next = pos_after;
        cos_t = cos_n;
        sin_t = sin_n;
    }
}

}  // namespace write
}  // namespace mla
