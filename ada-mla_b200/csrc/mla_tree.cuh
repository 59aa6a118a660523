// mla_tree.cuh -- the kernels around the draft-tree decode (tc::tc_decode_kernel
// with kTree): the drafts each row tile sees, and the merge of its split partials.
#pragma once

#include "mla_combine.cuh"
#include "mla_tc.cuh"

namespace mla {
namespace tree {

constexpr int kMergeWarps = 8;  // warps of a merge block

// seen[v] = the drafts that some draft of row tile v sees (bits at and past
// `drafts` clear); mask null: a chain, draft i sees drafts 0..i.  A thread per tile.
__global__ void __launch_bounds__(256) seen_kernel(const unsigned long long *__restrict__ mask, int mask_stride,
                                                   int drafts, int tiles, int tile_drafts, int ntiles,
                                                   unsigned long long *__restrict__ seen) {
    griddep_launch();
    griddep_wait();
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= ntiles) return;
    const int b = v / tiles, d0 = (v - b * tiles) * tile_drafts;
    const int d1 = min(d0 + tile_drafts, drafts);
    unsigned long long m = 0;
    if (mask == nullptr) m = (2ull << (d1 - 1)) - 1;
    else
        for (int d = d0; d < d1; ++d) m |= mask[(long long)b * mask_stride + d];
    seen[v] = drafts < 64 ? m & ((1ull << drafts) - 1) : m;
}

// O = sum_i e^(lse_i - M) O_i / sum_i e^(lse_i - M), M = max_i lse_i, over the
// items i of tile v that hold row r's partials (fp32: a 16-bit partial would add a
// third rounding of the size of the output's own).  kRowWarps warps share a row
// (each every kRowWarps-th split, joined in shared memory in a fixed order): 8
// where a few tiles have many splits, else 1.  Rows of tiles that were one item are
// complete already.  Bound by the partials' bytes, 2 KB a row and split.
template <typename OutT, int kRowWarps>
__global__ void __launch_bounds__(32 * kMergeWarps) merge_kernel(const float *__restrict__ part_o,
                                                                 const float *__restrict__ part_lse, WorkList wl,
                                                                 tc::TcTreeParams p, OutT *__restrict__ out,
                                                                 float *__restrict__ out_lse) {
    constexpr int kRows = kMergeWarps / kRowWarps;  // rows per block
    __shared__ __align__(16) float acc_s[kRowWarps > 1 ? kRowWarps - 1 : 1][kDV];
    __shared__ float sum_s[kMergeWarps];
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int v = blockIdx.y;
    const int r = blockIdx.x * kRows + warp / kRowWarps, g = warp % kRowWarps;
    long long row0;
    int rows;
    tc::tree_rows(p, v, row0, rows);
    int i0, i1;
    item_range(wl, v, i0, i1);
    if (i1 - i0 == 1) return;               // the same for the whole block
    if (r >= rows) return;                  // (with kRowWarps > 1 a block has one row)
    const int n = i1 - i0;
    const float *lse0 = part_lse + (size_t)i0 * p.num_heads + r;
    float mx = -INFINITY;
    for (int s = lane; s < n; s += 32) mx = fmaxf(mx, lse0[(size_t)s * p.num_heads]);
    mx = warp_max(mx);
    float acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    float wsum = 0.f;
    if (mx != -INFINITY) {
        const float4 *src = reinterpret_cast<const float4 *>(part_o + ((size_t)i0 * p.num_heads + r) * kDV) + lane;
        const size_t step = (size_t)p.num_heads * (kDV / 4);
        constexpr int kAhead = 4;
        for (int s = g; s < n; s += kRowWarps * kAhead) {
            float4 u[kAhead][4];
            float w[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int sj = s + j * kRowWarps;
                w[j] = 0.f;
                if (sj < n) {
                    w[j] = __expf(lse0[(size_t)sj * p.num_heads] - mx);  // exp(-inf) = 0
#pragma unroll
                    for (int q = 0; q < 4; ++q) u[j][q] = __ldg(src + (size_t)sj * step + q * 32);
                }
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (w[j] > 0.f) {  // (a split that saw nothing holds zeros)
                    wsum += w[j];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        acc[4 * q] = fmaf(w[j], u[j][q].x, acc[4 * q]);
                        acc[4 * q + 1] = fmaf(w[j], u[j][q].y, acc[4 * q + 1]);
                        acc[4 * q + 2] = fmaf(w[j], u[j][q].z, acc[4 * q + 2]);
                        acc[4 * q + 3] = fmaf(w[j], u[j][q].w, acc[4 * q + 3]);
                    }
                }
            }
        }
    }
    if constexpr (kRowWarps > 1) {
        if (g > 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                reinterpret_cast<float4 *>(acc_s[g - 1])[lane + q * 32] =
                    make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
            if (lane == 0) sum_s[g] = wsum;
        }
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int k = 1; k < kRowWarps; ++k) {
            wsum += sum_s[k];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 a = reinterpret_cast<const float4 *>(acc_s[k - 1])[lane + q * 32];
                acc[4 * q] += a.x;
                acc[4 * q + 1] += a.y;
                acc[4 * q + 2] += a.z;
                acc[4 * q + 3] += a.w;
            }
        }
    }
    const float inv = wsum > 0.f ? 1.f / wsum : 0.f;
    OutT *dst = out + (row0 + r) * kDV + lane * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float a = acc[4 * q] * inv, b = acc[4 * q + 1] * inv, c = acc[4 * q + 2] * inv, d = acc[4 * q + 3] * inv;
        if constexpr (sizeof(OutT) == 4)
            *reinterpret_cast<float4 *>(dst + q * 128) = make_float4(a, b, c, d);
        else
            *reinterpret_cast<uint2 *>(dst + q * 128) = make_uint2(pack_out2<OutT>(a, b), pack_out2<OutT>(c, d));
    }
    if (out_lse != nullptr && lane == 0) out_lse[row0 + r] = wsum > 0.f ? mx + __logf(wsum) : -INFINITY;
}

}  // namespace tree
}  // namespace mla
