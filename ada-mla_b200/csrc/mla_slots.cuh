// mla_slots.cuh -- pages and slot maps for the tokens a step appends to its
// requests, from the requests' lengths.
//
//   have_b = ceil(L_b / P), need_b = ceil((L_b + N_b) / P) - have_b (both within the
//   table's width), off_b = sum of need over the requests before b;
//   table[b, have_b + i] = free[head + off_b + i] for i < need_b, -1 past the list;
//   token t of request b, at position p = L_b + t: slot = table[b, p / P] * P + p % P.
//
// One launch.  A few bytes per request and 12 per token: a decode step's call is
// all latency, so nothing is handed from one kernel to the next: every block scans
// the requests' lengths itself (8 bytes each, from L2 after the first block) and
// then expands its own tokens, 1024 at a time, one per thread.  The request of a
// token comes from a second scan: each request that starts in (or reaches into) the
// 1024 tokens marks its first one, and a running maximum of the marks gives every
// token the last mark before it.  256 requests of one token: 8.8 us a call, which is its
// checks, one allocation and the launch (the kernel, with cold caches, takes 8.0); 93
// prompts, 381 000 tokens, 4.6 MB: 10.2 us (0.45 TB/s; 12.6 with cold caches).
#pragma once

#include "mla_common.cuh"

namespace mla {
namespace slots {

constexpr int kThreads = 1024;

struct SlotParams {
    const int32_t *seq_lens, *new_lens;
    int32_t *table;
    const int32_t *free_pages, *free_head;  // free_head null: 0
    long long table_stride;
    int batch, max_blocks, num_free, page_size;
    long long num_tokens;  // tokens that slots / positions have room for
    long long *slots;
    int32_t *positions, *cu_new, *new_seq_lens, *new_free_head;
};

struct Sums {
    long long tokens, pages;
};

__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }

__device__ __forceinline__ Sums shfl_up(Sums v, int o) {
    return {__shfl_up_sync(0xffffffffu, v.tokens, o), __shfl_up_sync(0xffffffffu, v.pages, o)};
}

struct Request {
    int len, add, have, need;
};

// ceil(n / page_size), at most `most`; the division in 32 bits where that holds n.
__device__ __forceinline__ int pages_of(unsigned long long n, int page_size, int most) {
    const unsigned long long up = n + (unsigned)(page_size - 1);
    const unsigned long long q = up >> 32 ? up / (unsigned)page_size : (unsigned)up / (unsigned)page_size;
    return (int)min(q, (unsigned long long)most);
}

__device__ __forceinline__ Request request_of(const SlotParams &p, int b) {
    Request r;
    r.len = max(p.seq_lens[b], 0);
    r.add = max(p.new_lens[b], 0);
    r.have = pages_of(r.len, p.page_size, p.max_blocks);
    r.need = pages_of((unsigned long long)r.len + r.add, p.page_size, p.max_blocks) - r.have;
    return r;
}

__device__ __forceinline__ int clamp_i32(long long v) { return (int)min(v, 0x7fffffffll); }

__global__ void __launch_bounds__(kThreads) build_slots_kernel(const SlotParams p) {
    __shared__ Sums warp_sum[32];
    __shared__ int warp_mark[32];
    __shared__ int mark[kThreads];           // 1 + index of the request record that starts at this token
    __shared__ long long rec_tok[kThreads];  // the request's first token ...
    __shared__ long long rec_page[kThreads]; // ... and its first new page's place in the free list
    __shared__ int rec_b[kThreads], rec_len[kThreads], rec_have[kThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // the sums before this thread's requests
    const int per = (p.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    const long long head = p.free_head != nullptr ? p.free_head[0] : 0;
    Sums own = {0, 0};
    Request first = {0, 0, 0, 0};  // (kept: with up to 1024 requests it is the only one)
    for (int b = b0; b < b1; ++b) {
        const Request r = request_of(p, b);
        if (b == b0) first = r;
        own = own + Sums{r.add, r.need};
    }
    Sums v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums u = shfl_up(v, o);
        if (lane >= o) v = v + u;
    }
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    if (warp == 0) {
        Sums w = warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const Sums u = shfl_up(w, o);
            if (lane >= o) w = w + u;
        }
        warp_sum[lane] = w;
    }
    __syncthreads();
    const long long total = warp_sum[31].tokens;
    Sums before = {v.tokens - own.tokens, v.pages - own.pages};
    if (warp > 0) before = before + warp_sum[warp - 1];

    // what is written once per request, dealt over the blocks
    if (tid % gridDim.x == blockIdx.x) {
        Sums s = before;
        for (int b = b0; b < b1; ++b) {
            const Request r = b == b0 ? first : request_of(p, b);
            p.cu_new[b] = clamp_i32(s.tokens);
            p.new_seq_lens[b] = clamp_i32((long long)r.len + r.add);
            s = s + Sums{r.add, r.need};
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.cu_new[p.batch] = clamp_i32(total);
        p.new_free_head[0] = clamp_i32(head + warp_sum[31].pages);
    }

    const long long end = max(total, p.num_tokens);
    for (long long t0 = (long long)blockIdx.x * kThreads; t0 < end; t0 += (long long)gridDim.x * kThreads) {
        __syncthreads();
        mark[tid] = 0;
        __syncthreads();
        {
            Sums s = before;
            for (int b = b0; b < b1 && s.tokens < t0 + kThreads; ++b) {
                const Request r = b == b0 ? first : request_of(p, b);
                if (r.add > 0 && s.tokens + r.add > t0) {
                    const int at = (int)max(s.tokens - t0, 0ll);  // its own: requests do not overlap
                    mark[at] = at + 1;
                    rec_tok[at] = s.tokens;
                    rec_page[at] = head + s.pages;
                    rec_b[at] = b;
                    rec_len[at] = r.len;
                    rec_have[at] = r.have;
                }
                s = s + Sums{r.add, r.need};
            }
        }
        __syncthreads();
        int m = mark[tid];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, m, o);
            if (lane >= o) m = max(m, u);
        }
        if (lane == 31) warp_mark[warp] = m;
        __syncthreads();
        if (warp == 0) {
            int w = warp_mark[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w = max(w, u);
            }
            warp_mark[lane] = w;
        }
        __syncthreads();
        if (warp > 0) m = max(m, warp_mark[warp - 1]);
        const long long t = t0 + tid;
        if (t < total) {
            const int b = rec_b[m - 1], have = rec_have[m - 1];
            const long long pos = rec_len[m - 1] + (t - rec_tok[m - 1]);
            const long long block = pos >> 32 ? pos / p.page_size : (long long)((unsigned)pos / (unsigned)p.page_size);
            const int in_page = (int)(pos - block * p.page_size);
            int page = -1;
            if (block < p.max_blocks) {
                int32_t *entry = p.table + (long long)b * p.table_stride + block;
                if (block < have) {
                    page = *entry;  // not one that this call writes
                } else {
                    const long long i = rec_page[m - 1] + (block - have);
                    if (i >= 0 && i < p.num_free) page = p.free_pages[i];
                    if (in_page == 0) *entry = page;
                }
            }
            if (t < p.num_tokens) {
                p.slots[t] = page < 0 ? -1 : (long long)page * p.page_size + in_page;
                p.positions[t] = clamp_i32(pos);
            }
        } else if (t < p.num_tokens) {
            p.slots[t] = -1;
            p.positions[t] = 0;
        }
    }
}

}  // namespace slots
}  // namespace mla
