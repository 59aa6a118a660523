// mla_prefill.cuh -- attention over prompts in expanded form, tcgen05:
//
//   s[h, i, j] = scale (q_nope[i, h] . k_nope[j, h] + q_rope[i, h] . k_rope[j])
//   o[i, h]    = softmax_j(s) v[j, h]          (j <= i + Lk - Lq when causal)
//
// q [.., 128 + 64], k_nope and v 128 wide per head, k_rope ONE 64-wide vector per
// token shared by all heads: its tile is loaded straight into the third K-block of
// the key tile, so the 192-wide keys never exist in memory.
//
// A work item is 256 query rows of one (sequence, head), two tiles of 128, on one
// persistent CTA per SM.  Both tiles read each key / value tile of 128 tokens once.
// While the tensor core works on one tile, the other tile's softmax runs:
//
//   tensor core:  PV0(j)  QK0(j+1)  PV1(j)  QK1(j+1)  PV0(j+1) ...
//   softmax 0:            [ tile 0, j+1 ......... ]
//   softmax 1:                               [ tile 1, j+1 ......... ]
//
// TMEM (512 columns): S0 S1 [128 x 128] fp32, O0 O1 [128 x 128] fp32; P (16-bit)
// overwrites the first half of its S and is PV's A operand.  A tile of the pair costs
// 768 cycles of QK (K = 192) and 512 of PV at the tensor rate, against 1024 cycles of
// exponentials (16 per cycle and SM), so the tensor core can be the bound.
//
// Shared memory: Q0 Q1 (2 x 48 KB) and a ring of eight 16 KB slots, a slot being one
// 64-column block of 128 keys or 64 tokens of V: K(0) V(0) K(1) V(1) .. in 3 + 2
// slots each.  Slots of one size let the two kinds share 128 KB (1.6 tiles).
//
// Roles (384 threads): warp 0 TMA producer, warps 1 and 3 MMA issuers (one per query
// tile), warp 2 TMEM owner and V tail, warps 4-7 softmax of tile 0, warps 8-11 of tile 1 (a thread per row: no
// shuffles).  The softmax warps rescale O themselves, rarely: the running maximum is
// only raised when it grew by more than 2^8.  Every wait is bounded.
//
// A call among others on inputs that change: 2048 queries over 8192 keys, 128 heads: 1177
// us, 1.02 PFLOP/s; six prompts of 262-1884 tokens, 128 heads: 597 us, 0.60 PFLOP/s, where
// an item's start and end (11 key tiles long on average) cost a quarter; 77 queries, 128
// heads: 10.3 us.  In a loop the power cap (990 W) holds the clock at 1575-1600 MHz of 1965.
// That is not all: also in one launch alone (1.05 ms) the tensor pipe is active 59 % of the
// cycles, as a tile's S waits for the last PV and its P for the softmax.
//
// A key's values reach the products of all queries of its tile pair, with weight 0 where the
// mask hides it: they have to be finite.  (What lies past a sequence's end may be anything.)
#pragma once

#include "mla_combine.cuh"
#include "mla_tc.cuh"

namespace mla {
namespace prefill {

constexpr int kQK = MLA_B200_HEAD_DIM + MLA_B200_HEAD_DIM_ROPE;  // 192
constexpr int kV = MLA_B200_HEAD_DIM;                            // 128
constexpr int kTileQ = 128;
constexpr int kItemQ = 2 * kTileQ;
constexpr int kTileK = 128;
constexpr int kKBlk = kQK / 64;                 // 3
constexpr int kBox = kTileQ * 128;              // 16 KB: 128 rows x 64 columns
constexpr int kQBytes = kKBlk * kBox;           // 48 KB
constexpr int kVHalf = kTileK / 2;              // tokens of a V slot
constexpr int kVBox = kVHalf * 128;             // 8 KB: 64 tokens x 64 columns
constexpr int kSlots = 8;
constexpr int kSlotsPerTile = kKBlk + 2;        // 5
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;
constexpr int kOffRing = 2 * kQBytes;
constexpr int kOffBar = kOffRing + kSlots * kBox;
enum : int {
    kBarFull = 0,
    kBarEmpty = kSlots,
    kBarQFull = 2 * kSlots,      // [2] Q tile landed
    kBarQEmpty = kBarQFull + 2,  // [2] last QK of the item done
    kBarS = kBarQEmpty + 2,      // [2] S tile complete
    kBarP = kBarS + 2,           // [2][2] half a P tile written, O corrected (128 threads)
    kBarO = kBarP + 4,           // [2] PV done
    kBarTail = kBarO + 2,        // [2] a sequence's last V tile landed, rows past its end not yet zeroed
    kBarDrain = kBarTail + 2,    // [2]
    kBarItem = kBarDrain + 2,    // [4] an item is in the queue
    kBarItemFree = kBarItem + 4, // [4] every role has read it (11 warps)
    kNumBars = kBarItemFree + 4
};
constexpr int kOffSlot = kOffBar + kNumBars * 8;
constexpr int kOffAbort = kOffSlot + 4;
constexpr int kQueue = 4;                        // items
constexpr int kQueueReaders = 11;                // producer, two MMA issuers, eight softmax warps
constexpr int kOffItems = (kOffAbort + 4 + 15) / 16 * 16;
constexpr int kItemBytes = 48;
constexpr int kSmemBytes = kOffItems + kQueue * kItemBytes + 1024;  // + 1024 alignment slack
static_assert(kSmemBytes <= 232448, "dynamic shared memory limit");
// 384 threads x 168 registers at launch = 64512; the softmax warpgroups take 208
// each and the first one keeps 88: 2 x 128 x 208 + 128 x 88 = 64512.
constexpr int kRegsLaunch = 168, kRegsSoftmax = 208, kRegsOther = 88;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsOther <= kThreads * kRegsLaunch, "register split");
constexpr float kRescaleLog2 = 8.f;
constexpr int kPlanBuckets = 1024;
constexpr uint64_t kAbortWaitNs = 10000000ull;  // after an error: for copies in flight
constexpr uint32_t kMaxIdle = 200000000;  // tries of 40 ns and more: 8 s and more

struct PrefillParams {
    const int32_t *cu_q, *cu_k;  // null: dense
    int batch, heads, max_q, max_k;
    int total_q, total_k;
    int causal;
    float scale_log2;
    const int2 *pairs;      // {sequence, first query row}, longest first; null: at most an item for each CTA
    const int *num_pairs;
    int *next_item;         // with pairs: items given out
    int blocks;             // without pairs: 256-row blocks per sequence
    int head_group;         // heads walked together
    int splits;             // without pairs: shares of the keys, an item each, joined by merge_kernel
    float *part_o;          // [splits, total_q, heads, 128], normalized
    float *part_lse;        // [splits, total_q, heads]
    void *out;              // [total_q, heads, 128]
    float *out_lse;         // [total_q, heads] or null
};

struct Seq {
    int q0, k0;  // first rows (all rows are below 2^31)
    int lq, lk;
};

__device__ __forceinline__ Seq seq_of(const PrefillParams &p, int b) {
    Seq s;
    if (p.cu_q == nullptr) {
        s.q0 = b * p.max_q;
        s.k0 = b * p.max_k;
        s.lq = p.max_q;
        s.lk = p.max_k;
    } else {
        s.q0 = min(max(p.cu_q[b], 0), p.total_q);
        s.k0 = min(max(p.cu_k[b], 0), p.total_k);
        s.lq = min(p.max_q, max(0, min(p.cu_q[b + 1], p.total_q) - s.q0));
        s.lk = min(p.max_k, max(0, min(p.cu_k[b + 1], p.total_k) - s.k0));
    }
    return s;
}

// Key tiles that rows [row, row + 128) of a sequence see.
__device__ __forceinline__ int tiles_of(const PrefillParams &p, const Seq &s, int row) {
    if (row >= s.lq) return 0;
    int end = s.lk;
    if (p.causal) end = min(end, min(row + kTileQ, s.lq) + s.lk - s.lq);
    return end > 0 ? (end + kTileK - 1) / kTileK : 0;
}

struct Item {
    Seq s;        // (a split's keys start at its own share's first)
    int h, row;   // head, first query row of the item in its sequence
    int n[2];     // key tiles of its two query tiles (n[0] <= n[1] unless tile 1 has no rows)
    int nmax;
    int ahead;    // keys of the share before and at query row 0 of the sequence, less one (causal)
    int split;
};

// Item u of the launch, if it has rows.  Items are laid out by head group (so that the
// keys and values of the heads in flight stay in L2), within a group by pair, longest
// first.
__device__ __forceinline__ bool item_at(const PrefillParams &p, int pairs, int u, Item &it) {
    int b;
    it.split = 0;
    if (p.pairs != nullptr) {
        const int per = pairs * p.head_group;
        const int grp = u / per, r = u - grp * per;
        const int heads = min(p.head_group, p.heads - grp * p.head_group);
        const int pair = r / heads;
        it.h = grp * p.head_group + (r - pair * heads);
        const int2 pr = p.pairs[pair];
        b = pr.x;
        it.row = pr.y;
    } else {
        it.split = u % p.splits;
        u /= p.splits;
        const int pair = u / p.heads;
        it.h = u - pair * p.heads;
        b = pair / p.blocks;
        it.row = (pair - b * p.blocks) * kItemQ;
    }
    it.s = seq_of(p, b);
    if (it.row >= it.s.lq) return false;
    it.n[0] = tiles_of(p, it.s, it.row);
    it.n[1] = tiles_of(p, it.s, it.row + kTileQ);
    it.nmax = max(it.n[0], it.n[1]);
    it.ahead = it.s.lk - it.s.lq;
    if (p.splits > 1) {
        const int share = (it.nmax + p.splits - 1) / p.splits, j0 = it.split * share;
        it.n[0] = min(max(it.n[0] - j0, 0), share);
        it.n[1] = min(max(it.n[1] - j0, 0), share);
        it.nmax = max(it.n[0], it.n[1]);
        it.s.k0 += j0 * kTileK;
        it.s.lk -= j0 * kTileK;
        it.ahead -= j0 * kTileK;
    }
    return true;
}
static_assert(sizeof(Item) <= kItemBytes, "item queue");
constexpr int kNoMore = -1;  // nmax of the queue's last entry

// A role's place in the CTA's item queue (whole warps).
struct Cursor {
    uint32_t n = 0;
    __device__ __forceinline__ bool next(uint8_t *smem, uint32_t bar0, volatile int *abort_flag, Item &it);
};

// {sequence, first row} of every 256-row block, most key tiles first (a counting
// sort; blocks of one bucket come in any order, which no result depends on).  One
// block, a warp per sequence.
__global__ void __launch_bounds__(1024) plan_kernel(const PrefillParams p, int cap, int2 *__restrict__ pairs,
                                                    int *__restrict__ num_pairs, int *__restrict__ next_item) {
    __shared__ int count[kPlanBuckets];
    __shared__ int warp_tot[32];
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    count[tid] = 0;
    __syncthreads();
    const long long most = ((long long)p.max_k + kTileK - 1) / kTileK + 1;  // (above every n: no bucket below 0)
    auto bucket = [&](const Seq &s, int row) {
        const int n = max(tiles_of(p, s, row), tiles_of(p, s, row + kTileQ));
        return kPlanBuckets - 1 - (int)((long long)n * kPlanBuckets / (most + 1));
    };
    for (int pass = 0; pass < 2; ++pass) {
        for (int b = warp; b < p.batch; b += 32) {
            const Seq s = seq_of(p, b);
            for (int row = lane * kItemQ; row < s.lq; row += 32 * kItemQ) {
                const int at = atomicAdd(&count[bucket(s, row)], 1);
                if (pass == 1 && at < cap) pairs[at] = make_int2(b, row);
            }
        }
        __syncthreads();
        if (pass == 0) {  // counts -> starts
            const int own = count[tid];
            int v = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (lane == 31) warp_tot[warp] = v;
            __syncthreads();
            if (warp == 0) {
                int w = warp_tot[lane];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, w, o);
                    if (lane >= o) w += u;
                }
                warp_tot[lane] = w;
            }
            __syncthreads();
            count[tid] = (warp > 0 ? warp_tot[warp - 1] : 0) + v - own;
            if (tid == 1023) {
                *num_pairs = min(warp_tot[31], cap);
                *next_item = 0;
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------
// Packed fp32 pairs.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// The V tail warp may have nothing to do for the whole of a long item: its limit
// starts anew while the other roles are at work, and an abort ends it.
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    for (uint32_t n = 0; n < kMaxIdle; ++n) {
        if (*abort_flag) return false;
        if (ptx::mbar_try_wait(bar, parity)) return true;
        __nanosleep(40);
    }
    set_device_error(kErrWaitFull);
    return false;
}

__device__ __forceinline__ void store32(void *dst, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ bool Cursor::next(uint8_t *smem, uint32_t bar0, volatile int *abort_flag, Item &it) {
    const uint32_t e = n % kQueue;
    bool ok = wait_or_abort(bar0 + 8 * (kBarItem + e), (n / kQueue) & 1, abort_flag);
    if (!__all_sync(0xffffffffu, ok)) return false;
    it = *reinterpret_cast<const Item *>(smem + kOffItems + e * kItemBytes);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar0 + 8 * (kBarItemFree + e));
    ++n;
    return it.nmax != kNoMore;
}

// qmap: q as (192, heads, rows), box (64, 1, 128); kmap: k_nope as (128, heads,
// rows), box (64, 1, 128); rmap: k_rope as (64, rows), box (64, 128); vmap: v as
// (128, heads, rows), box (64, 1, 64).  128-byte swizzle.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap rmap, const __grid_constant__ CUtensorMap vmap,
                   const PrefillParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = ptx::smem_u32(smem);
    auto bar = [&](int id) -> uint32_t { return sbase + kOffBar + 8u * id; };
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + kOffAbort);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < kNumBars; ++i)  // (a ring slot is free when both MMA issuers are done with it)
            ptx::mbar_init(bar(i), i >= kBarP && i < kBarP + 4 ? 128 : i >= kBarEmpty && i < kBarEmpty + kSlots ? 2 : i >= kBarItemFree && i < kBarItemFree + kQueue ? kQueueReaders : 1);
        *abort_flag = 0;
        ptx::fence_mbarrier_init_cluster();
    }
    if (tid == 32) {
        ptx::tma_prefetch_desc(&qmap);
        ptx::tma_prefetch_desc(&kmap);
        ptx::tma_prefetch_desc(&rmap);
        ptx::tma_prefetch_desc(&vmap);
    }
    if (warp == 2) {
        ptx::tmem_alloc(sbase + kOffSlot, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + kOffSlot);
    griddep_launch();
    griddep_wait();

    Cursor cur;
    Item it{};
    auto next_item = [&]() -> bool { return cur.next(smem, sbase + kOffBar, abort_flag, it); };
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp == 0) {
            // ------------------------------------------------------ TMA producer
            // (This role and the next run as whole warps with uniform control flow and one
            // elected lane behind each instruction, so that descriptors and coordinates
            // stay in uniform registers.)
            const uint32_t e = ptx::elect_one();
            uint32_t at = 0;           // slots filled so far
            uint32_t qn[2] = {0, 0};   // Q tiles loaded so far
            uint32_t tails = 0;        // V tiles handed to the V tail warp so far
            bool ok = true;
            auto acquire = [&]() -> uint32_t {  // the next slot, once it is free
                const uint32_t s = at % kSlots;
                ok = ok && !*abort_flag && ptx::mbar_wait_now(bar(kBarEmpty + s), ((at / kSlots) & 1) ^ 1, kErrWaitEmpty);
                ok = __all_sync(0xffffffffu, ok);
                if (ok) ++at;
                return s;
            };
            while (ok && next_item()) {
                if (it.nmax <= 0) continue;
                const int nmax = __shfl_sync(0xffffffffu, it.nmax, 0), h = __shfl_sync(0xffffffffu, it.h, 0);
                const int k0 = __shfl_sync(0xffffffffu, it.s.k0, 0), q0 = __shfl_sync(0xffffffffu, it.s.q0 + it.row, 0);
                const int lk = __shfl_sync(0xffffffffu, it.s.lk, 0);
                const bool has[2] = {it.n[0] > 0, it.n[1] > 0};
                // Q0 K(0) Q1 | V(0) K(1) | V(1) K(2) | ..
#pragma unroll 1
                for (int j = -1; ok && j < nmax; ++j) {
                    if (j >= 0) {
                        const int row = k0 + j * kTileK;
                        const bool tail = (j + 1) * kTileK > lk;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t s = acquire();
                            if (!ok) break;
                            const uint32_t full = bar(tail ? kBarTail + (tails & 1) : kBarFull + s);
                            const uint32_t dst = sbase + kOffRing + s * kBox;
                            if (!tail || c == 0) ptx::mbar_arrive_expect_tx_if(e, full, tail ? 2 * kBox : kBox);
                            ptx::tma_load_3d_if(e, dst, &vmap, 0, h, row + c * kVHalf, full);
                            ptx::tma_load_3d_if(e, dst + kVBox, &vmap, 64, h, row + c * kVHalf, full);
                        }
                        if (tail) ++tails;
                        if (!ok) break;
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j < 0 && has[t]) {
                            ok = ok && !*abort_flag && ptx::mbar_wait_now(bar(kBarQEmpty + t), (qn[t] & 1) ^ 1, kErrWaitEmpty);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            ++qn[t];
                            ptx::mbar_arrive_expect_tx_if(e, bar(kBarQFull + t), kQBytes);
#pragma unroll
                            for (int c = 0; c < kKBlk; ++c)
                                ptx::tma_load_3d_if(e, sbase + t * kQBytes + c * kBox, &qmap, c * 64, h, q0 + t * kTileQ,
                                                    bar(kBarQFull + t));
                        }
                        if (t == 0 && j + 1 < nmax) {
                            const int row = k0 + (j + 1) * kTileK;
#pragma unroll
                            for (int c = 0; c < kKBlk; ++c) {
                                const uint32_t s = acquire();
                                if (!ok) break;
                                const uint32_t full = bar(kBarFull + s), dst = sbase + kOffRing + s * kBox;
                                ptx::mbar_arrive_expect_tx_if(e, full, kBox);
                                if (c < 2) ptx::tma_load_3d_if(e, dst, &kmap, c * 64, h, row, full);
                                else ptx::tma_load_2d_if(e, dst, &rmap, 0, row, full);
                            }
                            if (!ok) break;
                        }
                    }
                }
            }
            if (!ok) *abort_flag = 1;
            // every load has landed before this CTA's shared memory goes (the slots' own
            // barriers, and those of tails not yet zeroed)
            if (ok) {
                for (uint32_t k = at > kSlots ? at - kSlots : 0; k < at; ++k)
                    ptx::mbar_wait(bar(kBarFull + k % kSlots), (k / kSlots) & 1, kErrWaitFull);
            } else {
                for (uint32_t k = at > kSlots ? at - kSlots : 0; k < at; ++k)
                    ptx::mbar_wait(bar(kBarFull + k % kSlots), (k / kSlots) & 1, kErrWaitFull, kAbortWaitNs);
            }
            for (uint32_t k = tails > 2 ? tails - 2 : 0; k < tails; ++k)
                ptx::mbar_wait(bar(kBarTail + (k & 1)), (k >> 1) & 1, kErrWaitFull, ok ? kWaitLimitNs : kAbortWaitNs);
            for (int t = 0; t < 2; ++t)
                if (qn[t] > 0) ptx::mbar_wait(bar(kBarQFull + t), (qn[t] - 1) & 1, kErrWaitFull);
        } else if (warp == 1 || warp == 3) {
            // ------------------------------------------------------ MMA issuers
            // Warp 1 issues for query tile 0, warp 3 for tile 1: one thread's waits, fences
            // and issue slots took 2250 cycles a tile, the products themselves need 1280.
            // (A wait that runs out does not branch off: the tile is finished on whatever
            // the buffers hold and then given up, its slots not freed: a load may still be
            // on its way to one.)
            const int t = warp == 1 ? 0 : 1;
            const uint32_t e = ptx::elect_one();
            constexpr uint32_t idesc_qk = ptx::idesc_f16_f32(kTileQ, kTileK, 0, 0, kBf16);
            constexpr uint32_t idesc_pv = ptx::idesc_f16_f32(kTileQ, kV, 0, 1, kBf16);
            const uint32_t s_col = tmem + t * kTileK, o_col = tmem + kTmemO + t * kV;
            uint32_t at = 0;  // ring slots of the items before this one
            uint32_t qn = 0, pn = 0;
            bool ok = true;
            auto full = [&](uint32_t k) {
                ok &= ptx::mbar_spin(bar(kBarFull + k % kSlots), (k / kSlots) & 1, kErrWaitFull);
            };
            // S = Q . K(j)^T (the slots have landed)
            auto qk = [&](int j, bool last) {
                const uint32_t k0 = at + j * kSlotsPerTile;
#pragma unroll
                for (int c = 0; c < kKBlk; ++c) {
                    const uint32_t slot = (k0 + c) % kSlots;
                    const uint64_t a = ptx::sdesc_sw128(sbase + t * kQBytes + c * kBox, 16, 1024);
                    const uint64_t b = ptx::sdesc_sw128(sbase + kOffRing + slot * kBox, 16, 1024);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        ptx::mma_ss_if(e, s_col, a + (uint64_t)(k * 2), b + (uint64_t)(k * 2), idesc_qk,
                                       (c > 0 || k > 0) ? 1u : 0u);
                    ptx::mma_commit_if(ok ? e : 0u, bar(kBarEmpty + slot));
                }
                ptx::mma_commit_if(e, bar(kBarS + t));
                if (last) ptx::mma_commit_if(e, bar(kBarQEmpty + t));
            };
            // half c of O += P . V(j)
            auto pv = [&](int j, int c) {
                const uint32_t slot = (at + j * kSlotsPerTile + kKBlk + c) % kSlots;
                ok &= ptx::mbar_spin(bar(kBarP + 2 * t + c), pn & 1, kErrWaitMma);
                ptx::tc_fence_after();  // P (and a corrected O) were stored by other threads
                const uint64_t b = ptx::sdesc_sw128(sbase + kOffRing + slot * kBox, kVBox, 1024);
#pragma unroll
                for (int k = 0; k < kVHalf / 16; ++k)
                    ptx::mma_ts_if(e, o_col, s_col + (c * 4 + k) * 8, b + (uint64_t)((k * 16 * 128) >> 4), idesc_pv,
                                   (j > 0 || c > 0 || k > 0) ? 1u : 0u);
                ptx::mma_commit_if(ok ? e : 0u, bar(kBarEmpty + slot));
            };
            // the slots of a key tile that this query tile does not see
            auto skip = [&](uint32_t k0, int n) {
                for (int c = 0; c < n; ++c) {
                    full(k0 + c);
                    if (ok && e) ptx::mbar_arrive(bar(kBarEmpty + (k0 + c) % kSlots));
                }
            };
            while (ok && next_item()) {
                if (it.nmax <= 0) continue;
                const int n = __shfl_sync(0xffffffffu, it.n[t], 0), nmax = __shfl_sync(0xffffffffu, it.nmax, 0);
                if (n > 0) {
                    ok &= ptx::mbar_spin(bar(kBarQFull + t), qn & 1, kErrWaitFull);
                    ++qn;
                    for (int c = 0; c < kKBlk; ++c) full(at + c);
                    qk(0, n == 1);
                }
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    ok = ok && !*abort_flag;
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    // (the waits for what the ring brings go before those for P)
                    const uint32_t k0 = at + j * kSlotsPerTile;
                    full(k0 + kKBlk);
                    full(k0 + kKBlk + 1);
                    pv(j, 0);
                    if (j + 1 < n)
                        for (int c = 0; c < kKBlk; ++c) full(k0 + kSlotsPerTile + c);
                    pv(j, 1);
                    ++pn;
                    ptx::mma_commit_if(e, bar(kBarO + t));
                    if (j + 1 < n) qk(j + 1, j + 2 == n);
                }
                if (ok && n < nmax) skip(at + n * kSlotsPerTile, (nmax - n) * kSlotsPerTile);
                at += nmax * kSlotsPerTile;
                // (a wait runs out by each lane's own clock: the lanes go on to the next
                // item's vote, or to the end, together)
                ok = __all_sync(0xffffffffu, ok);
            }
            if (!ok) *abort_flag = 1;
            // every MMA has retired before TMEM and shared memory go
            ptx::mma_commit_if(e, bar(kBarDrain + t));
            ptx::mbar_wait(bar(kBarDrain + t), 0, kErrWaitMma);
        } else if (warp == 2) {
            // ------------------------------------------------------ V tail
            // The rows of a sequence's last V tile past its end hold the next
            // sequence's values, or none: P is 0 there, but 0 x NaN is not.  Such a
            // tile lands on a barrier of this warp, which zeroes those rows and then
            // completes the slots' own barriers.  Two barriers in turn: the producer
            // may be one item ahead, but not two, as the ring does not hold the
            // second's values before the first's are used.
            //
            // It also keeps the item queue filled, two ahead of the item it is at: each CTA
            // takes the next item that nobody has (dealt out in advance, the CTAs ended up to
            // 30 % apart).
            uint32_t at = 0, tails = 0, put = 0;
            bool ok = true, more = true;
            const int pairs = p.pairs != nullptr ? *p.num_pairs : p.batch * p.blocks, total = pairs * p.heads * p.splits;
            auto publish = [&]() {
                if (!more || !ok) return;
                const uint32_t q = put % kQueue;
                ok = __all_sync(0xffffffffu, wait_or_abort(bar(kBarItemFree + q), ((put / kQueue) & 1) ^ 1, abort_flag));
                if (!ok) return;
                Item next{};
                for (;;) {  // (items without rows are left out)
                    int u = p.pairs != nullptr ? 0 : put == 0 && more ? (int)blockIdx.x : total;
                    if (p.pairs != nullptr && lane == 0) u = atomicAdd(p.next_item, 1);
                    u = __shfl_sync(0xffffffffu, u, 0);
                    if (u >= total) {
                        more = false;
                        next.nmax = kNoMore;
                        break;
                    }
                    if (item_at(p, pairs, u, next)) break;
                    if (p.pairs == nullptr) {  // (its only item)
                        more = false;
                        next.nmax = kNoMore;
                        break;
                    }
                }
                if (lane == 0) {
                    *reinterpret_cast<Item *>(smem + kOffItems + q * kItemBytes) = next;
                    ptx::mbar_arrive(bar(kBarItem + q));
                }
                __syncwarp();
                ++put;
            };
            publish();
            publish();
            for (uint32_t n = 0; ok; ++n) {
                publish();
                if (!ok) break;
                it = *reinterpret_cast<const Item *>(smem + kOffItems + (n % kQueue) * kItemBytes);
                if (it.nmax == kNoMore) break;
                if (it.nmax <= 0) continue;
                const int left = it.s.lk - (it.nmax - 1) * kTileK;  // tokens in the last tile
                if (left < kTileK) {
                    const uint32_t k0 = at + (it.nmax - 1) * kSlotsPerTile + kKBlk;
                    ok = wait_or_abort(bar(kBarTail + (tails & 1)), (tails >> 1) & 1, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    ++tails;
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {
                        const int keep = min(max(left - c * kVHalf, 0), kVHalf);
                        const uint32_t base = sbase + kOffRing + ((k0 + c) % kSlots) * kBox;
                        // 16-byte pieces of rows keep.. of both 64-column boxes
                        for (int q = lane; q < (kVHalf - keep) * 16; q += 32)
                            ptx::st_shared_v4(base + ((q >> 3) & 1) * kVBox + (keep + (q >> 4)) * 128 + (q & 7) * 16, 0u, 0u, 0u, 0u);
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane < 2) ptx::mbar_arrive(bar(kBarFull + (k0 + lane) % kSlots));
                }
                at += it.nmax * kSlotsPerTile;
            }
            if (!ok) *abort_flag = 1;
        }
    } else {
        // ---------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int t = warp >= 8 ? 1 : 0;
        const int r = tid - 128 - t * 128;  // row of the tile = TMEM lane
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lanes + t * kTileK, o_addr = tmem + lanes + kTmemO + t * kV;
        uint32_t sn = 0;  // S tiles so far (PV tile k completes phase k of kBarO)
        bool ok = true;
        const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
        while (ok && next_item()) {
            const int row = it.row + t * kTileQ + r;
            if (it.row + t * kTileQ >= it.s.lq) continue;
            const int n = it.n[t];
            // keys this row sees (rows past the sequence's end: like its last row)
            int sees = it.s.lk;
            if (p.causal) sees = min(sees, min(row, it.s.lq - 1) + 1 + it.ahead);
            float m_used = -INFINITY, l_run = 0.f;
            for (int j = 0; j < n; ++j, ++sn) {
                ok = !*abort_flag && ptx::mbar_wait_now(bar(kBarS + t), sn & 1, kErrWaitMma);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ptx::tc_fence_after();
                uint32_t s[kTileK];
#pragma unroll
                for (int q = 0; q < 4; ++q) ptx::tmem_ld_x32(s_addr + q * 32, *reinterpret_cast<uint32_t(*)[32]>(s + q * 32));
                ptx::tmem_wait_ld();
                const int valid = sees - j * kTileK;
                if (valid < kTileK) {
#pragma unroll
                    for (int k = 0; k < kTileK; ++k)
                        if (k >= valid) s[k] = tc::u32_of(-INFINITY);
                }
                float m8[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) m8[k] = fmaxf(tc::f32_of(s[k]), tc::f32_of(s[8 + k]));
#pragma unroll
                for (int k = 16; k < kTileK; k += 16)
#pragma unroll
                    for (int i = 0; i < 8; ++i) m8[i] = max3(m8[i], tc::f32_of(s[k + i]), tc::f32_of(s[k + 8 + i]));
                const float mx = max3(max3(m8[0], m8[1], m8[2]), max3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7])) * p.scale_log2;
                float alpha = 1.f;
                if (mx > m_used + kRescaleLog2) {
                    alpha = m_used == -INFINITY ? 0.f : ptx::ex2(m_used - mx);
                    m_used = mx;
                }
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_now(bar(kBarO + t), (sn - 1) & 1, kErrWaitMma));
                    if (!ok) break;
                    ptx::tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < kV / 32; ++c) {
                        uint32_t o[32];
                        ptx::tmem_ld_x32(o_addr + c * 32, o);
                        ptx::tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = tc::u32_of(tc::f32_of(o[k]) * alpha);
                        ptx::tmem_st_x32(o_addr + c * 32, o);
                    }
                }
                // (a row that has seen nothing keeps m_used = -inf: its weights are 0)
                const float nm = m_used == -INFINITY ? 0.f : -m_used;
                const float2 neg = make_float2(nm, nm);
                float2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t pk[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        float2 x = make_float2(tc::f32_of(s[hf * 64 + 2 * k]), tc::f32_of(s[hf * 64 + 2 * k + 1]));
                        x = fma2(x, sl2, neg);
                        x.x = ptx::ex2(x.x);
                        x.y = ptx::ex2(x.y);
                        sum[k & 3] = add2(sum[k & 3], x);
                        pk[k] = tc::pack2<kBf16>(x.x, x.y);
                    }
                    ptx::tmem_st_x32(s_addr + hf * 32, pk);
                    // (the first half's product runs under the second half's exponentials)
                    ptx::tmem_wait_st();
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(bar(kBarP + 2 * t + hf));
                }
                const float2 a = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
                l_run = l_run * alpha + (a.x + a.y);
            }
            if (!ok) break;
            // ------------------------------------------------------ epilogue
            const bool real = row < it.s.lq;
            const bool part = p.splits > 1;
            const long long orow = ((long long)it.split * p.total_q + it.s.q0 + row) * p.heads + it.h;
            uint8_t *dst = part ? reinterpret_cast<uint8_t *>(p.part_o + orow * kV)
                                : static_cast<uint8_t *>(p.out) + orow * (kV * 2);
            const float inv = l_run != 0.f ? 1.f / l_run : 0.f;  // (NaN stays NaN)
            if (n > 0) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait_now(bar(kBarO + t), (sn - 1) & 1, kErrWaitMma));
                if (!ok) break;
                ptx::tc_fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < kV / 32; ++c) {
                uint32_t o[32];
                if (n > 0) {
                    ptx::tmem_ld_x32(o_addr + c * 32, o);
                    ptx::tmem_wait_ld();
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = 0u;
                }
                if (part) {
                    uint32_t w[4][8];
#pragma unroll
                    for (int k = 0; k < 32; ++k) w[k >> 3][k & 7] = tc::u32_of(tc::f32_of(o[k]) * inv);
                    if (real) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) store32(dst + c * 128 + k * 32, w[k]);
                    }
                } else {
                    uint32_t w[2][8];
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        w[k >> 3][k & 7] = tc::pack2<kBf16>(tc::f32_of(o[2 * k]) * inv, tc::f32_of(o[2 * k + 1]) * inv);
                    if (real) {
                        store32(dst + c * 64, w[0]);
                        store32(dst + c * 64 + 32, w[1]);
                    }
                }
            }
            ptx::tc_fence_before();  // O is read before this thread's next P arrival lets a PV overwrite it
            float *lse = part ? p.part_lse : p.out_lse;
            if (real && lse != nullptr)
                lse[orow] = l_run != 0.f ? (m_used + __log2f(l_run)) * kLn2 : -INFINITY;
        }
        if (!ok) *abort_flag = 1;
    }

    ptx::tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 2) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the shares of the keys: out = sum_s e^(lse_s - M) o_s / sum_s e^(lse_s - M).  A
// warp per (query, head), 4 columns a lane; the shares are few and small (they are made
// only where there are fewer items than SMs).
template <typename OutT>
__global__ void __launch_bounds__(256) merge_kernel(const PrefillParams p) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)p.total_q * p.heads, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    // (a row outside every sequence has no shares)
    if (p.cu_q != nullptr) {
        const int i = (int)(row / p.heads);
        bool in = false;
        for (int b = lane; b < p.batch; b += 32) {
            const Seq s = seq_of(p, b);
            in |= i >= s.q0 && i < s.q0 + s.lq;
        }
        if (!__any_sync(0xffffffffu, in)) return;
    }
    const float mine = lane < p.splits ? p.part_lse[lane * rows + row] : -INFINITY;
    const float mx = __any_sync(0xffffffffu, mine != mine) ? NAN : warp_max(mine);
    const float w = mx == -INFINITY ? 0.f : __expf(mine - mx);  // exp(-inf) = 0
    const float total = warp_sum(w);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
        const float ws = __shfl_sync(0xffffffffu, w, s);
        const float4 o = reinterpret_cast<const float4 *>(p.part_o + (s * rows + row) * kV)[lane];
        if (ws != 0.f) {
            acc.x = fmaf(ws, o.x, acc.x);
            acc.y = fmaf(ws, o.y, acc.y);
            acc.z = fmaf(ws, o.z, acc.z);
            acc.w = fmaf(ws, o.w, acc.w);
        }
    }
    const float inv = total != 0.f ? 1.f / total : 0.f;
    *reinterpret_cast<uint2 *>(static_cast<OutT *>(p.out) + row * kV + 4 * lane) =
        make_uint2(pack_out2<OutT>(acc.x * inv, acc.y * inv), pack_out2<OutT>(acc.z * inv, acc.w * inv));
    if (lane == 0 && p.out_lse != nullptr) p.out_lse[row] = total != 0.f ? mx + __logf(total) : -INFINITY;
}
constexpr int kMaxSplits = 32;  // a lane each

}  // namespace prefill
}  // namespace mla
