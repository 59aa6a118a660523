// mla_tree.cuh -- attention of a tree of drafted tokens over the paged latent cache.
//
//   O[b, i, h] = softmax(scale Q*[b, i, h] . C_b^T + M[b, i]) . C_b[:, :512]
//
// for drafts i < k of sequence b, whose own rows are the last k of C_b: M hides draft
// row j from draft i unless bit j of i's mask is set, and nothing else.
//
// (draft, head) rows fill tiles of 128 rows: as many whole drafts as fit, dealt
// evenly over a sequence's tiles.  A tile is a "sequence" of the work list (WorkList:
// split by cost over the clusters, partials merged below), and reads its sequence's
// pages once.  Per cached token a tile needs 1152 bytes and 2 x 128 x (576 + 512)
// flop, so one tile is bound by HBM (1152 B / 6.5 TB/s over 74 clusters = 13 ns) about
// as much as by the tensor cores (12.6 ns); a sequence's further tiles find its rows in
// L2.
//
// The two products do not fit one SM's TMEM (O alone is all of it), so a tile runs on
// a cluster of two, as in the decode of one token per sequence (tc_decode_kernel): the
// S-CTA keeps Q in TMEM, computes S = Q C^T for 96 tokens at a time and the softmax,
// and sends P to the O-CTA, which accumulates O += P C_N.  Different here:
//
//   * the softmax of a tile is shared by two warpgroups, 48 columns each: with one,
//     its 1.2 us a tile were longer than everything else on the S-CTA.  They exchange
//     row maxima in shared memory behind one barrier; a warp of its own sends the
//     messages, so that nobody else waits for the O-CTA;
//   * the producer warp holds the block-table entries of ten tiles (30 pieces of 32
//     rows), a lane each, and loads the next ten ahead;
//   * rows of a C tile that no draft of the tile may see (past the sequence's end, or
//     padded drafts that may never have been written) are zeroed by a warp of their own
//     before GEMM2 (0 x NaN is not 0): such tiles land on that warp's barrier, which
//     then completes the slot's.  No other tile pays for it;
//   * partials are fp32, in two planes: the upper 16 bits of each value and what is kept of
//     the lower ones, all 16 for fp32 output, 8 for 16-bit output.  24 bits keep every value
//     to 2^-15 of itself (1/16 of fp16's rounding, whatever its neighbours hold) at three
//     quarters of the bytes (128 rows over 4104 tokens 23.3 us a call, 24.8 with 32 bits; 64
//     sequences x 112 rows 121.6, 124).  Each plane lies 16 columns (32 or 16 bytes) of all
//     rows together, so a warp's stores are whole kilobytes in a row;
//
//   * the schedule is made inside the kernel (plan_here).
//
// Roles (384 threads): warp 0 TMA producer, warps 1 and 3 MMA issuers (GEMM1 alternates
// between them; GEMM2 has one), warp 2 TMEM owner and message sender (S-CTA) or row
// zeroing (O-CTA), warps 4-11 math: thread h of each warpgroup owns row h.  Every wait
// is bounded.
//
// A call among others, with its merge, on inputs that change (a loop of such calls runs at
// the power cap, the larger ones near 1.5 GHz): 64 sequences of 1024-8192 tokens x 112 rows
// (356 MB of rows) 121 us, 2.9 TB/s and 0.6 PFLOP/s at once; 8 x 1536 rows 154 us, 0.89
// PFLOP/s; 512 rows over 131072 tokens 178 us, 0.82 PFLOP/s; 128 rows over 4104 tokens 23 us,
// one tile through the pair after the other.  The loop is bound by shared memory: an S
// tile's rows are written and read once on either SM (220 KB) and its weights as well (50
// KB), 2110 cycles at 128 bytes a cycle; 2550-2900 are measured, GEMM1 alone needs 1728.
// Over a whole launch there are 2950 cycles an S tile in long items (131072 tokens), 3270
// with 8 x 1536 rows and 3900 with 64 x 112, two items a cluster: what an item's start (Q,
// first tile) and end (its partial leaves one SM) add to the loop.
#pragma once

#include "mla_combine.cuh"
#include "mla_tc.cuh"

namespace mla {
namespace tree {

using tc::kBoxO;
using tc::kBoxS;
using tc::kKBlocks;
using tc::kKbPerSlot;
using tc::kOPerS;
using tc::kPieceS;
using tc::kQBoxBytes;
using tc::kQSlots;
using tc::kSlotO;
using tc::kSlotS;
using tc::kSlotsO;
using tc::kSlotsPerTile;
using tc::kSlotsS;
using tc::kSubP;
using tc::kTO;
using tc::kTS;
using tc::kVBlocks;

constexpr int kThreads = 384;
constexpr int kMath = 256;        // threads of the two math warpgroups
constexpr int kHalf = kTS / 2;    // columns of one warpgroup
constexpr int kRowTiles = 10;     // tiles whose block-table entries the producer warp holds
constexpr int kMergeWarps = 8;    // warps of a merge block
constexpr uint64_t kTailWaitNs = 20000000000ull;  // the zeroing warp waits through whole items

// Message S-CTA -> O-CTA, one per S tile: P as three SW64 K-major sub-tiles of [128
// rows x 32 tokens], then per row alpha, the two warpgroups' sums, m.
constexpr int kMsgP = kOPerS * kSubP;          // 24576
constexpr int kMsgAlpha = kMsgP;
constexpr int kMsgL = kMsgP + 512;             // [2][128]
constexpr int kMsgM = kMsgP + 1536;
constexpr int kMsgBytes = kMsgP + 2048;        // 26624
constexpr int kMsgSlots = 3;

enum BarId {
    kBarFull = 0,                       // ring slot landed (and its hidden rows zeroed); S-CTA: one of issuer 0's
    kBarEmpty = kSlotsS,                // ring slot consumed
    kBarSFull = 2 * kSlotsS,            // [2] S-CTA: S tile in TMEM
    kBarSEmpty = kBarSFull + 2,         // [2] S-CTA: S tile read (256)
    kBarQFree = kBarSEmpty + 2,         // [2] S-CTA: an issuer's GEMM1s reading Q done
    kBarQReady = kBarQFree + 2,         //     S-CTA: a tile's Q copied into TMEM
    kBarPFree = kBarQReady + 1,         // [3] GEMM2 done with a message slot (in both CTAs)
    kBarPFull = kBarPFree + kMsgSlots,  // [3] O-CTA: message landed
    kBarCorr = kBarPFull + kMsgSlots,   // [3] O-CTA: O ready for GEMM2 (256)
    kBarMmaDone = kBarCorr + kMsgSlots, // [3] O-CTA: GEMM2 of a message done
    kBarTail = kBarMmaDone + kMsgSlots, // [4] O-CTA: slot landed, hidden rows not yet zeroed
    kBarDrain = kBarTail + kSlotsO,     // [2] an issuer's operations retired
    kBarStaged = kBarDrain + 2,         //     S-CTA: a message is in the staging buffer (256)
    kBarStgFree = kBarStaged + 1,       //     S-CTA: it has left it
    kBarFull1 = kBarStgFree + 1,        //     S-CTA: ring slot of issuer 1's landed
    kNumBars = kBarFull1 + kSlotsS
};
static_assert(kSlotsS >= kSlotsO, "ring barriers");

constexpr int kOffRing = 0;
constexpr int kOffStg = kSlotsS * kSlotS;                   // S-CTA: message staging
constexpr int kOffMsg = kSlotsO * kSlotO;                   // O-CTA: received messages [3]
constexpr int kOffBar = kOffStg + kMsgBytes;
static_assert(kOffMsg + kMsgSlots * kMsgBytes <= kOffBar, "O-CTA layout");
static_assert(kMsgBytes % 1024 == 0, "swizzle atoms of the message slots");
constexpr int kOffSlot = kOffBar + kNumBars * 8;
constexpr int kOffAbort = kOffSlot + 4;
constexpr int kOffMax = (kOffAbort + 4 + 15) / 16 * 16;     // S-CTA: row maxima [2 tiles][2 halves][128]
// The plan of up to kPlanMax row tiles, made by every CTA for itself: offsets of the
// tiles' sequences on a virtual packed axis, places on the cost line, drafts seen.
constexpr int kPlanMax = 960;
// Up to here every warp makes it (plan_few): 1 tile of 43 S tiles, 22.9 us against 24.2; 31
// tiles 63.8 against 65.4; with 64 tiles there is no difference.
constexpr int kPlanFew = 31;
constexpr int kOffSeen = kOffMax + 2 * 2 * 128 * 4;
constexpr int kOffCu = kOffSeen + kPlanMax * 8;
constexpr int kOffCost = kOffCu + (kPlanMax + 4) * 4;
constexpr int kSmemBytes = kOffCost + (kPlanMax + 4) * 4 + 1024;
static_assert(kSmemBytes <= 232448, "dynamic shared memory limit");
static_assert(2 * (kPlanFew + 1) <= kPlanMax, "two warps' drafts seen");
constexpr uint32_t kTmemCols = 512, kTmemQ = 0, kTmemS = 288;

struct TreeParams {
    WorkList wl;
    int num_heads;     // rows of a full tile = rows between partials: tile_drafts * heads
    float scale_log2;  // softmax scale * log2(e)
    uint8_t *part_hi;  // [slots, 32 pieces, num_heads, 16] upper 16 bits: see part_piece
    uint8_t *part_lo;  // the same of the lower 16 bits (fp32 output), or the upper 8 of them
    float *part_lse;   // [slots, num_heads]
    void *out;         // [batch, drafts, heads, 512]: written directly for tiles of one item
    int out_kind;      // tc::OutKind
    float *out_lse;    // [batch, drafts, heads] or null
    int chain;         // the merge after this launch is a programmatic dependent
    const int32_t *block_table;
    int max_blocks, page_size, num_pages;
    const unsigned long long *mask;   // [batch or 1, drafts]; null: a chain
    const unsigned long long *seen;   // [tiles of all sequences], made by a plan kernel; or, with
    const int32_t *seq_lens;          // seq_lens, made in the kernel (null: by a plan kernel)
    int max_seq_len;
    int2 *plan_range;                 // with seq_lens: every tile's items, for the merge kernel
    int mask_stride;                  // drafts, or 0 (one mask for all)
    int drafts, heads, tiles, tile_drafts;
};

// Rows of query, output and LSE before tile v, and the rows it has.
__device__ __forceinline__ void tree_rows(const TreeParams &p, int v, long long &row0, int &rows) {
    const int b = v / p.tiles, d0 = (v - b * p.tiles) * p.tile_drafts;
    row0 = ((long long)b * p.drafts + d0) * p.heads;
    rows = min(p.tile_drafts, p.drafts - d0) * p.heads;
}

// Which of the 32 tokens [t, t + 32) a row sees whose drafts start at token `start`:
// all before `start`, then the bits of `mask` (clear at and past the number of
// drafts), so none past the sequence's end.
__device__ __forceinline__ uint32_t tree_word(unsigned long long mask, int start, int t) {
    const int s = start - t;
    if (s >= 32) return 0xffffffffu;
    if (s >= 0) return ((1u << s) - 1u) | (uint32_t)(mask << s);
    return s > -64 ? (uint32_t)(mask >> -s) : 0u;
}

// First token of the drafts of tile v's sequence (below 0 when it is shorter).
__device__ __forceinline__ int draft_start(const WorkList &wl, const TreeParams &p, int v) {
    return wl.cu_seqlens[v + 1] - wl.cu_seqlens[v] - p.drafts;
}

// Draft i of the tiles' drafts in a row (tile i / tile_drafts): the drafts it sees.
__device__ __forceinline__ unsigned long long draft_mask(const TreeParams &p, int ntiles, int i) {
    const int v = i / p.tile_drafts, b = v / p.tiles;
    const int d = (v - b * p.tiles) * p.tile_drafts + (i - v * p.tile_drafts);
    if (i >= ntiles * p.tile_drafts || d >= p.drafts) return 0;
    const unsigned long long m = p.mask != nullptr ? p.mask[(long long)b * p.mask_stride + d] : (2ull << d) - 1;
    return p.drafts < 64 ? m & ((1ull << p.drafts) - 1) : m;
}

// plan_here's tables for a few tiles, by every warp for itself (all write the same cu and
// cost; `seen`, where asked for, is the warp's own): one round of loads and a warp's scan
// instead of four barriers of the CTA.
__device__ void plan_few(const TreeParams &p, int ntiles, int item_cost, int *cu, int *cost, unsigned long long *seen) {
    constexpr int kPer = (kPlanFew + 1) / 32;
    const int lane = threadIdx.x & 31;
    int2 own[kPer], sum = make_int2(0, 0);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int v = lane * kPer + k;
        const int len = v < ntiles ? min(max(p.seq_lens[v / p.tiles], 0), p.max_seq_len) : 0;
        own[k] = make_int2(len, len > 0 ? (len + kTile - 1) / kTile + item_cost : 0);
    }
    if (seen != nullptr) {
        for (int v = lane; v < ntiles; v += 32) seen[v] = 0;
        __syncwarp();
        for (int i = lane; i < ntiles * p.tile_drafts; i += 32) {
            const unsigned long long m = draft_mask(p, ntiles, i);
            if (m != 0) atomicOr(seen + i / p.tile_drafts, m);
        }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        sum.x += own[k].x;
        sum.y += own[k].y;
    }
    int2 at = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, at.x, o), y = __shfl_up_sync(0xffffffffu, at.y, o);
        if (lane >= o) {
            at.x += x;
            at.y += y;
        }
    }
    at.x -= sum.x;
    at.y -= sum.y;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int v = lane * kPer + k;
        if (v <= ntiles) {  // the entry after the last tile is the total
            cu[v] = at.x;
            cost[v] = at.y;
        }
        at.x += own[k].x;
        at.y += own[k].y;
    }
    __syncwarp();
}

// The balanced schedule's tables (lens_to_offsets, plan_balanced_kernel and plan_tree in
// one) in this CTA's shared memory, by all its threads: a scan over up to kPlanMax
// tiles takes about a microsecond, a plan kernel before this one cost four and a launch.
__device__ void plan_here(const TreeParams &p, int ntiles, int item_cost, int *cu, int *cost,
                          unsigned long long *seen) {
    constexpr int kPer = (kPlanMax + kThreads - 1) / kThreads;
    __shared__ int2 warp_tot[kThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int2 own[kPer], sum = make_int2(0, 0);
    int lens[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int v = tid * kPer + k;
        lens[k] = v < ntiles ? p.seq_lens[v / p.tiles] : 0;
    }
    // the drafts seen, a thread per (tile, draft): one round of loads, beside the lengths'
    unsigned long long mine = draft_mask(p, ntiles, tid);
    for (int v = tid; v < ntiles; v += kThreads) seen[v] = 0;
    __syncthreads();
    for (int i = tid; i < ntiles * p.tile_drafts; i += kThreads) {
        if (i != tid) mine = draft_mask(p, ntiles, i);
        if (mine != 0) atomicOr(seen + i / p.tile_drafts, mine);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int len = min(max(lens[k], 0), p.max_seq_len);
        own[k] = make_int2(len, len > 0 ? (len + kTile - 1) / kTile + item_cost : 0);
        sum.x += own[k].x;
        sum.y += own[k].y;
    }
    int2 v2 = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v2.x, o), y = __shfl_up_sync(0xffffffffu, v2.y, o);
        if (lane >= o) {
            v2.x += x;
            v2.y += y;
        }
    }
    if (lane == 31) warp_tot[warp] = v2;
    __syncthreads();
    int2 at = make_int2(v2.x - sum.x, v2.y - sum.y);
    for (int k = 0; k < warp; ++k) {
        at.x += warp_tot[k].x;
        at.y += warp_tot[k].y;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int v = tid * kPer + k;
        if (v <= ntiles) {  // the entry after the last tile is the total
            cu[v] = at.x;
            cost[v] = at.y;
        }
        at.x += own[k].x;
        at.y += own[k].y;
    }
    __syncthreads();
}
static_assert(((kPlanMax + kThreads - 1) / kThreads) * kThreads > kPlanMax, "a thread for the total's entry");

// Pool row of the 32-row piece at token t of sequence b; pieces past the item's last
// token re-read its last piece (the softmax hides them).
__device__ __forceinline__ int pool_row(const TreeParams &p, int b, int t, int last) {
    const int tc = min(t, last & ~(kTO - 1));
    const int blk = tc / p.page_size;
    // (an entry that is no page: the row after the pool, which TMA reads as zeros)
    const int pg = (int)min((unsigned)p.block_table[(long long)b * p.max_blocks + blk], (unsigned)p.num_pages);
    return pg * p.page_size + (tc - blk * p.page_size);
}

// Partial slot of item `id`, the `s`-th of tile v.  The balanced schedule gives worker w
// the items id = v + w (items_next): of a split tile's items the later ones are their
// worker's first and the first one its worker's last, so two slots a worker hold all
// partials, however many tiles there are.
__device__ __forceinline__ size_t part_slot(const WorkList &wl, bool balanced, int v, int id, int s) {
    return balanced ? id - v + (s == 0 ? wl.nworkers : 0) : id;
}

// Place of 16 columns (16 piece ..) of row r of a partial, in units of 16 columns.
__device__ __forceinline__ size_t part_piece(const TreeParams &p, size_t slot, int piece, int r) {
    return (slot * (kDV / 16) + piece) * p.num_heads + r;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ void load32(const void *src, uint32_t (&v)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(src));
}

__device__ __forceinline__ void load16(const void *src, uint32_t (&v)[4]) {
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "l"(src));
}

__device__ __forceinline__ void store16(void *dst, const uint32_t *v) {
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
}

__device__ __forceinline__ void store32(void *dst, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// cmap_s: the pool as (64, 8 rows, 9 K-blocks, row groups), one box = 3 K-blocks x 32
// rows, three boxes to a ring slot (its K-blocks interleaved per 8-row group); cmap_o:
// the pool as (64, rows, 9), one box = 8 K-blocks x 32 rows; qmap: the queries
// [batch * drafts * heads, 576], box 64 x 128.  128-byte swizzle.
template <int kSched, bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap cmap_s, const __grid_constant__ CUtensorMap cmap_o,
                  const __grid_constant__ CUtensorMap qmap, const TreeParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = ptx::smem_u32(smem);
    auto bar = [&](int id) -> uint32_t { return sbase + kOffBar + 8u * id; };
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + kOffAbort);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t role = ptx::cluster_ctarank();  // 0 = S-CTA, 1 = O-CTA
    const int cid = (int)ptx::cluster_id_x(), ncl = (int)ptx::nclusters_x();

    if (tid == 0) {
        for (int i = 0; i < kNumBars; ++i) {
            const bool math = (i >= kBarSEmpty && i < kBarSEmpty + 2) || (i >= kBarCorr && i < kBarCorr + kMsgSlots) ||
                              i == kBarStaged;
            ptx::mbar_init(bar(i), math ? kMath : 1);
        }
        *abort_flag = 0;
        ptx::fence_mbarrier_init_cluster();
    }
    if (warp == 0 && lane == 0) {
        ptx::tma_prefetch_desc(role == 0 ? &cmap_s : &cmap_o);
        if (role == 0) ptx::tma_prefetch_desc(&qmap);
    }
    if (warp == 2) {
        ptx::tmem_alloc(sbase + kOffSlot, kTmemCols);
        ptx::tmem_relinquish();
    }
    // The cluster barrier is .aligned: a warp that came to it in parts (lanes 1-31 of warp 0
    // while lane 0 still initialises barriers) would be counted too early, and the partner
    // could then use barriers that are not there yet.
    __syncwarp();
    ptx::tc_fence_before();
    ptx::cluster_sync();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + kOffSlot);
    if (p.chain) griddep_launch();  // the chained merge may place its CTAs
    griddep_wait();                 // the plan kernel's work list
    WorkList wl = p.wl;
    const unsigned long long *seen_of = p.seen;
    if (kSched == kSchedBalanced && p.seq_lens != nullptr) {
        int *cu = reinterpret_cast<int *>(smem + kOffCu), *cost = reinterpret_cast<int *>(smem + kOffCost);
        unsigned long long *seen = reinterpret_cast<unsigned long long *>(smem + kOffSeen);
        const bool few = wl.batch <= kPlanFew;
        if (few) {
            // (read by the O-CTA's producer and its warp of hidden rows)
            if (warp == 2) seen += kPlanFew + 1;
            plan_few(p, wl.batch, wl.item_cost, cu, cost, role == 1 && (warp == 0 || warp == 2) ? seen : nullptr);
        } else {
            plan_here(p, wl.batch, wl.item_cost, cu, cost, seen);
        }
        wl.cu_seqlens = cu;
        wl.cost_off = cost;
        seen_of = seen;
        if (blockIdx.x == 0 && (!few || warp == 2)) {
            for (int v = few ? lane : tid; v < wl.batch; v += few ? 32 : kThreads) {
                int i0, i1;
                item_range<kSched>(wl, v, i0, i1);
                p.plan_range[v] = make_int2(i0, i1);
            }
        }
    }
    ItemCursor cur = items_begin<kSched>(wl, cid, ncl);
    Item it;
    int id;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        // (a whole warp with one elected lane, as the MMA issuers below)
        const uint32_t e = ptx::elect_one();
        const int nslots = role == 0 ? kSlotsS : kSlotsO;
        tc::Ring rg;
        int prev_b = -1;
        uint32_t jt = 0;
        bool ok = true;
        auto acquire = [&]() {
            ok = ok && !*abort_flag && ptx::mbar_wait_now(bar(kBarEmpty + rg.slot), rg.phase ^ 1, kErrWaitEmpty);
            ok = __all_sync(0xffffffffu, ok);
        };
        while (ok && items_next<kSched>(wl, cur, it, id)) {
            const int len = __shfl_sync(0xffffffffu, it.len, 0), tok0 = __shfl_sync(0xffffffffu, it.tok0, 0);
            const int v = __shfl_sync(0xffffffffu, it.b, 0), b = v / p.tiles, last = tok0 + len - 1;
            auto rows_from = [&](int piece) -> int {  // this lane's piece of ten tiles
                return pool_row(p, b, tok0 + (piece + min(lane, kRowTiles * kOPerS - 1)) * kTO, last);
            };
            int row = 0, row_next = rows_from(0);
            const int start = draft_start(wl, p, v);
            const unsigned long long seen = role == 1 ? seen_of[v] : 0;
            // Q of a new row tile goes through the ring too, two 128 x 64 boxes (K-blocks) to
            // a slot, in front of the first S tile's slots that need them: Q01 Q23 C012 Q45
            // C345 Q67 Q8 C678, so that the two come in together.
            const bool new_q = role == 0 && v != prev_b;
            prev_b = v;
            long long q_row = 0;
            if (new_q) {
                int n;
                tree_rows(p, v, q_row, n);
            }
            for (int t0 = 0; ok && t0 < len; t0 += kTS, ++jt) {
                const int piece = t0 / kTO, at = piece % (kRowTiles * kOPerS);
                if (at == 0) {
                    row = row_next;
                    row_next = rows_from(piece + kRowTiles * kOPerS);
                }
                int pr[kOPerS];
#pragma unroll
                for (int c = 0; c < kOPerS; ++c) pr[c] = __shfl_sync(0xffffffffu, row, at + c);
                if (role == 0) {
                    const int full = (jt & 1) ? kBarFull1 : kBarFull;  // the tile's issuer's
#pragma unroll 1
                    for (int sl = 0; sl < kSlotsPerTile; ++sl) {
                        if (new_q && t0 == 0) {
                            int kb = sl == 0 ? 0 : sl == 1 ? 4 : 6;
#pragma unroll 1
                            for (int c = sl == 1 ? 1 : 0; c < 2 && ok; ++c, kb += 2) {
                                acquire();
                                if (!ok) break;
                                const int nb = min(2, kKBlocks - kb);
                                const uint32_t dst = sbase + kOffRing + rg.slot * kSlotS;
                                ptx::mbar_arrive_expect_tx_if(e, bar(full + rg.slot), nb * kQBoxBytes);
                                for (int j = 0; j < nb; ++j)
                                    ptx::tma_load_2d_if(e, dst + j * kQBoxBytes, &qmap, (kb + j) * 64, (int)q_row,
                                                        bar(full + rg.slot));
                                rg.next(nslots);
                            }
                        }
                        acquire();
                        if (!ok) break;
                        const uint32_t dst = sbase + kOffRing + rg.slot * kSlotS;
                        ptx::mbar_arrive_expect_tx_if(e, bar(full + rg.slot), kSlotS);
#pragma unroll
                        for (int c = 0; c < kOPerS; ++c)
                            ptx::tma_load_4d_if(e, dst + c * kPieceS, &cmap_s, 0, 0, sl * kKbPerSlot, pr[c] >> 3,
                                                bar(full + rg.slot));
                        rg.next(nslots);
                    }
                } else {
                    const int nct = (min(kTS, len - t0) + kTO - 1) / kTO;
#pragma unroll
                    for (int ct = 0; ct < kOPerS; ++ct) {
                        if (ct >= nct) break;
                        acquire();
                        if (!ok) break;
                        const int t = tok0 + t0 + ct * kTO;
                        const bool hidden = t + kTO > start && tree_word(seen, start, t) != 0xffffffffu;
                        const uint32_t full = bar((hidden ? kBarTail : kBarFull) + rg.slot);
                        ptx::mbar_arrive_expect_tx_if(e, full, kSlotO);
                        ptx::tma_load_3d_if(e, sbase + kOffRing + rg.slot * kSlotO, &cmap_o, 0, pr[ct], 0, full);
                        rg.next(nslots);
                    }
                }
            }
        }
        if (!ok) *abort_flag = 1;
        // drain: every issued load has been consumed (or the wait expires)
        for (int k = 0; k < nslots; ++k, rg.next(nslots))
            ptx::mbar_wait(bar(kBarEmpty + rg.slot), rg.phase ^ 1, kErrWaitEmpty);
    } else if (warp == 1 && role == 1) {
        // ------------------------------------------------------------ O-CTA: GEMM2
        // (The issuing warps run as whole warps with uniform control flow and one elected
        // lane behind each instruction, so that descriptors stay in uniform registers: 48
        // cycles an MMA of N = 96 against 53 from a branch of lane 0, and ~100 there when
        // math warps share the scheduler.  So a wait that runs out does not branch off
        // either: the tile is finished on whatever the buffers hold and then given up, its
        // slots not freed: a load may still be on its way to one.)
        const uint32_t e = ptx::elect_one();
        tc::Ring rg;
        uint32_t jt = 0;
        bool ok = true;
        while (ok && items_next<kSched>(wl, cur, it, id)) {
            const int len = __shfl_sync(0xffffffffu, it.len, 0);
            for (int t0 = 0; t0 < len; t0 += kTS, ++jt) {
                const uint32_t ms = jt % kMsgSlots, mu = jt / kMsgSlots;
                ok = !*abort_flag && ptx::mbar_wait<true>(bar(kBarPFull + ms), mu & 1, kErrWaitPeer);
                ok = ok && ptx::mbar_spin(bar(kBarCorr + ms), mu & 1, kErrWaitMma);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                const int nct = (min(kTS, len - t0) + kTO - 1) / kTO;
                ptx::tc_fence_after();  // the correction's TMEM stores to O come first
                const uint64_t p0 = ptx::sdesc_sw64(sbase + kOffMsg + ms * kMsgBytes, 16, 512);
                for (int ct = 0; ct < nct; ++ct) {
                    ok &= ptx::mbar_spin(bar(kBarFull + rg.slot), rg.phase, kErrWaitFull);
                    const uint32_t acc0 = (t0 > 0 || ct > 0) ? 1u : 0u;
                    const uint64_t c0 = ptx::sdesc_sw128(sbase + kOffRing + rg.slot * kSlotO, kBoxO, 1024);
                    const uint64_t pa = p0 + (uint64_t)(ct * (kSubP >> 4));
#pragma unroll
                    for (int kk = 0; kk < kTO / 16; ++kk)
#pragma unroll
                        for (int nh = 0; nh < 2; ++nh)
                            ptx::mma_ss_if(e, tmem + nh * 256, pa + (uint64_t)((kk * 32) >> 4),
                                           c0 + (uint64_t)((nh * 4 * kBoxO + kk * 16 * 128) >> 4), tc::idesc_o<kBf16>(),
                                           kk > 0 ? 1u : acc0);
                    ptx::mma_commit_if(ok ? e : 0u, bar(kBarEmpty + rg.slot));
                    rg.next(kSlotsO);
                }
                // (in this order: once a message has come through a freed slot, the slot's
                // last kBarMmaDone phase is known to be complete)
                ptx::mma_commit_if(e, bar(kBarMmaDone + ms));
                ptx::mma_commit_mc_if(e, bar(kBarPFree + ms), 0x3);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            }
        }
        if (!ok) *abort_flag = 1;
        ptx::mma_commit_if(e, bar(kBarDrain));
        ptx::mbar_wait(bar(kBarDrain), 0, kErrWaitMma);
    } else if ((warp == 1 || warp == 3) && role == 0) {
        // ------------------------------------------------------------ S-CTA: GEMM1
        // Two warps take alternate S tiles (and S buffers).  At the first S tile of a
        // row tile its issuer copies Q into TMEM once every GEMM1 of the previous one
        // is done; the other waits for the copy before its next S tile.
        //
        // A wait by parity is exact only while the phase before the awaited one is known
        // to be complete, and an issuer does not wait for the other's slots: a load that
        // comes in late would let it take the slot's next use for landed.  So each has
        // its own set of barriers for the slots, and waits on the barriers they share
        // (kBarSFull, kBarQReady) only after kBarSEmpty: then the softmax has read tile
        // jt - 2, so every GEMM1 and copy of Q up to that tile is complete.
        const uint32_t e = ptx::elect_one();
        const uint32_t me = warp == 1 ? 0u : 1u;
        tc::Ring rg;
        uint32_t jt = 0, qphase = 0, nseq = 0, qready_seq = 0;
        uint32_t phases = 0;  // per slot: parity of this issuer's next use
        int prev_b = -1;
        bool ok = true;
        auto full = [&]() {
            ok &= ptx::mbar_spin(bar((me == 0 ? kBarFull : kBarFull1) + rg.slot), (phases >> rg.slot) & 1, kErrWaitFull);
            phases ^= 1u << rg.slot;
        };
        while (ok && items_next<kSched>(wl, cur, it, id)) {
            const int len = __shfl_sync(0xffffffffu, it.len, 0), v = __shfl_sync(0xffffffffu, it.b, 0);
            const bool new_seq = v != prev_b;
            prev_b = v;
            for (int t0 = 0; t0 < len; t0 += kTS, ++jt) {
                const bool mine = (jt & 1u) == me;
                const uint32_t sb = jt & 1, use = jt >> 1;
                if (mine) {
                    ok = ok && !*abort_flag && ptx::mbar_spin(bar(kBarSEmpty + sb), (use & 1) ^ 1, kErrWaitMma);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                }
                if (new_seq && t0 == 0) {
                    ++nseq;
                    if (mine) {
                        if (jt > 0) {
                            // an MMA is not ordered before a later tcgen05.cp: every GEMM1
                            // that reads the old Q completes first
                            ptx::mma_commit_if(e, bar(kBarQFree + me));
                            ok = ptx::mbar_spin(bar(kBarQFree + me), qphase, kErrWaitMma);
                            qphase ^= 1;
                            const uint32_t pj = jt - 1;  // the other issuer's last tile
                            ok = ok && ptx::mbar_spin(bar(kBarSFull + (pj & 1)), (pj >> 1) & 1, kErrWaitMma);
                            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                            ptx::tc_fence_after();
                        }
                        qready_seq = nseq;
                    } else {
                        for (int q = 0; q < kQSlots; ++q) rg.next(kSlotsS);
                    }
                }
                if (!mine) {
                    for (int sl = 0; sl < kSlotsPerTile; ++sl) rg.next(kSlotsS);
                    continue;
                }
                const bool copy_q = new_seq && t0 == 0;  // this issuer copies Q on the way
                if (qready_seq != nseq) {  // the other issuer copied this tile's Q
                    ok &= ptx::mbar_spin(bar(kBarQReady), (nseq - 1) & 1, kErrWaitMma);
                    qready_seq = nseq;
                }
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                ptx::tc_fence_after();  // the softmax's loads of this S buffer (and Q's copy) come first
                const uint32_t d = tmem + kTmemS + sb * kTS;
                for (int sl = 0; sl < kSlotsPerTile; ++sl) {
                    if (copy_q) {  // K-blocks 0-3, 4-5, 6-8 of Q (see the producer)
                        const int kb0 = sl == 0 ? 0 : sl == 1 ? 4 : 6, kb1 = sl == 0 ? 4 : sl == 1 ? 6 : kKBlocks;
                        for (int kb = kb0; kb < kb1; kb += 2) {
                            full();
                            const uint32_t slot = sbase + kOffRing + rg.slot * kSlotS;
                            const int nb = min(2, kKBlocks - kb);
                            for (int j = 0; j < nb; ++j) {
#pragma unroll
                                for (int c = 0; c < 4; ++c)
                                    ptx::tmem_cp_128x256b_if(e, tmem + kTmemQ + ((kb + j) * 4 + c) * 8,
                                                             ptx::sdesc_sw128(slot + j * kQBoxBytes + c * 32, 16, 1024));
                            }
                            ptx::mma_commit_if(ok ? e : 0u, bar(kBarEmpty + rg.slot));
                            rg.next(kSlotsS);
                        }
                        if (sl == kSlotsPerTile - 1) ptx::mma_commit_if(e, bar(kBarQReady));
                    }
                    full();
                    const uint32_t acc0 = sl > 0 ? 1u : 0u;
                    // the slot's K-blocks interleave per 8-row group: groups 3 KB apart
                    const uint64_t b0 = ptx::sdesc_sw128(sbase + kOffRing + rg.slot * kSlotS, 16, kKbPerSlot * 1024);
                    const uint32_t a0 = tmem + kTmemQ + sl * (kKbPerSlot * 32);
#pragma unroll
                    for (int k = 0; k < kKbPerSlot * 4; ++k)
                        ptx::mma_ts_if(e, d, a0 + k * 8, b0 + (uint64_t)(((k >> 2) * 1024 + (k & 3) * 32) >> 4),
                                       tc::idesc_s<kBf16>(), k > 0 ? 1u : acc0);
                    ptx::mma_commit_if(ok ? e : 0u, bar(kBarEmpty + rg.slot));
                    rg.next(kSlotsS);
                }
                ptx::mma_commit_if(e, bar(kBarSFull + sb));
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            }
        }
        if (!ok) *abort_flag = 1;
        ptx::mma_commit_if(e, bar(kBarDrain + me));
        ptx::mbar_wait(bar(kBarDrain + me), 0, kErrWaitMma);
    } else if (warp == 2 && role == 1) {
        // ------------------------------------------------------------ O-CTA: hidden rows
        uint32_t at = 0;        // ring slots of the items before this one
        uint32_t uses = 0;      // per slot: parity of its next hidden tile
        bool ok = true;
        while (ok && items_next<kSched>(wl, cur, it, id)) {
            const int start = draft_start(wl, p, it.b);
            const int pieces = (it.len + kTO - 1) / kTO;
            if (it.tok0 + it.len > start) {
                const unsigned long long seen = seen_of[it.b];
                for (int q = max(0, (start - it.tok0) / kTO - 1); ok && q < pieces; ++q) {
                    const int t = it.tok0 + q * kTO;
                    if (t + kTO <= start) continue;
                    const uint32_t keep = tree_word(seen, start, t);
                    if (keep == 0xffffffffu) continue;
                    const uint32_t slot = (at + q) % kSlotsO;
                    ok = !*abort_flag && ptx::mbar_wait(bar(kBarTail + slot), (uses >> slot) & 1, kErrWaitFull, kTailWaitNs);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    uses ^= 1u << slot;
                    const uint32_t tile = sbase + kOffRing + slot * kSlotO;
                    for (int i = lane; i < kTO * kVBlocks * 8; i += 32) {  // 16-byte pieces, 64 a row
                        const int row = i >> 6;
                        if (!((keep >> row) & 1u))
                            ptx::st_shared_v4(tile + ((i >> 3) & (kVBlocks - 1)) * kBoxO + row * 128 + (i & 7) * 16, 0u, 0u, 0u, 0u);
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(bar(kBarFull + slot));
                }
            }
            at += pieces;
        }
        if (!ok) *abort_flag = 1;
    } else if (warp == 2) {
        // ------------------------------------------------------------ S-CTA: message sender
        if (lane == 0) {
            const uint32_t peer_pfull0 = ptx::mapa(bar(kBarPFull), 1);
            const uint32_t peer_msg0 = ptx::mapa(sbase + kOffMsg, 1);
            uint32_t jt = 0;
            bool ok = true;
            while (ok && items_next<kSched>(wl, cur, it, id)) {
                for (int t0 = 0; t0 < it.len; t0 += kTS, ++jt) {
                    const uint32_t ms = jt % kMsgSlots, mu = jt / kMsgSlots;
                    // the O-CTA's slot is free once GEMM2 of S tile jt - 3 finished
                    ok = !*abort_flag && ptx::mbar_wait<true>(bar(kBarPFree + ms), (mu & 1) ^ 1, kErrWaitPeer) &&
                         ptx::mbar_wait(bar(kBarStaged), jt & 1, kErrWaitMma);
                    if (!ok) break;
                    const uint32_t rbar = peer_pfull0 + 8u * ms;
                    ptx::mbar_remote_arrive_expect_tx(rbar, kMsgBytes);
                    ptx::bulk_copy_s2cluster(peer_msg0 + ms * kMsgBytes, sbase + kOffStg, kMsgBytes, rbar);
                    ptx::bulk_commit_group();
                    ptx::bulk_wait_group_read<0>();
                    ptx::mbar_arrive(bar(kBarStgFree));
                }
            }
            if (!ok) *abort_flag = 1;
            // The last messages were consumed by the peer's GEMM2 (so no remote arrival is
            // still in flight towards this CTA).
            for (uint32_t k = (jt >= (uint32_t)kMsgSlots ? jt - kMsgSlots : 0); k < jt; ++k)
                ptx::mbar_wait<true>(bar(kBarPFree + (k % kMsgSlots)), (k / kMsgSlots) & 1, kErrWaitPeer);
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------ math warpgroups
        const int h = (tid - 128) & 127;            // row = TMEM lane
        const int half = (tid - 128) >> 7;
        const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint32_t jt = 0;
        bool ok = true;
        if (role == 0) {
            // ------------------------------------------------ S-CTA: softmax
            float *maxima = reinterpret_cast<float *>(smem + kOffMax);
            const float sl2 = p.scale_log2;
            while (ok && items_next<kSched>(wl, cur, it, id)) {
                float m_used = -INFINITY, l_run = 0.f;
                // the drafts this row sees, and where they start from this warpgroup's column 0
                const int b = it.b / p.tiles;
                const int d = min((it.b - b * p.tiles) * p.tile_drafts + h / p.heads, p.drafts - 1);
                unsigned long long mask = p.mask != nullptr ? p.mask[(long long)b * p.mask_stride + d] : (2ull << d) - 1;
                if (p.drafts < 64) mask &= (1ull << p.drafts) - 1;
                const int start = draft_start(wl, p, it.b) - it.tok0 - half * kHalf;
                for (int t0 = 0; t0 < it.len; t0 += kTS, ++jt) {
                    const uint32_t sb = jt & 1, use = jt >> 1;
                    const bool last = t0 + kTS >= it.len;
                    // Every decision is uniform over the warpgroups (bar.red below), so an
                    // expired wait never splits a warp at a .sync.aligned instruction.
                    bool w = !*abort_flag && ptx::mbar_wait(bar(kBarSFull + sb), use & 1, kErrWaitMma);
                    w = __all_sync(0xffffffffu, w);
                    uint32_t r[kHalf];
                    float own = -INFINITY;
                    if (w) {
                        ptx::tc_fence_after();
                        const uint32_t s_addr = trow + kTmemS + sb * kTS + half * kHalf;
                        ptx::tmem_ld_x32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(r));
                        tmem_ld_x16(s_addr + 32, *reinterpret_cast<uint32_t(*)[16]>(r + 32));
                        ptx::tmem_wait_ld();
                        ptx::tc_fence_before();
                        ptx::mbar_arrive(bar(kBarSEmpty + sb));
                        if (t0 + kHalf > start) {  // the columns reach into the drafts
                            const uint32_t w0 = tree_word(mask, start, t0), w1 = tree_word(mask, start, t0 + 32);
#pragma unroll
                            for (int k = 0; k < kHalf; ++k)
                                if (!(((k < 32 ? w0 : w1) >> (k & 31)) & 1u)) r[k] = tc::u32_of(-INFINITY);
                        }
                        float m4[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) m4[k] = tc::f32_of(r[k]);
#pragma unroll
                        for (int k = 4; k < kHalf; ++k) m4[k & 3] = fmaxf(m4[k & 3], tc::f32_of(r[k]));
                        own = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                        maxima[(sb * 2 + half) * 128 + h] = own;
                    }
                    if (!ptx::named_barrier_and(1, kMath, w)) { ok = false; break; }
                    const float mx = fmaxf(own, maxima[(sb * 2 + (half ^ 1)) * 128 + h]) * sl2;
                    float alpha = 1.f;
                    if (mx > m_used + tc::kRescaleLog2) {
                        alpha = m_used == -INFINITY ? 0.f : ptx::ex2(m_used - mx);
                        m_used = mx;
                    }
                    // (a row that has seen nothing keeps m_used = -inf: its weights are 0)
                    const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
                    float s4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t pk[kHalf / 2];
#pragma unroll
                    for (int k = 0; k < kHalf; k += 2) {
                        const float p0 = ptx::ex2(fmaf(tc::f32_of(r[k]), sl2, neg_m));
                        const float p1 = ptx::ex2(fmaf(tc::f32_of(r[k + 1]), sl2, neg_m));
                        s4[(k >> 1) & 3] += p0 + p1;
                        pk[k >> 1] = tc::pack2<kBf16>(p0, p1);
                    }
                    l_run = l_run * alpha + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
                    // the previous message has left the staging buffer (a wait that runs out
                    // is noticed at the next tile's barrier)
                    if (!ptx::mbar_wait(bar(kBarStgFree), (jt & 1) ^ 1, kErrWaitPeer)) *abort_flag = 1;
                    uint8_t *msg = smem + kOffStg;
#pragma unroll
                    for (int q = 0; q < kHalf / 8; ++q) {  // 16-byte pieces of 8 tokens
                        const int c = half * (kHalf / 8) + q, st = c >> 2, c4 = c & 3;
                        reinterpret_cast<uint4 *>(msg + st * kSubP + h * 64)[c4 ^ ((h >> 1) & 3)] =
                            make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
                    }
                    if (half == 0) reinterpret_cast<float *>(msg + kMsgAlpha)[h] = alpha;
                    if (last) {
                        reinterpret_cast<float *>(msg + kMsgL)[half * 128 + h] = l_run;
                        if (half == 0) reinterpret_cast<float *>(msg + kMsgM)[h] = m_used;
                    }
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive(bar(kBarStaged));
                }
            }
            if (!ok) *abort_flag = 1;
        } else {
            // ------------------------------------------------ O-CTA: correction + epilogue
            // (each warpgroup its half of O's columns)
            const uint32_t o_addr = trow + half * (kDV / 2);
            auto gemm2_done = [&](uint32_t x) -> bool {
                return ptx::mbar_wait(bar(kBarMmaDone + x % kMsgSlots), (x / kMsgSlots) & 1, kErrWaitMma);
            };
            while (ok && items_next<kSched>(wl, cur, it, id)) {
                for (int t0 = 0; t0 < it.len; t0 += kTS, ++jt) {
                    const uint32_t ms = jt % kMsgSlots, mu = jt / kMsgSlots;
                    bool w = !*abort_flag && ptx::mbar_wait<true>(bar(kBarPFull + ms), mu & 1, kErrWaitPeer);
                    const uint8_t *msg = smem + kOffMsg + ms * kMsgBytes;
                    const bool last = t0 + kTS >= it.len;
                    float alpha = 1.f, l_fin = 0.f, m_fin = 0.f;
                    if (w) {
                        alpha = reinterpret_cast<const float *>(msg + kMsgAlpha)[h];
                        if (last) {
                            l_fin = reinterpret_cast<const float *>(msg + kMsgL)[h] +
                                    reinterpret_cast<const float *>(msg + kMsgL)[128 + h];
                            m_fin = reinterpret_cast<const float *>(msg + kMsgM)[h];
                        }
                    } else {
                        *abort_flag = 1;
                    }
                    // one barrier: does any row need its O corrected, or did any wait fail?
                    if (ptx::named_barrier_or(2, kMath, !w || (t0 > 0 && alpha != 1.f))) {
                        w = !*abort_flag && gemm2_done(jt - 1);
                        if (!ptx::named_barrier_and(2, kMath, w)) { ok = false; break; }
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < kDV / 64; ++c) {
                            uint32_t r[32];
                            ptx::tmem_ld_x32(o_addr + c * 32, r);
                            ptx::tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) r[k] = tc::u32_of(tc::f32_of(r[k]) * alpha);
                            ptx::tmem_st_x32(o_addr + c * 32, r);
                        }
                        ptx::tmem_wait_st();
                    }
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(bar(kBarCorr + ms));
                    if (last) {
                        w = gemm2_done(jt);
                        if (!ptx::named_barrier_and(2, kMath, w)) { ok = false; break; }
                        ptx::tc_fence_after();
                        // A tile of one item gets its final output here, else its partial
                        // goes to the workspace.  32 bytes (a whole sector) a store.
                        int i0, i1, nrows;
                        item_range<kSched>(wl, it.b, i0, i1);
                        const bool single = i1 - i0 == 1;
                        long long row0;
                        tree_rows(p, it.b, row0, nrows);
                        const float inv_l = l_fin != 0.f ? 1.f / l_fin : 0.f;  // (NaN stays NaN)
                        const bool f32 = p.out_kind == tc::kOutF32;
                        const size_t slot = part_slot(wl, kSched == kSchedBalanced, it.b, id, id - i0);
                        const size_t row = single ? (size_t)row0 + h : slot * p.num_heads + h;
                        uint8_t *dst = static_cast<uint8_t *>(p.out) + (row * kDV + half * (kDV / 2)) * (f32 ? 4 : 2);
#pragma unroll 1
                        for (int c = 0; c < kDV / 64; ++c) {
                            uint32_t r[32];
                            ptx::tmem_ld_x32(o_addr + c * 32, r);
                            ptx::tmem_wait_ld();
                            if (!single) {
                                const int piece = half * (kDV / 32) + 2 * c;
                                const size_t at = part_piece(p, slot, piece, h), next = part_piece(p, slot, piece + 1, h);
                                uint32_t o[16];
#pragma unroll
                                for (int k = 0; k < 32; ++k) r[k] = tc::u32_of(tc::f32_of(r[k]) * inv_l);
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __byte_perm(r[2 * k], r[2 * k + 1], 0x7632);
                                if (h < nrows) {
                                    store32(p.part_hi + at * 32, o);
                                    store32(p.part_hi + next * 32, o + 8);
                                }
                                if (f32) {
#pragma unroll
                                    for (int k = 0; k < 16; ++k) o[k] = __byte_perm(r[2 * k], r[2 * k + 1], 0x5410);
                                    if (h < nrows) {
                                        store32(p.part_lo + at * 32, o);
                                        store32(p.part_lo + next * 32, o + 8);
                                    }
                                } else {  // cut, not rounded: a carry could turn a NaN into a number
#pragma unroll
                                    for (int k = 0; k < 8; ++k)
                                        o[k] = __byte_perm(__byte_perm(r[4 * k], r[4 * k + 1], 0x0051),
                                                           __byte_perm(r[4 * k + 2], r[4 * k + 3], 0x0051), 0x5410);
                                    if (h < nrows) {
                                        store16(p.part_lo + at * 16, o);
                                        store16(p.part_lo + next * 16, o + 4);
                                    }
                                }
                            } else if (f32) {
#pragma unroll
                                for (int k = 0; k < 32; ++k) r[k] = tc::u32_of(tc::f32_of(r[k]) * inv_l);
                                if (h < nrows) {
#pragma unroll
                                    for (int k = 0; k < 4; ++k) store32(dst + c * 128 + k * 32, r + 8 * k);
                                }
                            } else {
                                uint32_t o[16];
#pragma unroll
                                for (int k = 0; k < 16; ++k)
                                    o[k] = tc::pack2<kBf16>(tc::f32_of(r[2 * k]) * inv_l, tc::f32_of(r[2 * k + 1]) * inv_l);
                                if (h < nrows) {
                                    store32(dst + c * 64, o);
                                    store32(dst + c * 64 + 32, o + 8);
                                }
                            }
                        }
                        if (half == 0 && h < nrows) {
                            const float lse = l_fin != 0.f ? (m_fin + __log2f(l_fin)) * kLn2 : -INFINITY;
                            if (!single) p.part_lse[row] = lse;
                            else if (p.out_lse != nullptr) p.out_lse[row] = lse;
                        }
                        ptx::tc_fence_before();
                    }
                }
            }
            if (!ok) *abort_flag = 1;
        }
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    __syncwarp();
    ptx::cluster_sync();  // neither CTA leaves while its partner may still target it
    if (warp == 2) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

// O = sum_i e^(lse_i - M) O_i / sum_i e^(lse_i - M), M = max_i lse_i, over the items i
// of tile v that hold row r's partials.  A lane per row and a warp per piece of 16
// columns, as the partials lie: every load is whole kilobytes (the weights' 128 bytes)
// in a row.  (With a warp per row, its 32 pieces 4 KB apart, the loads took 5 of this
// kernel's 8 us.)  kRowWarps warps share a piece's splits, each every kRowWarps-th with its
// own maximum, joined in shared memory in a fixed order: 8 where a few tiles have many
// splits, else 1.  Rows of tiles that were one item are complete already.  Bound by the
// latency of two dependent loads, then by the partials' bytes, 1.5 KB a row and split (2
// for fp32 output).
// (Plain loads, not the read-only path: it may be resident while the decode writes.)
template <typename OutT, int kRowWarps>
__global__ void __launch_bounds__(32 * kMergeWarps) merge_kernel(const TreeParams p) {
    constexpr int kPieces = kMergeWarps / kRowWarps;  // of a block
    constexpr int kBlocks = kDV / 16 / kPieces;       // that share 32 rows
    __shared__ float acc_s[kRowWarps > 1 ? kRowWarps - 1 : 1][16][32];
    __shared__ float max_s[kMergeWarps][32], sum_s[kMergeWarps][32];
    griddep_launch();
    griddep_wait();
    const WorkList &wl = p.wl;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int v = blockIdx.y, group = blockIdx.x / kBlocks, g = warp % kRowWarps;
    const int piece = (blockIdx.x - group * kBlocks) * kPieces + warp / kRowWarps;
    long long row0;
    int rows;
    tree_rows(p, v, row0, rows);
    int i0, i1;
    if (p.plan_range != nullptr) {
        const int2 range = p.plan_range[v];
        i0 = range.x;
        i1 = range.y;
    } else {
        item_range(wl, v, i0, i1);
    }
    // (both the same for the whole block)
    if (i1 - i0 == 1) return;
    if (group * 32 >= rows) return;
    const int n = i1 - i0, r = group * 32 + lane, rr = min(r, rows - 1);
    auto slot = [&](int s) { return part_slot(wl, wl.chunk == 0, v, i0 + s, s); };
    auto lse = [&](int s) { return p.part_lse[slot(s) * p.num_heads + rr]; };
    constexpr bool kWhole = sizeof(OutT) == 4;  // 32 bits of a partial, else 24
    constexpr int kLo = kWhole ? 32 : 16;        // bytes of 16 columns' lower plane
    constexpr int kAhead = 4;
    uint32_t hi[kAhead][8], lo[kAhead][kLo / 4];
    auto fetch = [&](int s) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int sj = s + j * kRowWarps;
            if (sj < n) {
                const size_t at = part_piece(p, slot(sj), piece, rr);
                load32(p.part_hi + at * 32, hi[j]);
                if constexpr (kWhole) load32(p.part_lo + at * kLo, lo[j]);
                else load16(p.part_lo + at * kLo, lo[j]);
            }
        }
    };
    fetch(g);
    float mx = -INFINITY;  // NaN if any weight is
#pragma unroll 4
    for (int s = g; s < n; s += kRowWarps) mx = max_nan(mx, lse(s));
    float acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    float wsum = 0.f;
    for (int s = g; s < n; s += kRowWarps * kAhead) {
        if (s != g) fetch(s);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int sj = s + j * kRowWarps;
            // (exp(-inf) = 0; nothing is added where no split has seen anything)
            const float w = sj < n && mx != -INFINITY ? __expf(lse(sj) - mx) : 0.f;
            if (w != 0.f) {  // (a split that saw nothing holds zeros)
                wsum += w;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t up = hi[j][e / 2];
                    uint32_t x;
                    if constexpr (kWhole) x = __byte_perm(lo[j][e / 2], up, e & 1 ? 0x7632 : 0x5410);
                    else x = __byte_perm(lo[j][e / 4], up, (e & 1 ? 0x7600 : 0x5400) + (e & 3) * 16) & 0xffffff00u;
                    acc[e] = fmaf(w, tc::f32_of(x), acc[e]);
                }
            }
        }
    }
    if constexpr (kRowWarps > 1) {
        max_s[g][lane] = mx;
        sum_s[g][lane] = wsum;
        if (g > 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc_s[g - 1][e][lane] = acc[e];
        }
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int k = 1; k < kRowWarps; ++k) mx = max_nan(mx, max_s[k][lane]);
        wsum = 0.f;
#pragma unroll
        for (int k = 0; k < kRowWarps; ++k) {
            const float f = mx == -INFINITY ? 0.f : __expf(max_s[k][lane] - mx);
            wsum = fmaf(f, sum_s[k][lane], wsum);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = k == 0 ? acc[e] * f : fmaf(f, acc_s[k > 0 ? k - 1 : 0][e][lane], acc[e]);
        }
    }
    if (r >= rows) return;
    const float inv = wsum != 0.f ? 1.f / wsum : 0.f;
    OutT *dst = static_cast<OutT *>(p.out) + (row0 + r) * kDV + piece * 16;
    uint32_t o[16];
    if constexpr (sizeof(OutT) == 4) {
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = tc::u32_of(acc[e] * inv);
        store32(dst, o);
        store32(dst + 8, o + 8);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = pack_out2<OutT>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
        store32(dst, o);
    }
    if (p.out_lse != nullptr && piece == 0) p.out_lse[row0 + r] = wsum != 0.f ? mx + __logf(wsum) : -INFINITY;
}

}  // namespace tree
}  // namespace mla
