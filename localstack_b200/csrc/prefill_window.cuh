// prefill_window.cuh - paged flash-attention over a sliding window with sinks for prompt chunks, on
// the tcgen05 tensor cores.
//
// Query p sees keys i <= p, i < kv_len, with i > p - window or i < n_sink. The operand layouts are
// those of prefill.cuh (128 query rows = 128 / G tokens x the G query heads of one KV head; tiles of
// 128 keys = 4 pages; UMMA descriptors, softmax arithmetic); what differs is the schedule.
//
// Work item: (sequence, pair of adjacent query tiles, KV head). Its keys are the sinks' pages
// followed by the pages from the first query's window to the last query's position; key tiles are
// taken over that list of pages, so pages between the two are neither loaded nor multiplied, and each
// warp masks its two pages of a key tile by a bit mask per row.
//
// Two query tiles per CTA, because one leaves the tensor core waiting: a tile's chain S = Q K^T ->
// softmax -> O += P V -> next S is serial (P lies over S in tensor memory), about half of it softmax.
// With two chains one tile's products run under the other's softmax, and K and V are loaded once for
// both. A window bounds every item to about the same work, so pairs balance well over the SMs (for a
// whole causal prompt, where they do not, prefill.cuh keeps one tile with two S buffers).
//
// What bounds it. Per key tile and pair, three units need about 2048 cycles each: the tensor core
// (4 x 8 MMAs of 64 cycles), the MUFU (2 x 128 x 128 exponentials at 16 a cycle) and shared memory
// (256 KiB: the K and V tiles in, Q and K read for S, V for PV). Measured are about 3.7 k cycles: the
// chain of one tile (S 512-900 as the issuing thread competes with the softmax warps for issue slots,
// its latency to the softmax 300, max 440, exponentials 1360, P to the last MMA 200, PV's completion
// 600) is longer than two turns of the exponentials. 8192 tokens, window 4096, 32 / 4 heads: 490 us =
// 0.52 of the measured bf16 peak, against 528 us with one tile per CTA (prefill.cuh's schedule with the
// same masks). Steps that paid, in that measure: turns at the exponentials (623 -> 539 us), P in
// quarters (-> 526), a warp-uniform issuer (-> 497), f32 exponentials with packed sums (-> 482), sorted
// sequences (8 chunks behind contexts of up to 16 k: 337 -> 301). Steps that did not: a quarter of the
// exponentials by a cubic on the FMA pipe (6 % slower: it takes issue slots from the MMA issuers),
// handing the turn on after half of the exponentials (6 %), taking the turn before the row maxima (3 %),
// keeping the last 32 scores in registers between maximum and exponentials (5 %).
//
// Persistent: one CTA per SM, 20 warps:
//   warps 0-15  softmax: tile w / 8, key half (w / 4) % 2 (64 score columns), TMEM quadrant w % 4 (32
//               rows). The halves of a tile share one O, so they agree on the running max: a barrier
//               reduction per key tile says whether any row's max exceeds it by more than 2^8, and
//               only then do they exchange maxima and rescale O (each half its 64 columns). Each half
//               keeps its part of the row sum until the end. The tiles take turns at the exponentials.
//   warp 16     TMA: Q of both tiles per item, then K_0 V_0 K_1 V_1 ... through a ring of five 32 KiB
//               stages, running ahead into the next item.
//   warps 17,18 MMA issuers, one per tile: S_j once K_j has landed and PV_{j-1} (which read P from S's
//               columns) has completed; PV_j by quarters of P_j as they are written. Their two chains
//               interleave on the tensor core. (Queueing S_j behind PV_{j-1} without the wait, on the
//               tensor core's order of execution alone, would be 3 % faster; the ISA promises that order
//               only for products with one accumulator.)
//   warp 19     clears the V rows that no query of the item sees, in shared memory, before they are
//               multiplied (a cell outside the sequence or the window may hold anything: 0 * inf is
//               not 0), and passes the stage on.
// Few items (a handful of queries behind long contexts): the items' key tiles are split over the idle SMs
// and joined by log-sum-exp (prefill_join_kernel).
// TMEM: S_0 [0,128), S_1 [128,256), O_0 [256,384), O_1 [384,512); P_t in S_t's columns [0,32) and
// [64,96). Every wait is on a parity at most one phase from the arrivals, and bounded; a warp whose
// wait ran out keeps taking part in its tile's named barriers until the item ends.
// A non-finite K or V value that some query of an item sees may reach the item's other rows.
#pragma once

#include "prefill.cuh"

namespace lstk {
namespace prefill_window {

using prefill::kBM;
using prefill::kBN;
using prefill::kD;
using prefill::kPage;
using prefill::kSub;
using prefill::kTile;

struct Params : prefill::Params {  // n_qt counts pairs of query tiles
    int window, n_sink;
    // Few items: every item's key tiles are cut into n_split runs, each an item of its own whose rows' results
    // (normalised, f32) and log-sum-exps (log2 units) go to part_o / part_lse, row (split, token, head).
    int n_split;
    int max_q_len;
    float *part_o, *part_lse;
};
constexpr int kMaxSplit = 32;

constexpr int kStages = 5;
constexpr int kSoftmaxWarps = 16;
constexpr int kTileThreads = 256;  // softmax threads of one query tile
constexpr int kWarpTma = 16, kWarpMma0 = 17, kWarpClear = 19;
constexpr int kThreads = 640;
constexpr int kTmemCols = 512;

constexpr int kSorted = 128;  // sequences that the schedule sorts (more are taken in their order, in kSorted groups)

constexpr int kOffQ = 0;
constexpr int kOffKv = 2 * kTile;
constexpr int kOffBar = kOffKv + kStages * kTile;
constexpr int kSmemBytes = kOffBar + 3 * 1024;

struct Barriers {
    uint64_t q_full;            // Q of both tiles landed (one phase per item)
    uint64_t q_empty;           // both issuers' last S of the item has read Q
    uint64_t full[kStages];     // a K or V tile landed
    uint64_t ready[kStages];    // V tiles: hidden rows are cleared (every second use of a stage is a V tile)
    uint64_t empty[kStages];    // both issuers' products with the stage have completed
    uint64_t s_full[2];         // S_j of tile t (one phase per key tile)
    uint64_t p_full[2][4];      // quarters of P_j of tile t written (16 keys of each half), O rescaled: one arrival per warp
    uint64_t o_done[2];         // PV_j of tile t has completed
    uint64_t o_free[2];         // the softmax warps have read O out (one phase per item)
    uint64_t turn[2];           // the other tile is through its exponentials: one arrival per softmax warp
    uint64_t drain[2];
    uint32_t tmem_base;
    int abort;
    float row[2][2][kBM];       // per tile and key half: row maxima, and the row sums at the end
    int first_pair[kSorted + 1];  // schedule: pairs before each place of the order, or before each group of sequences
    uint8_t order[kSorted];       // sequences, the most key tiles per pair first
};
static_assert(sizeof(Barriers) <= 3 * 1024, "barrier block over its reserved bytes");
static_assert(kSmemBytes <= 232448, "shared memory over the 227 KiB limit");

// Bit i: key i of page pg is at a position below n.
__device__ __forceinline__ uint32_t below(int n, int pg) {
    const int r = n - pg * kPage;
    return r <= 0 ? 0u : r >= kPage ? 0xffffffffu : (1u << r) - 1u;
}
// First key of the window of the query at position pos, and one past its last key. Positions may pass 32
// bits (a first position of up to 2^31 - 1, keys only below it).
__device__ __forceinline__ int window_first(int64_t pos, int window) {
    return (int) min(max((int64_t) 0, pos + 1 - window), (int64_t) INT32_MAX);
}
__device__ __forceinline__ int keys_end(int64_t pos, int kv_len) { return (int) max(min(pos + 1, (int64_t) kv_len), (int64_t) 0); }
// Keys of page pg in [lo, hi) or below both n_sink and hi.
__device__ __forceinline__ uint32_t window_mask(int pg, int lo, int hi, int n_sink) {
    return below(hi, pg) & (~below(lo, pg) | below(n_sink, pg));
}

struct Item {
    int b, kvh, tok0, q_begin, n_q, kv_len, pos0, n_keys, n_tiles;
    bool bad_rows;     // the sequence's query rows are not inside [0, total_tokens): no rows, reported
    bool second;       // the pair's second tile has rows
    int split, tile0;  // this run of the item's key tiles: tile0 .. tile0 + n_tiles - 1
    int n_sink_pages, first_page, n_pages;  // pages: n_sink_pages from page 0, then those from first_page on
    int first;         // first key of the first query's window (at most n_keys)
    __device__ __forceinline__ int page(int v) const { return v < n_sink_pages ? v : v - n_sink_pages + first_page; }
};

// Pair `qt` of sequence b for KV head kvh.
__device__ __forceinline__ Item item_of(const Params &p, int b, int qt, int kvh) {
    Item it;
    const int tokens = 2 * (kBM / p.group);  // of a pair
    it.kvh = kvh;
    it.b = b;
    it.tok0 = qt * tokens;
    const int q0 = p.q_seq_start[b], q1 = p.q_seq_start[b + 1];
    it.pos0 = p.q_pos0[b];
    it.kv_len = max(0, min(p.kv_lens[b], p.max_blocks * kPage));
    it.q_begin = q0;
    it.bad_rows = q0 < 0 || q1 < q0 || q1 > p.total_tokens;
    it.n_q = it.bad_rows ? 0 : q1 - q0;
    it.second = it.tok0 + tokens / 2 < it.n_q;
    const int last = min(it.tok0 + tokens, it.n_q) - 1;
    it.n_keys = it.tok0 < it.n_q ? keys_end((int64_t) it.pos0 + last, it.kv_len) : 0;
    const int end_page = (it.n_keys + kPage - 1) / kPage;
    it.first = min(window_first((int64_t) it.pos0 + it.tok0, p.window), it.n_keys);
    it.first_page = it.first == it.n_keys ? end_page : it.first / kPage;
    it.n_sink_pages = min((min(p.n_sink, it.first) + kPage - 1) / kPage, it.first_page);
    it.n_pages = it.n_sink_pages + end_page - it.first_page;
    it.n_tiles = (it.n_pages * kPage + kBN - 1) / kBN;
    it.split = it.tile0 = 0;
    return it;
}

// Pairs of sequence b that have rows; one for bad rows, whose item reports them.
__device__ __forceinline__ int pairs_of(const Params &p, int b) {
    const int tokens = 2 * (kBM / p.group), q0 = p.q_seq_start[b], q1 = p.q_seq_start[b + 1];
    return q0 < 0 || q1 < q0 || q1 > p.total_tokens ? 1 : min((q1 - q0 + tokens - 1) / tokens, p.n_qt);
}

__device__ __forceinline__ int group_of(const Params &p) { return (p.n_seqs + kSorted - 1) / kSorted; }

// The schedule. Several sequences, up to kSorted, are ordered by the key tiles of their last pair, most first, and
// only the pairs that have rows are numbered: x counts the KV heads of a pair, the pairs of a sequence
// from the last, the sequences in that order. A CTA takes one item of each round of gridDim.x
// (index), so the long items are dealt out evenly and the short ones fill the last round.
// Eight chunks of 450 to 511 tokens behind contexts of up to 16 thousand keys (window 4096): a CTA's
// longest share is 4 x 33 key tiles dealt in the sequences' own order, 3 x 33 and a short item sorted. More
// sequences keep their order and are numbered in kSorted groups (a prompt of 2048 tokens and 199 single queries: 457 us with
// the pairs that have no rows numbered too, 114 without); those of a pair at most are taken as they come.
template <bool kSplit, bool kMany>
struct Schedule {
    const int *first_pair;  // shared memory; nullptr: every pair of every sequence
    const uint8_t *order;
    int n_items;
    __device__ __forceinline__ int index(int r) const {
        const int64_t g = gridDim.x;
        const int64_t idx = (int64_t) r * g + ((r & 1) ? g - 1 - (int64_t) blockIdx.x : (int64_t) blockIdx.x);
        return idx < n_items ? (int) idx : -1;
    }
    __device__ __forceinline__ Item item(const Params &p, int x) const {
        if constexpr (!kSplit) return whole(p, x);
        Item it = whole(p, x / p.n_split);
        it.split = x % p.n_split;
        it.tile0 = it.n_tiles * it.split / p.n_split;
        it.n_tiles = it.n_tiles * (it.split + 1) / p.n_split - it.tile0;
        return it;
    }
    __device__ __forceinline__ Item whole(const Params &p, int x) const {
        const int kvh = x % p.n_head_kv, y = x / p.n_head_kv;
        if (first_pair == nullptr) return item_of(p, y % p.n_seqs, p.n_qt - 1 - y / p.n_seqs, kvh);
        int lo = 0, hi = (kMany ? kSorted : p.n_seqs) - 1;  // the last place with first_pair <= y
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first_pair[mid] <= y) lo = mid; else hi = mid - 1;
        }
        if constexpr (kMany) {
            int rest = y - first_pair[lo], b = lo * group_of(p), pairs;
            while (rest >= (pairs = pairs_of(p, b))) rest -= pairs, b++;
            return item_of(p, b, pairs - 1 - rest, kvh);
        }
        return item_of(p, order[lo], first_pair[lo + 1] - 1 - y, kvh);
    }
};

// Fills the schedule's shared memory (every thread of the block; cost: scratch of kSorted ints).
template <bool kSplit, bool kMany>
__device__ __forceinline__ Schedule<kSplit, kMany> make_schedule(const Params &p, int *first_pair, uint8_t *order, int *cost, int *pairs) {
    if (p.n_seqs == 1 || (!kMany && p.n_seqs > kSorted)) return {nullptr, nullptr, p.n_items * (kSplit ? p.n_split : 1)};
    const int b = threadIdx.x;
    if constexpr (kMany) {
        const int per = group_of(p);
        if (b < kSorted) {
            int n = 0;
            for (int c = b * per; c < min((b + 1) * per, p.n_seqs); c++) n += pairs_of(p, c);
            pairs[b] = n;
        }
        __syncthreads();
        if (b < kSorted) {
            int before = 0;
            for (int c = 0; c < b; c++) before += pairs[c];
            first_pair[b] = before;
            if (b == kSorted - 1) first_pair[kSorted] = before + pairs[b];
        }
        __syncthreads();
        return {first_pair, nullptr, first_pair[kSorted] * p.n_head_kv * (kSplit ? p.n_split : 1)};
    }
    if (b < p.n_seqs) {
        pairs[b] = pairs_of(p, b);
        cost[b] = pairs[b] == 0 ? 0 : item_of(p, b, pairs[b] - 1, 0).n_tiles;  // 0 for bad rows
    }
    __syncthreads();
    if (b < p.n_seqs) {
        int rank = 0, before = 0;
        for (int c = 0; c < p.n_seqs; c++) {
            const bool ahead = cost[c] > cost[b] || (cost[c] == cost[b] && c < b);
            rank += ahead;
            before += ahead ? pairs[c] : 0;
        }
        order[rank] = (uint8_t) b;
        first_pair[rank] = before;
        if (rank == p.n_seqs - 1) first_pair[p.n_seqs] = before + pairs[b];
    }
    __syncthreads();
    return {first_pair, order, first_pair[p.n_seqs] * p.n_head_kv * (kSplit ? p.n_split : 1)};
}

// 32 score columns of this thread's row - page v of the item's list - with the keys that the row's query
// does not see at -inf.
__device__ __forceinline__ void load_scores(float (&sc)[32], uint32_t col, const Item &I, int v, int lo, int hi, int n_sink) {
    tmem_ld32(col, sc);
    tmem_wait_ld();
    const int pg = I.page(v), at = pg * kPage;
    if (at < lo || at + kPage > hi || v >= I.n_pages) {  // not wholly inside the window
        const uint32_t vis = v < I.n_pages ? window_mask(pg, lo, hi, n_sink) : 0u;
#pragma unroll
        for (int c = 0; c < 32; c++) sc[c] = (vis >> c) & 1u ? sc[c] : -INFINITY;
    }
}

// Softmax numerators of two adjacent scores: x = s * scale_log2 - mu (one packed FMA), 2^x in f32, both
// added to the packed row sums, and the pair rounded to f16 for the PV product. ex2.approx.f16x2 would not
// be faster (16 cycles of a sub-partition per warp, as two f32 ones) and rounds x to f16 first.
__device__ __forceinline__ uint32_t softmax_pair(float s0, float s1, uint64_t scale2, uint64_t neg_mu2, uint64_t &sum2) {
    uint32_t p;
    asm("{\n\t"
        ".reg .b64 x;\n\t"
        ".reg .f32 a, b;\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "fma.rn.f32x2 x, x, %4, %5;\n\t"
        "mov.b64 {a, b}, x;\n\t"
        "ex2.approx.ftz.f32 a, a;\n\t"
        "ex2.approx.ftz.f32 b, b;\n\t"
        "mov.b64 x, {a, b};\n\t"
        "add.rn.f32x2 %1, %1, x;\n\t"
        "cvt.rn.f16x2.f32 %0, b, a;\n\t"
        "}"
        : "=r"(p), "+l"(sum2)
        : "f"(s0), "f"(s1), "l"(scale2), "l"(neg_mu2));
    return p;
}
// Pairs 8 q .. 8 q + 7 of 32 scores.
template <int kQ>
__device__ __forceinline__ void eight_pairs(uint32_t *pk, const float (&sc)[32], uint64_t scale2, uint64_t neg_mu2,
                                            uint64_t (&sum2)[2]) {
#pragma unroll
    for (int c = 0; c < 8; c++)
        pk[c] = softmax_pair(sc[16 * kQ + 2 * c], sc[16 * kQ + 2 * c + 1], scale2, neg_mu2, sum2[c & 1]);
}

// True on one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// Max of the raw scores (the scale is positive): 4 independent max3 chains.
__device__ __forceinline__ float row_max(const float (&sc)[32]) {
    float mx[4];
#pragma unroll
    for (int i = 0; i < 4; i++) mx[i] = fmaxf(sc[i], sc[4 + i]);
#pragma unroll
    for (int c = 8; c < 32; c += 8)
#pragma unroll
        for (int i = 0; i < 4; i++) mx[i] = prefill::max3(mx[i], sc[c + i], sc[c + 4 + i]);
    return prefill::max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
}

extern __shared__ __align__(1024) uint8_t dyn_smem[];

// kOut16: out is bf16, each f32 result rounded once. kSplit: items are runs of key tiles (Params::n_split),
// whose results go to part_o and part_lse (kOut16 does not matter). kMany: more than kSorted sequences,
// some of several pairs (an instantiation of its own: its search costs the others 3 % in registers).
template <bool kOut16, bool kSplit, bool kMany>
__global__ void __launch_bounds__(kThreads, 1) prefill_window_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                     const __grid_constant__ CUtensorMap kmap,
                                                                     const __grid_constant__ CUtensorMap vmap,
                                                                     const Params p) {
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    uint8_t *base = dyn_smem;
    if ((smem_u32(base) & 1023u) != 0) {  // the 128-byte swizzle needs 1024-byte aligned tiles
        if (threadIdx.x == 0) report(p.status, kStatusBadIndex, kSitePrefillSmem, (int) (smem_u32(base) & 1023u));
        return;
    }
    Barriers *bars = reinterpret_cast<Barriers *>(base + kOffBar);
    const uint32_t sQ = smem_u32(base + kOffQ), sKv = smem_u32(base + kOffKv);
    volatile int *abort_flag = &bars->abort;

    if (threadIdx.x == 0) {
        bars->abort = 0;
        mbar_init(smem_u32(&bars->q_full), 1);
        mbar_init(smem_u32(&bars->q_empty), 2);
        for (int i = 0; i < kStages; i++) {
            mbar_init(smem_u32(&bars->full[i]), 1);
            mbar_init(smem_u32(&bars->ready[i]), 1);
            mbar_init(smem_u32(&bars->empty[i]), 2);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(smem_u32(&bars->s_full[t]), 1);
            for (int c = 0; c < 4; c++) mbar_init(smem_u32(&bars->p_full[t][c]), kSoftmaxWarps / 2);
            mbar_init(smem_u32(&bars->o_done[t]), 1);
            mbar_init(smem_u32(&bars->o_free[t]), kSoftmaxWarps / 2);
            mbar_init(smem_u32(&bars->turn[t]), kSoftmaxWarps / 2);
            mbar_init(smem_u32(&bars->drain[t]), 1);
        }
        fence_barrier_init();
    }
    if (warp == kWarpMma0) {
        tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    // The set-up above overlaps the previous kernel in the stream (programmatic dependent
    // launch); everything below reads what earlier work produced.
    pdl_wait();
    pdl_launch_dependents();
    const int G = p.group;
    const Schedule<kSplit, kMany> sched = make_schedule<kSplit, kMany>(
        p, bars->first_pair, bars->order, reinterpret_cast<int *>(bars->row[0][0]), reinterpret_cast<int *>(bars->row[0][1]));

    // Every role walks the same items. Barrier phases come from running counts: key tile g of this CTA
    // has K in ring use 2 g and V in use 2 g + 1 (stage use % 5, parity (use / 5) % 2) and is phase g of
    // s_full, p_full and o_done of a tile that takes part; items with tiles count the phases of q_full,
    // q_empty and o_free.
    if (warp == kWarpTma) {
        if (lane == 0) {
            prefetch_tensormap(&qmap);
            prefetch_tensormap(&kmap);
            prefetch_tensormap(&vmap);
        }
        int use = 0, n_items_t = 0;
        bool ok = true;
        if (p.start_flag != nullptr) {
            if (lane == 0 && !(ok = flag_wait_bounded(p.start_flag, abort_flag, p.wait_ns))) {
                report(p.status, kStatusTimeout, kSitePrefillWaitStart, warp);
                *abort_flag = 1;
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        for (int r = 0; ok; r++) {
            const int x = sched.index(r);
            if (x < 0) break;
            const Item I = sched.item(p, x);
            if (I.n_tiles == 0) continue;
            if (lane == 0) {
                if (n_items_t > 0)
                    ok = mbar_wait_bounded(smem_u32(&bars->q_empty), (uint32_t) (n_items_t - 1) & 1, abort_flag, p.wait_ns);
                if (ok) {
                    const int tiles = I.second ? 2 : 1;
                    mbar_arrive_expect_tx(smem_u32(&bars->q_full), (uint32_t) (tiles * kTile));
                    for (int t = 0; t < tiles; t++)
                        for (int h = 0; h < 2; h++)
                            tma_load_3d(sQ + t * kTile + h * kSub, &qmap, smem_u32(&bars->q_full), h * 64, I.kvh * G,
                                        I.q_begin + I.tok0 + t * (kBM / G));
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            n_items_t++;
            const int32_t *bt = p.block_tables + (int64_t) I.b * p.max_blocks;
            // The block table is read a warp at a time (lane i: page 32 c + i of the list), one chunk ahead.
            auto load_chunk = [&](int chunk) -> int {
                const int v = chunk * 32 + lane;
                int cell = (int) p.n_cells;  // out of bounds: TMA fills zeros
                if (v < I.n_pages) {
                    const int32_t pid = bt[I.page(v)];
                    if (pid >= 0 && pid < p.n_pages) cell = pid * kPage;
                    else report(p.status, kStatusBadIndex, kSitePrefillPage, pid);
                }
                return cell;
            };
            const int tile0 = kSplit ? I.tile0 : 0;
            int cur = load_chunk(tile0 / 8);
            int nxt = (tile0 / 8 + 1) * 32 < I.n_pages ? load_chunk(tile0 / 8 + 1) : (int) p.n_cells;
            for (int j = tile0; j < tile0 + I.n_tiles; j++) {
                if (j > tile0 && (j & 7) == 0) {  // next 32 pages: 8 tiles
                    cur = nxt;
                    nxt = (j / 8 + 1) * 32 < I.n_pages ? load_chunk(j / 8 + 1) : (int) p.n_cells;
                }
                int cell0[4];
#pragma unroll
                for (int q = 0; q < 4; q++) cell0[q] = __shfl_sync(0xffffffffu, cur, (j & 7) * 4 + q);
                for (int kv = 0; kv < 2; kv++) {
                    if (lane == 0) {
                        const int s = use % kStages;
                        const uint32_t n = (uint32_t) (use / kStages);
                        if (n > 0) ok = mbar_wait_bounded(smem_u32(&bars->empty[s]), (n - 1) & 1, abort_flag, p.wait_ns);
                        if (ok) {
                            const uint32_t fb = smem_u32(&bars->full[s]);
                            mbar_arrive_expect_tx(fb, kTile);
                            for (int q = 0; q < 4; q++)
                                for (int h = 0; h < 2; h++)
                                    tma_load_3d(sKv + s * kTile + h * kSub + q * (kPage * 128), kv ? &vmap : &kmap, fb, h * 64,
                                                I.kvh, cell0[q]);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) break;
                    use++;
                }
                if (!ok) break;
            }
        }
        if (lane == 0) {
            if (!ok) {
                report(p.status, kStatusTimeout, kSitePrefillWait, warp);
                *abort_flag = 1;
            }
            if (*abort_flag) {
                // Drain: every load still in flight lands before shared memory is released.
                if (n_items_t > 0)
                    mbar_wait_bounded(smem_u32(&bars->q_full), (uint32_t) (n_items_t - 1) & 1, nullptr);
                for (int u = max(0, use - kStages); u < use; u++)
                    mbar_wait_bounded(smem_u32(&bars->full[u % kStages]), (uint32_t) (u / kStages) & 1, nullptr);
            }
        }
    } else if (warp == kWarpMma0 || warp == kWarpMma0 + 1) {
        // The whole warp walks the tiles and one elected lane issues: control flow and descriptors stay
        // warp-uniform, so they sit in uniform registers, which the MMA instructions read; a branch on
        // lane 0 had every operand moved there for every MMA.
        {
            const int t = __shfl_sync(0xffffffffu, warp, 0) - kWarpMma0;
            const bool leader = elect_one();
            constexpr uint32_t idesc_qk = prefill::idesc_f16(false), idesc_pv = prefill::idesc_f16(true);
            // Descriptors as (low, high) words: the high word is fixed, the low one holds address >> 4.
            const uint64_t dq0 = sdesc_sw128(sQ + t * kTile, 16, 1024), dk0 = sdesc_sw128(sKv, 16, 1024);
            const uint64_t dv0 = sdesc_sw128(sKv, kSub, 1024);
            const uint32_t lq = (uint32_t) dq0, lk = (uint32_t) dk0, lv = (uint32_t) dv0;
            const uint64_t hq = dq0 & 0xFFFFFFFF00000000ull, hk = dk0 & 0xFFFFFFFF00000000ull;
            const uint64_t hv = dv0 & 0xFFFFFFFF00000000ull;
            const uint32_t ts = tmem + (uint32_t) t * 128, to = tmem + 256u + (uint32_t) t * 128;
            int g = 0;          // key tiles of the ring
            int mine = 0;       // key tiles of this tile: the phases of s_full, p_full, o_done
            int n_items_t = 0, n_items_mine = 0;
            bool ok = true, issued = false;
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                return __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(bar), parity & 1u, abort_flag, p.wait_ns)) != 0;
            };
            for (int r = 0; ok; r++) {
                const int x = sched.index(r);
                if (x < 0) break;
                const Item I = sched.item(p, x);
                const int n_tiles = __shfl_sync(0xffffffffu, I.n_tiles, 0);
                if (n_tiles == 0) continue;
                const bool part = t == 0 || __shfl_sync(0xffffffffu, (int) I.second, 0) != 0;
                ok = wait(&bars->q_full, (uint32_t) n_items_t);
                for (int j = 0; ok && j < n_tiles; j++, g++) {
                    const int uk = 2 * g, uv = 2 * g + 1;
                    const int sk = uk % kStages, sv = uv % kStages;
                    ok = wait(&bars->full[sk], (uint32_t) (uk / kStages));
                    if (!ok) break;
                    if (!part) {  // the pair has one tile here: pass the stages on
                        if (leader) mbar_arrive(smem_u32(&bars->empty[sk]));
                        if (!(ok = wait(&bars->ready[sv], (uint32_t) (uv / (2 * kStages))))) break;
                        if (leader) mbar_arrive(smem_u32(&bars->empty[sv]));
                        continue;
                    }
                    // S_j: PV_{j-1} has completed (it read P from these columns), and the softmax has read S_{j-1}
                    // (PV_{j-1} was issued after P_{j-1} was written).
                    if (mine > 0) ok = wait(&bars->o_done[t], (uint32_t) (mine - 1));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t lkb = lk + (uint32_t) sk * (kTile >> 4);
                    if (leader) {
                        mma_f16_ss_k<0>(ts, hq | lq, hk | lkb, idesc_qk);
#pragma unroll
                        for (int kk = 1; kk < 8; kk++) {
                            const uint32_t off = (uint32_t) (((kk >> 2) * kSub + (kk & 3) * 32) >> 4);
                            mma_f16_ss_k<1>(ts, hq | (lq + off), hk | (lkb + off), idesc_qk);
                        }
                        mma_commit(smem_u32(&bars->s_full[t]));
                        mma_commit(smem_u32(&bars->empty[sk]));
                        if (j == n_tiles - 1) mma_commit(smem_u32(&bars->q_empty));
                    }
                    __syncwarp();
                    issued = true;
                    // PV_j
                    ok = wait(&bars->ready[sv], (uint32_t) (uv / (2 * kStages)));
                    if (ok && j == 0 && n_items_mine > 0)  // the item's first PV overwrites O
                        ok = wait(&bars->o_free[t], (uint32_t) (n_items_mine - 1));
                    if (!ok) break;
                    const uint32_t lvb = lv + (uint32_t) sv * (kTile >> 4);
#pragma unroll
                    for (int i = 0; i < 4 && ok; i++) {  // a quarter: 16 keys of either half, in the order they are written
                        const int c = (i + 2) & 3;
                        ok = wait(&bars->p_full[t][c], (uint32_t) mine);
                        if (!ok) break;
                        tc_fence_after();
                        if (!leader) continue;
#pragma unroll
                        for (int h = 0; h < 2; h++) {  // 16 keys: 8 columns of P, 128 descriptor units of V
                            const uint32_t a = ts + (uint32_t) (h * 64 + c * 8);
                            const uint64_t v = hv | (lvb + (uint32_t) (4 * h + c) * 128u);
                            if (i == 0 && h == 0) mma_f16_ts(to, a, v, idesc_pv, j > 0 ? 1u : 0u);
                            else mma_f16_ts_k<1>(to, a, v, idesc_pv);
                        }
                    }
                    if (!ok) break;
                    if (leader) {
                        mma_commit(smem_u32(&bars->o_done[t]));
                        mma_commit(smem_u32(&bars->empty[sv]));
                    }
                    __syncwarp();
                    mine++;
                }
                if (!part && ok && leader) mbar_arrive(smem_u32(&bars->q_empty));
                n_items_t++;
                n_items_mine += part;
            }
            if (!ok && leader) {
                report(p.status, kStatusTimeout, kSitePrefillWait, warp);
                *abort_flag = 1;
            }
            // Every MMA this thread issued completes before TMEM can be released.
            if (issued && leader) {
                mma_commit(smem_u32(&bars->drain[t]));
                mbar_wait_bounded(smem_u32(&bars->drain[t]), 0, nullptr);
            }
        }
    } else if (warp == kWarpClear) {
        int g = 0;
        bool ok = true;
        for (int r = 0; ok; r++) {
            const int x = sched.index(r);
            if (x < 0) break;
            const Item I = sched.item(p, x);
            for (int j = 0; ok && j < I.n_tiles; j++, g++) {
                const int u = 2 * g + 1, s = u % kStages;
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&bars->full[s]), (uint32_t) (u / kStages) & 1,
                                                                abort_flag, p.wait_ns));
                if (!ok) break;
                bool cleared = false;
                for (int q = 0; q < 4; q++) {
                    const int v = 4 * ((kSplit ? I.tile0 : 0) + j) + q;  // pages past the list are zeros already
                    const uint32_t m = v < I.n_pages ? window_mask(I.page(v), I.first, I.n_keys, p.n_sink) : 0xffffffffu;
                    if (m == 0xffffffffu) continue;
                    cleared = true;
                    // lane: 16 bytes of every second row (from lane / 16), dim half (lane / 8) % 2
                    uint8_t *page = base + kOffKv + s * kTile + ((lane >> 3) & 1) * kSub + q * (kPage * 128) + (lane & 7) * 16;
                    for (int k = lane >> 4; k < kPage; k += 2)
                        if (!((m >> k) & 1u)) *reinterpret_cast<uint4 *>(page + k * 128) = make_uint4(0, 0, 0, 0);
                }
                if (cleared) fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars->ready[s]));
            }
        }
        if (!ok && lane == 0) {
            report(p.status, kStatusTimeout, kSitePrefillWait, warp);
            *abort_flag = 1;
        }
    } else {
        // ---- softmax ----
        const int t = warp >> 3, hf = (warp >> 2) & 1, quad = warp & 3;
        const int r = quad * 32 + lane;  // row within the tile
        const uint32_t lane_base = tmem + ((uint32_t) (quad * 32) << 16);
        const uint32_t scol = lane_base + (uint32_t) (t * 128 + 64 * hf);
        const uint32_t ocol = lane_base + 256u + (uint32_t) (t * 128 + 64 * hf);
        const uint64_t scale2 = prefill::pack_f32x2(p.scale_log2, p.scale_log2);
        const int bar = 1 + t;  // the tile's named barrier
        auto any_of_tile = [&](bool v) {
            int any;
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %1, 0;\n\t"
                         "barrier.red.or.pred p, %2, %3, p;\n\tselp.s32 %0, 1, 0, p;\n\t}"
                         : "=r"(any)
                         : "r"(v ? 1 : 0), "r"(bar), "r"(kTileThreads)
                         : "memory");
            return any != 0;
        };
        auto sync_tile = [&]() { asm volatile("barrier.sync %0, %1;" ::"r"(bar), "r"(kTileThreads) : "memory"); };
        int g = 0;       // key tiles of this query tile
        int n_turn = 0;  // key tiles that both query tiles took part in
        for (int it = 0;; it++) {
            const int x = sched.index(it);
            if (x < 0) break;
            const Item I = sched.item(p, x);
            if (I.bad_rows && threadIdx.x == 0) report(p.status, kStatusBadIndex, kSitePrefillRows, I.b);
            if (t == 1 && !I.second) continue;
            const int tq = I.tok0 + t * (kBM / G) + r / G;  // query token index within the sequence
            const int head = I.kvh * G + r % G;
            const int hi = keys_end((int64_t) I.pos0 + tq, I.kv_len);  // keys [lo, hi) and sinks below hi are visible
            const int lo = window_first((int64_t) I.pos0 + tq, p.window);
            const bool live = tq < I.n_q;
            bool ok = true;
            float m = -INFINITY, l = 0.f;  // the tile's running max (log2 units); this half's row sum
            for (int j = 0; j < I.n_tiles; j++, g++, n_turn += I.second) {
                // Warp-uniform outcomes: tcgen05.ld / st below are warp-collective.
                if (ok)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&bars->s_full[t]), (uint32_t) g & 1, abort_flag,
                                                                    p.wait_ns));
                // The scores are taken 32 at a time, once for the maximum and once for the exponentials, to stay
                // within the registers of 20 warps.
                float sc[32];
                float m_half = -INFINITY;
                const int v0 = 4 * ((kSplit ? I.tile0 : 0) + j) + 2 * hf;  // this warp's first page of the tile
                if (ok) {
                    tc_fence_after();
                    load_scores(sc, scol, I, v0, lo, hi, p.n_sink);
                    m_half = row_max(sc);
                    load_scores(sc, scol + 32, I, v0 + 1, lo, hi, p.n_sink);
                    m_half = fmaxf(m_half, row_max(sc)) * p.scale_log2;
                }
                if (any_of_tile(m_half > m + prefill::kRescaleThreshold)) {
                    bars->row[t][hf][r] = m_half;
                    sync_tile();
                    const float m_tile = fmaxf(m_half, bars->row[t][hf ^ 1][r]);
                    const bool up = m_tile > m + prefill::kRescaleThreshold;  // always for the first visible keys
                    const float alpha = up ? fast_exp2(m - m_tile) : 1.f;
                    if (up) m = m_tile;
                    l *= alpha;
                    if (ok && j > 0) {  // S_j is there, so PV_{j-1} has completed: O is stable
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            float o[32];
                            tmem_ld32(ocol + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] *= alpha;
                            tmem_st32(ocol + c * 32, o);
                        }
                    }
                }
                // The tiles take turns at the exponentials (tile 0 first), so that they stay half a period apart:
                // side by side both would wait for the MUFU, and then both for the tensor core.
                if (ok && I.second && n_turn + t > 0)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&bars->turn[t]), (uint32_t) (n_turn + t - 1) & 1,
                                                                    abort_flag, p.wait_ns));
                if (ok) {
                    const float mu = m == -INFINITY ? 0.f : m;
                    const uint64_t neg_mu2 = prefill::pack_f32x2(-mu, -mu);
                    uint64_t sum2[2] = {0, 0};  // packed f32 partial row sums
                    // P row r in quarters of 16 keys (8 packed columns, over the first 32 of this warp's own 64 score
                    // columns), each handed to the PV MMAs while the next one is computed.
                    uint32_t pk[16];
                    load_scores(sc, scol + 32, I, v0 + 1, lo, hi, p.n_sink);
                    eight_pairs<0>(pk, sc, scale2, neg_mu2, sum2);  // keys 32 .. 63 first: their columns are not P's
                    eight_pairs<1>(pk + 8, sc, scale2, neg_mu2, sum2);
                    load_scores(sc, scol, I, v0, lo, hi, p.n_sink);
                    tmem_st8(scol + 16, pk);
                    tmem_st8(scol + 24, pk + 8);
                    auto written = [&](int c) {
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&bars->p_full[t][c]));
                    };
                    eight_pairs<0>(pk, sc, scale2, neg_mu2, sum2);
                    written(2), written(3);
                    tmem_st8(scol, pk);
                    eight_pairs<1>(pk + 8, sc, scale2, neg_mu2, sum2);
                    written(0);
                    tmem_st8(scol + 8, pk + 8);
                    if (I.second) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&bars->turn[t ^ 1]));
                    }
                    written(1);
                    l += (__uint_as_float((uint32_t) sum2[0]) + __uint_as_float((uint32_t) (sum2[0] >> 32))) +
                         (__uint_as_float((uint32_t) sum2[1]) + __uint_as_float((uint32_t) (sum2[1] >> 32)));
                }
            }
            if (I.n_tiles > 0) {
                // Epilogue: the item's last PV has completed; the halves add their row sums, and each
                // writes its 64 output columns.
                if (ok)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&bars->o_done[t]), (uint32_t) (g - 1) & 1,
                                                                    abort_flag, p.wait_ns));
                bars->row[t][hf][r] = l;
                sync_tile();
                const float sum = l + bars->row[t][hf ^ 1][r];
                const bool none = sum == 0.f;  // the row saw no key; a sum of NaN makes the row NaN
                const float inv = 1.f / sum;
                const int64_t row = (int64_t) (I.q_begin + tq) * p.n_head + head;
                const int64_t part = kSplit ? (int64_t) I.split * p.total_tokens * p.n_head + row : row;
                if (kSplit && live && ok && hf == 0) p.part_lse[part] = none ? -INFINITY : sum != sum ? INFINITY : m + __log2f(sum);
                tc_fence_after();
                if (ok) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float o[32];
                        tmem_ld32(ocol + c * 32, o);
                        tmem_wait_ld();
                        if (live) {
                            // a row that saw no key is zero, whatever its O holds
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = none ? 0.f : o[i] * inv;
                            const int64_t at = part * kD + 64 * hf + 32 * c;
                            if constexpr (kOut16 && !kSplit) {
                                uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + at);
#pragma unroll
                                for (int ch = 0; ch < 4; ch++) {
                                    uint32_t w[4];
#pragma unroll
                                    for (int i = 0; i < 4; i++) {
                                        const __nv_bfloat162 h = __floats2bfloat162_rn(o[8 * ch + 2 * i], o[8 * ch + 2 * i + 1]);
                                        w[i] = *reinterpret_cast<const uint32_t *>(&h);
                                    }
                                    dst[ch] = make_uint4(w[0], w[1], w[2], w[3]);
                                }
                            } else {
                                float4 *dst = reinterpret_cast<float4 *>((kSplit ? p.part_o : p.out) + at);
#pragma unroll
                                for (int ch = 0; ch < 8; ch++)
                                    dst[ch] = make_float4(o[4 * ch], o[4 * ch + 1], o[4 * ch + 2], o[4 * ch + 3]);
                            }
                        }
                        __syncwarp();  // the tensor-memory loads are warp-collective
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars->o_free[t]));
            } else if (kSplit && live) {  // an empty run
                if (hf == 0)
                    p.part_lse[((int64_t) I.split * p.total_tokens + I.q_begin + tq) * p.n_head + head] = -INFINITY;
            } else if (live) {
                // no visible keys: the row's output is zero
                const int64_t at = ((int64_t) (I.q_begin + tq) * p.n_head + head) * kD + 64 * hf;
                uint4 *dst = kOut16 ? reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + at)
                                    : reinterpret_cast<uint4 *>(p.out + at);
#pragma unroll
                for (int i = 0; i < (kOut16 ? 8 : 16); i++) dst[i] = make_uint4(0, 0, 0, 0);
            }
            // The tile's warps stop at the same item if any of them failed.
            if (any_of_tile(!ok)) {
                if ((warp & 7) == 0 && lane == 0) {
                    report(p.status, kStatusTimeout, kSitePrefillWait, warp);
                    *abort_flag = 1;
                }
                break;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kWarpMma0) tmem_dealloc(tmem, kTmemCols);
}

// Joins the runs of split items: a warp per row (token of a sequence, head), lane s the log-sum-exp of
// run s, then each lane four dims of every run that saw a key.
template <bool kOut16>
__global__ void __launch_bounds__(256) prefill_join_kernel(const Params p) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t per_seq = (int64_t) p.max_q_len * p.n_head;
    const int64_t b = w / per_seq;
    if (b >= p.n_seqs) return;
    const int tq = (int) ((w - b * per_seq) / p.n_head), head = (int) (w % p.n_head);
    const int q0 = p.q_seq_start[b], q1 = p.q_seq_start[b + 1];
    if (q0 < 0 || q1 < q0 || q1 > p.total_tokens || tq >= q1 - q0) return;  // no row of a sequence
    const int64_t rows = (int64_t) p.total_tokens * p.n_head, row = (int64_t) (q0 + tq) * p.n_head + head;
    const float l = lane < p.n_split ? p.part_lse[lane * rows + row] : -INFINITY;
    const float M = warp_max_xor(l, 1);
    const float wt = M == -INFINITY ? 0.f : fast_exp2(l - M);  // 0 for an empty run, NaN for a run of NaN (+inf)
    const float den = warp_sum_xor(wt, 1);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.n_split; s++) {
        const float ws = __shfl_sync(0xffffffffu, wt, s);
        if (ws == 0.f) continue;  // its part_o was not written
        const float4 v = reinterpret_cast<const float4 *>(p.part_o + (s * rows + row) * kD)[lane];
        o.x += ws * v.x, o.y += ws * v.y, o.z += ws * v.z, o.w += ws * v.w;
    }
    const float inv = M == -INFINITY ? 0.f : 1.f / den;
    o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if constexpr (kOut16) {
        const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(o.x, o.y), __floats2bfloat162_rn(o.z, o.w)};
        reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + row * kD)[lane] =
            make_uint2(*reinterpret_cast<const uint32_t *>(&h[0]), *reinterpret_cast<const uint32_t *>(&h[1]));
    } else {
        reinterpret_cast<float4 *>(p.out + row * kD)[lane] = o;
    }
}

}  // namespace prefill_window
}  // namespace lstk
