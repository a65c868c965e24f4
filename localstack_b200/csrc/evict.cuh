// evict.cuh - eviction from the paged cache by accumulated attention weight.
//
// A row (sequence slot) with more than `budget` keys keeps the `budget` keys that rank first by
//   1. protected: the first n_sink tokens of the sequence and its last n_recent,
//   2. the larger accumulated weight acc (NaN below everything, -0 equal to +0),
//   3. the lower index.
// Attention does not depend on the order of the cached keys (RoPE is in K already), so the kept keys
// are not shifted together: kept keys at indexes >= budget ("movers") go to the indexes < budget that
// lost their key ("holes"), the j-th mover to the j-th hole in index order. That moves at most
// min(budget, len - budget) rows of K and V, each read and written once, and no row is both a source
// and a destination, so the moves are independent. The tokens' order is kept on the side: pos[i] is
// the position of the token at index i < held, and tokens appended since (i >= held) are at position
// i + shift, shift being the number of tokens the row has lost so far.
//
//   select_kernel   - the moves of every row (changes nothing else);
//   move_kernel     - carries them out on one layer's K and V planes;
//   finish_kernel   - the same on acc and pos, and clears acc behind the budget;
//   truncate_kernel - KvCache::truncate_seq(row, budget) for every row over its budget, in row order
//                     (src/kv_cache.cpp:85-132): blocks back on the free stack, length, high-water mark.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"
#include "kv_pages.cuh"

namespace lstk {
namespace evict {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kBins = 256;  // 8 bits of a key at a time

struct Weights {
    float *acc;      // [n_rows][row_cells]
    int32_t *pos;    // [n_rows][row_cells], the first held[b] entries
    int32_t *held;   // [n_rows]
    int32_t *shift;  // [n_rows]
    int n_rows, row_cells;
};

struct SelectParams {
    Weights w;
    const int32_t *seq_lens;
    int budget, n_sink, n_recent;
    int max_moves;
    int cap;  // keys of a CTA's share kept in shared memory; the others are formed again at each use
    int32_t *n_moves;
    int32_t *src, *dst;  // [n_rows][max_moves], -1 behind a row's moves
    DeviceStatus *status;
};

// One row's inputs. key(i): a 32-bit number that orders the row's keys by rules 1 and 2.
struct Row {
    const float *acc;
    const int32_t *pos;
    int len, held, n_sink;
    int64_t shift, recent;  // positions >= recent are protected
    __device__ __forceinline__ uint32_t key(int i) const {
        const float a = acc[i];  // both loads at once
        const int64_t at = i < held ? (int64_t) pos[i] : i + shift;
        const uint32_t u = __float_as_uint(a + 0.f);  // -0 + 0 = +0
        const uint32_t k = a != a ? 0u : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
        return at < n_sink || at >= recent ? 0xffffffffu : k;
    }
};

// The length of row b: 0 (and a report) if it is not in [0, max_len].
__device__ __forceinline__ int row_len(const int32_t *seq_lens, int b, int max_len, DeviceStatus *status) {
    const int len = seq_lens[b];
    if (len >= 0 && len <= max_len) return len;
    if (threadIdx.x == 0) report(status, kStatusBadIndex, kSiteEvictLen, b);
    return 0;
}

// Exclusive scan of v over a block of kWarps warps (a row of warp totals in shared memory); *total gets
// the sum.
template <int kWarps>
__device__ __forceinline__ int exclusive_scan(int v, int *warp_sums, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int w = lane < kWarps ? warp_sums[lane] : 0;  // every warp scans the totals for itself
#pragma unroll
    for (int off = 1; off < kWarps; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, off);
        if (lane >= off) w += y;
    }
    *total = __shfl_sync(0xffffffffu, w, kWarps - 1);
    const int before = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
    __syncthreads();  // warp_sums is reused by the next scan
    return before + x - v;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kShare = 8192;  // keys of a CTA before a row is split over more CTAs

// Counts of a stretch of keys against the threshold: above it and equal to it, below the budget's
// index (low) and past it (high).
struct __align__(16) Counts {
    int gt_low, eq_low, gt_high, eq_high;
    __device__ __forceinline__ void add(const Counts &o) {
        gt_low += o.gt_low, eq_low += o.eq_low, gt_high += o.gt_high, eq_high += o.eq_high;
    }
};

// A row per cluster of C CTAs (kMulti: C > 1), each with a contiguous share of the row's keys, and each
// warp with a contiguous stretch of its CTA's. The budget-th largest key is found 8 bits at a time:
// shared-memory histograms of the keys that match the bits found so far (one array per step, so that no
// CTA clears what another still reads), copied once from the cluster's other CTAs (1 KiB each, through
// distributed shared memory), summed and scanned by one warp. The ranks of equal keys, of holes and of
// movers come from ballots, the warps' counts, and one exchange of the CTAs' counts (an equal key's rank
// decides whether it stays, and equal keys in low indexes come before those in high ones, so the counts
// of kept keys follow from Counts alone).
// The weights and positions are read once; the rest is latency: the launch, two round trips to memory,
// and the barriers of four steps and one exchange. Measured with the moves, as a call of both: one row of
// 544 keys 11 us, 64 rows of 4 k 13 us, 16 rows of up to 32 k cut to 8 k 56 us (moves 36). Steps that paid
// there: 8 bits at a time instead of 11 (the cluster's 8 KiB histograms cost more to read than a fourth
// step), plain atomics instead of aggregating equal keys first, 1024 threads instead of 512 (18.0 -> 16.0
// and 66.7 -> 61.4 us), one warp scanning instead of all 32 (14.4 -> 12.9 and 60.5 -> 56.3 us).
// The loops are kept rolled: code that runs once per launch costs its instruction fetches.
template <bool kMulti>
__global__ void __launch_bounds__(kSelectThreads, 1) select_kernel(const SelectParams p) {
    extern __shared__ uint32_t keys_s[];
    __shared__ __align__(16) int hist[4][kBins];  // read as int4
    __shared__ __align__(16) int parts[kMulti ? kMaxCluster : 1][kBins];
    __shared__ Counts warp_counts[kSelectWarps], cta_counts;
    __shared__ uint32_t found_s[2];  // the bits found so far, and the keys still to be taken
    cg::cluster_group cluster = cg::this_cluster();
    const int C = kMulti ? (int) cluster.num_blocks() : 1, rank = kMulti ? (int) cluster.block_rank() : 0;
    const int b = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < 4 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    const int held = p.w.held[b], shift_b = p.w.shift[b];  // in flight with the length
    const int len = row_len(p.seq_lens, b, p.w.row_cells, p.status);
    int32_t *src = p.src + (int64_t) b * p.max_moves, *dst = p.dst + (int64_t) b * p.max_moves;
    if (len <= p.budget) {  // the whole cluster: nothing to evict
        for (int j = rank * kSelectThreads + tid; j < p.max_moves; j += C * kSelectThreads) src[j] = dst[j] = -1;
        if (rank == 0 && tid == 0) p.n_moves[b] = 0;
        return;
    }
    Row row;
    row.acc = p.w.acc + (int64_t) b * p.w.row_cells;
    row.pos = p.w.pos + (int64_t) b * p.w.row_cells;
    row.len = len;
    row.held = min(max(held, 0), len);
    row.n_sink = p.n_sink;
    row.shift = shift_b;
    row.recent = len + row.shift - p.n_recent;
    const int share = (len + C - 1) / C;
    const int first = min(rank * share, len), n = min(share, len - first);
    const int stretch = ((n + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32;
    const int lo = min(warp * stretch, n), hi = min(lo + stretch, n);  // this warp's keys
    // Each lane forms the keys it reads again below (those beyond cap again at each use).
#pragma unroll 4
    for (int i = lo + lane; i < min(hi, p.cap); i += 32) keys_s[i] = row.key(first + i);
    const bool cached = hi <= p.cap;
    auto key = [&](int i) { return cached || i < p.cap ? keys_s[i] : row.key(first + i); };

    uint32_t prefix = 0;
    int need = p.budget;  // keys still to be taken among those that match the prefix
    __syncthreads();      // the histograms are clear
#pragma unroll 1
    for (int d = 0; d < 4; d++) {
        const int shift = 24 - 8 * d;
        // One shared-memory atomic per key: runs of equal keys (protected tokens, weights of zero) conflict,
        // which costs less than aggregating them would for all the others.
        for (int i = lo + lane; i < hi; i += 32) {
            const uint32_t k = key(i);
            if (d == 0 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[d][(k >> shift) & (kBins - 1)], 1);
        }
        if constexpr (kMulti) {
            cluster.sync();
            // thread t: four bins of CTA t / 64
            const int r = tid >> 6, q = tid & 63;
            if (r < C) reinterpret_cast<int4 *>(parts[r])[q] = reinterpret_cast<const int4 *>(cluster.map_shared_rank(&hist[d][0], r))[q];
        }
        __syncthreads();
        if (warp == 0) {  // one warp: 32 that scan for themselves take 1300 cycles of issue slots, this 500
            // lane l: bins 255 - 8 l down to 248 - 8 l
            int c[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0;
#pragma unroll
            for (int r = 0; r < (kMulti ? kMaxCluster : 1); r++) {
                if (kMulti && r >= C) break;
                const int4 *h = reinterpret_cast<const int4 *>(kMulti ? parts[r] : hist[d]) + 2 * (31 - lane);
                const int4 u = h[0], v = h[1];
                c[0] += v.w, c[1] += v.z, c[2] += v.y, c[3] += v.x, c[4] += u.w, c[5] += u.z, c[6] += u.y, c[7] += u.x;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) sum += c[e];
            int above = sum;  // of the bins over this lane's
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, above, off);
                if (lane >= off) above += y;
            }
            above -= sum;
            const uint32_t has = __ballot_sync(0xffffffffu, above < need && need <= above + sum);  // exactly one lane
            int digit = 255 - 8 * lane;
#pragma unroll
            for (int e = 0; e < 7; e++) {
                if (need > above + c[e] && digit == 255 - 8 * lane - e) above += c[e], digit--;
            }
            const int from = __ffs((int) has) - 1;
            if (lane == from) {
                found_s[0] = (prefix << 8) | (uint32_t) digit;
                found_s[1] = (uint32_t) (need - above);
            }
        }
        __syncthreads();
        prefix = found_s[0];
        need = (int) found_s[1];
    }
    // Kept: key > prefix, and the first `need` keys equal to it.
    const int edge = p.budget - first;  // indexes below it are low
    Counts mine = {0, 0, 0, 0};
    for (int i = lo + lane; i < hi; i += 32) {
        const uint32_t k = key(i);
        const int gt = k > prefix, eq = k == prefix;
        if (i < edge) mine.gt_low += gt, mine.eq_low += eq;
        else mine.gt_high += gt, mine.eq_high += eq;
    }
    mine = {__reduce_add_sync(0xffffffffu, mine.gt_low), __reduce_add_sync(0xffffffffu, mine.eq_low),
            __reduce_add_sync(0xffffffffu, mine.gt_high), __reduce_add_sync(0xffffffffu, mine.eq_high)};
    if (lane == 0) warp_counts[warp] = mine;
    __syncthreads();
    // Every warp: lane w the counts of warp w, scanned; `before` of this warp, `all` of the CTA.
    Counts scan = lane < kSelectWarps ? warp_counts[lane] : Counts{0, 0, 0, 0};
#pragma unroll
    for (int off = 1; off < kSelectWarps; off <<= 1) {
        const Counts o = {__shfl_up_sync(0xffffffffu, scan.gt_low, off), __shfl_up_sync(0xffffffffu, scan.eq_low, off),
                          __shfl_up_sync(0xffffffffu, scan.gt_high, off), __shfl_up_sync(0xffffffffu, scan.eq_high, off)};
        if (lane >= off) scan.add(o);
    }
    auto of_lane = [&](int l) {
        return Counts{__shfl_sync(0xffffffffu, scan.gt_low, l), __shfl_sync(0xffffffffu, scan.eq_low, l),
                      __shfl_sync(0xffffffffu, scan.gt_high, l), __shfl_sync(0xffffffffu, scan.eq_high, l)};
    };
    const Counts all = of_lane(kSelectWarps - 1), upto = of_lane(warp);
    const Counts before = {upto.gt_low - mine.gt_low, upto.eq_low - mine.eq_low, upto.gt_high - mine.gt_high,
                           upto.eq_high - mine.eq_high};
    if (kMulti) {
        if (tid == 0) cta_counts = all;
        cluster.sync();
    }
    // eq keys, holes and movers of the CTAs before this one; all movers
    int eq_at = 0, hole_at = 0, mover_at = 0, n_moves = 0, eq_seen = 0;
    Counts other[kMulti ? kMaxCluster : 1];
    if constexpr (kMulti) {
#pragma unroll
        for (int r = 0; r < kMaxCluster; r++)
            if (r < C) other[r] = *cluster.map_shared_rank(&cta_counts, r);
        // Waited for at the end: no CTA leaves while another reads its counts. (The arrival orders the
        // loads above before it.)
        cluster.barrier_arrive();
    } else {
        other[0] = all;
    }
    auto kept_of = [&](int eq_before, int eq) { return max(0, min(eq, need - eq_before)); };
#pragma unroll
    for (int r = 0; r < (kMulti ? kMaxCluster : 1); r++) {
        if (r >= C) break;
        const int r_first = min(r * share, len), r_end = r_first + min(share, len - r_first);
        const int n_low = max(0, min(r_end, p.budget) - r_first);
        const int kept_low = other[r].gt_low + kept_of(eq_seen, other[r].eq_low);
        const int kept_high = other[r].gt_high + kept_of(eq_seen + other[r].eq_low, other[r].eq_high);
        if (r == rank) eq_at = eq_seen, mover_at = n_moves;
        if (r < rank) hole_at += n_low - kept_low;
        eq_seen += other[r].eq_low + other[r].eq_high;
        n_moves += kept_high;
    }
    // ... and of the warps before this one
    {
        const int n_low = max(0, min(lo, edge));
        hole_at += n_low - before.gt_low - kept_of(eq_at, before.eq_low);
        mover_at += before.gt_high + kept_of(eq_at + before.eq_low, before.eq_high);
        eq_at += before.eq_low + before.eq_high;
    }
    const uint32_t lower = (1u << lane) - 1u;
    const bool some_eq = mine.eq_low + mine.eq_high > 0;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t k = i < hi ? key(i) : 0u;
        bool kept = k > prefix;
        if (some_eq) {
            const uint32_t eq = __ballot_sync(0xffffffffu, i < hi && k == prefix);
            kept = kept || (k == prefix && eq_at + __popc(eq & lower) < need);
            eq_at += __popc(eq);
        }
        if (i0 < edge) {
            const bool hole = i < hi && i < edge && !kept;
            const uint32_t holes = __ballot_sync(0xffffffffu, hole);
            if (hole) dst[hole_at + __popc(holes & lower)] = first + i;
            hole_at += __popc(holes);
        }
        if (i0 + 32 > edge) {
            const bool mover = i < hi && i >= edge && kept;
            const uint32_t movers = __ballot_sync(0xffffffffu, mover);
            if (mover) src[mover_at + __popc(movers & lower)] = first + i;
            mover_at += __popc(movers);
        }
    }
    for (int j = n_moves + rank * kSelectThreads + tid; j < p.max_moves; j += C * kSelectThreads) src[j] = dst[j] = -1;
    if (rank == 0 && tid == 0) p.n_moves[b] = n_moves;
    if constexpr (kMulti) cluster.barrier_wait();
}

// Planes whose rows (one cell each) a move copies: K and V, or the four planes of a q8_0 cache.
struct MoveParams {
    uint8_t *k, *v, *kd, *vd;
    int row_bytes;    // of k and v, a multiple of 16
    int small_bytes;  // of the scale planes, a multiple of 8; 0 = none
    const int32_t *block_tables;
    int n_rows, max_blocks;
    int64_t n_pages;
    const int32_t *n_moves;
    const int32_t *src, *dst;
    int max_moves;
    int batch;  // moves of a warp, 1 .. 16
    DeviceStatus *status;
};

constexpr int kMoveThreads = 256;

// The cell of index i of a row, or -1 (reported) when the index or its page is out of range.
__device__ __forceinline__ int64_t move_cell(const MoveParams &p, int b, int i) {
    if (i < 0 || i >= p.max_blocks * pages::kBlock) {
        report(p.status, kStatusBadIndex, kSiteEvictMove, i);
        return -1;
    }
    const int32_t pid = p.block_tables[(int64_t) b * p.max_blocks + i / pages::kBlock];
    if (pid < 0 || pid >= p.n_pages) {
        report(p.status, kStatusBadIndex, kSiteEvictPage, pid);
        return -1;
    }
    return (int64_t) pid * pages::kBlock + i % pages::kBlock;
}

// Bound by DRAM with rows of 512 bytes in scattered order: 16 rows of up to 32 k q8_0 keys cut to 8 k move
// 170 MB (read and written) in 36 us, 4.7 TB/s. A move per warp, its lookups one after the other, took 51.
//
// A warp takes `batch` consecutive moves of a row: its lanes look up all their cells at once, then the
// moves are copied four at a time (16 bytes a lane, K and V together: 8 loads in flight), and the scale
// planes with several moves to a pass.
__device__ __forceinline__ void move_big(uint8_t *k, uint8_t *v, int bytes, int64_t cell, int count) {
    const int lane = threadIdx.x & 31;
    for (int m0 = 0; m0 < count; m0 += 4) {
        int64_t from[4], to[4];
        bool go[4];
#pragma unroll
        for (int m = 0; m < 4; m++) {
            from[m] = __shfl_sync(0xffffffffu, cell, (m0 + m) & 15) * bytes;
            to[m] = __shfl_sync(0xffffffffu, cell, 16 + ((m0 + m) & 15)) * bytes;
            go[m] = m0 + m < count && from[m] >= 0 && to[m] >= 0;
        }
        for (int o = lane * 16; o < bytes; o += 512) {
            uint4 a[4], b[4];
#pragma unroll
            for (int m = 0; m < 4; m++)
                if (go[m]) {
                    a[m] = *reinterpret_cast<const uint4 *>(k + from[m] + o);
                    b[m] = *reinterpret_cast<const uint4 *>(v + from[m] + o);
                }
#pragma unroll
            for (int m = 0; m < 4; m++)
                if (go[m]) {
                    *reinterpret_cast<uint4 *>(k + to[m] + o) = a[m];
                    *reinterpret_cast<uint4 *>(v + to[m] + o) = b[m];
                }
        }
    }
}
__device__ __forceinline__ void move_small(uint8_t *k, uint8_t *v, int bytes, int64_t cell, int count) {
    const int lane = threadIdx.x & 31, units = bytes / 8;  // 8-byte units of a row
    for (int u0 = 0; u0 < count * units; u0 += 32) {
        const int u = u0 + lane, m = min(u / units, 15);
        const int64_t from = __shfl_sync(0xffffffffu, cell, m), to = __shfl_sync(0xffffffffu, cell, 16 + m);
        if (u < count * units && from >= 0 && to >= 0) {
            const int o = (u - m * units) * 8;
            const uint2 a = *reinterpret_cast<const uint2 *>(k + from * bytes + o);
            const uint2 b = *reinterpret_cast<const uint2 *>(v + from * bytes + o);
            *reinterpret_cast<uint2 *>(k + to * bytes + o) = a;
            *reinterpret_cast<uint2 *>(v + to * bytes + o) = b;
        }
    }
}

__global__ void __launch_bounds__(kMoveThreads, 3) move_kernel(const MoveParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t per_row = (p.max_moves + p.batch - 1) / p.batch, total = per_row * p.n_rows;
    for (int64_t x = (int64_t) blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); x < total;
         x += (int64_t) gridDim.x * (kMoveThreads / 32)) {
        const int b = (int) (x / per_row), j0 = (int) (x - (int64_t) b * per_row) * p.batch;
        const int count = min(min(p.n_moves[b], p.max_moves) - j0, p.batch);
        if (count <= 0) continue;
        // lane m: the source cell of move j0 + m; lane 16 + m: its destination; -1 where out of range
        const int m = lane & 15;
        int64_t cell = -1;
        if (m < count) cell = move_cell(p, b, (lane < 16 ? p.src : p.dst)[(int64_t) b * p.max_moves + j0 + m]);
        move_big(p.k, p.v, p.row_bytes, cell, count);
        if (p.small_bytes) move_small(p.kd, p.vd, p.small_bytes, cell, count);
    }
}

struct FinishParams {
    Weights w;
    const int32_t *seq_lens;
    int max_len;  // cells of a block table's row
    int budget;
    const int32_t *n_moves;
    const int32_t *src, *dst;
    int max_moves;
    DeviceStatus *status;
};

// A row per CTA: records the positions of the tokens that stay below the budget, moves acc and pos,
// clears acc behind the budget, and sets held and shift.
__global__ void __launch_bounds__(kThreads) finish_kernel(const FinishParams p) {
    pdl_wait();
    const int b = blockIdx.x, tid = threadIdx.x;
    const int len = row_len(p.seq_lens, b, p.max_len, p.status);
    if (len <= p.budget) return;
    float *acc = p.w.acc + (int64_t) b * p.w.row_cells;
    int32_t *pos = p.w.pos + (int64_t) b * p.w.row_cells;
    const int held = min(max(p.w.held[b], 0), len), shift = p.w.shift[b];
    const int n = min(p.n_moves[b], p.max_moves);
    for (int i = held + tid; i < p.budget; i += kThreads) pos[i] = i + shift;
    __syncthreads();  // holes among them are written below; held and shift have been read
    for (int j = tid; j < n; j += kThreads) {
        const int s = p.src[(int64_t) b * p.max_moves + j], d = p.dst[(int64_t) b * p.max_moves + j];
        if (s < p.budget || s >= len || d < 0 || d >= p.budget) {  // not a move of this row as it is now
            report(p.status, kStatusBadIndex, kSiteEvictMove, s < p.budget || s >= len ? s : d);
            continue;
        }
        acc[d] = acc[s];
        pos[d] = s < held ? pos[s] : s + shift;
    }
    __syncthreads();
    for (int i = p.budget + tid; i < len; i += kThreads) acc[i] = 0.f;
    if (tid == 0) {
        p.w.held[b] = p.budget;
        p.w.shift[b] = shift + (len - p.budget);
    }
}

// KvCache::truncate_seq(row, budget) for the rows over their budget, in row order. One CTA; a warp
// pushes a row's blocks (its last block first) at the offset that the rows before it leave. Latency: of
// lengths, scan, tables and the walk over every slot's blocks for the high-water mark. Together with
// finish_kernel: 1 row 10 us, 64 rows of 4160 cut to 4096 keys 12 us, 16 rows of 32 k cut to 8 k 32 us, 1024 rows
// of 300 cut to 256 49 us.
__global__ void __launch_bounds__(kThreads) truncate_kernel(pages::State st, int budget) {
    __shared__ int warp_sums[32];
    __shared__ int at_s[kThreads];
    __shared__ int hwm_s;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int keep_blocks = pages::n_blocks_for(budget);
    const int cells = st.max_blocks * pages::kBlock;
    int top = *st.free_top;
    if (tid == 0) hwm_s = 0;
    for (int r0 = 0; r0 < st.n_slots; r0 += kThreads) {
        const int rows = min(kThreads, st.n_slots - r0);
        const int len = tid < rows ? st.seq_lens[r0 + tid] : 0;
        const int freed = len > budget && len <= cells ? pages::n_blocks_for(len) - keep_blocks : 0;
        int total;
        at_s[tid] = exclusive_scan<kThreads / 32>(freed, warp_sums, &total);
        __syncthreads();
        for (int r = warp; r < rows; r += kThreads / 32) {
            const int l = st.seq_lens[r0 + r];
            if (l <= budget || l > cells) continue;
            const int32_t *bt = st.block_tables + (int64_t) (r0 + r) * st.max_blocks;
            const int last = pages::n_blocks_for(l) - 1;
            for (int k = lane; k <= last - keep_blocks; k += 32)
                st.free_blocks[top + at_s[r] + k] = (uint32_t) bt[last - k];
        }
        __syncthreads();  // every warp has read the lengths
        if (tid < rows && len > budget && len <= cells) st.seq_lens[r0 + tid] = budget;
        top += total;
        __syncthreads();
    }
    if (tid == 0) *st.free_top = top;
    // high-water mark: one past the highest occupied cell over every slot
    int hwm = 0;
    for (int s = warp; s < st.n_slots; s += kThreads / 32) {
        const int len = min(st.seq_lens[s], cells);
        const int32_t *bt = st.block_tables + (int64_t) s * st.max_blocks;
        for (int k = lane; k * pages::kBlock < len; k += 32)
            hwm = max(hwm, bt[k] * pages::kBlock + min(pages::kBlock, len - k * pages::kBlock));
    }
    atomicMax(&hwm_s, hwm);
    __syncthreads();
    if (tid == 0) *st.used_hwm = hwm_s;
}

}  // namespace evict
}  // namespace lstk
