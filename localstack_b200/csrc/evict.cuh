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
constexpr int kBins = 2048;

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
    __device__ __forceinline__ int64_t position(int i) const { return i < held ? (int64_t) pos[i] : i + shift; }
    __device__ __forceinline__ uint32_t key(int i) const {
        const int64_t at = position(i);
        if (at < n_sink || at >= recent) return 0xffffffffu;
        const float a = acc[i];
        if (a != a) return 0u;
        const uint32_t u = __float_as_uint(a + 0.f);  // -0 + 0 = +0
        return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
    }
};

// The length of row b: 0 (and a report) if it is not in [0, max_len].
__device__ __forceinline__ int row_len(const int32_t *seq_lens, int b, int max_len, DeviceStatus *status) {
    const int len = seq_lens[b];
    if (len >= 0 && len <= max_len) return len;
    if (threadIdx.x == 0) report(status, kStatusBadIndex, kSiteEvictLen, b);
    return 0;
}

__device__ __forceinline__ int exclusive_scan(int v, int *warp_sums, int *total) {
    return pages::block_exclusive_scan(v, warp_sums, total);
}

// A row per cluster of C CTAs, each with a contiguous share of the row's keys. The budget-th largest
// key is found digit by digit (11, 11 and 10 bits): shared-memory histograms of the keys that match the
// digits found so far, summed over the cluster's CTAs through distributed shared memory, one array per
// digit so that no CTA clears what another still reads. Then the ranks of equal keys, of holes and of
// movers come from block scans plus the totals of the CTAs before. The weights and positions are read
// once; the time is that of a dozen block and cluster barriers.
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectParams p) {
    extern __shared__ uint32_t keys_s[];
    __shared__ int hist[3][kBins];
    __shared__ int warp_sums[32];
    __shared__ int digit_s, before_s;
    __shared__ int eq_total, hole_total, mover_total;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    const int b = blockIdx.x / C;
    const int tid = threadIdx.x;
    for (int i = tid; i < 3 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    const int len = row_len(p.seq_lens, b, p.w.row_cells, p.status);
    int32_t *src = p.src + (int64_t) b * p.max_moves, *dst = p.dst + (int64_t) b * p.max_moves;
    if (len <= p.budget) {  // the whole cluster: nothing to evict
        for (int j = rank * kThreads + tid; j < p.max_moves; j += C * kThreads) src[j] = dst[j] = -1;
        if (rank == 0 && tid == 0) p.n_moves[b] = 0;
        return;
    }
    Row row;
    row.acc = p.w.acc + (int64_t) b * p.w.row_cells;
    row.pos = p.w.pos + (int64_t) b * p.w.row_cells;
    row.len = len;
    row.held = min(max(p.w.held[b], 0), len);
    row.n_sink = p.n_sink;
    row.shift = p.w.shift[b];
    row.recent = len + row.shift - p.n_recent;
    const int share = (len + C - 1) / C;
    const int first = min(rank * share, len), n = min(share, len - first);
    auto key = [&](int i) { return i < p.cap ? keys_s[i] : row.key(first + i); };
    for (int i = tid; i < min(n, p.cap); i += kThreads) keys_s[i] = row.key(first + i);
    __syncthreads();

    uint32_t prefix = 0;
    int need = p.budget;  // keys still to be taken among those that match the prefix
#pragma unroll
    for (int d = 0; d < 3; d++) {
        constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
        const int shift = kShift[d], bins = 1 << kBits[d];
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t k = key(i);
            if (d == 0 || (k >> (shift + kBits[d])) == prefix) atomicAdd(&hist[d][(k >> shift) & (bins - 1)], 1);
        }
        cluster.sync();
        // thread t: bins of descending digit, 2 t and 2 t + 1 from the top
        int c[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int bin = bins - 1 - (2 * tid + e);
            if (bin >= 0)
                for (int r = 0; r < C; r++) c[e] += *cluster.map_shared_rank(&hist[d][bin], r);
        }
        int total;
        int above = exclusive_scan(c[0] + c[1], warp_sums, &total);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (above < need && need <= above + c[e]) {  // exactly one bin of the block
                digit_s = bins - 1 - (2 * tid + e);
                before_s = above;
            }
            above += c[e];
        }
        __syncthreads();
        prefix = (prefix << kBits[d]) | (uint32_t) digit_s;
        need -= before_s;
        __syncthreads();  // digit_s, before_s are written again
    }
    // Kept: key > prefix, and the first `need` keys equal to it. Thread t walks `per` consecutive keys.
    const int per = (n + kThreads - 1) / kThreads;
    const int lo = min(tid * per, n), hi = min(lo + per, n);
    int eq = 0;
    for (int i = lo; i < hi; i++) eq += key(i) == prefix;
    int total;
    int eq_rank = exclusive_scan(eq, warp_sums, &total);
    if (tid == 0) eq_total = total;
    cluster.sync();
    for (int r = 0; r < rank; r++) eq_rank += *cluster.map_shared_rank(&eq_total, r);
    int holes = 0, movers = 0, rk = eq_rank;
    for (int i = lo; i < hi; i++) {
        const uint32_t k = key(i);
        const bool kept = k > prefix || (k == prefix && rk++ < need);
        if (first + i < p.budget) holes += !kept;
        else movers += kept;
    }
    int hole_at = exclusive_scan(holes, warp_sums, &total);
    if (tid == 0) hole_total = total;
    int mover_at = exclusive_scan(movers, warp_sums, &total);
    if (tid == 0) mover_total = total;
    cluster.sync();
    int n_moves = 0;
    for (int r = 0; r < C; r++) {
        const int m = *cluster.map_shared_rank(&mover_total, r);
        if (r < rank) {
            mover_at += m;
            hole_at += *cluster.map_shared_rank(&hole_total, r);
        }
        n_moves += m;
    }
    cluster.sync();  // no CTA leaves while another reads its totals
    rk = eq_rank;
    for (int i = lo; i < hi; i++) {
        const uint32_t k = key(i);
        const bool kept = k > prefix || (k == prefix && rk++ < need);
        if (first + i < p.budget) {
            if (!kept) dst[hole_at++] = first + i;
        } else if (kept) {
            src[mover_at++] = first + i;
        }
    }
    for (int j = n_moves + rank * kThreads + tid; j < p.max_moves; j += C * kThreads) src[j] = dst[j] = -1;
    if (rank == 0 && tid == 0) p.n_moves[b] = n_moves;
}

// Planes whose rows (one cell each) a move copies: K and V, or the four planes of a q8_0 cache.
struct MoveParams {
    uint8_t *plane[4];
    int row_bytes[4];  // multiples of 8; planes 0 and 1 of 16
    int n_planes;
    const int32_t *block_tables;
    int n_rows, max_blocks;
    int64_t n_pages;
    const int32_t *n_moves;
    const int32_t *src, *dst;
    int max_moves;
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

// A warp per move.
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MoveParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t total = (int64_t) p.n_rows * p.max_moves;
    for (int64_t x = (int64_t) blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); x < total;
         x += (int64_t) gridDim.x * (kMoveThreads / 32)) {
        const int b = (int) (x / p.max_moves), j = (int) (x - (int64_t) b * p.max_moves);
        if (j >= p.n_moves[b]) continue;
        const int64_t from = move_cell(p, b, p.src[x]), to = move_cell(p, b, p.dst[x]);
        if (from < 0 || to < 0) continue;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k >= p.n_planes) break;
            const int bytes = p.row_bytes[k];
            const uint8_t *s = p.plane[k] + from * bytes;
            uint8_t *d = p.plane[k] + to * bytes;
            if (k < 2) {
                for (int o = lane * 16; o < bytes; o += 512)
                    *reinterpret_cast<uint4 *>(d + o) = *reinterpret_cast<const uint4 *>(s + o);
            } else {
                for (int o = lane * 8; o < bytes; o += 256)
                    *reinterpret_cast<uint2 *>(d + o) = *reinterpret_cast<const uint2 *>(s + o);
            }
        }
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
// pushes a row's blocks (its last block first) at the offset that the rows before it leave.
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
        at_s[tid] = exclusive_scan(freed, warp_sums, &total);
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
