// Embedding lookup with scaling and its gradient by sorted tokens.
//
//   forward    out[t, :] = scale * W[id[t], :]
//   backward   gW[v, :]  = scale * sum over t with id[t] == v, ascending t, of g[t, :]
//
// The gradient is a segmented sum over the tokens in sorted order, without atomics on values, so it is the same
// bits on every run:
//   1. with the lookup: a stable radix sort of (id, position) by one cluster of thread blocks, which also marks the ids
//      that occur, while the other blocks of the launch look up (a lookup is bound by memory, the sort by latency);
//   2. one warp per range of sorted tokens and slab of columns adds the gradient rows in fp32 registers and writes
//      every segment that begins in its range; among these blocks others write the zero rows of ids that do not
//      occur, so each row of gW is written once;
//   3. segments that go on far behind their range are joined from their fp32 partial sums, in range order.
//
// Measured, 65536 tokens of 1024 bf16 features (ids as in text: few frequent, many rare) into a table of 65536 rows:
//   1. 38 us: the sort takes 31 alone (latency of two passes of a cluster of eight blocks), the lookup beside it reads 35 MB
//      of rows and writes 134 MB from the other SMs, 4.5 TB/s;
//   2. 52 us for 134 MB of gradients read and 134 MB of table written: 5.2 TB/s, 0.8 of the copy rate.  The rows on
//      their way to shared memory instead of registers made 69 us 63, neighbouring warps on the slabs of a row 52;
//   3. 12 us: most blocks find nothing to join, the others wait for up to a few hundred partial rows.
// 5003 tokens of 515 fp32 features: 11 + 17 + 4.5 us.
// Above 65536 tokens the sort goes through the workspace, every pass reading its tokens twice, still on the eight SMs of one
// cluster: the first launch takes 32 us for 65536 tokens of 16 fp32 features, 64 for 65537, 180 for 2^18 and 690 for 2^20
// (the other two 16 + 15, 16 + 15, 30 + 21 and 78 + 27 us).
// For one step of generation (32 tokens) the lookup is a launch of 1.8 us.
#include <cooperative_groups.h>

#include "elements.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_KEYS = 8;  // per thread and tile
constexpr int SORT_TILE = SORT_KEYS * SORT_THREADS;
constexpr int SORT_DIGIT_BITS = 9;  // two passes sort tables of up to 2^18 - 1 rows
constexpr int SORT_BINS = 1 << SORT_DIGIT_BITS;
constexpr int MAX_CLUSTER = 8;  // the largest portable one

// id as stored, or -1 when it is outside [0, V)
template <typename I>
__device__ __forceinline__ int64_t checked_id(const I* ids, int64_t t, int64_t V) {
    const int64_t id = (int64_t)ids[t];
    return id >= 0 && id < V ? id : -1;
}

// ------------------------------------------------------------------------------------------ forward
template <typename T, typename I>
struct Lookup {
    const I* ids;
    const T* weight;
    T* out;
    int64_t tokens, V;
    int nvec;        // vectors per row
    int lanes_log2;  // 2^lanes_log2 threads per row, up to four accesses in flight each
    float scale;
};

// rows of block `block` of `blocks`, each of 2^threads_log2 threads
template <typename T, int W, typename I>
__device__ __forceinline__ void look_up(const Lookup<T, I>& p, int64_t block, int64_t blocks, int threads_log2) {
    const int lanes = 1 << p.lanes_log2, rows = 1 << (threads_log2 - p.lanes_log2);
    for (int64_t t = block * rows + (threadIdx.x >> p.lanes_log2); t < p.tokens; t += blocks * rows) {
        const int64_t id = checked_id(p.ids, t, p.V);
        const DlVec<T, W>* src = reinterpret_cast<const DlVec<T, W>*>(p.weight) + (id < 0 ? 0 : id) * p.nvec;
        DlVec<T, W>* dst = reinterpret_cast<DlVec<T, W>*>(p.out) + t * p.nvec;
        const float factor = id < 0 ? __int_as_float(0x7fffffff) : p.scale;  // NaN rows for ids that do not exist
        for (int v0 = threadIdx.x & (lanes - 1); v0 < p.nvec; v0 += 4 * lanes) {
            DlVec<T, W> r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (v0 + u * lanes < p.nvec) r[u] = src[v0 + u * lanes];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (v0 + u * lanes >= p.nvec) break;
                float f[W];
                dl_unpack(r[u], f);
#pragma unroll
                for (int e = 0; e < W; ++e) f[e] *= factor;
                dl_pack(f, r[u]);
                dst[v0 + u * lanes] = r[u];
            }
        }
    }
}

template <typename T, int W, typename I>
__global__ void __launch_bounds__(256) embedding_kernel(Lookup<T, I> p) {
    look_up<T, W, I>(p, blockIdx.x, gridDim.x, 8);
}

// ------------------------------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (key, position); ids that take no gradient get the key V and end up
// last.  Block r of the sorting cluster (the grid's first) owns the r-th run of tokens.  Per pass a warp ranks its
// tokens among its own by matching digits, a column scan over the warps ranks them in the block, and the blocks'
// digit counts are added up through distributed shared memory.  A run of one tile (all there is up to 65536 tokens)
// stays on the chip: between the passes the tokens go straight to the shared memory of the block that ranks them next.
// Longer runs are counted first and go through the workspace.
struct SortShared {
    uint2 tile[SORT_TILE];                       // the block's run as the last pass left it
    uint16_t warp_count[SORT_WARPS][SORT_BINS];  // first counts, then offsets inside the tile
    uint32_t totals[SORT_BINS];                  // of the block's run; read by the other blocks
    uint32_t base[SORT_BINS];                    // where the block's next token with this digit goes
    uint32_t start[SORT_BINS];                   // where its first one lies among the block's own, by digit
    uint32_t warp_sum[2][SORT_BINS / 32];
};

// The lanes that hold the same digit (NO_KEY included), by one vote per bit: the match instruction walks the distinct
// values, which took 7 us for a tile of random digits.
__device__ __forceinline__ uint32_t same_digit(uint32_t digit) {
    const bool valid = digit != NO_KEY;
    const uint32_t votes = __ballot_sync(0xffffffffu, valid);
    uint32_t same = valid ? votes : ~votes;
#pragma unroll
    for (int b = 0; b < SORT_DIGIT_BITS; ++b) {
        const bool set = (digit >> b) & 1;
        const uint32_t v = __ballot_sync(0xffffffffu, set);
        same &= set ? v : ~v;
    }
    return same;
}

template <typename T, int W, typename I>
__global__ void __launch_bounds__(SORT_THREADS)
embedding_sorting_kernel(Lookup<T, I> lookup, int64_t padding, uint2* a, uint2* b, uint8_t* present, int passes,
                         int digit_bits, int64_t per, int per_log2) {
    extern __shared__ __align__(16) unsigned char dynamic_shared[];
    SortShared& sh = *reinterpret_cast<SortShared*>(dynamic_shared);
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if ((int)blockIdx.x >= ranks) {
        look_up<T, W, I>(lookup, blockIdx.x - ranks, gridDim.x - ranks, 10);
        return;
    }
    const I* ids = lookup.ids;
    const int64_t tokens = lookup.tokens, V = lookup.V;
    uint32_t* present_words = reinterpret_cast<uint32_t*>(present);  // the workspace holds whole words
    for (int64_t i = (int64_t)rank * SORT_THREADS + tid; i < (V + 3) / 4; i += (int64_t)ranks * SORT_THREADS)
        present_words[i] = 0;  // before the first cluster barrier; set in the last pass
    const int64_t lo = rank * per < tokens ? rank * per : tokens;
    const int64_t hi = lo + per < tokens ? lo + per : tokens;
    const bool one_tile = per_log2 >= 0;  // then per is 2^per_log2
    const int keys = one_tile ? (int)((per + SORT_THREADS - 1) / SORT_THREADS) : SORT_KEYS;  // of a thread: all warps work
    const int bins = 1 << digit_bits;
    const uint32_t mask = (uint32_t)bins - 1;

    const uint2* src = nullptr;
    uint2* dst = a;
    uint2 entry[SORT_KEYS];
    uint32_t digit[SORT_KEYS], slot[SORT_KEYS];
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        auto load = [&](int64_t i) {
            if (pass > 0) return one_tile ? sh.tile[i - lo] : __ldcg(src + i);  // others wrote it: read past L1
            const int64_t id = checked_id(ids, i, V);
            return make_uint2(id < 0 || id == padding ? (uint32_t)V : (uint32_t)id, (uint32_t)i);
        };
        // reads a tile and ranks its tokens inside their warps; warp_count holds the warps' counts afterwards
        auto rank_tile = [&](int64_t t0) {
#pragma unroll
            for (int j = 0; j < SORT_KEYS; ++j) {
                const int64_t i = j < keys ? t0 + warp * (32 * keys) + j * 32 + lane : hi;
                entry[j] = i < hi ? load(i) : make_uint2(0, 0);
                digit[j] = i < hi ? (entry[j].x >> shift) & mask : NO_KEY;
            }
            uint32_t* words = reinterpret_cast<uint32_t*>(&sh.warp_count[warp][0]);
#pragma unroll
            for (int k = 0; k < SORT_BINS / 64; ++k) words[k * 32 + lane] = 0;
            // the votes of all keys first: they do not depend on one another, the counting behind them does
#pragma unroll
            for (int j = 0; j < SORT_KEYS; ++j)
                if (j < keys) slot[j] = same_digit(digit[j]);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < SORT_KEYS; ++j) {
                if (j >= keys) break;
                const uint32_t same = slot[j], below = same & ((1u << lane) - 1);
                uint32_t held = 0;
                if (digit[j] != NO_KEY) held = sh.warp_count[warp][digit[j]];
                __syncwarp();
                if (digit[j] != NO_KEY && below == 0) sh.warp_count[warp][digit[j]] = (uint16_t)(held + __popc(same));
                __syncwarp();
                slot[j] = held + __popc(below);
            }
            __syncthreads();
        };
        // counts -> offsets inside the tile; returns the tile's count of digit `tid`
        auto scan_columns = [&]() {
            uint32_t run = 0;
            if (tid < bins) {
#pragma unroll
                for (int w = 0; w < SORT_WARPS; ++w) {
                    const uint32_t c = sh.warp_count[w][tid];
                    sh.warp_count[w][tid] = (uint16_t)run;
                    run += c;
                }
            }
            return run;
        };
        auto scatter_tile = [&]() {
#pragma unroll
            for (int j = 0; j < SORT_KEYS; ++j)
                if (digit[j] != NO_KEY) {
                    const uint32_t at = sh.base[digit[j]] + sh.warp_count[warp][digit[j]] + slot[j];
                    if (one_tile)
                        cluster.map_shared_rank(sh.tile, at >> per_log2)[at & (uint32_t)(per - 1)] = entry[j];
                    else
                        dst[at] = entry[j];
                    if (pass == passes - 1 && entry[j].x < V) present[entry[j].x] = 1;
                }
        };
        // the last pass of a run of one tile: put in order on the chip first, so that neighbouring threads write
        // neighbouring entries, and only the first of equal ids marks it
        auto write_tile = [&]() {
#pragma unroll
            for (int j = 0; j < SORT_KEYS; ++j)
                if (digit[j] != NO_KEY)
                    sh.tile[sh.start[digit[j]] + sh.warp_count[warp][digit[j]] + slot[j]] = entry[j];
            __syncthreads();
            const int n = (int)(hi - lo);
            for (int i = tid; i < n; i += SORT_THREADS) {
                const uint2 e = sh.tile[i];
                const uint32_t d = (e.x >> shift) & mask;
                dst[sh.base[d] + i - sh.start[d]] = e;
                if (e.x < V && (i == 0 || sh.tile[i - 1].x != e.x)) present[e.x] = 1;
            }
        };

        if (one_tile) {
            rank_tile(lo);
            const uint32_t n = scan_columns();
            if (tid < bins) sh.totals[tid] = n;
        } else {
            if (tid < SORT_BINS) sh.totals[tid] = 0;
            __syncthreads();
            for (int64_t i0 = lo; i0 < hi; i0 += SORT_THREADS) {
                const int64_t i = i0 + tid;
                const uint32_t d = i < hi ? (load(i).x >> shift) & mask : NO_KEY;
                const uint32_t same = same_digit(d);
                if (d != NO_KEY && lane == __ffs(same) - 1) atomicAdd(&sh.totals[d], (uint32_t)__popc(same));
            }
        }
        cluster.sync();
        uint32_t all = 0, before = 0, inclusive = 0, own = 0, own_inclusive = 0;
        if (tid < SORT_BINS) {
            if (tid < bins) {
#pragma unroll
                for (int r = 0; r < MAX_CLUSTER; ++r) {  // all loads in flight at once
                    const uint32_t c = r < ranks ? *cluster.map_shared_rank(&sh.totals[tid], r) : 0;
                    all += c;
                    if (r < rank) before += c;
                }
                own = sh.totals[tid];
            }
            inclusive = all;
            own_inclusive = own;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, inclusive, s);
                const uint32_t oo = __shfl_up_sync(0xffffffffu, own_inclusive, s);
                if (lane >= s) {
                    inclusive += o;
                    own_inclusive += oo;
                }
            }
            if (lane == 31) {
                sh.warp_sum[0][warp] = inclusive;
                sh.warp_sum[1][warp] = own_inclusive;
            }
        }
        __syncthreads();
        if (tid < bins) {
            uint32_t lower = 0, own_lower = 0;
            for (int w = 0; w < warp; ++w) {
                lower += sh.warp_sum[0][w];
                own_lower += sh.warp_sum[1][w];
            }
            sh.base[tid] = lower + inclusive - all + before;
            sh.start[tid] = own_lower + own_inclusive - own;
        }
        __syncthreads();
        if (one_tile && pass == passes - 1) {
            write_tile();
        } else if (one_tile) {
            scatter_tile();
        } else {
            for (int64_t t0 = lo; t0 < hi; t0 += SORT_TILE) {
                rank_tile(t0);
                const uint32_t n = scan_columns();
                __syncthreads();
                scatter_tile();
                __syncthreads();
                if (tid < bins) sh.base[tid] += n;
                __syncthreads();
            }
        }
        cluster.sync();  // the pass is complete, and every block has read the other blocks' totals
        src = dst;
        dst = dst == a ? b : a;
    }
}

// ------------------------------------------------------------------------------------------ segmented sum
constexpr int SUM_WARPS = 4;
constexpr int ZERO_ROWS = 32 * SUM_WARPS;  // rows looked at per block: a flag per lane
constexpr int ROWS_IN_FLIGHT = 16;  // per warp, as copies to shared memory: 24 warps of an SM have up to 196 KB under way
// A segment that goes on behind its range for fewer tokens than this is finished by the warp that began it; the next
// range leaves them out.  Both sides read the same entry of the sorted list to decide.
constexpr int REACH = 32;
constexpr int JOIN_WARPS = 8;
// Ranges looked at per block; few have something to join.  (16 warps and 4 ranges: 11.6 instead of 12.4 us for 65536 tokens of
// 1024 bf16, but 9.1 instead of 4.5 for 5003 of 515 fp32.)
constexpr int JOIN_RANGES = 8;

// does the segment of `key` reach REACH tokens behind position `at`?
__device__ __forceinline__ bool reaches_far(const uint2* sorted, int64_t at, int64_t tokens, uint32_t key) {
    return at + REACH - 1 < tokens && sorted[at + REACH - 1].x == key;
}

// 4, 8 or 16 bytes from global to shared memory in the background (2 bytes at once: there is no such copy)
template <typename T, int W>
__device__ __forceinline__ void copy_async(DlVec<T, W>* dst, const DlVec<T, W>* src) {
    constexpr int BYTES = (int)sizeof(T) * W;
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                     : "memory");
    else if constexpr (BYTES >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                     "l"(src), "n"(BYTES)
                     : "memory");
    else
        *dst = *src;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <typename T, int W>
__device__ __forceinline__ void store_scaled(T* dst, const float (&acc)[W], float scale) {
    DlVec<T, W> r;
    float f[W];
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] = acc[e] * scale;
    dl_pack(f, r);
    *reinterpret_cast<DlVec<T, W>*>(dst) = r;
}

// head[r]: what range r adds to a far-reaching segment that began in an earlier range.
// tail[r]: what range r adds to a far-reaching segment that begins in it.
template <typename T, int W>
__global__ void __launch_bounds__(32 * SUM_WARPS)
embedding_sum_kernel(const uint2* __restrict__ sorted, const T* __restrict__ g, T* __restrict__ gw,
                     const uint8_t* __restrict__ present, float* __restrict__ head, float* __restrict__ tail,
                     int64_t tokens, int64_t V, int64_t D, int64_t range_len, int64_t ranges, int slabs,
                     int64_t zero_blocks, float scale) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the zero blocks are spread evenly among the others: reads and writes then overlap all along
    const int64_t zero_before = (int64_t)blockIdx.x * zero_blocks / gridDim.x;
    if (((int64_t)blockIdx.x + 1) * zero_blocks / gridDim.x > zero_before) {
        DlVec<T, W> zero;
#pragma unroll
        for (int e = 0; e < W; ++e) zero.v[e] = dl_from_float<T>(0.0f);
        const int64_t row0 = zero_before * ZERO_ROWS + warp * 32;
        uint32_t absent = __ballot_sync(0xffffffffu, row0 + lane < V && !present[row0 + lane]);
        for (; absent; absent &= absent - 1) {
            DlVec<T, W>* row = reinterpret_cast<DlVec<T, W>*>(gw + (row0 + __ffs(absent) - 1) * D);
            for (int64_t c = lane; c < D / W; c += 32) row[c] = zero;
        }
        return;
    }
    // the slabs of a range are neighbouring warps: they read the same rows at the same time
    const int64_t item = ((int64_t)blockIdx.x - zero_before) * SUM_WARPS + warp, range = item / slabs;
    const int slab = (int)(item - range * slabs);
    if (range >= ranges) return;
    const int64_t col = ((int64_t)slab * 32 + lane) * W;
    const bool live = col < D;
    const int64_t partial_at = range * ((int64_t)slabs * 32 * W) + col;
    int64_t start = range * range_len;
    int64_t stop = start + range_len < tokens ? start + range_len : tokens;
    uint32_t key = sorted[start].x;
    bool open = false;  // in a far-reaching segment that began in an earlier range
    if (start > 0 && sorted[start - 1].x == key) {
        open = reaches_far(sorted, start, tokens, key);
        if (!open) {
            // the earlier range finishes this segment: begin behind it
            const uint32_t k = start + lane < tokens ? sorted[start + lane].x : NO_KEY;
            start += __popc(__ballot_sync(0xffffffffu, k == key));
            if (start >= stop) return;
            key = sorted[start].x;
        }
    }
    if (key >= (uint64_t)V) return;  // only ids without gradient from here on
    bool goes_on = false;            // the last segment reaches far behind the range
    if (stop < tokens) {
        const uint32_t last = sorted[stop - 1].x;
        if (last < (uint64_t)V && sorted[stop].x == last) {
            goes_on = reaches_far(sorted, stop, tokens, last);
            if (!goes_on) {
                const uint32_t k = stop + lane < tokens ? sorted[stop + lane].x : NO_KEY;
                stop += __popc(__ballot_sync(0xffffffffu, k == last));
            }
        }
    }
    float acc[W];
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] = 0.0f;

    // a ring of gradient pieces; every lane copies and reads its own slots only
    __shared__ DlVec<T, W> ring[SUM_WARPS][ROWS_IN_FLIGHT][32];
    const int n = (int)(stop - start);
    uint2 now = lane < n ? sorted[start + lane] : make_uint2(NO_KEY, 0);
    uint2 next = 32 + lane < n ? sorted[start + 32 + lane] : make_uint2(NO_KEY, 0);
    const DlVec<T, W>* column = reinterpret_cast<const DlVec<T, W>*>(g + col);
    const int64_t row_vectors = D / W;
    // i counts from the first entry of `now`; one group is committed per entry, copied or not
    auto request = [&](int i) {
        const uint32_t k = __shfl_sync(0xffffffffu, i < 32 ? now.x : next.x, i & 31);
        const uint32_t t = __shfl_sync(0xffffffffu, i < 32 ? now.y : next.y, i & 31);
        if (k < (uint64_t)V && live) copy_async<T, W>(&ring[warp][i % ROWS_IN_FLIGHT][lane], column + t * row_vectors);
        copy_commit();
    };
    for (int i = 0; i < ROWS_IN_FLIGHT - 1; ++i) request(i);
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int m = n - i0 < 32 ? n - i0 : 32;
        for (int i = 0; i < m; ++i) {
            request(i + ROWS_IN_FLIGHT - 1);
            copy_wait<ROWS_IN_FLIGHT - 1>();
            const uint32_t k = __shfl_sync(0xffffffffu, now.x, i);
            if (k != key) {
                if (live) {
                    if (open) {
#pragma unroll
                        for (int e = 0; e < W; ++e) head[partial_at + e] = acc[e];
                    } else {
                        store_scaled<T, W>(gw + (int64_t)key * D + col, acc, scale);
                    }
                }
                if (k >= (uint64_t)V) {
                    copy_wait<0>();
                    return;
                }
                key = k;
                open = false;
#pragma unroll
                for (int e = 0; e < W; ++e) acc[e] = 0.0f;
            }
            if (live) {
                float f[W];
                dl_unpack(ring[warp][i % ROWS_IN_FLIGHT][lane], f);
#pragma unroll
                for (int e = 0; e < W; ++e) acc[e] += f[e];
            }
        }
        now = next;
        next = i0 + 64 + lane < n ? sorted[start + i0 + 64 + lane] : make_uint2(NO_KEY, 0);
    }
    if (!live) return;
    if (open || goes_on) {
        float* p = (open ? head : tail) + partial_at;
#pragma unroll
        for (int e = 0; e < W; ++e) p[e] = acc[e];
    } else {
        store_scaled<T, W>(gw + (int64_t)key * D + col, acc, scale);
    }
}

// One block per JOIN_RANGES ranges and slab: a warp each looks for a far-reaching segment that begins in its range, then
// the block joins the found ones in turn.
template <typename T, int W>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
embedding_join_kernel(const uint2* __restrict__ sorted, T* __restrict__ gw, const float* __restrict__ head,
                      const float* __restrict__ tail, int64_t tokens, int64_t V, int64_t D, int64_t range_len,
                      int64_t ranges, int slabs, float scale) {
    __shared__ float sums[JOIN_WARPS][32 * W];
    __shared__ long long last_range[JOIN_RANGES];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t range0 = (int64_t)(blockIdx.x / slabs) * JOIN_RANGES;
    const int slab = (int)(blockIdx.x % slabs);
    if (warp < JOIN_RANGES) {
        const int64_t start = (range0 + warp) * range_len, stop = start + range_len;
        long long last = -1;  // the last range that adds to the segment; -1: nothing to join here
        if (stop < tokens) {
            const uint32_t key = sorted[stop - 1].x;
            const bool begins = start == 0 || sorted[start].x != key || sorted[start - 1].x != key;
            if (key < (uint64_t)V && begins && reaches_far(sorted, stop, tokens, key)) {
                for (int64_t r0 = range0 + warp + 1; last < 0; r0 += 32) {
                    // range r is the last one when the segment does not reach far behind it; the list's last range is one
                    const int64_t next = (r0 + lane + 1) * range_len;
                    const bool ends = next >= tokens || !reaches_far(sorted, next, tokens, key) || sorted[next - 1].x != key;
                    const uint32_t found = __ballot_sync(0xffffffffu, ends);
                    if (found) last = r0 + __ffs(found) - 1;
                }
            }
        }
        if (lane == 0) last_range[warp] = last;
    }
    __syncthreads();
    const int64_t row_len = (int64_t)slabs * 32 * W, col = ((int64_t)slab * 32 + lane) * W;
    for (int f = 0; f < JOIN_RANGES; ++f) {
        if (last_range[f] < 0) continue;
        const int64_t range = range0 + f;
        const int64_t n = (int64_t)last_range[f] - range;  // partial sums of ranges range + 1 .. range + n
        const int64_t share = (n + JOIN_WARPS - 1) / JOIN_WARPS;
        const int64_t from = warp * share < n ? warp * share : n, to = from + share < n ? from + share : n;
        float acc[W];
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] = 0.0f;
        const float* p = head + (range + 1 + from) * row_len + col;
        if (col < D) {
#pragma unroll 8
            for (int64_t i = from; i < to; ++i, p += row_len) {
                const DlVec<float, W> row = *reinterpret_cast<const DlVec<float, W>*>(p);
#pragma unroll
                for (int e = 0; e < W; ++e) acc[e] += row.v[e];
            }
        }
#pragma unroll
        for (int e = 0; e < W; ++e) sums[warp][e * 32 + lane] = acc[e];
        __syncthreads();
        if (warp == 0 && col < D) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                acc[e] = tail[range * row_len + col + e];
                for (int w = 0; w < JOIN_WARPS; ++w) acc[e] += sums[w][e * 32 + lane];
            }
            store_scaled<T, W>(gw + (int64_t)sorted[(range + 1) * range_len].x * D + col, acc, scale);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------ host
int64_t aligned256(int64_t n) { return (n + 255) / 256 * 256; }

// The sorted tokens, kept from the lookup to the backward pass.
struct OrderPlan {
    int passes, digit_bits;
    int64_t off_b, off_present, bytes;
    int64_t off_sorted() const { return passes % 2 ? 0 : off_b; }
};

OrderPlan order_plan(int64_t tokens, int64_t V) {
    OrderPlan p;
    int key_bits = 1;  // of the keys 0 .. V
    while (((int64_t)1 << key_bits) <= V) ++key_bits;
    p.passes = (key_bits + SORT_DIGIT_BITS - 1) / SORT_DIGIT_BITS;
    p.digit_bits = (key_bits + p.passes - 1) / p.passes;
    p.off_b = aligned256(tokens * 8);
    p.off_present = 2 * p.off_b;
    p.bytes = p.off_present + aligned256(V);
    return p;
}

// How the backward pass cuts its work; a function of the sizes alone.
struct BackwardPlan {
    int64_t range_len;  // sorted tokens per warp
    int64_t ranges;
    int64_t off_tail, bytes;
};

BackwardPlan backward_plan(int64_t tokens, int64_t D, int64_t dtype) {
    BackwardPlan p;
    const int64_t width = 16 / dl_dtype_size(dtype);
    const int64_t slabs = dl_ceil_div(D, 32 * width);
    // 48 warps for each SM, two rounds of what is resident: ranges differ in what they add to or leave out of their ends
    // (65536 tokens of 2 KB: 56 us, with half as many 63 us).  Ranges of fewer than 8 tokens would mostly be joining.
    p.range_len = dl_min64(dl_max64(dl_ceil_div(tokens * slabs, (int64_t)DL_NUM_SMS * 48), 8), 1024);
    p.ranges = dl_ceil_div(tokens, p.range_len);
    const int64_t row_len = slabs * 32 * width;  // floats per partial row: enough for every vector width
    p.off_tail = aligned256(p.ranges * row_len * 4);
    p.bytes = 2 * p.off_tail;
    return p;
}

template <typename T, int W, typename I>
int launch_forward(const void* ids, const void* weight, void* out, int64_t tokens, int64_t V, int64_t D, float scale,
                   int64_t padding, char* order, cudaStream_t s) {
    Lookup<T, I> look;
    const int64_t nvec = D / W;
    if (nvec > 0x7fffffff) return DL_ERR_TOO_LARGE;
    look.ids = static_cast<const I*>(ids);
    look.weight = static_cast<const T*>(weight);
    look.out = static_cast<T*>(out);
    look.tokens = tokens;
    look.V = V;
    look.nvec = (int)nvec;
    look.scale = scale;
    // four accesses per thread when there are rows enough to fill the GPU, else as many threads as the row has vectors
    const int64_t wanted = tokens >= DL_NUM_SMS * 16 ? dl_ceil_div(nvec, 4) : nvec;
    look.lanes_log2 = 0;
    while (look.lanes_log2 < 8 && (1 << look.lanes_log2) < wanted) ++look.lanes_log2;
    if (order == nullptr) {
        const int64_t blocks = dl_ceil_div(tokens, 256 >> look.lanes_log2);
        if (blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
        embedding_kernel<T, W, I><<<(unsigned)blocks, 256, 0, s>>>(look);
        return dl_launch_status();
    }
    const OrderPlan p = order_plan(tokens, V);
    // runs of 1024 tokens (a key per thread) while the cluster is not full, longer ones from 8192 tokens on
    int per_log2 = 10;
    while (((int64_t)MAX_CLUSTER << per_log2) < tokens) ++per_log2;
    int ranks = 1;
    while (((int64_t)ranks << per_log2) < tokens) ranks *= 2;
    int64_t per = (int64_t)1 << per_log2;
    if (per > SORT_TILE) {
        per = dl_ceil_div(tokens, ranks);
        per_log2 = -1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ranks);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = sizeof(SortShared);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const auto kernel = embedding_sorting_kernel<T, W, I>;
    static DlKernelLimits limits;
    if (!dl_allow(reinterpret_cast<const void*>(kernel), limits, sizeof(SortShared))) return DL_ERR_LAUNCH;
    // as many clusters look up beside the one that sorts as are resident with it, as far as there are rows for them: a
    // cluster that has to wait would start its share when the others have finished theirs (65536 rows of 2 KB: 52 us)
    static std::atomic<int> resident[64][4];  // per device and log2 of the cluster; asked for once
    int device = 0, log2 = 0;
    while (1 << log2 < ranks) ++log2;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return DL_ERR_LAUNCH;
    int clusters = resident[device][log2].load(std::memory_order_relaxed);
    if (clusters == 0) {
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) return DL_ERR_LAUNCH;
        resident[device][log2].store(clusters, std::memory_order_relaxed);
    }
    const int64_t lookers = dl_ceil_div(tokens, (int64_t)(SORT_THREADS >> look.lanes_log2) * ranks);
    cfg.gridDim.x = (unsigned)((1 + dl_max64(dl_min64(lookers, clusters - 1), 1)) * ranks);
    const cudaError_t e = cudaLaunchKernelEx(
        &cfg, kernel, look, padding, reinterpret_cast<uint2*>(order), reinterpret_cast<uint2*>(order + p.off_b),
        reinterpret_cast<uint8_t*>(order + p.off_present), p.passes, p.digit_bits, per, per_log2);
    return e == cudaSuccess ? dl_launch_status() : DL_ERR_LAUNCH;
}

template <typename T, typename I>
int forward_width(const void* ids, const void* weight, void* out, int64_t tokens, int64_t V, int64_t D, float scale,
                  int64_t padding, char* order, cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), D, dl_address(weight) | dl_address(out));
    if (w == 16 / (int)sizeof(T))
        return launch_forward<T, 16 / sizeof(T), I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
    if (w == 4) return launch_forward<T, 4, I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
    if (w == 2) return launch_forward<T, 2, I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
    return launch_forward<T, 1, I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
}

template <typename I>
int forward_type(const void* ids, const void* weight, void* out, int64_t tokens, int64_t V, int64_t D, int64_t dtype,
                 float scale, int64_t padding, char* order, cudaStream_t s) {
    if (dtype == DL_DTYPE_F32)
        return forward_width<float, I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
    if (dtype == DL_DTYPE_BF16)
        return forward_width<__nv_bfloat16, I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
    return forward_width<__half, I>(ids, weight, out, tokens, V, D, scale, padding, order, s);
}

template <typename T, int W>
int launch_sums(const char* order, const void* g, void* gw, char* scratch, int64_t tokens, int64_t V, int64_t D,
                int64_t dtype, float scale, cudaStream_t s) {
    const OrderPlan o = order_plan(tokens, V);
    const BackwardPlan p = backward_plan(tokens, D, dtype);
    const uint2* sorted = reinterpret_cast<const uint2*>(order + o.off_sorted());
    const uint8_t* present = reinterpret_cast<const uint8_t*>(order + o.off_present);
    float* head = reinterpret_cast<float*>(scratch);
    float* tail = reinterpret_cast<float*>(scratch + p.off_tail);
    const int slabs = (int)dl_ceil_div(D, 32 * W);
    const int64_t zero_blocks = dl_ceil_div(V, ZERO_ROWS);
    const int64_t blocks = dl_ceil_div(p.ranges * slabs, SUM_WARPS) + zero_blocks;
    const int64_t join_blocks = dl_ceil_div(p.ranges, JOIN_RANGES) * slabs;
    if (blocks > 0x7fffffff || join_blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
    embedding_sum_kernel<T, W><<<(unsigned)blocks, 32 * SUM_WARPS, 0, s>>>(
        sorted, static_cast<const T*>(g), static_cast<T*>(gw), present, head, tail, tokens, V, D, p.range_len, p.ranges,
        slabs, zero_blocks, scale);
    if (cudaPeekAtLastError() != cudaSuccess) return DL_ERR_LAUNCH;
    if (p.range_len + REACH <= tokens)  // else no segment can reach far behind a range
        embedding_join_kernel<T, W><<<(unsigned)join_blocks, 32 * JOIN_WARPS, 0, s>>>(
            sorted, static_cast<T*>(gw), head, tail, tokens, V, D, p.range_len, p.ranges, slabs, scale);
    return dl_launch_status();
}

template <typename T>
int sums_width(const char* order, const void* g, void* gw, char* scratch, int64_t tokens, int64_t V, int64_t D,
               int64_t dtype, float scale, cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), D, dl_address(g) | dl_address(gw));
    if (w == 16 / (int)sizeof(T))
        return launch_sums<T, 16 / sizeof(T)>(order, g, gw, scratch, tokens, V, D, dtype, scale, s);
    if (w == 4) return launch_sums<T, 4>(order, g, gw, scratch, tokens, V, D, dtype, scale, s);
    if (w == 2) return launch_sums<T, 2>(order, g, gw, scratch, tokens, V, D, dtype, scale, s);
    return launch_sums<T, 1>(order, g, gw, scratch, tokens, V, D, dtype, scale, s);
}

bool sizes_ok(int64_t tokens, int64_t V, int64_t D, int64_t dtype) {
    return tokens >= 0 && V > 0 && D > 0 && dl_dtype_known(dtype);
}

// keys and positions are 32-bit words, and the key V stands for "no gradient"
bool order_fits(int64_t tokens, int64_t V, int64_t D) {
    return tokens < ((int64_t)1 << 31) && V < ((int64_t)1 << 31) && D < ((int64_t)1 << 31);
}

}  // namespace

DL_EXPORT int64_t dl_embedding_order_bytes(int64_t tokens, int64_t V, int64_t D, int64_t dtype) {
    if (!sizes_ok(tokens, V, D, dtype) || !order_fits(tokens, V, D)) return 0;
    return order_plan(tokens, V).bytes;
}

DL_EXPORT int dl_embedding(const void* ids, int64_t id_bits, const void* weight, void* out, int64_t tokens, int64_t V,
                           int64_t D, int64_t dtype, float scale, int64_t padding_idx, void* order, dl_stream_t stream) {
    DL_REQUIRE(sizes_ok(tokens, V, D, dtype) && (id_bits == 32 || id_bits == 64));
    if (tokens == 0 && order == nullptr) return DL_OK;
    DL_REQUIRE(tokens == 0 || (ids && weight && out));
    DL_REQUIRE_ALIGNED(ids, id_bits / 8);
    DL_REQUIRE_ALIGNED(weight, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(out, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(order, 256);
    if (order != nullptr && !order_fits(tokens, V, D)) return DL_ERR_TOO_LARGE;
    cudaStream_t s = dl_cast(stream);
    char* mem = static_cast<char*>(order);
    return id_bits == 64 ? forward_type<int64_t>(ids, weight, out, tokens, V, D, dtype, scale, padding_idx, mem, s)
                         : forward_type<int32_t>(ids, weight, out, tokens, V, D, dtype, scale, padding_idx, mem, s);
}

DL_EXPORT int64_t dl_embedding_bwd_scratch_bytes(int64_t tokens, int64_t V, int64_t D, int64_t dtype) {
    if (!sizes_ok(tokens, V, D, dtype) || !order_fits(tokens, V, D)) return 0;
    return dl_max64(backward_plan(tokens, D, dtype).bytes, 256);  // 0 means "not supported"
}

DL_EXPORT int dl_embedding_bwd(const void* order, const void* g, void* gw, int64_t tokens, int64_t V, int64_t D,
                               int64_t dtype, float scale, void* scratch, dl_stream_t stream) {
    DL_REQUIRE(sizes_ok(tokens, V, D, dtype));
    DL_REQUIRE(order && gw && scratch && (tokens == 0 || g));
    if (!order_fits(tokens, V, D)) return DL_ERR_TOO_LARGE;
    DL_REQUIRE_ALIGNED(order, 256);
    DL_REQUIRE_ALIGNED(scratch, 256);
    DL_REQUIRE_ALIGNED(g, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(gw, dl_dtype_size(dtype));
    const char* sorted = static_cast<const char*>(order);
    char* mem = static_cast<char*>(scratch);
    cudaStream_t s = dl_cast(stream);
    if (dtype == DL_DTYPE_F32) return sums_width<float>(sorted, g, gw, mem, tokens, V, D, dtype, scale, s);
    if (dtype == DL_DTYPE_BF16) return sums_width<__nv_bfloat16>(sorted, g, gw, mem, tokens, V, D, dtype, scale, s);
    return sums_width<__half>(sorted, g, gw, mem, tokens, V, D, dtype, scale, s);
}
