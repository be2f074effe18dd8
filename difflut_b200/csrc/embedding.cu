// Embedding lookup with scaling and its gradient by sorted tokens.
//
//   forward    out[t, :] = scale * W[id[t], :]
//   backward   gW[v, :]  = scale * sum over t with id[t] == v, ascending t, of g[t, :]
//
// The gradient is a segmented sum over the tokens in sorted order, without atomics on values, so it is the same
// bits on every run.  Three launches:
//   1. a stable radix sort of (id, position) by one cluster of thread blocks, which also marks the ids that occur;
//   2. one warp per range of sorted tokens and slab of columns adds the gradient rows in fp32 registers and writes
//      every segment that lies inside its range; blocks behind those write the zero rows of ids that do not occur,
//      so each row of gW is written once;
//   3. segments that cross range borders are joined from their fp32 partial sums, in range order.
#include <cooperative_groups.h>

#include "elements.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_TILE = 4 * SORT_THREADS;
constexpr int SORT_BINS = 256;
constexpr int MAX_CLUSTER = 8;

// id as stored, or -1 when it is outside [0, V)
template <typename I>
__device__ __forceinline__ int64_t checked_id(const I* ids, int64_t t, int64_t V) {
    const int64_t id = (int64_t)ids[t];
    return id >= 0 && id < V ? id : -1;
}

// ------------------------------------------------------------------------------------------ forward
// 2^lanes_log2 threads per row, up to four accesses in flight each
template <typename T, int W, typename I>
__global__ void __launch_bounds__(256)
embedding_kernel(const I* __restrict__ ids, const T* __restrict__ weight, T* __restrict__ out, int64_t tokens, int64_t V,
                 int nvec, int lanes_log2, float scale) {
    const int lanes = 1 << lanes_log2;
    const int64_t t = (int64_t)blockIdx.x * (256 >> lanes_log2) + (threadIdx.x >> lanes_log2);
    if (t >= tokens) return;
    const int64_t id = checked_id(ids, t, V);
    const DlVec<T, W>* src = reinterpret_cast<const DlVec<T, W>*>(weight) + (id < 0 ? 0 : id) * nvec;
    DlVec<T, W>* dst = reinterpret_cast<DlVec<T, W>*>(out) + t * nvec;
    const float factor = id < 0 ? __int_as_float(0x7fffffff) : scale;  // NaN rows for ids that do not exist
    for (int v0 = threadIdx.x & (lanes - 1); v0 < nvec; v0 += 4 * lanes) {
        DlVec<T, W> r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (v0 + u * lanes < nvec) r[u] = src[v0 + u * lanes];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (v0 + u * lanes >= nvec) break;
#pragma unroll
            for (int e = 0; e < W; ++e) r[u].v[e] = dl_from_float<T>(dl_to_float(r[u].v[e]) * factor);
            dst[v0 + u * lanes] = r[u];
        }
    }
}

// ------------------------------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (key, position); ids that take no gradient get the key V and end up
// last.  Block r of the cluster owns the r-th run of tokens; per pass it counts its digits, adds up the other blocks'
// counts through distributed shared memory, and scatters its tokens tile by tile in order.
template <typename I>
__global__ void __launch_bounds__(SORT_THREADS)
embedding_sort_kernel(const I* __restrict__ ids, int64_t tokens, int64_t V, int64_t padding, uint2* a, uint2* b,
                      uint8_t* present, int passes, int digit_bits) {
    __shared__ uint32_t warp_count[SORT_THREADS / 32][SORT_BINS];
    __shared__ uint32_t totals[SORT_BINS];
    __shared__ uint32_t base[SORT_BINS];
    __shared__ uint32_t warp_sum[SORT_BINS / 32];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t per = (tokens + ranks - 1) / ranks;
    const int64_t lo = rank * per < tokens ? rank * per : tokens;
    const int64_t hi = lo + per < tokens ? lo + per : tokens;
    const uint32_t bins_mask = (1u << digit_bits) - 1;

    uint32_t* present_words = reinterpret_cast<uint32_t*>(present);  // the scratch holds whole words
    for (int64_t i = (int64_t)rank * SORT_THREADS + tid; i < (V + 3) / 4; i += (int64_t)ranks * SORT_THREADS)
        present_words[i] = 0;

    const uint2* src = nullptr;
    uint2* dst = a;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        // entries of other blocks' writing are read past L1
        auto load = [&](int64_t i) {
            if (pass > 0) return __ldcg(src + i);
            const int64_t id = checked_id(ids, i, V);
            return make_uint2(id < 0 || id == padding ? (uint32_t)V : (uint32_t)id, (uint32_t)i);
        };
        if (tid < SORT_BINS) totals[tid] = 0;
        __syncthreads();
        for (int64_t i0 = lo; i0 < hi; i0 += SORT_THREADS) {
            const int64_t i = i0 + tid;
            const uint32_t digit = i < hi ? (load(i).x >> shift) & bins_mask : NO_KEY;
            const uint32_t same = __match_any_sync(0xffffffffu, digit);
            if (digit != NO_KEY && lane == __ffs(same) - 1) atomicAdd(&totals[digit], (uint32_t)__popc(same));
        }
        cluster.sync();
        uint32_t all = 0, before = 0, inclusive = 0;
        if (tid < SORT_BINS) {
            for (int r = 0; r < ranks; ++r) {
                const uint32_t c = *cluster.map_shared_rank(&totals[tid], r);
                all += c;
                if (r < rank) before += c;
            }
            inclusive = all;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, inclusive, s);
                if (lane >= s) inclusive += o;
            }
            if (lane == 31) warp_sum[warp] = inclusive;
        }
        __syncthreads();
        if (tid < SORT_BINS) {
            uint32_t lower = 0;
            for (int w = 0; w < warp; ++w) lower += warp_sum[w];
            base[tid] = lower + inclusive - all + before;
        }
        const bool last = pass == passes - 1;
        for (int64_t t0 = lo; t0 < hi; t0 += SORT_TILE) {
#pragma unroll
            for (int k = 0; k < SORT_BINS / 32; ++k) (&warp_count[0][0])[k * SORT_THREADS + tid] = 0;
            __syncthreads();
            uint2 entry[4];
            uint32_t digit[4], slot[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t i = t0 + warp * 128 + j * 32 + lane;
                entry[j] = i < hi ? load(i) : make_uint2(0, 0);
                digit[j] = i < hi ? (entry[j].x >> shift) & bins_mask : NO_KEY;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t same = __match_any_sync(0xffffffffu, digit[j]);
                uint32_t held = 0;
                if (digit[j] != NO_KEY) held = warp_count[warp][digit[j]];
                __syncwarp();
                if (digit[j] != NO_KEY && lane == __ffs(same) - 1) warp_count[warp][digit[j]] = held + __popc(same);
                __syncwarp();
                slot[j] = held + __popc(same & ((1u << lane) - 1));
            }
            __syncthreads();
            if (tid < SORT_BINS) {
                uint32_t run = base[tid];
#pragma unroll 8
                for (int w = 0; w < SORT_THREADS / 32; ++w) {
                    const uint32_t c = warp_count[w][tid];
                    warp_count[w][tid] = run;
                    run += c;
                }
                base[tid] = run;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (digit[j] == NO_KEY) continue;
                dst[warp_count[warp][digit[j]] + slot[j]] = entry[j];
                if (last && entry[j].x < V) present[entry[j].x] = 1;
            }
            __syncthreads();
        }
        cluster.sync();  // the pass is complete, and every block has read the other blocks' totals
        src = dst;
        dst = dst == a ? b : a;
    }
}

// ------------------------------------------------------------------------------------------ segmented sum
constexpr int SUM_WARPS = 4;
constexpr int ROWS_IN_FLIGHT = 8;
constexpr int ZERO_ROWS = 32;
constexpr int JOIN_WARPS = 8;

template <typename T, int W>
__device__ __forceinline__ void store_scaled(T* dst, const float (&acc)[W], float scale) {
    DlVec<T, W> r;
#pragma unroll
    for (int e = 0; e < W; ++e) r.v[e] = dl_from_float<T>(acc[e] * scale);
    *reinterpret_cast<DlVec<T, W>*>(dst) = r;
}

// partial sums have the padded row length slabs * 32 * W
template <int W>
__device__ __forceinline__ void store_partial(float* dst, const float (&acc)[W]) {
#pragma unroll
    for (int e = 0; e < W; ++e) dst[e] = acc[e];
}

template <typename T, int W>
__global__ void __launch_bounds__(32 * SUM_WARPS)
embedding_sum_kernel(const uint2* __restrict__ sorted, const T* __restrict__ g, T* __restrict__ gw,
                     const uint8_t* __restrict__ present, float* __restrict__ head, float* __restrict__ tail,
                     int64_t tokens, int64_t V, int64_t D, int64_t range_len, int64_t ranges, int slabs,
                     int64_t sum_blocks, float scale) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if ((int64_t)blockIdx.x >= sum_blocks) {
        const int64_t row0 = ((int64_t)blockIdx.x - sum_blocks) * ZERO_ROWS;
        DlVec<T, W> zero;
#pragma unroll
        for (int e = 0; e < W; ++e) zero.v[e] = dl_from_float<T>(0.0f);
        for (int64_t v = row0 + warp; v < row0 + ZERO_ROWS && v < V; v += SUM_WARPS) {
            if (present[v]) continue;
            for (int64_t c = lane; c < D / W; c += 32) reinterpret_cast<DlVec<T, W>*>(gw + v * D)[c] = zero;
        }
        return;
    }
    const int slab = (int)(blockIdx.x % slabs);
    const int64_t range = (int64_t)(blockIdx.x / slabs) * SUM_WARPS + warp;
    if (range >= ranges) return;
    const int64_t col = ((int64_t)slab * 32 + lane) * W;
    const bool live = col < D;
    const int64_t start = range * range_len;
    const int64_t stop = start + range_len < tokens ? start + range_len : tokens;
    const int64_t partial_at = range * ((int64_t)slabs * 32 * W) + col;
    const uint32_t ahead = start > 0 ? sorted[start - 1].x : NO_KEY;
    const uint32_t behind = stop < tokens ? sorted[stop].x : NO_KEY;
    uint32_t key = sorted[start].x;
    if (key >= (uint64_t)V) return;  // only ids without gradient from here on
    bool open = key == ahead;        // the segment began in an earlier range
    float acc[W];
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] = 0.0f;

    for (int64_t i0 = start; i0 < stop; i0 += 32) {
        const uint2 mine = i0 + lane < stop ? sorted[i0 + lane] : make_uint2(NO_KEY, 0);
        const int n = (int)(stop - i0 < 32 ? stop - i0 : 32);
        for (int j0 = 0; j0 < n; j0 += ROWS_IN_FLIGHT) {
            DlVec<T, W> row[ROWS_IN_FLIGHT];
#pragma unroll
            for (int u = 0; u < ROWS_IN_FLIGHT; ++u) {
                const uint32_t k = __shfl_sync(0xffffffffu, mine.x, (j0 + u) & 31);
                const uint32_t t = __shfl_sync(0xffffffffu, mine.y, (j0 + u) & 31);
                if (j0 + u < n && k < (uint64_t)V && live)
                    row[u] = *reinterpret_cast<const DlVec<T, W>*>(g + (int64_t)t * D + col);
            }
#pragma unroll
            for (int u = 0; u < ROWS_IN_FLIGHT; ++u) {
                const uint32_t k = __shfl_sync(0xffffffffu, mine.x, (j0 + u) & 31);
                if (j0 + u >= n) break;
                if (k != key) {
                    if (live) {
                        if (open) store_partial<W>(head + partial_at, acc);
                        else store_scaled<T, W>(gw + (int64_t)key * D + col, acc, scale);
                    }
                    if (k >= (uint64_t)V) return;
                    key = k;
                    open = false;
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[e] = 0.0f;
                }
                if (live) {
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[e] += dl_to_float(row[u].v[e]);
                }
            }
        }
    }
    if (!live) return;
    if (open) store_partial<W>(head + partial_at, acc);
    else if (key == behind) store_partial<W>(tail + partial_at, acc);
    else store_scaled<T, W>(gw + (int64_t)key * D + col, acc, scale);
}

// One block per (range, slab); it works only where a segment begins in the range and goes on behind it.
template <typename T, int W>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
embedding_join_kernel(const uint2* __restrict__ sorted, T* __restrict__ gw, const float* __restrict__ head,
                      const float* __restrict__ tail, int64_t tokens, int64_t V, int64_t D, int64_t range_len,
                      int64_t ranges, int slabs, float scale) {
    __shared__ float sums[JOIN_WARPS][32 * W];
    __shared__ unsigned long long last_range;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t range = blockIdx.x / slabs;
    const int slab = (int)(blockIdx.x % slabs);
    const int64_t start = range * range_len, stop = start + range_len;
    if (stop >= tokens) return;
    const uint32_t key = sorted[stop - 1].x;
    if (key >= (uint64_t)V || sorted[stop].x != key) return;
    if (start > 0 && sorted[start].x == key && sorted[start - 1].x == key) return;
    if (threadIdx.x == 0) last_range = ~0ull;
    __syncthreads();
    for (int64_t r0 = range + 1;; r0 += blockDim.x) {
        const int64_t r = r0 + threadIdx.x;
        const int64_t next = (r + 1) * range_len;
        const bool ends = r < ranges && (next >= tokens || sorted[next].x != key);
        if (ends) atomicMin(&last_range, (unsigned long long)r);
        // the last range always ends its segment, so some thread finds one
        if (__syncthreads_or(ends)) break;
    }
    const int64_t n = (int64_t)last_range - range;  // partial sums of ranges range + 1 .. range + n
    const int64_t row_len = (int64_t)slabs * 32 * W, col = ((int64_t)slab * 32 + lane) * W;
    const int64_t share = (n + JOIN_WARPS - 1) / JOIN_WARPS;
    const int64_t from = warp * share < n ? warp * share : n, to = from + share < n ? from + share : n;
    float acc[W];
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] = 0.0f;
    const float* p = head + (range + 1 + from) * row_len + col;
    if (col < D) {
#pragma unroll 4
        for (int64_t i = from; i < to; ++i, p += row_len) {
#pragma unroll
            for (int e = 0; e < W; ++e) acc[e] += p[e];
        }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) sums[warp][e * 32 + lane] = acc[e];
    __syncthreads();
    if (warp != 0 || col >= D) return;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        acc[e] = tail[range * row_len + col + e];
        for (int w = 0; w < JOIN_WARPS; ++w) acc[e] += sums[w][e * 32 + lane];
    }
    store_scaled<T, W>(gw + (int64_t)key * D + col, acc, scale);
}

// ------------------------------------------------------------------------------------------ host
// How the backward pass cuts its work; a function of the sizes alone.
struct BackwardPlan {
    int slabs;           // of 32 * nominal vector width columns
    int64_t range_len;   // sorted tokens per warp
    int64_t ranges;
    int64_t row_len;     // floats per partial row: enough for every vector width
    int64_t off_b, off_present, off_head, off_tail, bytes;
};

int64_t aligned256(int64_t n) { return (n + 255) / 256 * 256; }

BackwardPlan backward_plan(int64_t tokens, int64_t V, int64_t D, int64_t dtype) {
    BackwardPlan p;
    const int64_t width = 16 / dl_dtype_size(dtype);
    p.slabs = (int)dl_ceil_div(D, 32 * width);
    // about 32 warps for each SM; short ranges would spend their time on joining, long ones leave SMs idle
    p.range_len = dl_min64(dl_max64(dl_ceil_div(tokens * p.slabs, (int64_t)DL_NUM_SMS * 32), 8), 1024);
    p.ranges = dl_ceil_div(tokens, p.range_len);
    p.row_len = p.slabs * 32 * width;
    p.off_b = aligned256(tokens * 8);
    p.off_present = p.off_b + aligned256(tokens * 8);
    p.off_head = p.off_present + aligned256(V);
    p.off_tail = p.off_head + aligned256(p.ranges * p.row_len * 4);
    p.bytes = p.off_tail + aligned256(p.ranges * p.row_len * 4);
    return p;
}

template <typename T, int W, typename I>
int launch_forward(const void* ids, const void* weight, void* out, int64_t tokens, int64_t V, int64_t D, float scale,
                   cudaStream_t s) {
    const int64_t nvec = D / W;
    if (nvec > 0x7fffffff) return DL_ERR_TOO_LARGE;
    // four accesses per thread when there are rows enough to fill the GPU, else as many threads as the row has vectors
    const int64_t wanted = tokens >= DL_NUM_SMS * 16 ? dl_ceil_div(nvec, 4) : nvec;
    int lanes_log2 = 0;
    while (lanes_log2 < 8 && (1 << lanes_log2) < wanted) ++lanes_log2;
    const int64_t blocks = dl_ceil_div(tokens, 256 >> lanes_log2);
    if (blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
    embedding_kernel<T, W, I><<<(unsigned)blocks, 256, 0, s>>>(static_cast<const I*>(ids), static_cast<const T*>(weight),
                                                              static_cast<T*>(out), tokens, V, (int)nvec, lanes_log2,
                                                              scale);
    return dl_launch_status();
}

template <typename T, typename I>
int forward_width(const void* ids, const void* weight, void* out, int64_t tokens, int64_t V, int64_t D, float scale,
                  cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), D, dl_address(weight) | dl_address(out));
    if (w == 16 / (int)sizeof(T)) return launch_forward<T, 16 / sizeof(T), I>(ids, weight, out, tokens, V, D, scale, s);
    if (w == 4) return launch_forward<T, 4, I>(ids, weight, out, tokens, V, D, scale, s);
    if (w == 2) return launch_forward<T, 2, I>(ids, weight, out, tokens, V, D, scale, s);
    return launch_forward<T, 1, I>(ids, weight, out, tokens, V, D, scale, s);
}

template <typename I>
int forward_type(const void* ids, const void* weight, void* out, int64_t tokens, int64_t V, int64_t D, int64_t dtype,
                 float scale, cudaStream_t s) {
    if (dtype == DL_DTYPE_F32) return forward_width<float, I>(ids, weight, out, tokens, V, D, scale, s);
    if (dtype == DL_DTYPE_BF16) return forward_width<__nv_bfloat16, I>(ids, weight, out, tokens, V, D, scale, s);
    return forward_width<__half, I>(ids, weight, out, tokens, V, D, scale, s);
}

template <typename T, int W>
int launch_sums(const uint2* sorted, const void* g, void* gw, const uint8_t* present, float* head, float* tail,
                int64_t tokens, int64_t V, int64_t D, const BackwardPlan& p, float scale, cudaStream_t s) {
    const int slabs = (int)dl_ceil_div(D, 32 * W);
    const int64_t sum_blocks = dl_ceil_div(p.ranges, SUM_WARPS) * slabs;
    const int64_t blocks = sum_blocks + dl_ceil_div(V, ZERO_ROWS);
    if (blocks > 0x7fffffff || p.ranges * slabs > 0x7fffffff) return DL_ERR_TOO_LARGE;
    embedding_sum_kernel<T, W><<<(unsigned)blocks, 32 * SUM_WARPS, 0, s>>>(
        sorted, static_cast<const T*>(g), static_cast<T*>(gw), present, head, tail, tokens, V, D, p.range_len, p.ranges,
        slabs, sum_blocks, scale);
    if (cudaPeekAtLastError() != cudaSuccess) return DL_ERR_LAUNCH;
    if (p.ranges > 1)
        embedding_join_kernel<T, W><<<(unsigned)(p.ranges * slabs), 32 * JOIN_WARPS, 0, s>>>(
            sorted, static_cast<T*>(gw), head, tail, tokens, V, D, p.range_len, p.ranges, slabs, scale);
    return dl_launch_status();
}

template <typename T>
int sums_width(const uint2* sorted, const void* g, void* gw, const uint8_t* present, float* head, float* tail,
               int64_t tokens, int64_t V, int64_t D, const BackwardPlan& p, float scale, cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), D, dl_address(g) | dl_address(gw));
    if (w == 16 / (int)sizeof(T))
        return launch_sums<T, 16 / sizeof(T)>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
    if (w == 4) return launch_sums<T, 4>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
    if (w == 2) return launch_sums<T, 2>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
    return launch_sums<T, 1>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
}

template <typename I>
int launch_sort(const void* ids, int64_t tokens, int64_t V, int64_t padding, uint2* a, uint2* b, uint8_t* present,
                int passes, int digit_bits, cudaStream_t s) {
    int ranks = 1;  // one tile per block and pass while the cluster is not full
    while (ranks < MAX_CLUSTER && (int64_t)ranks * SORT_TILE < tokens) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ranks);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, embedding_sort_kernel<I>, static_cast<const I*>(ids), tokens, V,
                                             padding, a, b, present, passes, digit_bits);
    return e == cudaSuccess ? dl_launch_status() : DL_ERR_LAUNCH;
}

bool sizes_ok(int64_t tokens, int64_t V, int64_t D, int64_t dtype) {
    return tokens >= 0 && V > 0 && D > 0 && dl_dtype_known(dtype);
}

// keys and positions are 32-bit words, and the key V stands for "no gradient"
bool backward_fits(int64_t tokens, int64_t V, int64_t D) {
    return tokens < ((int64_t)1 << 31) && V < ((int64_t)1 << 31) && D < ((int64_t)1 << 31);
}

}  // namespace

DL_EXPORT int dl_embedding(const void* ids, int64_t id_bits, const void* weight, void* out, int64_t tokens, int64_t V,
                           int64_t D, int64_t dtype, float scale, dl_stream_t stream) {
    DL_REQUIRE(sizes_ok(tokens, V, D, dtype) && (id_bits == 32 || id_bits == 64));
    if (tokens == 0) return DL_OK;
    DL_REQUIRE(ids && weight && out);
    DL_REQUIRE_ALIGNED(ids, id_bits / 8);
    DL_REQUIRE_ALIGNED(weight, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(out, dl_dtype_size(dtype));
    cudaStream_t s = dl_cast(stream);
    return id_bits == 64 ? forward_type<int64_t>(ids, weight, out, tokens, V, D, dtype, scale, s)
                         : forward_type<int32_t>(ids, weight, out, tokens, V, D, dtype, scale, s);
}

DL_EXPORT int64_t dl_embedding_bwd_scratch_bytes(int64_t tokens, int64_t V, int64_t D, int64_t dtype) {
    if (!sizes_ok(tokens, V, D, dtype) || !backward_fits(tokens, V, D)) return 0;
    return backward_plan(tokens, V, D, dtype).bytes;
}

DL_EXPORT int dl_embedding_bwd(const void* ids, int64_t id_bits, const void* g, void* gw, int64_t tokens, int64_t V,
                               int64_t D, int64_t dtype, float scale, int64_t padding_idx, void* scratch,
                               dl_stream_t stream) {
    DL_REQUIRE(sizes_ok(tokens, V, D, dtype) && (id_bits == 32 || id_bits == 64));
    DL_REQUIRE(gw && scratch && (tokens == 0 || (ids && g)));
    if (!backward_fits(tokens, V, D)) return DL_ERR_TOO_LARGE;
    DL_REQUIRE_ALIGNED(scratch, 256);
    DL_REQUIRE_ALIGNED(ids, id_bits / 8);
    DL_REQUIRE_ALIGNED(g, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(gw, dl_dtype_size(dtype));
    const BackwardPlan p = backward_plan(tokens, V, D, dtype);
    char* mem = static_cast<char*>(scratch);
    uint2* a = reinterpret_cast<uint2*>(mem);
    uint2* b = reinterpret_cast<uint2*>(mem + p.off_b);
    uint8_t* present = reinterpret_cast<uint8_t*>(mem + p.off_present);
    float* head = reinterpret_cast<float*>(mem + p.off_head);
    float* tail = reinterpret_cast<float*>(mem + p.off_tail);
    int key_bits = 1;  // of the keys 0 .. V
    while (((int64_t)1 << key_bits) <= V) ++key_bits;
    const int passes = (key_bits + 7) / 8, digit_bits = (key_bits + passes - 1) / passes;
    cudaStream_t s = dl_cast(stream);
    const int rc = id_bits == 64 ? launch_sort<int64_t>(ids, tokens, V, padding_idx, a, b, present, passes, digit_bits, s)
                                 : launch_sort<int32_t>(ids, tokens, V, padding_idx, a, b, present, passes, digit_bits, s);
    if (rc != DL_OK) return rc;
    const uint2* sorted = passes % 2 ? a : b;
    if (dtype == DL_DTYPE_F32) return sums_width<float>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
    if (dtype == DL_DTYPE_BF16)
        return sums_width<__nv_bfloat16>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
    return sums_width<__half>(sorted, g, gw, present, head, tail, tokens, V, D, p, scale, s);
}
