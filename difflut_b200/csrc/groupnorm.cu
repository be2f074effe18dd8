// Group norm with an activation over channels-last data x (N, S, C), G groups of C / G channels.
//
//   xh = (x - mean) * rstd per (sample, group), z = xh * weight + bias, y = act(z)
//   dz = gy * act'(z);  gbias = sum dz;  gweight = sum dz * xh;
//   gx = rstd * (weight * dz - (s1 + xh * s2) / m),  s1 = sum weight * dz,  s2 = sum weight * dz * xh,  m = S * C / G
//
// Both directions read their tensors twice, first for the sums, then to write the result.  A sample is cut into chunks of
// rows, one thread block each, such that all blocks are resident at once: one launch leaves every chunk's sums, the next
// one adds up its sample's (a few hundred numbers) and writes.  Where samples alone fill the GPU a chunk is a sample and
// one launch does both.  The second reading comes from L2 as far as the tensor fits there.  (Holding a sample in the shared
// memory of a cluster, so that it is read once, was slower: all blocks load, then all compute, then all store, and each
// sample costs a cluster barrier: 51 us instead of 43 us forward, 90 instead of 73 us backward for 16 x 4096 x 512 bf16.)
// A thread keeps to its own channels (a vector of W).  Rows without positions (S = 1) take kernels of their own, in which a
// group is a few lanes of a warp and stays in registers.
//
// A thread takes its values in runs of up to 32 rows and sums their squares relative to the mean of all that came before the
// run.  A run is no longer than what came before it, so these squares add up to no more than twice the squares around the
// thread's mean, wherever its first values lie: a run of n values costs at most 2 n * 2^-24 of the variance.  (The first
// run of 8 rows is taken relative to the mean of its first row: 9 n.)  Runs, threads and chunks are joined by their means and
// their squares, moved to the joint mean: only additions.  No atomics: the same bits on every call.
//
// Measured with nothing of the inputs in L2, 16 x 4096 x 512 bf16 with 32 groups and silu (67 MB a tensor): sums 19.9 us
// (3.4 TB/s; without the runs 19.8), writing 28.4 us (4.7 TB/s read and written; the exponential and the reciprocal keep
// their pipe 60 % busy); backward sums 34 us (3.9 TB/s), writing 35 us (5.7 TB/s), the parameters' sums 4 us.  8192 rows of
// 1024 bf16 features, 32 groups, sigmoid (17 MB a tensor): 15.2 us forward and 24.1 + 3.6 us backward: a round of loads,
// shuffles and stores after the other, no unit above half of its rate (issue slots 51 %).  Maps of 128 x 576 x 32 fp32
// (9 MB): 5.9 + 5.6 us forward, 7.7 + 6.3 + 2.4 us backward, mostly the latency of the launches.  Many samples of few
// positions are slow for their size: 8192 x 6 x 16 fp32 (3 MB) 37.9 us forward, 49.8 + 12.4 backward, as every sample is
// a block of one warp here, which holds the shared memory of eight.
#include <type_traits>

#include "elements.cuh"

namespace {

constexpr int MAX_LANES = 256;  // threads across the channels of one block

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_SIGMOID = 3 };

// 1 / (1 + e^-z).  The approximate exponential (2^x with x rounded to fp32: its error grows with |z|, where the sigmoid
// no longer depends on it) is for 16-bit results.  Results below 2^-126 become 0.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float z) {
    float e, s;
    if (sizeof(T) == 4) e = expf(-z);
    else asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + e));
    return s;
}

template <typename T, int ACT>
__device__ __forceinline__ float activate(float z) {
    if (ACT == ACT_NONE) return z;
    if (ACT == ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    const float s = sigmoid_of<T>(z);
    return ACT == ACT_SILU ? z * s : s;
}

template <typename T, int ACT>
__device__ __forceinline__ float slope(float z) {
    if (ACT == ACT_NONE) return 1.0f;
    if (ACT == ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    const float s = sigmoid_of<T>(z), rest = 1.0f - s;
    return ACT == ACT_SILU ? s * fmaf(z, rest, 1.0f) : s * rest;
}

// calls f with the activation as a compile-time constant: inside the loops over rows the switch would cost a branch
// per value
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
    if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>());
    else if (act == ACT_SIGMOID) f(std::integral_constant<int, ACT_SIGMOID>());
    else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>());
    else f(std::integral_constant<int, ACT_NONE>());
}

struct Norm {
    const void* weight;  // null: ones
    const void* bias;    // null: zeros
    int param_dtype;
    int64_t N, S;
    int C, G;
    int per_group;  // channels
    float eps;
    int act;
};

// parameters c .. c + W - 1, c a multiple of W; by vectors where their addresses allow
template <int W>
__device__ __forceinline__ void load_param(const void* p, int dtype, float missing, int c, float (&f)[W]) {
    constexpr int BYTES32 = W * 4 < 16 ? W * 4 : 16;
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < W; ++e) f[e] = missing;
    } else if (dtype == DL_DTYPE_F32 && reinterpret_cast<uintptr_t>(p) % BYTES32 == 0) {
        dl_unpack(*reinterpret_cast<const DlVec<float, W>*>(static_cast<const float*>(p) + c), f);
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) f[e] = dl_load_as_float(p, dtype, c + e);
    }
}
template <int W>
__device__ __forceinline__ void load_params(const Norm& p, int c, float (&w)[W], float (&b)[W]) {
    load_param<W>(p.weight, p.param_dtype, 1.0f, c, w);
    load_param<W>(p.bias, p.param_dtype, 0.0f, c, b);
}

// ------------------------------------------------------------------------------------------ chunks of rows
constexpr int CHUNK_THREADS = 256;

// How the tensor is cut; a function of sizes, type and alignment.
struct Cut {
    int lanes;       // vectors across one group
    int groups;      // per block of channels, whole ones; 1 when a group is wider than a block
    int split;       // blocks of channels per group
    int tx, ty;      // threads across channels and down the rows of one block
    int blocks_c;    // blocks of channels
    int chunks;      // of rows per sample
    int rows;        // per chunk
};

// What a thread works on.  A part is one (chunk, block of channels of the group): the partial sums of a sample's group are
// chunks * split numbers.
struct Place {
    int tx, ty;
    int64_t n;
    int chunk, piece;     // which of the group's blocks of channels
    int group0, groups;   // first group of the block, how many it has
    int group;            // of the thread, from group0
    int group_lanes;      // of a group in this block
    int channel;          // first of the thread's W
    int row0, rows;
    int mine;             // rows of the thread: ty, ty + k.ty, ...
    bool live;
    __device__ __forceinline__ Place(const Norm& p, const Cut& k, int W) {
        tx = threadIdx.x % k.tx;
        ty = threadIdx.x / k.tx;
        const int64_t unit = blockIdx.x / k.chunks;
        chunk = (int)(blockIdx.x - unit * k.chunks);
        n = unit / k.blocks_c;
        const int block_c = (int)(unit - n * k.blocks_c), set = block_c / k.split;
        piece = block_c - set * k.split;
        group0 = set * k.groups;
        groups = p.G - group0 < k.groups ? p.G - group0 : k.groups;
        group_lanes = lanes_of(k, piece);
        const int lane = piece * k.tx + tx;  // piece is 0 when the block holds whole groups
        group = k.split > 1 ? 0 : tx / k.lanes;
        live = ty < k.ty && (k.split > 1 ? lane < k.lanes : group < groups);
        channel = (group0 * k.lanes + lane) * W;
        row0 = chunk * k.rows;
        rows = rows_of(p, k, chunk);
        mine = live && ty < rows ? (rows - ty + k.ty - 1) / k.ty : 0;
    }
    __device__ __forceinline__ static int lanes_of(const Cut& k, int piece) {
        if (k.split == 1) return k.lanes;
        const int left = k.lanes - piece * k.tx;
        return left < k.tx ? left : k.tx;
    }
    __device__ __forceinline__ static int rows_of(const Norm& p, const Cut& k, int chunk) {
        const int64_t behind = p.S - (int64_t)chunk * k.rows;
        return (int)(behind < k.rows ? (behind > 0 ? behind : 0) : k.rows);
    }
    __device__ __forceinline__ int part(const Cut& k) const { return chunk * k.split + piece; }
};

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// rows of every tensor that a thread has on their way to its slots of shared memory, at 16 bytes each
template <int TENSORS>
struct Ring {
    static constexpr int AHEAD = TENSORS == 1 ? 8 : 4;  // 32 KB per block
    template <typename V>
    static constexpr size_t bytes() {
        return sizeof(V) < 4 ? 0 : (size_t)AHEAD * TENSORS * CHUNK_THREADS * sizeof(V);
    }
};

constexpr int FIRST_RUN = 8, LONGEST_RUN = 32;  // rows

// What each_row tells about the runs of rows: begin(first row) before f gets it, end(rows) behind every run
template <typename B, typename E>
struct Runs {
    static constexpr bool ARE = true;
    B begin;
    E end;
};
template <typename B, typename E>
Runs(B, E) -> Runs<B, E>;
struct NoRuns {
    static constexpr bool ARE = false;
};

// f(vectors...) for every row of the thread in order; src points to its first row.  The rows come through a ring in shared
// memory, of which every thread fills and reads its own slots: loads go on while it computes, without holding registers.
// Runs are 8, 8, 16, 32, 32, .. rows long, the last one what is left.
template <typename T, int W, typename R, typename F, typename... Src>
__device__ __forceinline__ void each_row(const Place& at, int64_t step, R runs, F f, const Src*... src) {
    int begun = 0, end = FIRST_RUN;  // of the run
    auto end_run = [&](int i) {
        if constexpr (R::ARE) {
            runs.end(i - begun);
            begun = i;
            end += end < LONGEST_RUN ? end : LONGEST_RUN;
        }
    };
    if constexpr (sizeof(DlVec<T, W>) < 4) {  // there is no such copy of two bytes
        if constexpr (R::ARE) {
            if (at.mine > 0) runs.begin(*reinterpret_cast<const DlVec<T, W>*>(src)...);
        }
        for (int i = 0; i < at.mine;) {
            const int stop = R::ARE && end < at.mine ? end : at.mine;
            for (; i < stop; ++i) f(*reinterpret_cast<const DlVec<T, W>*>(src + i * step)...);
            end_run(i);
        }
    } else {
        constexpr int TENSORS = (int)sizeof...(Src), AHEAD = Ring<TENSORS>::AHEAD, BYTES = (int)sizeof(DlVec<T, W>);
        static_assert(FIRST_RUN % AHEAD == 0 && LONGEST_RUN % AHEAD == 0, "runs end between two rounds of the ring");
        extern __shared__ __align__(16) unsigned char ring_of_block[];
        const DlVec<T, W>* ring = reinterpret_cast<const DlVec<T, W>*>(ring_of_block) + threadIdx.x;
        const uint32_t slots = (uint32_t)__cvta_generic_to_shared(ring);
        const T* from[] = {src...};
        auto request = [&](int i, int slot) {
            if (i < at.mine) {
#pragma unroll
                for (int s = 0; s < TENSORS; ++s) {
                    const uint32_t to = slots + (slot * TENSORS + s) * CHUNK_THREADS * BYTES;
                    if constexpr (BYTES == 16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from[s]) : "memory");
                    else
                        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from[s]), "n"(BYTES) : "memory");
                    from[s] += step;
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) request(d, d);
        if constexpr (R::ARE) {
            copy_wait<AHEAD - 1>();
            if (at.mine > 0) runs.begin(ring[0]);
        }
        for (int i = 0; i < at.mine; i += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (i + u >= at.mine) break;
                copy_wait<AHEAD - 1>();
                const DlVec<T, W>* here = ring + u * TENSORS * CHUNK_THREADS;
                if constexpr (TENSORS == 1) f(here[0]);
                else f(here[0], here[CHUNK_THREADS]);
                request(i + u + AHEAD, u);
            }
            if (i + AHEAD == end || i + AHEAD >= at.mine) end_run(i + AHEAD < at.mine ? i + AHEAD : at.mine);
        }
        copy_wait<0>();  // nothing is under way into slots that are used again
    }
}

// Joins sets of values given by count, mean and squares around their means: set(i, count, mean, squares) for i < sets, by a
// warp.  First their mean, relative to one of the sets' (`centre`), then the squares around it.
template <typename F>
__device__ __forceinline__ void join_sets(int sets, float centre, float total, F set, float& mean, float& squares) {
    const int lane = threadIdx.x & 31;
    float count0 = 0.0f, m0 = 0.0f, around0 = 0.0f, count, m, around;  // a lane's first set stays in registers
    if (lane < sets) set(lane, count0, m0, around0);
    float moved = lane < sets ? count0 * (m0 - centre) : 0.0f;
    for (int i = lane + 32; i < sets; i += 32) {
        set(i, count, m, around);
        moved = fmaf(count, m - centre, moved);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) moved += __shfl_xor_sync(0xffffffffu, moved, s);
    mean = centre + __fdividef(moved, total);
    const float d0 = m0 - mean;
    float sum = lane < sets ? fmaf(count0 * d0, d0, around0) : 0.0f;
    for (int i = lane + 32; i < sets; i += 32) {
        set(i, count, m, around);
        const float d = m - mean;
        sum += fmaf(count * d, d, around);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    squares = sum;
}

// calls f(group, entry) for every thread of every group of the block, a warp per group; then done(group) in every lane
template <typename F, typename D, typename B>
__device__ __forceinline__ void warp_per_group(const Place& at, const Cut& k, B begin, F f, D done) {
    const int lane = threadIdx.x & 31, entries = at.group_lanes * k.ty;
    for (int g = threadIdx.x / 32; g < at.groups; g += blockDim.x / 32) {
        begin(g);
        for (int e = lane; e < entries; e += 32) {
            const int y = e / at.group_lanes;
            f(g, y * k.tx + g * at.group_lanes + (e - y * at.group_lanes));
        }
        done(g);
    }
}

enum { SUMS = 1, WRITE = 2 };  // what a launch does; both when a chunk is a sample

// sums (N, G, parts, 2): mean and squares around it of every part
template <typename T, int W, int DO>
__global__ void __launch_bounds__(CHUNK_THREADS, 4)
norm_chunk_kernel(const T* __restrict__ x, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                  float* __restrict__ sums, const __grid_constant__ Norm p, const __grid_constant__ Cut k) {
    __shared__ float red[3][CHUNK_THREADS];
    __shared__ float stats[2][MAX_LANES];  // mean and rstd of the block's groups
    const Place at(p, k, W);
    const int64_t pitch = p.C, first = (at.n * p.S + at.row0 + at.ty) * pitch + at.channel, step = k.ty * pitch;
    const int lane = threadIdx.x & 31, parts = k.chunks * k.split;
    const float values = (float)p.S * (float)p.per_group;
    if (DO & SUMS) {
        float count = 0.0f, moved = 0.0f, squares = 0.0f;  // of the runs so far; moved: their mean, from `origin`
        float origin = 0.0f;                                // the mean of the first row: exact where all values are equal
        float centre = 0.0f, s1 = 0.0f, s2 = 0.0f;  // of the run, from `centre`
        const auto begin = [&](const DlVec<T, W>& v) {
            float f[W], sum = 0.0f;
            dl_unpack(v, f);
#pragma unroll
            for (int e = 1; e < W; ++e) sum += f[e] - f[0];
            centre = origin = f[0] + sum * (1.0f / W);
        };
        const auto end = [&](int rows) {
            const float n = (float)rows * W, all = count + n;
            const float off = __fdividef(s1, n), share = __fdividef(n, all), d = centre - origin + off - moved;
            float around = s2 - off * s1;
            around = around < 0.0f ? 0.0f : around;  // NaN stays
            squares += fmaf(count * share * d, d, around);
            moved = fmaf(d, share, moved);
            count = all;
            centre = origin + moved;
            s1 = s2 = 0.0f;
        };
        each_row<T, W>(at, step, Runs{begin, end}, [&](const DlVec<T, W>& v) {
            float f[W];
            dl_unpack(v, f);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float d = f[e] - centre;
                s1 += d;
                s2 = fmaf(d, d, s2);
            }
        }, x + first);
        red[0][threadIdx.x] = count;
        red[1][threadIdx.x] = origin + moved;
        red[2][threadIdx.x] = squares;
        __syncthreads();
        const int entries = at.group_lanes * k.ty;
        for (int g = threadIdx.x / 32; g < at.groups; g += blockDim.x / 32) {
            float mean, around;
            // the group's first thread has the first row
            join_sets(entries, red[1][g * at.group_lanes], (float)at.rows * (float)(at.group_lanes * W),
                      [&](int e, float& n, float& m, float& q) {
                          const int y = e / at.group_lanes, i = y * k.tx + g * at.group_lanes + (e - y * at.group_lanes);
                          n = red[0][i];
                          m = red[1][i];
                          q = red[2][i];
                      }, mean, around);
            if (lane != 0) continue;
            if (DO & WRITE) {  // the only part
                stats[0][g] = mean;
                stats[1][g] = around;
            } else {
                float* out = sums + ((at.n * p.G + at.group0 + g) * parts + at.part(k)) * 2;
                out[0] = mean;
                out[1] = around;
            }
        }
    }
    if (!(DO & WRITE)) return;
    float w[W], b[W];
    if (at.live) load_params<W>(p, at.channel, w, b);
    if (!(DO & SUMS)) {
        for (int g = threadIdx.x / 32; g < at.groups; g += blockDim.x / 32) {
            const float2* in = reinterpret_cast<const float2*>(sums) + (at.n * p.G + at.group0 + g) * parts;
            float mean, around;
            join_sets(parts, in[0].x, values, [&](int i, float& n, float& m, float& q) {
                const int chunk = i / k.split;
                n = (float)Place::rows_of(p, k, chunk) * (float)(Place::lanes_of(k, i - chunk * k.split) * W);
                m = in[i].x;
                q = in[i].y;
            }, mean, around);
            if (lane == 0) {
                stats[0][g] = mean;
                stats[1][g] = around;
            }
        }
    }
    __syncthreads();
    if (at.chunk == 0 && at.piece == 0 && mean_out != nullptr) {
        for (int g = threadIdx.x; g < at.groups; g += blockDim.x) {
            mean_out[at.n * p.G + at.group0 + g] = stats[0][g];
            rstd_out[at.n * p.G + at.group0 + g] = rsqrtf(stats[1][g] / values + p.eps);
        }
    }
    if (!at.live) return;
    // z = a * x + c
    const float mean = stats[0][at.group], rstd = rsqrtf(stats[1][at.group] / values + p.eps);
#pragma unroll
    for (int e = 0; e < W; ++e) {
        w[e] *= rstd;
        b[e] = fmaf(-mean, w[e], b[e]);
    }
    T* dst = y + first;
    with_activation(p.act, [&](auto act) {
        each_row<T, W>(at, step, NoRuns(), [&](const DlVec<T, W>& v) {
            float f[W];
            dl_unpack(v, f);
#pragma unroll
            for (int e = 0; e < W; ++e) f[e] = activate<T, act.value>(fmaf(f[e], w[e], b[e]));
            DlVec<T, W> out;
            dl_pack(f, out);
            *reinterpret_cast<DlVec<T, W>*>(dst) = out;
            dst += step;
        }, x + first);
    });
}

// sums (N, G, parts, 2): the parts of s1 and s2.  partial (N * chunks, 2, C): the sums of dz and dz * xh of every channel
template <typename T, int W, int DO>
__global__ void __launch_bounds__(CHUNK_THREADS, 3)
norm_chunk_bwd_kernel(const T* __restrict__ x, const T* __restrict__ gy, const float* __restrict__ mean_in,
                      const float* __restrict__ rstd_in, T* __restrict__ gx, float* __restrict__ sums,
                      float* __restrict__ partial, const __grid_constant__ Norm p, const __grid_constant__ Cut k) {
    __shared__ float red[CHUNK_THREADS * (W > 2 ? W : 2)];
    __shared__ float stats[2][MAX_LANES];  // s1 and s2 of the block's groups
    const Place at(p, k, W);
    const int64_t pitch = p.C, first = (at.n * p.S + at.row0 + at.ty) * pitch + at.channel, step = k.ty * pitch;
    const int lane = threadIdx.x & 31, parts = k.chunks * k.split;
    float w[W], b[W], rstd = 0.0f, off = 0.0f;  // xh = rstd * x + off
    if (at.live) {
        load_params<W>(p, at.channel, w, b);
        rstd = rstd_in[at.n * p.G + at.group0 + at.group];
        off = -mean_in[at.n * p.G + at.group0 + at.group] * rstd;
    }
    if (DO & SUMS) {
        float dz_sum[W], dzx_sum[W], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int e = 0; e < W; ++e) dz_sum[e] = dzx_sum[e] = 0.0f;
        if (at.live) {
            with_activation(p.act, [&](auto act) {
                each_row<T, W>(at, step, NoRuns(), [&](const DlVec<T, W>& v, const DlVec<T, W>& vg) {
                    float f[W], d[W];
                    dl_unpack(v, f);
                    dl_unpack(vg, d);
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const float xh = fmaf(f[e], rstd, off), dz = d[e] * slope<T, act.value>(fmaf(xh, w[e], b[e]));
                        dz_sum[e] += dz;
                        dzx_sum[e] = fmaf(dz, xh, dzx_sum[e]);
                    }
                }, x + first, gy + first);
            });
#pragma unroll
            for (int e = 0; e < W; ++e) {
                s1 = fmaf(dz_sum[e], w[e], s1);
                s2 = fmaf(dzx_sum[e], w[e], s2);
            }
        }
        red[threadIdx.x] = s1;
        red[CHUNK_THREADS + threadIdx.x] = s2;
        __syncthreads();
        warp_per_group(at, k, [&](int) { s1 = s2 = 0.0f; },
            [&](int, int i) {
                s1 += red[i];
                s2 += red[CHUNK_THREADS + i];
            },
            [&](int g) {
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) {
                    s1 += __shfl_xor_sync(0xffffffffu, s1, s);
                    s2 += __shfl_xor_sync(0xffffffffu, s2, s);
                }
                if (lane != 0) return;
                if (DO & WRITE) {  // the only part
                    stats[0][g] = s1;
                    stats[1][g] = s2;
                } else {
                    float* out = sums + ((at.n * p.G + at.group0 + g) * parts + at.part(k)) * 2;
                    out[0] = s1;
                    out[1] = s2;
                }
            });
        if (partial != nullptr) {  // per channel over the rows of threads
            const int channels = k.tx * W, valid = k.split > 1 ? at.group_lanes * W : at.groups * k.lanes * W;
            float* out = partial + (at.n * k.chunks + at.chunk) * 2 * pitch + (at.channel - at.tx * W);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                __syncthreads();
                if (at.ty < k.ty) {
#pragma unroll
                    for (int e = 0; e < W; ++e) red[(at.ty * k.tx + at.tx) * W + e] = v == 0 ? dz_sum[e] : dzx_sum[e];
                }
                __syncthreads();
                for (int c = threadIdx.x; c < valid; c += blockDim.x) {
                    float sum = 0.0f;
                    for (int r = 0; r < k.ty; ++r) sum += red[r * channels + c];
                    out[v * pitch + c] = sum;
                }
            }
        }
    }
    if (!(DO & WRITE)) return;
    if (!(DO & SUMS)) {
        for (int g = threadIdx.x / 32; g < at.groups; g += blockDim.x / 32) {
            const float2* in = reinterpret_cast<const float2*>(sums) + (at.n * p.G + at.group0 + g) * parts;
            float s1 = 0.0f, s2 = 0.0f;
            for (int i = lane; i < parts; i += 32) {
                s1 += in[i].x;
                s2 += in[i].y;
            }
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) {
                s1 += __shfl_xor_sync(0xffffffffu, s1, s);
                s2 += __shfl_xor_sync(0xffffffffu, s2, s);
            }
            if (lane == 0) {
                stats[0][g] = s1;
                stats[1][g] = s2;
            }
        }
    }
    __syncthreads();
    if (!at.live) return;
    // gx = rstd * w * dz - rstd * (s1 + xh * s2) / m
    const float over_m = 1.0f / ((float)p.S * (float)p.per_group);
    const float k1 = -rstd * stats[0][at.group] * over_m, k2 = -rstd * stats[1][at.group] * over_m;
    T* dst = gx + first;
    with_activation(p.act, [&](auto act) {
        each_row<T, W>(at, step, NoRuns(), [&](const DlVec<T, W>& v, const DlVec<T, W>& vg) {
            float f[W], d[W];
            dl_unpack(v, f);
            dl_unpack(vg, d);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float xh = fmaf(f[e], rstd, off), dz = d[e] * slope<T, act.value>(fmaf(xh, w[e], b[e]));
                f[e] = fmaf(dz * w[e], rstd, fmaf(xh, k2, k1));
            }
            DlVec<T, W> out;
            dl_pack(f, out);
            *reinterpret_cast<DlVec<T, W>*>(dst) = out;
            dst += step;
        }, x + first, gy + first);
    });
}

// ------------------------------------------------------------------------------------------ rows without positions
// S = 1: a group is `lanes` lanes (padded to 2^lanes_log2 <= 32) of a warp, a block covers tx lanes of ty rows.
// Vectors of four channels at most: parameters, sums and the rows in flight then fit the registers.
constexpr int ROW_THREADS = 256;
constexpr int ROW_WIDTH = 4;

struct RowCut {
    int lanes, lanes_log2;
    int tx, ty;
    int rows;          // per block
    int64_t blocks_x;  // down the rows
    int blocks_c;      // across the channels
};

template <int ITEMS>
__device__ __forceinline__ void sum_lanes(float (&v)[ITEMS], int lanes_log2) {
    for (int s = 1 << lanes_log2 >> 1; s > 0; s >>= 1) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], s);
    }
}

struct RowPlace {
    int tx, ty, group, channel, first_lane;
    int64_t row0;
    int rows;  // of the block
    bool live;
    __device__ __forceinline__ RowPlace(const Norm& p, const RowCut& k, int W) {
        tx = threadIdx.x % k.tx;
        ty = threadIdx.x / k.tx;
        const int slot = blockIdx.y * k.tx + tx, j = slot & ((1 << k.lanes_log2) - 1);
        group = slot >> k.lanes_log2;
        live = group < p.G && j < k.lanes && ty < k.ty;
        channel = group * p.per_group + j * W;
        first_lane = j == 0;
        row0 = (int64_t)blockIdx.x * k.rows;
        rows = (int)(p.N - row0 < k.rows ? p.N - row0 : k.rows);
    }
};

template <typename T, int W, int ITEMS>
__global__ void __launch_bounds__(ROW_THREADS, 4)
norm_rows_kernel(const T* __restrict__ x, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                 const __grid_constant__ Norm p, const __grid_constant__ RowCut k) {
    const RowPlace at(p, k, W);
    const T* src = x + (at.row0 + at.ty) * p.C + at.channel;
    T* dst = y + (at.row0 + at.ty) * p.C + at.channel;
    const int64_t step = (int64_t)k.ty * p.C;
    float w[W], b[W];
    const float over_m = 1.0f / (float)p.per_group;
    with_activation(p.act, [&](auto act) {
        for (int r0 = 0; r0 < at.rows; r0 += k.ty * ITEMS, src += ITEMS * step, dst += ITEMS * step) {
            DlVec<T, W> in[ITEMS];
            bool here[ITEMS];
            float mean[ITEMS], square[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                here[i] = at.live && r0 + i * k.ty + at.ty < at.rows;
                if (here[i]) in[i] = *reinterpret_cast<const DlVec<T, W>*>(src + i * step);
            }
            if (r0 == 0 && at.live) load_params<W>(p, at.channel, w, b);  // behind the first rows' loads
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                mean[i] = 0.0f;
                if (!here[i]) continue;
                float f[W];
                dl_unpack(in[i], f);
#pragma unroll
                for (int e = 0; e < W; ++e) mean[i] += f[e];
            }
            sum_lanes(mean, k.lanes_log2);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                mean[i] *= over_m;
                square[i] = 0.0f;
                if (!here[i]) continue;
                float f[W];
                dl_unpack(in[i], f);
#pragma unroll
                for (int e = 0; e < W; ++e) square[i] = fmaf(f[e] - mean[i], f[e] - mean[i], square[i]);
            }
            sum_lanes(square, k.lanes_log2);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                if (!here[i]) continue;
                const float rstd = rsqrtf(fmaf(square[i], over_m, p.eps));
                if (at.first_lane && mean_out != nullptr) {
                    const int64_t n = at.row0 + r0 + i * k.ty + at.ty;
                    mean_out[n * p.G + at.group] = mean[i];
                    rstd_out[n * p.G + at.group] = rstd;
                }
                float f[W];
                dl_unpack(in[i], f);
#pragma unroll
                for (int e = 0; e < W; ++e) f[e] = activate<T, act.value>(fmaf((f[e] - mean[i]) * rstd, w[e], b[e]));
                DlVec<T, W> out;
                dl_pack(f, out);
                *reinterpret_cast<DlVec<T, W>*>(dst + i * step) = out;
            }
        }
    });
}

template <typename T, int W, int ITEMS>
__global__ void __launch_bounds__(ROW_THREADS, 4)
norm_rows_bwd_kernel(const T* __restrict__ x, const T* __restrict__ gy, const float* __restrict__ mean_in,
                     const float* __restrict__ rstd_in, T* __restrict__ gx, float* __restrict__ partial,
                     const __grid_constant__ Norm p, const __grid_constant__ RowCut k) {
    __shared__ float red[ROW_THREADS * W];
    const RowPlace at(p, k, W);
    const int64_t first = (at.row0 + at.ty) * p.C + at.channel, step = (int64_t)k.ty * p.C;
    const T *src = x + first, *src_g = gy + first;
    T* dst = gx + first;
    const float *mean = mean_in + (at.row0 + at.ty) * p.G + at.group, *rstd = rstd_in + (at.row0 + at.ty) * p.G + at.group;
    const int64_t group_step = (int64_t)k.ty * p.G;
    float w[W], b[W], sum_dz[W], sum_dzx[W];
#pragma unroll
    for (int e = 0; e < W; ++e) sum_dz[e] = sum_dzx[e] = 0.0f;
    const float over_m = 1.0f / (float)p.per_group;
    with_activation(p.act, [&](auto act) {
        for (int r0 = 0; r0 < at.rows; r0 += k.ty * ITEMS) {
            DlVec<T, W> in[ITEMS], in_g[ITEMS];
            bool here[ITEMS];
            float mu[ITEMS], rs[ITEMS], s1[ITEMS], s2[ITEMS], xh[ITEMS][W], dzw[ITEMS][W];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                here[i] = at.live && r0 + i * k.ty + at.ty < at.rows;
                if (here[i]) {
                    in[i] = *reinterpret_cast<const DlVec<T, W>*>(src + i * step);
                    in_g[i] = *reinterpret_cast<const DlVec<T, W>*>(src_g + i * step);
                    mu[i] = mean[i * group_step];
                    rs[i] = rstd[i * group_step];
                }
            }
            if (r0 == 0 && at.live) load_params<W>(p, at.channel, w, b);  // behind the first rows' loads
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                s1[i] = s2[i] = 0.0f;
                if (!here[i]) continue;
                const float off = -mu[i] * rs[i];
                dl_unpack(in[i], xh[i]);
                dl_unpack(in_g[i], dzw[i]);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    xh[i][e] = fmaf(xh[i][e], rs[i], off);
                    const float dz = dzw[i][e] * slope<T, act.value>(fmaf(xh[i][e], w[e], b[e]));
                    sum_dz[e] += dz;
                    sum_dzx[e] = fmaf(dz, xh[i][e], sum_dzx[e]);
                    dzw[i][e] = dz * w[e];
                    s1[i] += dzw[i][e];
                    s2[i] = fmaf(dzw[i][e], xh[i][e], s2[i]);
                }
            }
            sum_lanes(s1, k.lanes_log2);
            sum_lanes(s2, k.lanes_log2);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                if (!here[i]) continue;
                const float a = s1[i] * over_m, c = s2[i] * over_m;
#pragma unroll
                for (int e = 0; e < W; ++e) xh[i][e] = rs[i] * (dzw[i][e] - fmaf(xh[i][e], c, a));
                DlVec<T, W> out;
                dl_pack(xh[i], out);
                *reinterpret_cast<DlVec<T, W>*>(dst + i * step) = out;
            }
            src += ITEMS * step;
            src_g += ITEMS * step;
            dst += ITEMS * step;
            mean += ITEMS * group_step;
            rstd += ITEMS * group_step;
        }
    });
    if (partial == nullptr) return;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        __syncthreads();
        if (at.ty < k.ty) {
#pragma unroll
            for (int e = 0; e < W; ++e) red[(at.ty * k.tx + at.tx) * W + e] = v == 0 ? sum_dz[e] : sum_dzx[e];
        }
        __syncthreads();
        if (at.live && at.ty == 0) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                float sum = 0.0f;
                for (int r = 0; r < k.ty; ++r) sum += red[(r * k.tx + at.tx) * W + e];
                partial[((int64_t)blockIdx.x * 2 + v) * p.C + at.channel + e] = sum;
            }
        }
    }
}

// gbias / gweight[c] = sum over parts of partial[part][0 / 1][c]; 8 channels (a sector) x 128 threads down the parts
constexpr int PARAM_CHANNELS = 8, PARAM_ROWS = 128;

__global__ void __launch_bounds__(PARAM_CHANNELS * PARAM_ROWS)
norm_params_kernel(const float* __restrict__ partial, int64_t parts, int C, void* gweight, void* gbias, int param_dtype) {
    __shared__ float red[2][PARAM_ROWS / 4][PARAM_CHANNELS];
    const int x = threadIdx.x % PARAM_CHANNELS, y = threadIdx.x / PARAM_CHANNELS, c = blockIdx.x * PARAM_CHANNELS + x;
    float sum[2] = {0.0f, 0.0f};
    if (c < C) {
#pragma unroll 4
        for (int64_t i = y; i < parts; i += PARAM_ROWS) {
            sum[0] += partial[(i * 2) * C + c];
            sum[1] += partial[(i * 2 + 1) * C + c];
        }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        sum[v] += __shfl_xor_sync(0xffffffffu, sum[v], 8);
        sum[v] += __shfl_xor_sync(0xffffffffu, sum[v], 16);
        if (y % 4 == 0) red[v][y / 4][x] = sum[v];  // a warp holds four rows
    }
    __syncthreads();
    if (threadIdx.x < 2 * PARAM_CHANNELS) {
        const int v = threadIdx.x / PARAM_CHANNELS;
        float total = 0.0f;
#pragma unroll
        for (int r = 0; r < PARAM_ROWS / 4; ++r) total += red[v][r][x];
        void* out = v == 0 ? gbias : gweight;
        if (c < C && out != nullptr) dl_store_from_float(out, param_dtype, c, total);
    }
}

// ------------------------------------------------------------------------------------------ host
// `resident` blocks of a launch fit an SM
Cut cut_chunks(const Norm& p, int W, int resident) {
    Cut k;
    k.lanes = p.per_group / W;
    k.split = (int)dl_ceil_div(k.lanes, MAX_LANES);
    k.groups = k.split > 1 ? 1 : (int)dl_min64(MAX_LANES / k.lanes, p.G);
    k.tx = k.split > 1 ? (int)dl_ceil_div(k.lanes, k.split) : k.groups * k.lanes;
    k.ty = (int)dl_min64(CHUNK_THREADS / k.tx, p.S);
    k.blocks_c = (int)(dl_ceil_div(p.G, k.groups) * k.split);
    // as many chunks as are resident at once, but rows enough in each to keep the loads going; a sample whose groups are split
    // over blocks of channels always takes two launches
    const int64_t units = p.N * k.blocks_c, slots = (int64_t)DL_NUM_SMS * resident;
    const int64_t most = dl_max64(p.S / ((int64_t)k.ty * 8), 1);
    k.chunks = (int)dl_max64(dl_min64(slots / dl_max64(units, 1), most), 1);
    k.rows = (int)dl_ceil_div(p.S, k.chunks);
    k.chunks = (int)dl_ceil_div(p.S, k.rows);
    return k;
}
constexpr int RESIDENT = 4, RESIDENT_BWD = 3;  // the kernels' launch bounds

unsigned threads_of(const Cut& k) { return (unsigned)(dl_ceil_div(k.tx * k.ty, 32) * 32); }
bool one_launch(const Cut& k) { return k.chunks == 1 && k.split == 1; }
int64_t sums_floats(const Norm& p, const Cut& k) {
    return one_launch(k) ? 0 : p.N * p.G * (int64_t)k.chunks * k.split * 2;
}
bool grid_fits(const Norm& p, const Cut& k) { return p.N * k.blocks_c * (int64_t)k.chunks <= 0x7fffffff; }

// W as the kernel takes it, at most ROW_WIDTH
bool cut_rows(const Norm& p, int W, int items, int64_t most_blocks, RowCut& k) {
    if (p.S != 1 || p.N == 0 || p.per_group / W > 32) return false;  // without rows there is nothing to divide by
    k.lanes = p.per_group / W;
    k.lanes_log2 = 0;
    while ((1 << k.lanes_log2) < k.lanes) ++k.lanes_log2;
    const int64_t slots = (int64_t)p.G << k.lanes_log2;
    k.tx = (int)dl_min64(slots, ROW_THREADS);
    k.ty = ROW_THREADS / k.tx;
    const int64_t across = dl_ceil_div(slots, k.tx);
    if (across > 65535) return false;
    k.blocks_c = (int)across;
    // one round of resident blocks, each with as many rows as the others
    const int64_t rows =
        dl_ceil_div(p.N, dl_min64(dl_ceil_div(p.N, (int64_t)k.ty * items), dl_max64(most_blocks / across, 1)));
    if (rows > 0x3fffffff) return false;
    k.rows = (int)rows;
    k.blocks_x = dl_ceil_div(p.N, rows);
    return true;
}

constexpr int row_width(int W) { return W < ROW_WIDTH ? W : ROW_WIDTH; }
constexpr int ROW_ITEMS = 4, ROW_ITEMS_BWD = 2;   // rows a thread loads before it uses the first
constexpr int64_t ROW_BLOCKS = DL_NUM_SMS * 4;    // resident: the kernels' launch bounds

template <typename T, int W>
int launch_forward(const void* x, void* y, float* mean, float* rstd, float* sums, const Norm& p, cudaStream_t s) {
    const T* src = static_cast<const T*>(x);
    T* dst = static_cast<T*>(y);
    RowCut r;
    if (cut_rows(p, row_width(W), ROW_ITEMS, ROW_BLOCKS, r)) {
        norm_rows_kernel<T, row_width(W), ROW_ITEMS><<<dim3((unsigned)r.blocks_x, (unsigned)r.blocks_c), ROW_THREADS, 0, s>>>(
            src, dst, mean, rstd, p, r);
        return dl_launch_status();
    }
    const Cut k = cut_chunks(p, W, RESIDENT);
    if (!grid_fits(p, k)) return DL_ERR_TOO_LARGE;
    const unsigned blocks = (unsigned)(p.N * k.blocks_c * k.chunks);
    constexpr size_t ring = Ring<1>::template bytes<DlVec<T, W>>();
    if (one_launch(k)) {
        norm_chunk_kernel<T, W, SUMS | WRITE><<<blocks, threads_of(k), ring, s>>>(src, dst, mean, rstd, sums, p, k);
        return dl_launch_status();
    }
    norm_chunk_kernel<T, W, SUMS><<<blocks, threads_of(k), ring, s>>>(src, dst, mean, rstd, sums, p, k);
    if (cudaPeekAtLastError() != cudaSuccess) return DL_ERR_LAUNCH;
    norm_chunk_kernel<T, W, WRITE><<<blocks, threads_of(k), ring, s>>>(src, dst, mean, rstd, sums, p, k);
    return dl_launch_status();
}

// floats of workspace: sums of the chunks, then the partial sums of the parameters' gradients
int64_t forward_floats(const Norm& p, int W) {
    RowCut r;
    if (cut_rows(p, row_width(W), ROW_ITEMS, ROW_BLOCKS, r)) return 0;
    return sums_floats(p, cut_chunks(p, W, RESIDENT));
}
int64_t backward_floats(const Norm& p, int W, int64_t& parts) {
    RowCut r;
    if (cut_rows(p, row_width(W), ROW_ITEMS_BWD, ROW_BLOCKS, r)) {
        parts = r.blocks_x;
        return 0;
    }
    const Cut k = cut_chunks(p, W, RESIDENT_BWD);
    parts = p.N * k.chunks;
    return sums_floats(p, k);
}

template <typename T, int W>
int launch_backward(const void* x, const void* g, const float* mean, const float* rstd, void* gx, void* gweight,
                    void* gbias, float* scratch, const Norm& p, cudaStream_t s) {
    const T *src = static_cast<const T*>(x), *src_g = static_cast<const T*>(g);
    T* dst = static_cast<T*>(gx);
    int64_t parts;
    float* partial = scratch + backward_floats(p, W, parts);
    if (gweight == nullptr && gbias == nullptr) partial = nullptr;
    RowCut r;
    if (cut_rows(p, row_width(W), ROW_ITEMS_BWD, ROW_BLOCKS, r)) {
        norm_rows_bwd_kernel<T, row_width(W), ROW_ITEMS_BWD>
            <<<dim3((unsigned)r.blocks_x, (unsigned)r.blocks_c), ROW_THREADS, 0, s>>>(src, src_g, mean, rstd, dst, partial,
                                                                                     p, r);
    } else {
        const Cut k = cut_chunks(p, W, RESIDENT_BWD);
        if (!grid_fits(p, k)) return DL_ERR_TOO_LARGE;
        const unsigned blocks = (unsigned)(p.N * k.blocks_c * k.chunks);
        constexpr size_t ring = Ring<2>::template bytes<DlVec<T, W>>();
        if (one_launch(k)) {
            norm_chunk_bwd_kernel<T, W, SUMS | WRITE><<<blocks, threads_of(k), ring, s>>>(src, src_g, mean, rstd, dst, scratch,
                                                                                      partial, p, k);
        } else {
            norm_chunk_bwd_kernel<T, W, SUMS><<<blocks, threads_of(k), ring, s>>>(src, src_g, mean, rstd, dst, scratch, partial,
                                                                              p, k);
            if (cudaPeekAtLastError() != cudaSuccess) return DL_ERR_LAUNCH;
            norm_chunk_bwd_kernel<T, W, WRITE><<<blocks, threads_of(k), ring, s>>>(src, src_g, mean, rstd, dst, scratch,
                                                                               partial, p, k);
        }
    }
    if (cudaPeekAtLastError() != cudaSuccess) return DL_ERR_LAUNCH;
    if (partial != nullptr)
        norm_params_kernel<<<(unsigned)dl_ceil_div(p.C, PARAM_CHANNELS), PARAM_CHANNELS * PARAM_ROWS, 0, s>>>(
            partial, parts, p.C, gweight, gbias, p.param_dtype);
    return dl_launch_status();
}

template <typename T>
int forward_width(const void* x, void* y, float* mean, float* rstd, float* sums, const Norm& p, cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), p.per_group, dl_address(x) | dl_address(y));
    if (w == 16 / (int)sizeof(T)) return launch_forward<T, 16 / sizeof(T)>(x, y, mean, rstd, sums, p, s);
    if (w == 4) return launch_forward<T, 4>(x, y, mean, rstd, sums, p, s);
    if (w == 2) return launch_forward<T, 2>(x, y, mean, rstd, sums, p, s);
    return launch_forward<T, 1>(x, y, mean, rstd, sums, p, s);
}

template <typename T>
int backward_width(const void* x, const void* g, const float* mean, const float* rstd, void* gx, void* gw, void* gb,
                   float* partial, const Norm& p, cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), p.per_group, dl_address(x) | dl_address(g) | dl_address(gx));
    if (w == 16 / (int)sizeof(T))
        return launch_backward<T, 16 / sizeof(T)>(x, g, mean, rstd, gx, gw, gb, partial, p, s);
    if (w == 4) return launch_backward<T, 4>(x, g, mean, rstd, gx, gw, gb, partial, p, s);
    if (w == 2) return launch_backward<T, 2>(x, g, mean, rstd, gx, gw, gb, partial, p, s);
    return launch_backward<T, 1>(x, g, mean, rstd, gx, gw, gb, partial, p, s);
}

bool describe(int64_t N, int64_t S, int64_t C, int64_t G, int64_t dtype, Norm& p) {
    if (N < 0 || S <= 0 || C <= 0 || G <= 0 || C % G != 0 || !dl_dtype_known(dtype)) return false;
    if (C > 0x3fffffff || S > 0x3fffffff) return false;
    p.weight = p.bias = nullptr;
    p.param_dtype = DL_DTYPE_F32;
    p.N = N;
    p.S = S;
    p.C = (int)C;
    p.G = (int)G;
    p.per_group = (int)(C / G);
    p.eps = 0.0f;
    p.act = 0;
    return true;
}

}  // namespace

// Addresses may rule out the wider vectors: the workspaces are large enough for every width that the sizes allow.
DL_EXPORT int64_t dl_group_norm_scratch_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int64_t dtype) {
    Norm p;
    if (!describe(N, S, C, G, dtype, p)) return -1;
    int64_t floats = 0;
    for (int w = dl_vector_width(dl_dtype_size(dtype), p.per_group, 0); w >= 1; w /= 2)
        floats = dl_max64(floats, forward_floats(p, w));
    return floats * 4;
}

DL_EXPORT int64_t dl_group_norm_bwd_scratch_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int64_t dtype) {
    Norm p;
    if (!describe(N, S, C, G, dtype, p)) return -1;
    int64_t floats = 0, parts;
    for (int w = dl_vector_width(dl_dtype_size(dtype), p.per_group, 0); w >= 1; w /= 2) {
        const int64_t sums = backward_floats(p, w, parts);
        floats = dl_max64(floats, sums + parts * 2 * C);
    }
    return floats * 4;
}

DL_EXPORT int dl_group_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                            void* scratch, int64_t N, int64_t S, int64_t C, int64_t G, int64_t dtype, int64_t param_dtype,
                            int64_t activation, float eps, dl_stream_t stream) {
    Norm p;
    DL_REQUIRE(describe(N, S, C, G, dtype, p) && dl_dtype_known(param_dtype));
    DL_REQUIRE(activation >= ACT_NONE && activation <= ACT_SIGMOID && eps >= 0.0f);
    if (N == 0) return DL_OK;
    DL_REQUIRE(x && y && (mean == nullptr) == (rstd == nullptr));
    DL_REQUIRE(scratch || dl_group_norm_scratch_bytes(N, S, C, G, dtype) == 0);
    DL_REQUIRE_ALIGNED(scratch, 16);
    DL_REQUIRE_ALIGNED(x, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(y, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(weight, dl_dtype_size(param_dtype));
    DL_REQUIRE_ALIGNED(bias, dl_dtype_size(param_dtype));
    DL_REQUIRE_ALIGNED(mean, 4);
    DL_REQUIRE_ALIGNED(rstd, 4);
    p.weight = weight;
    p.bias = bias;
    p.param_dtype = (int)param_dtype;
    p.eps = eps;
    p.act = (int)activation;
    cudaStream_t s = dl_cast(stream);
    float* sums = static_cast<float*>(scratch);
    if (dtype == DL_DTYPE_F32) return forward_width<float>(x, y, mean, rstd, sums, p, s);
    if (dtype == DL_DTYPE_BF16) return forward_width<__nv_bfloat16>(x, y, mean, rstd, sums, p, s);
    return forward_width<__half>(x, y, mean, rstd, sums, p, s);
}

DL_EXPORT int dl_group_norm_bwd(const void* x, const void* g, const void* weight, const void* bias, const float* mean,
                                const float* rstd, void* gx, void* gweight, void* gbias, void* scratch, int64_t N,
                                int64_t S, int64_t C, int64_t G, int64_t dtype, int64_t param_dtype, int64_t activation,
                                dl_stream_t stream) {
    Norm p;
    DL_REQUIRE(describe(N, S, C, G, dtype, p) && dl_dtype_known(param_dtype));
    DL_REQUIRE(activation >= ACT_NONE && activation <= ACT_SIGMOID);
    cudaStream_t s = dl_cast(stream);
    if (N == 0) {  // no samples: the parameters' gradients are zero
        const size_t bytes = (size_t)(C * dl_dtype_size(param_dtype));
        if (gweight && cudaMemsetAsync(gweight, 0, bytes, s) != cudaSuccess) return DL_ERR_LAUNCH;
        if (gbias && cudaMemsetAsync(gbias, 0, bytes, s) != cudaSuccess) return DL_ERR_LAUNCH;
        return DL_OK;
    }
    DL_REQUIRE(x && g && mean && rstd && gx && scratch);
    DL_REQUIRE_ALIGNED(x, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(g, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(gx, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(weight, dl_dtype_size(param_dtype));
    DL_REQUIRE_ALIGNED(bias, dl_dtype_size(param_dtype));
    DL_REQUIRE_ALIGNED(gweight, dl_dtype_size(param_dtype));
    DL_REQUIRE_ALIGNED(gbias, dl_dtype_size(param_dtype));
    DL_REQUIRE_ALIGNED(mean, 4);
    DL_REQUIRE_ALIGNED(rstd, 4);
    DL_REQUIRE_ALIGNED(scratch, 16);
    p.weight = weight;
    p.bias = bias;
    p.param_dtype = (int)param_dtype;
    p.act = (int)activation;
    float* partial = static_cast<float*>(scratch);
    if (dtype == DL_DTYPE_F32) return backward_width<float>(x, g, mean, rstd, gx, gweight, gbias, partial, p, s);
    if (dtype == DL_DTYPE_BF16)
        return backward_width<__nv_bfloat16>(x, g, mean, rstd, gx, gweight, gbias, partial, p, s);
    return backward_width<__half>(x, g, mean, rstd, gx, gweight, gbias, partial, p, s);
}
