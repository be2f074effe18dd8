// Group norm with an activation over channels-last data x (N, S, C), G groups of C / G channels.
//
//   xh = (x - mean) * rstd per (sample, group), z = xh * weight + bias, y = act(z)
//   dz = gy * act'(z);  gbias = sum dz;  gweight = sum dz * xh;
//   gx = rstd * (weight * dz - (s1 + xh * s2) / m),  s1 = sum weight * dz,  s2 = sum weight * dz * xh,  m = S * C / G
//
// Both directions are bound by memory, so every tensor is read once: a unit (one sample, a block of whole groups at
// least 128 bytes wide) is held in the shared memory of a thread block, or of a cluster when it is larger, while its sums
// are formed; the blocks of a cluster exchange their sums through distributed shared memory.  What does not fit is read
// twice.  Every thread keeps to its own channels (a vector of W) and to its own slots of shared memory.  Rows without
// positions (S = 1) take kernels of their own, in which a group is a few lanes of a warp and stays in registers.
// Statistics are centred sums in fp32: the mean first, then the squares around it; parts are combined by
// (count, mean, squares).  No atomics: the same bits on every run.
#include <cooperative_groups.h>

#include <type_traits>

#include "elements.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int MAX_CLUSTER = 8;
constexpr int MAX_LANES = 512;  // threads across the channels of one block

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_SIGMOID = 3 };

// e^-z.  16-bit results have no use for the last bits of the exponential.
template <typename T>
__device__ __forceinline__ float exp_minus(float z) {
    return sizeof(T) == 4 ? expf(-z) : __expf(-z);
}

template <typename T, int ACT>
__device__ __forceinline__ float activate(float z) {
    if (ACT == ACT_NONE) return z;
    if (ACT == ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    const float s = __fdividef(1.0f, 1.0f + exp_minus<T>(z));
    return ACT == ACT_SILU ? z * s : s;
}

template <typename T, int ACT>
__device__ __forceinline__ float slope(float z) {
    if (ACT == ACT_NONE) return 1.0f;
    if (ACT == ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    const float s = __fdividef(1.0f, 1.0f + exp_minus<T>(z)), rest = 1.0f - s;
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

template <typename T, int W>
__device__ __forceinline__ void copy_async(DlVec<T, W>* dst, const DlVec<T, W>* src) {
    constexpr int BYTES = (int)sizeof(T) * W;
    if constexpr (BYTES >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                     "l"(src), "n"(BYTES)
                     : "memory");
    else
        *dst = *src;
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ------------------------------------------------------------------------------------------ units in shared memory
// How the tensor is cut; a function of sizes, type and alignment.
struct Cut {
    int groups;      // per block of channels (one unit)
    int lanes;       // vectors across one group, all blocks of the cluster together
    int tx, ty;      // threads across channels and down the rows of one block
    int threads;
    int cluster;     // blocks per unit
    int by_channel;  // the cluster splits the channels of a single group instead of the rows
    int rows;        // of a unit per block
    int cached;      // of them in shared memory
    int blocks_c;    // blocks of channels
    int64_t teams;   // clusters per block of channels; each takes every teams-th sample
    size_t shared;
};

// What a thread of a unit works on.
struct Place {
    int tx, ty;
    int rank;
    int group;      // of the block, 0 .. groups - 1
    int channel;    // first of the thread's W
    bool live;
    int group_lanes;  // of a group in this block
    int row0, rows;
    __device__ __forceinline__ Place(const Norm& p, const Cut& k, int W) {
        const int lanes_here = k.by_channel ? 0 : k.groups * k.lanes;
        tx = threadIdx.x % k.tx;
        ty = threadIdx.x / k.tx;
        rank = blockIdx.x % k.cluster;
        const int block_c = (int)(blockIdx.x / k.cluster % k.blocks_c);
        const int lane = k.by_channel ? rank * k.tx + tx : tx;
        live = ty < k.ty && lane < (k.by_channel ? k.lanes : lanes_here);
        group = k.by_channel ? 0 : tx / k.lanes;
        channel = (block_c * k.groups * k.lanes + lane) * W;
        const int left = k.lanes - rank * k.tx;
        group_lanes = k.by_channel ? (left < k.tx ? (left > 0 ? left : 0) : k.tx) : k.lanes;
        row0 = k.by_channel ? 0 : rank * k.rows;
        const int64_t behind = p.S - row0;
        rows = (int)(behind < k.rows ? (behind > 0 ? behind : 0) : k.rows);
    }
};

// out[v][g] = sum of value[v] over the threads of group g; all threads call it, `red` holds 2 * threads floats
template <int NV>
__device__ __forceinline__ void sum_groups(const float (&value)[NV], const Place& at, const Cut& k, float* red, float* out) {
    __syncthreads();  // `red` and `out` may still be read from the last time
#pragma unroll
    for (int v = 0; v < NV; ++v) red[v * k.threads + threadIdx.x] = at.live ? value[v] : 0.0f;
    __syncthreads();
    const int lane = threadIdx.x & 31, warps = k.threads / 32;
    const int entries = at.group_lanes * k.ty;
    for (int g = threadIdx.x / 32; g < k.groups; g += warps) {
        float sum[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) sum[v] = 0.0f;
        for (int e = lane; e < entries; e += 32) {
            const int y = e / at.group_lanes, i = y * k.tx + g * at.group_lanes + (e - y * at.group_lanes);
#pragma unroll
            for (int v = 0; v < NV; ++v) sum[v] += red[v * k.threads + i];
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) sum[v] += __shfl_xor_sync(0xffffffffu, sum[v], s);
            if (lane == 0) out[v * k.groups + g] = sum[v];
        }
    }
    __syncthreads();
}

template <typename T, int W>
__global__ void __launch_bounds__(MAX_LANES)
norm_unit_kernel(const T* __restrict__ x, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                 const __grid_constant__ Norm p, const __grid_constant__ Cut k) {
    extern __shared__ __align__(16) unsigned char shared_bytes[];
    DlVec<T, W>* tile = reinterpret_cast<DlVec<T, W>*>(shared_bytes);
    float* red = reinterpret_cast<float*>(shared_bytes + (size_t)k.cached * k.tx * sizeof(DlVec<T, W>) / 16 * 16 + 16);
    float* sums = red + 2 * k.threads;       // [2][groups]
    float* stats = sums + 2 * k.groups;      // [2][groups] mean and rstd of the unit
    float* shared_parts = stats + 2 * k.groups;  // [2][3][groups] count, mean, squares, read by the other blocks
    cg::cluster_group cluster = cg::this_cluster();
    const Place at(p, k, W);
    float w[W], b[W];
    if (at.live) load_params<W>(p, at.channel, w, b);
    const int cached = at.rows < k.cached ? at.rows : k.cached;
    const int64_t team = blockIdx.x / k.cluster / k.blocks_c;
    const int group0 = (int)(blockIdx.x / k.cluster % k.blocks_c) * k.groups;
    const int64_t pitch = p.C;
    int parity = 0;
    for (int64_t n = team; n < p.N; n += k.teams, parity ^= 1) {
        const T* src = x + (n * p.S + at.row0) * pitch + at.channel;
        T* dst = y + (n * p.S + at.row0) * pitch + at.channel;
        float part[2] = {0.0f, 0.0f};
        if (at.live) {
            for (int r = at.ty; r < cached; r += k.ty)
                copy_async<T, W>(&tile[r * k.tx + at.tx], reinterpret_cast<const DlVec<T, W>*>(src + r * pitch));
            copy_wait_all();
            for (int r = at.ty; r < cached; r += k.ty) {
                float f[W];
                dl_unpack(tile[r * k.tx + at.tx], f);
#pragma unroll
                for (int e = 0; e < W; ++e) part[0] += f[e];
            }
        }
        {
            const float one[1] = {part[0]};
            sum_groups<1>(one, at, k, red, sums);
        }
        const float width = (float)(at.group_lanes * W);
        const float centre = cached > 0 && at.group_lanes > 0 ? sums[at.group] / ((float)cached * width) : 0.0f;
        part[0] = part[1] = 0.0f;
        if (at.live) {
            for (int r = at.ty; r < at.rows; r += k.ty) {
                float f[W];
                if (r < cached)
                    dl_unpack(tile[r * k.tx + at.tx], f);
                else
                    dl_unpack(*reinterpret_cast<const DlVec<T, W>*>(src + r * pitch), f);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float d = f[e] - centre;
                    part[0] += d;
                    part[1] += d * d;
                }
            }
        }
        float* parts = shared_parts + parity * 3 * k.groups;
        // `centre` of a group is the same in all its threads; thread g of the block still needs that of group g
        if (threadIdx.x < k.groups) parts[k.groups + threadIdx.x] = cached > 0 && at.group_lanes > 0 ? sums[threadIdx.x] / ((float)cached * width) : 0.0f;
        sum_groups<2>(part, at, k, red, sums);
        for (int g = threadIdx.x; g < k.groups; g += k.threads) {
            const float count = (float)at.rows * width, off = count > 0.0f ? sums[g] / count : 0.0f;
            parts[g] = count;
            parts[k.groups + g] += off;
            parts[2 * k.groups + g] = sums[k.groups + g] - off * sums[g];
        }
        if (k.cluster > 1) cluster.sync();
        else __syncthreads();
        for (int g = threadIdx.x; g < k.groups; g += k.threads) {
            float count = 0.0f, mean = 0.0f, squares = 0.0f;
            for (int r = 0; r < k.cluster; ++r) {
                const float* other = k.cluster > 1 ? cluster.map_shared_rank(parts, r) : parts;
                const float c = other[g], m = other[k.groups + g], q = other[2 * k.groups + g];
                if (c == 0.0f) continue;
                const float both = count + c, d = m - mean;
                mean += d * (c / both);
                squares += q + d * d * (count * (c / both));
                count = both;
            }
            const float rstd = rsqrtf((squares < 0.0f ? 0.0f : squares / count) + p.eps);
            stats[g] = mean;
            stats[k.groups + g] = rstd;
            if (at.rank == 0 && mean_out != nullptr) {
                mean_out[n * p.G + group0 + g] = mean;
                rstd_out[n * p.G + group0 + g] = rstd;
            }
        }
        __syncthreads();
        if (at.live) {
            // z = a * x + c
            const float mean = stats[at.group], rstd = stats[k.groups + at.group];
            float a[W], c[W];
#pragma unroll
            for (int e = 0; e < W; ++e) {
                a[e] = rstd * w[e];
                c[e] = fmaf(-mean, a[e], b[e]);
            }
            with_activation(p.act, [&](auto act) {
                for (int r = at.ty; r < at.rows; r += k.ty) {
                    float f[W];
                    if (r < cached)
                        dl_unpack(tile[r * k.tx + at.tx], f);
                    else
                        dl_unpack(*reinterpret_cast<const DlVec<T, W>*>(src + r * pitch), f);
#pragma unroll
                    for (int e = 0; e < W; ++e) f[e] = activate<T, act.value>(fmaf(f[e], a[e], c[e]));
                    DlVec<T, W> out;
                    dl_pack(f, out);
                    *reinterpret_cast<DlVec<T, W>*>(dst + r * pitch) = out;
                }
            });
        }
    }
    if (k.cluster > 1) cluster.sync();  // nobody leaves while others read its sums
}

// partial (parts, 2, C): per team and row slice the sums of dz and dz * xh of every channel
template <typename T, int W>
__global__ void __launch_bounds__(MAX_LANES)
norm_unit_bwd_kernel(const T* __restrict__ x, const T* __restrict__ gy, const float* __restrict__ mean_in,
                     const float* __restrict__ rstd_in, T* __restrict__ gx, float* __restrict__ partial,
                     const __grid_constant__ Norm p, const __grid_constant__ Cut k) {
    extern __shared__ __align__(16) unsigned char shared_bytes[];
    DlVec<T, W>* tile = reinterpret_cast<DlVec<T, W>*>(shared_bytes);
    DlVec<T, W>* tile_g = tile + (size_t)k.cached * k.tx;
    float* red = reinterpret_cast<float*>(shared_bytes + (size_t)2 * k.cached * k.tx * sizeof(DlVec<T, W>) / 16 * 16 + 16);
    float* sums = red + (size_t)k.threads * (W > 2 ? W : 2);  // [2][groups]
    float* shared_sums = sums + 2 * k.groups;                 // [2][2][groups], read by the other blocks
    cg::cluster_group cluster = cg::this_cluster();
    const Place at(p, k, W);
    float w[W], b[W], sum_dz[W], sum_dzx[W];
    if (at.live) load_params<W>(p, at.channel, w, b);
#pragma unroll
    for (int e = 0; e < W; ++e) sum_dz[e] = sum_dzx[e] = 0.0f;
    const int cached = at.rows < k.cached ? at.rows : k.cached;
    const int64_t team = blockIdx.x / k.cluster / k.blocks_c;
    const int group0 = (int)(blockIdx.x / k.cluster % k.blocks_c) * k.groups;
    const int64_t pitch = p.C;
    const float over_m = 1.0f / ((float)p.S * (float)p.per_group);
    int parity = 0;
    for (int64_t n = team; n < p.N; n += k.teams, parity ^= 1) {
        const int64_t from = (n * p.S + at.row0) * pitch + at.channel;
        const T *src = x + from, *src_g = gy + from;
        float part[2] = {0.0f, 0.0f}, rstd = 0.0f, off = 0.0f;  // xh = rstd * x + off
        if (at.live) {
            for (int r = at.ty; r < cached; r += k.ty) {
                copy_async<T, W>(&tile[r * k.tx + at.tx], reinterpret_cast<const DlVec<T, W>*>(src + r * pitch));
                copy_async<T, W>(&tile_g[r * k.tx + at.tx], reinterpret_cast<const DlVec<T, W>*>(src_g + r * pitch));
            }
            rstd = rstd_in[n * p.G + group0 + at.group];
            off = -mean_in[n * p.G + group0 + at.group] * rstd;
            float unit_dz[W], unit_dzx[W];
#pragma unroll
            for (int e = 0; e < W; ++e) unit_dz[e] = unit_dzx[e] = 0.0f;
            copy_wait_all();
            with_activation(p.act, [&](auto act) {
                for (int r = at.ty; r < at.rows; r += k.ty) {
                    float f[W], d[W];
                    if (r < cached) {
                        dl_unpack(tile[r * k.tx + at.tx], f);
                        dl_unpack(tile_g[r * k.tx + at.tx], d);
                    } else {
                        dl_unpack(*reinterpret_cast<const DlVec<T, W>*>(src + r * pitch), f);
                        dl_unpack(*reinterpret_cast<const DlVec<T, W>*>(src_g + r * pitch), d);
                    }
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const float xh = fmaf(f[e], rstd, off), dz = d[e] * slope<T, act.value>(fmaf(xh, w[e], b[e]));
                        unit_dz[e] += dz;
                        unit_dzx[e] = fmaf(dz, xh, unit_dzx[e]);
                    }
                }
            });
#pragma unroll
            for (int e = 0; e < W; ++e) {
                part[0] = fmaf(unit_dz[e], w[e], part[0]);
                part[1] = fmaf(unit_dzx[e], w[e], part[1]);
                sum_dz[e] += unit_dz[e];
                sum_dzx[e] += unit_dzx[e];
            }
        }
        float* mine = k.cluster > 1 ? shared_sums + parity * 2 * k.groups : sums;
        sum_groups<2>(part, at, k, red, mine);
        float s1 = 0.0f, s2 = 0.0f;
        if (k.cluster > 1) {
            cluster.sync();
            for (int r = 0; r < k.cluster; ++r) {
                const float* other = cluster.map_shared_rank(mine, r);
                s1 += other[at.group < k.groups ? at.group : 0];
                s2 += other[k.groups + (at.group < k.groups ? at.group : 0)];
            }
        } else if (at.live) {
            s1 = mine[at.group];
            s2 = mine[k.groups + at.group];
        }
        if (at.live) {
            // gx = rstd * w * dz - rstd * (s1 + xh * s2)
            const float k1 = -rstd * s1 * over_m, k2 = -rstd * s2 * over_m;
            float rw[W];
#pragma unroll
            for (int e = 0; e < W; ++e) rw[e] = rstd * w[e];
            T* dst = gx + from;
            with_activation(p.act, [&](auto act) {
                for (int r = at.ty; r < at.rows; r += k.ty) {
                    float f[W], d[W];
                    if (r < cached) {
                        dl_unpack(tile[r * k.tx + at.tx], f);
                        dl_unpack(tile_g[r * k.tx + at.tx], d);
                    } else {
                        dl_unpack(*reinterpret_cast<const DlVec<T, W>*>(src + r * pitch), f);
                        dl_unpack(*reinterpret_cast<const DlVec<T, W>*>(src_g + r * pitch), d);
                    }
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const float xh = fmaf(f[e], rstd, off), dz = d[e] * slope<T, act.value>(fmaf(xh, w[e], b[e]));
                        f[e] = fmaf(dz, rw[e], fmaf(xh, k2, k1));
                    }
                    DlVec<T, W> out;
                    dl_pack(f, out);
                    *reinterpret_cast<DlVec<T, W>*>(dst + r * pitch) = out;
                }
            });
        }
    }
    if (k.cluster > 1) cluster.sync();  // nobody leaves while others read its sums
    if (partial == nullptr) return;
    // per channel over the rows of threads
    const int channels = k.tx * W;
    const int64_t slice = k.by_channel ? team : team * k.cluster + at.rank;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        __syncthreads();
        if (at.live) {
#pragma unroll
            for (int e = 0; e < W; ++e) red[(at.ty * k.tx + at.tx) * W + e] = v == 0 ? sum_dz[e] : sum_dzx[e];
        }
        __syncthreads();
        const int first = (int)(blockIdx.x / k.cluster % k.blocks_c) * k.groups * k.lanes * W +
                          (k.by_channel ? at.rank * channels : 0);
        const int valid = k.by_channel ? at.group_lanes * W : channels;
        for (int c = threadIdx.x; c < valid; c += k.threads) {
            float sum = 0.0f;
            for (int r = 0; r < k.ty; ++r) sum += red[r * channels + c];
            partial[(slice * 2 + v) * p.C + first + c] = sum;
        }
    }
}

// ------------------------------------------------------------------------------------------ rows without positions
// S = 1: a group is `lanes` lanes (padded to 2^lanes_log2 <= 32) of a warp, a block covers tx lanes of ty rows.
struct RowCut {
    int lanes, lanes_log2;
    int tx, ty;
    int64_t blocks_x;  // down the rows
    int blocks_c;      // across the channels
};

__device__ __forceinline__ float sum_lanes(float v, int lanes_log2) {
    for (int s = 1 << lanes_log2 >> 1; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}

constexpr int ROW_THREADS = 256;

template <typename T, int W, int ITEMS>
__global__ void __launch_bounds__(ROW_THREADS)
norm_rows_kernel(const T* __restrict__ x, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                 const __grid_constant__ Norm p, const __grid_constant__ RowCut k) {
    const int slot = blockIdx.y * k.tx + threadIdx.x % k.tx, ty = threadIdx.x / k.tx;
    const int group = slot >> k.lanes_log2, j = slot & ((1 << k.lanes_log2) - 1);
    const bool live = group < p.G && j < k.lanes && ty < k.ty;
    const int channel = group * p.per_group + j * W;
    float w[W], b[W];
    bool first = true;
    const float over_m = 1.0f / (float)p.per_group;
    with_activation(p.act, [&](auto act) {
    for (int64_t n0 = (int64_t)blockIdx.x * k.ty * ITEMS; n0 < p.N; n0 += (int64_t)gridDim.x * k.ty * ITEMS) {
        DlVec<T, W> in[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t n = n0 + i * k.ty + ty;
            if (live && n < p.N) in[i] = *reinterpret_cast<const DlVec<T, W>*>(x + n * p.C + channel);
        }
        if (first && live) load_params<W>(p, channel, w, b);  // behind the first rows' loads
        first = false;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t n = n0 + i * k.ty + ty;
            const bool here = live && n < p.N;
            float f[W], sum = 0.0f, squares = 0.0f;
            if (here) {
                dl_unpack(in[i], f);
#pragma unroll
                for (int e = 0; e < W; ++e) sum += f[e];
            }
            const float mean = sum_lanes(sum, k.lanes_log2) * over_m;
            if (here) {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    f[e] -= mean;
                    squares = fmaf(f[e], f[e], squares);
                }
            }
            const float rstd = rsqrtf(sum_lanes(squares, k.lanes_log2) * over_m + p.eps);
            if (!here) continue;
            if (j == 0 && mean_out != nullptr) {
                mean_out[n * p.G + group] = mean;
                rstd_out[n * p.G + group] = rstd;
            }
#pragma unroll
            for (int e = 0; e < W; ++e) f[e] = activate<T, act.value>(fmaf(f[e] * rstd, w[e], b[e]));
            DlVec<T, W> out;
            dl_pack(f, out);
            *reinterpret_cast<DlVec<T, W>*>(y + n * p.C + channel) = out;
        }
    }
    });
}

template <typename T, int W, int ITEMS>
__global__ void __launch_bounds__(ROW_THREADS)
norm_rows_bwd_kernel(const T* __restrict__ x, const T* __restrict__ gy, const float* __restrict__ mean_in,
                     const float* __restrict__ rstd_in, T* __restrict__ gx, float* __restrict__ partial,
                     const __grid_constant__ Norm p, const __grid_constant__ RowCut k) {
    __shared__ float red[ROW_THREADS * W];
    const int tx = threadIdx.x % k.tx, slot = blockIdx.y * k.tx + tx, ty = threadIdx.x / k.tx;
    const int group = slot >> k.lanes_log2, j = slot & ((1 << k.lanes_log2) - 1);
    const bool live = group < p.G && j < k.lanes && ty < k.ty;
    const int channel = group * p.per_group + j * W;
    float w[W], b[W], sum_dz[W], sum_dzx[W];
    bool first = true;
#pragma unroll
    for (int e = 0; e < W; ++e) sum_dz[e] = sum_dzx[e] = 0.0f;
    const float over_m = 1.0f / (float)p.per_group;
    with_activation(p.act, [&](auto act) {
    for (int64_t n0 = (int64_t)blockIdx.x * k.ty * ITEMS; n0 < p.N; n0 += (int64_t)gridDim.x * k.ty * ITEMS) {
        DlVec<T, W> in[ITEMS], in_g[ITEMS];
        float mean[ITEMS], rstd[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t n = n0 + i * k.ty + ty;
            if (live && n < p.N) {
                in[i] = *reinterpret_cast<const DlVec<T, W>*>(x + n * p.C + channel);
                in_g[i] = *reinterpret_cast<const DlVec<T, W>*>(gy + n * p.C + channel);
                mean[i] = mean_in[n * p.G + group];
                rstd[i] = rstd_in[n * p.G + group];
            }
        }
        if (first && live) load_params<W>(p, channel, w, b);  // behind the first rows' loads
        first = false;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int64_t n = n0 + i * k.ty + ty;
            const bool here = live && n < p.N;
            float xh[W], dzw[W], s1 = 0.0f, s2 = 0.0f;
            if (here) {
                const float off = -mean[i] * rstd[i];
                dl_unpack(in[i], xh);
                dl_unpack(in_g[i], dzw);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    xh[e] = fmaf(xh[e], rstd[i], off);
                    const float dz = dzw[e] * slope<T, act.value>(fmaf(xh[e], w[e], b[e]));
                    sum_dz[e] += dz;
                    sum_dzx[e] = fmaf(dz, xh[e], sum_dzx[e]);
                    dzw[e] = dz * w[e];
                    s1 += dzw[e];
                    s2 = fmaf(dzw[e], xh[e], s2);
                }
            }
            s1 = sum_lanes(s1, k.lanes_log2) * over_m;
            s2 = sum_lanes(s2, k.lanes_log2) * over_m;
            if (!here) continue;
#pragma unroll
            for (int e = 0; e < W; ++e) xh[e] = rstd[i] * (dzw[e] - fmaf(xh[e], s2, s1));
            DlVec<T, W> out;
            dl_pack(xh, out);
            *reinterpret_cast<DlVec<T, W>*>(gx + n * p.C + channel) = out;
        }
    }
    });
    if (partial == nullptr) return;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        __syncthreads();
        if (ty < k.ty) {
#pragma unroll
            for (int e = 0; e < W; ++e) red[(ty * k.tx + tx) * W + e] = v == 0 ? sum_dz[e] : sum_dzx[e];
        }
        __syncthreads();
        if (live && ty == 0) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                float sum = 0.0f;
                for (int r = 0; r < k.ty; ++r) sum += red[(r * k.tx + tx) * W + e];
                partial[((int64_t)blockIdx.x * 2 + v) * p.C + channel + e] = sum;
            }
        }
    }
}

// gbias / gweight[c] = sum over parts of partial[part][0 / 1][c]; 32 channels x 32 threads down the parts per block
__global__ void __launch_bounds__(1024)
norm_params_kernel(const float* __restrict__ partial, int64_t parts, int C, void* gweight, void* gbias, int param_dtype) {
    __shared__ float red[2][32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
    float sum[2] = {0.0f, 0.0f};
    if (c < C) {
#pragma unroll 4
        for (int64_t i = y; i < parts; i += 32) {
            sum[0] += partial[(i * 2) * C + c];
            sum[1] += partial[(i * 2 + 1) * C + c];
        }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) red[v][y][threadIdx.x & 31] = sum[v];
    __syncthreads();
    if (y < 2) {  // warp 0: bias, warp 1: weight
        float total = 0.0f;
        for (int r = 0; r < 32; ++r) total += red[y][r][threadIdx.x & 31];
        void* out = y == 0 ? gbias : gweight;
        if (c < C && out != nullptr) dl_store_from_float(out, param_dtype, c, total);
    }
}

// ------------------------------------------------------------------------------------------ host
constexpr size_t SHARED_MOST = 227 * 1024;    // of a block
constexpr size_t SHARED_LIMIT = 190 * 1024;   // of these for tiles
constexpr size_t SHARED_WANTED = 64 * 1024;   // so that about three blocks share an SM and overlap their phases

// false: the groups are too wide.  `tensors` are held at once (1 forward, 2 backward).
bool cut_units(const Norm& p, int W, int64_t esize, int tensors, bool accumulate, Cut& k) {
    k.lanes = p.per_group / W;
    k.cluster = 1;
    k.by_channel = k.lanes > MAX_LANES;
    if (k.by_channel) {
        while (k.cluster < MAX_CLUSTER && dl_ceil_div(k.lanes, k.cluster) > MAX_LANES) k.cluster *= 2;
        if (dl_ceil_div(k.lanes, k.cluster) > MAX_LANES) return false;
        k.groups = 1;
        k.tx = (int)dl_ceil_div(k.lanes, k.cluster);
    } else {
        // the fewest groups that are 128 bytes wide together; 64 or 32 when the unit would not fit a cluster at the
        // wanted size, or when there would be too few units for the SMs
        for (int64_t width = 128; width >= 32; width /= 2) {
            k.groups = 1;
            while (k.groups < p.G && (p.G % k.groups != 0 || (int64_t)k.groups * p.per_group * esize < width)) ++k.groups;
            const int64_t unit = p.S * k.groups * p.per_group * esize * tensors;
            if (unit <= (int64_t)SHARED_WANTED * MAX_CLUSTER && p.N * (p.G / k.groups) * MAX_CLUSTER >= DL_NUM_SMS) break;
        }
        // all groups of a block need a lane each; wide groups of one-element vectors may not fit
        while (k.groups * k.lanes > MAX_LANES) {
            --k.groups;
            while (p.G % k.groups != 0) --k.groups;
        }
        k.tx = k.groups * k.lanes;
    }
    k.blocks_c = p.G / k.groups;
    const int64_t row_bytes = (int64_t)k.tx * W * esize * tensors;
    const int most_threads = k.tx > 256 ? MAX_LANES : 256;
    if (!k.by_channel) {
        // a cluster when the unit is large, or when there are too few units for all SMs
        const int64_t units = p.N * k.blocks_c;
        while (k.cluster < MAX_CLUSTER && p.S >= 16 * k.cluster &&
               (p.S * row_bytes > (int64_t)SHARED_WANTED * k.cluster ||
                (units * k.cluster < 2 * DL_NUM_SMS && p.S * k.tx > 2 * (int64_t)most_threads * k.cluster)))
            k.cluster *= 2;
    }
    const int64_t rows = k.by_channel ? p.S : dl_ceil_div(p.S, k.cluster);
    if (rows > 0x7fffffff / 2) return false;
    k.rows = (int)rows;
    k.cached = (int)dl_min64(rows, dl_max64((int64_t)SHARED_LIMIT / row_bytes, 1));
    k.ty = (int)dl_max64(dl_min64(rows, most_threads / k.tx), 1);
    k.threads = (int)dl_ceil_div(k.tx * k.ty, 32) * 32;
    // tiles (rounded up), sums of threads (of channels at the end of the backward pass), and a few floats per group
    k.shared = (size_t)(k.cached * row_bytes + 32) + (size_t)k.threads * 4 * (accumulate && W > 2 ? W : 2) +
               (size_t)k.groups * 4 * 10;
    k.teams = p.N;
    if (accumulate) {
        // as many clusters as are resident at once, each with the same number of samples, give or take one
        const int64_t resident = dl_max64(dl_min64((int64_t)(220 * 1024 / (k.shared + 1024)), 1024 / k.threads), 1);
        const int64_t at_once = dl_max64(DL_NUM_SMS * resident / ((int64_t)k.blocks_c * k.cluster), 1);
        k.teams = dl_ceil_div(p.N, dl_ceil_div(p.N, at_once));
    }
    return true;
}

bool cut_rows(const Norm& p, int W, int items, int64_t most_blocks, RowCut& k) {
    if (p.S != 1 || p.per_group / W > 32) return false;
    k.lanes = p.per_group / W;
    k.lanes_log2 = 0;
    while ((1 << k.lanes_log2) < k.lanes) ++k.lanes_log2;
    const int64_t slots = (int64_t)p.G << k.lanes_log2;
    k.tx = (int)dl_min64(slots, ROW_THREADS);
    k.ty = ROW_THREADS / k.tx;
    const int64_t across = dl_ceil_div(slots, k.tx);
    if (across > 65535) return false;
    k.blocks_c = (int)across;
    k.blocks_x = dl_min64(dl_ceil_div(p.N, (int64_t)k.ty * items), dl_max64(most_blocks / across, 1));
    return true;
}

constexpr int ROW_ITEMS = 4, ROW_ITEMS_BWD = 2;
constexpr int64_t ROW_BLOCKS = DL_NUM_SMS * 16, ROW_BLOCKS_BWD = DL_NUM_SMS * 4;

void unit_config(const Cut& k, cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, cudaStream_t s) {
    cfg.gridDim = dim3((unsigned)(k.teams * k.blocks_c * k.cluster));
    cfg.blockDim = dim3((unsigned)k.threads);
    cfg.dynamicSmemBytes = k.shared;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)k.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
}

template <typename T, int W>
int launch_forward(const void* x, void* y, float* mean, float* rstd, const Norm& p, cudaStream_t s) {
    const T* src = static_cast<const T*>(x);
    T* dst = static_cast<T*>(y);
    RowCut r;
    if (cut_rows(p, W, ROW_ITEMS, ROW_BLOCKS, r)) {
        norm_rows_kernel<T, W, ROW_ITEMS><<<dim3((unsigned)r.blocks_x, (unsigned)r.blocks_c), ROW_THREADS, 0, s>>>(
            src, dst, mean, rstd, p, r);
        return dl_launch_status();
    }
    Cut k;
    if (!cut_units(p, W, sizeof(T), 1, false, k)) return DL_ERR_TOO_LARGE;
    if (k.teams * k.blocks_c * k.cluster > 0x7fffffff) return DL_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const auto kernel = norm_unit_kernel<T, W>;
    static DlKernelLimits limits;
    if (!dl_allow(reinterpret_cast<const void*>(kernel), limits, SHARED_MOST, false)) return DL_ERR_LAUNCH;
    unit_config(k, cfg, attr, s);
    return cudaLaunchKernelEx(&cfg, kernel, src, dst, mean, rstd, p, k) == cudaSuccess ? dl_launch_status()
                                                                                      : DL_ERR_LAUNCH;
}

// rows of `partial` that the backward pass with vectors of W writes; 0: not supported
int64_t backward_parts(const Norm& p, int W, int64_t esize) {
    RowCut r;
    if (cut_rows(p, W, ROW_ITEMS_BWD, ROW_BLOCKS_BWD, r)) return r.blocks_x;
    Cut k;
    if (!cut_units(p, W, esize, 2, true, k)) return 0;
    return k.by_channel ? k.teams : k.teams * k.cluster;
}

template <typename T, int W>
int launch_backward(const void* x, const void* g, const float* mean, const float* rstd, void* gx, void* gweight,
                    void* gbias, float* partial, const Norm& p, cudaStream_t s) {
    const T *src = static_cast<const T*>(x), *src_g = static_cast<const T*>(g);
    T* dst = static_cast<T*>(gx);
    if (gweight == nullptr && gbias == nullptr) partial = nullptr;
    RowCut r;
    if (cut_rows(p, W, ROW_ITEMS_BWD, ROW_BLOCKS_BWD, r)) {
        norm_rows_bwd_kernel<T, W, ROW_ITEMS_BWD>
            <<<dim3((unsigned)r.blocks_x, (unsigned)r.blocks_c), ROW_THREADS, 0, s>>>(src, src_g, mean, rstd, dst, partial,
                                                                                     p, r);
        if (cudaPeekAtLastError() != cudaSuccess) return DL_ERR_LAUNCH;
    } else {
        Cut k;
        if (!cut_units(p, W, sizeof(T), 2, true, k)) return DL_ERR_TOO_LARGE;
        if (k.teams * k.blocks_c * k.cluster > 0x7fffffff) return DL_ERR_TOO_LARGE;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        const auto kernel = norm_unit_bwd_kernel<T, W>;
        static DlKernelLimits limits;
        if (!dl_allow(reinterpret_cast<const void*>(kernel), limits, SHARED_MOST, false)) return DL_ERR_LAUNCH;
        unit_config(k, cfg, attr, s);
        if (cudaLaunchKernelEx(&cfg, kernel, src, src_g, mean, rstd, dst, partial, p, k) != cudaSuccess)
            return DL_ERR_LAUNCH;
    }
    if (partial != nullptr)
        norm_params_kernel<<<(unsigned)dl_ceil_div(p.C, 32), 1024, 0, s>>>(partial, backward_parts(p, W, sizeof(T)), p.C,
                                                                         gweight, gbias, p.param_dtype);
    return dl_launch_status();
}

template <typename T>
int forward_width(const void* x, void* y, float* mean, float* rstd, const Norm& p, cudaStream_t s) {
    const int w = dl_vector_width(sizeof(T), p.per_group, dl_address(x) | dl_address(y));
    if (w == 16 / (int)sizeof(T)) return launch_forward<T, 16 / sizeof(T)>(x, y, mean, rstd, p, s);
    if (w == 4) return launch_forward<T, 4>(x, y, mean, rstd, p, s);
    if (w == 2) return launch_forward<T, 2>(x, y, mean, rstd, p, s);
    return launch_forward<T, 1>(x, y, mean, rstd, p, s);
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

DL_EXPORT int64_t dl_group_norm_bwd_scratch_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int64_t dtype) {
    Norm p;
    if (!describe(N, S, C, G, dtype, p)) return 0;
    if (N == 0) return 256;
    // the widest partial table of the vector widths that these sizes allow: addresses may rule out the wider ones
    int64_t parts = 0;
    for (int w = dl_vector_width(dl_dtype_size(dtype), p.per_group, 0); w >= 1; w /= 2)
        parts = dl_max64(parts, backward_parts(p, w, dl_dtype_size(dtype)));
    return parts * 2 * C * 4;
}

DL_EXPORT int dl_group_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                            int64_t N, int64_t S, int64_t C, int64_t G, int64_t dtype, int64_t param_dtype,
                            int64_t activation, float eps, dl_stream_t stream) {
    Norm p;
    DL_REQUIRE(describe(N, S, C, G, dtype, p) && dl_dtype_known(param_dtype));
    DL_REQUIRE(activation >= ACT_NONE && activation <= ACT_SIGMOID && eps >= 0.0f);
    if (N == 0) return DL_OK;
    DL_REQUIRE(x && y && (mean == nullptr) == (rstd == nullptr));
    DL_REQUIRE_ALIGNED(x, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(y, dl_dtype_size(dtype));
    p.weight = weight;
    p.bias = bias;
    p.param_dtype = (int)param_dtype;
    p.eps = eps;
    p.act = (int)activation;
    cudaStream_t s = dl_cast(stream);
    if (dtype == DL_DTYPE_F32) return forward_width<float>(x, y, mean, rstd, p, s);
    if (dtype == DL_DTYPE_BF16) return forward_width<__nv_bfloat16>(x, y, mean, rstd, p, s);
    return forward_width<__half>(x, y, mean, rstd, p, s);
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
    DL_REQUIRE(x && g && mean && rstd && gx && (scratch || (!gweight && !gbias)));
    DL_REQUIRE_ALIGNED(x, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(g, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(gx, dl_dtype_size(dtype));
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
