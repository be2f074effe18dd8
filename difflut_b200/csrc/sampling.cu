// Sampling a class per row of logits with temperature, top-k, top-p and min-p from given random numbers.
//
//   w_i = exp((l_i - max) / T);  top-k keeps the k largest (equal logits: lowest index first);  top-p keeps, of those in
//   descending order, the ones with less than p * (their total) before them;  min-p keeps w_i >= min_p;
//   the class is the first i, in ascending order, whose running sum of kept weights exceeds u * (total kept weight).
//
// Both cuts are one question: down to which (logit, index) does a running sum, of ones or of weights, stay below a
// target?  It is answered without sorting: a histogram over (max - l) / T in 2048 steps of 1/32 finds the step in which
// the target falls, and the few logits of that step are ranked among themselves by counting (or, when very many share the
// step, by histograms over the bits of their keys and, for equal ones, over their index).
//
// A class next to a border must not depend on the order of additions, so weights are whole numbers: exp in double
// precision, as fixed point with up to 50 fractional bits, chosen so that the sum of a row fits 62 bits.  Integer sums are
// exact in any order, so shared-memory atomics are harmless here.
//
// Rows of up to 512 classes take one warp and registers; longer ones a block of 512 threads, or a cluster of up to
// eight when there are few rows.  Each pass reads the logits again: after the first they come from L2.
#include <cooperative_groups.h>

#include "elements.cuh"

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int BINS = 2048;
constexpr int LIST = 512;  // most logits ranked by counting
constexpr int MAX_CLUSTER = 8;
constexpr int SMALL_V = 512;
constexpr int TABLE = 128;
constexpr uint32_t FULL = 0xffffffffu;

struct Settings {
    const float* temperature;  // per row; null: the scalar
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
};

struct Job {
    const void* u;
    int u_double;
    int64_t* out;
    int64_t R, V, pitch;
    int shift;  // weights have this many fractional bits
    Settings set;
};

// what one row asks for
struct Rule {
    double inverse_T, top_p, u;
    int64_t top_k;  // 0: off
    u64 least;      // min-p as a weight
    bool greedy;
    __device__ __forceinline__ Rule(const Job& j, int64_t r) {
        const double T = j.set.temperature ? (double)j.set.temperature[r] : j.set.temperature_all;
        inverse_T = 1.0 / T;
        greedy = !(T > 0.0) || inverse_T == INFINITY;
        const int64_t k = j.set.top_k ? (int64_t)j.set.top_k[r] : j.set.top_k_all;
        top_k = k > 0 && k < j.V ? k : 0;
        top_p = j.set.top_p ? (double)j.set.top_p[r] : j.set.top_p_all;
        double m = j.set.min_p ? (double)j.set.min_p[r] : j.set.min_p_all;
        m = m > 0.0 ? (m < 1.0 ? m : 1.0) : 0.0;
        least = (u64)ceil(m * (double)(1ull << j.shift));
        u = j.u_double ? static_cast<const double*>(j.u)[r] : (double)static_cast<const float*>(j.u)[r];
    }
};

// Ordered key of a logit: larger logits have larger keys, both zeros the same one; 0 for NaN and -inf, which are never
// taken.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return l > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp(-(top - l) / T) as fixed point.  With j = round(128 z / ln 2) and r = z - j ln 2 / 128, |r| < 0.0028,
// e^-z = 2^(-j / 128) e^-r: a table for the fraction of the power, four terms of the series for e^-r (the fifth is below
// 2^-49), the whole part of the power as an exponent.
struct Weigher {
    const double* table;  // 2^(shift - i / 128)
    double top, inverse_T, most_z;
    bool infinite;        // the largest logit is +inf
    u64 one;
    __device__ __forceinline__ Weigher(const double* table, uint32_t top_key, double inverse_T, int shift)
        : table(table), inverse_T(inverse_T) {
        const float t = logit_of(top_key);
        infinite = t == INFINITY;
        top = infinite ? 0.0 : (double)t;
        most_z = 0.6931471805599453 * (shift + 2);  // less than a quarter of the last bit from here on
        one = 1ull << shift;
    }
    __device__ __forceinline__ u64 operator()(uint32_t key) const {
        const float l = logit_of(key);
        if (infinite) return l == INFINITY ? one : 0ull;
        const double z = (top - (double)l) * inverse_T;
        if (!(z < most_z)) return 0ull;
        const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
        const double shifted = fma(z, 184.6649652337873, magic);
        const int j = __double2loint(shifted);
        const double r = fma(shifted - magic, -0.0054152123481245725, z);
        const double e = fma(fma(fma(fma(r, 1.0 / 24, -1.0 / 6), r, 0.5), r, -1.0), r, 1.0);
        double w = table[j & (TABLE - 1)] * e;
        w = __hiloint2double(__double2hiint(w) - ((j >> 7) << 20), __double2loint(w));
        return (u64)__double_as_longlong(w + 4503599627370496.0) - 0x4330000000000000ull;  // w < 2^52, rounded
    }
};

__device__ __forceinline__ void fill_table(double* table, int shift, int tid, int threads) {
    for (int i = tid; i < TABLE; i += threads) table[i] = exp2((double)shift - (double)i / TABLE);
}

// p * total rounded up: "before < p * total" for whole numbers
__device__ __forceinline__ u64 share_of(double p, u64 total) {
    const double t = ceil(p * (double)total);
    return t >= (double)total ? total : (t > 1.0 ? (u64)t : 1ull);
}
// the running sum must exceed this: floor(u * total), below total
__device__ __forceinline__ u64 point_of(double u, u64 total) {
    const double t = floor(u * (double)total);
    if (!(t > 0.0)) return 0ull;
    return t >= (double)total ? total - 1 : (u64)t;
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(FULL, v, s);
    return v;
}
__device__ __forceinline__ u64 warp_inclusive(u64 v, int lane) {
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const u64 o = __shfl_up_sync(FULL, v, s);
        if (lane >= s) v += o;
    }
    return v;
}

// ------------------------------------------------------------------------------------------ one warp per row
// Element j * 32 + lane sits in register j: index order is register, then lane.
template <typename T, int PER>
__global__ void __launch_bounds__(128)
sample_small_kernel(const T* __restrict__ logits, const __grid_constant__ Job job) {
    __shared__ double table[TABLE];
    const int lane = threadIdx.x & 31;
    fill_table(table, job.shift, threadIdx.x, blockDim.x);
    __syncthreads();
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= job.R) return;
    const Rule rule(job, row);
    const T* src = logits + row * job.pitch;
    const int V = (int)job.V;
    uint32_t key[PER], most = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = j * 32 + lane;
        key[j] = i < V ? key_of(dl_to_float(src[i])) : 0u;
        most = key[j] > most ? key[j] : most;
    }
    most = __reduce_max_sync(FULL, most);
    if (most == 0) {
        if (lane == 0) job.out[row] = -1;
        return;
    }
    uint32_t member = 0;  // bit j: element j is still in
#pragma unroll
    for (int j = 0; j < PER; ++j) member |= (key[j] != 0u) << j;
    if (rule.greedy) {
        int first = V;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j)
            if (key[j] == most) first = j * 32 + lane;
        first = __reduce_min_sync(FULL, first);
        if (lane == 0) job.out[row] = first;
        return;
    }
    if (rule.top_k > 0) {
        // the k-th largest key, bit by bit: the largest t with at least k keys >= t
        uint32_t t = 0;
        int valid = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) valid += key[j] != 0u;
        valid = __reduce_add_sync(FULL, valid);
        if (valid > rule.top_k) {
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t at = t | (1u << bit);
                if (at > most) continue;
                int n = 0;
#pragma unroll
                for (int j = 0; j < PER; ++j) n += key[j] >= at;
                if (__reduce_add_sync(FULL, n) >= rule.top_k) t = at;
            }
            int above = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) above += key[j] > t;
            int ties = (int)rule.top_k - __reduce_add_sync(FULL, above);  // of the keys equal to t these are in
            member = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint32_t equal = __ballot_sync(FULL, key[j] == t);
                const bool in = key[j] > t || (key[j] == t && __popc(equal & ((1u << lane) - 1)) < ties);
                ties -= __popc(equal);
                member |= (uint32_t)in << j;
            }
        }
    }
    const Weigher weigh(table, most, rule.inverse_T, job.shift);
    u64 w[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        w[j] = member >> j & 1 ? weigh(key[j]) : 0ull;
        mine += w[j];
    }
    u64 total = warp_sum(mine);
    if (rule.top_p < 1.0) {
        const u64 target = share_of(rule.top_p, total);
        // the smallest kept key: the largest t whose keys >= t weigh at least the target
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t at = t | (1u << bit);
            if (at > most) continue;
            u64 s = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) s += key[j] >= at ? w[j] : 0ull;
            if (warp_sum(s) >= target) t = at;
        }
        u64 above = 0, each = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            above += key[j] > t ? w[j] : 0ull;
            if (key[j] == t && (member >> j & 1)) each = w[j];
        }
        above = warp_sum(above);
        // equal keys weigh the same: so many of them start below the target
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) {
            const u64 o = __shfl_xor_sync(FULL, each, s);
            each = o > each ? o : each;
        }
        int64_t ties = each > 0 ? (int64_t)((target - above + each - 1) / each) : 0;
        mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool tie = key[j] == t && (member >> j & 1);
            const uint32_t equal = __ballot_sync(FULL, tie);
            const bool in = key[j] > t || (tie && __popc(equal & ((1u << lane) - 1)) < ties);
            ties -= __popc(equal);
            if (!in) w[j] = 0ull;
        }
    }
    mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (w[j] < rule.least) w[j] = 0ull;
        mine += w[j];
    }
    total = warp_sum(mine);
    const u64 point = point_of(rule.u, total);
    u64 run = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const u64 upto = run + warp_inclusive(w[j], lane);
        const uint32_t hit = __ballot_sync(FULL, upto > point);
        if (hit) {
            if (lane == 0) job.out[row] = j * 32 + __ffs(hit) - 1;
            return;
        }
        run = __shfl_sync(FULL, upto, 31);
    }
}

// ------------------------------------------------------------------------------------------ a block or cluster per row
struct Shared {
    double table[TABLE];
    uint32_t low[BINS], high[BINS];  // the two words of every step's sum
    u64 list_weight[LIST], all_weight[LIST];
    uint32_t list_key[LIST], list_index[LIST], all_key[LIST], all_index[LIST];
    u64 warp_value[WARPS];
    u64 found[4];
    u64 published[2][4];  // for the other blocks, two turns
    uint32_t list_count;
    u64 result;
};

// down to where a running sum stays below its target: keys above, and equal keys up to an index
struct Cut {
    uint32_t key;
    uint32_t last;  // index
    __device__ __forceinline__ bool holds(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

template <typename T>
struct Row {
    const T* logits;
    uint32_t from, to;  // this block's slice
    Shared& sh;
    cg::cluster_group cluster;
    int rank, ranks, tid, lane, warp, turn;

    __device__ __forceinline__ void barrier() {
        if (ranks > 1) cluster.sync();
        else __syncthreads();
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {  // f(index, key) over the slice, four loads in flight
        uint32_t i = from + tid;
        for (; i + 3 * THREADS < to; i += 4 * THREADS) {
            float l[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) l[k] = dl_to_float(logits[i + k * THREADS]);
#pragma unroll
            for (int k = 0; k < 4; ++k) f(i + k * THREADS, key_of(l[k]));
        }
        for (; i < to; i += THREADS) f(i, key_of(dl_to_float(logits[i])));
    }
    // over the whole row: `combine` of every thread's value
    template <typename F>
    __device__ __forceinline__ u64 reduce(u64 v, F combine) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) v = combine(v, __shfl_xor_sync(FULL, v, s));
        __syncthreads();
        if (lane == 0) sh.warp_value[warp] = v;
        __syncthreads();
        v = sh.warp_value[0];
        for (int k = 1; k < WARPS; ++k) v = combine(v, sh.warp_value[k]);
        if (ranks == 1) return v;
        if (tid == 0) sh.published[turn][0] = v;
        cluster.sync();
        v = *cluster.map_shared_rank(&sh.published[turn][0], 0);
        for (int r = 1; r < ranks; ++r) v = combine(v, *cluster.map_shared_rank(&sh.published[turn][0], r));
        turn ^= 1;
        return v;
    }
    // clears the histogram, adds value(i, key) at step(i, key) wherever that is not negative, and finds the step at which
    // the row's sum reaches target(total).  False: it never does.
    template <typename S, typename G>
    __device__ __forceinline__ bool crossing(S step, G target, int& at, u64& before, u64& total, u64& goal) {
        __syncthreads();
        for (int b = tid; b < BINS; b += THREADS) sh.low[b] = sh.high[b] = 0;
        if (tid == 0) sh.found[0] = BINS;
        __syncthreads();
        each([&](uint32_t i, uint32_t key) {
            u64 value;
            const int b = step(i, key, value);
            if (b < 0) return;
            const uint32_t lo = (uint32_t)value, old = atomicAdd(&sh.low[b], lo);
            const uint32_t hi = (uint32_t)(value >> 32) + (old + lo < old ? 1u : 0u);
            if (hi) atomicAdd(&sh.high[b], hi);
        });
        barrier();
        constexpr int PER = BINS / THREADS;
        u64 v[PER], sum = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            v[k] = 0;
            for (int r = 0; r < ranks; ++r) {
                const uint32_t* low = ranks > 1 ? cluster.map_shared_rank(sh.low, r) : sh.low;
                const uint32_t* high = ranks > 1 ? cluster.map_shared_rank(sh.high, r) : sh.high;
                v[k] += (u64)low[tid * PER + k] | (u64)high[tid * PER + k] << 32;
            }
            sum += v[k];
        }
        const u64 inclusive = warp_inclusive(sum, lane);
        if (lane == 31) sh.warp_value[warp] = inclusive;
        __syncthreads();
        u64 run = inclusive - sum;
        total = 0;
        for (int k = 0; k < WARPS; ++k) {
            if (k < warp) run += sh.warp_value[k];
            total += sh.warp_value[k];
        }
        goal = target(total);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            if (run < goal && run + v[k] >= goal) {
                sh.found[0] = tid * PER + k;
                sh.found[1] = run;
            }
            run += v[k];
        }
        barrier();  // also: nobody clears a histogram that others still read
        at = (int)sh.found[0];
        before = sh.found[1];
        return at < BINS;
    }
    // The cut at which the sum of value over the members stays below the target, members in descending order.
    // weight(key) is a member's value, goal_of the target from the members' total.
    template <typename M, typename W, typename S, typename G>
    __device__ __forceinline__ bool cut(M member, W weight, S coarse, G goal_of, Cut& out) {
        int at;
        u64 before, total, goal;
        const bool crosses = crossing(
            [&](uint32_t i, uint32_t key, u64& value) {
                if (!member(i, key)) return -1;
                value = weight(key);
                return coarse(key);
            },
            goal_of, at, before, total, goal);
        if (!crosses) return false;
        // the members of that step
        if (tid == 0) sh.list_count = 0;
        __syncthreads();
        each([&](uint32_t i, uint32_t key) {
            if (!member(i, key) || coarse(key) != at) return;
            const uint32_t n = atomicAdd(&sh.list_count, 1u);
            if (n < LIST) {
                sh.list_key[n] = key;
                sh.list_index[n] = i;
                sh.list_weight[n] = weight(key);
            }
        });
        barrier();
        uint32_t n = 0, here = 0;
        for (int r = 0; r < ranks; ++r) {
            const uint32_t c = ranks > 1 ? *cluster.map_shared_rank(&sh.list_count, r) : sh.list_count;
            n += c;
        }
        if (n <= LIST) {
            uint32_t start = 0;
            for (int r = 0; r < ranks; ++r) {
                const Shared* other = ranks > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
                here = other->list_count;
                if (tid < (int)here) {
                    sh.all_key[start + tid] = other->list_key[tid];
                    sh.all_index[start + tid] = other->list_index[tid];
                    sh.all_weight[start + tid] = other->list_weight[tid];
                }
                start += here;
            }
            barrier();
            u64 worst = ~0ull;
            if (tid < (int)n) {
                const uint32_t key = sh.all_key[tid], index = sh.all_index[tid];
                u64 ahead = before;
                for (uint32_t k = 0; k < n; ++k) {
                    const uint32_t other = sh.all_key[k];
                    if (other > key || (other == key && sh.all_index[k] < index)) ahead += sh.all_weight[k];
                }
                if (ahead < goal) worst = (u64)key << 32 | (uint32_t)~index;
            }
            __syncthreads();
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) {
                const u64 o = __shfl_xor_sync(FULL, worst, s);
                worst = o < worst ? o : worst;
            }
            if (lane == 0) sh.warp_value[warp] = worst;
            __syncthreads();
            worst = sh.warp_value[0];
            for (int k = 1; k < WARPS; ++k) worst = sh.warp_value[k] < worst ? sh.warp_value[k] : worst;
            out.key = (uint32_t)(worst >> 32);
            out.last = ~(uint32_t)worst;
            return true;
        }
        // very many in one step: narrow their keys down to one
        u64 least = ~0ull, most = 0;
        each([&](uint32_t i, uint32_t key) {
            if (!member(i, key) || coarse(key) != at) return;
            least = key < least ? key : least;
            most = key > most ? key : most;
        });
        uint32_t klo = (uint32_t)reduce(least, [](u64 a, u64 b) { return a < b ? a : b; });
        uint32_t khi = (uint32_t)reduce(most, [](u64 a, u64 b) { return a > b ? a : b; });
        // three rounds of 11 bits are enough for 32; the limit also ends them should the logits change meanwhile
        for (int round = 0; klo < khi && round < 4; ++round) {
            int width = 0;
            while (((khi - klo) >> width) >= BINS) ++width;
            int sub;
            u64 upto, unused_total, unused_goal;
            const u64 wanted = goal - before;
            crossing(
                [&](uint32_t i, uint32_t key, u64& value) {
                    if (!member(i, key) || coarse(key) != at || key < klo || key > khi) return -1;
                    value = weight(key);
                    return (int)((khi - key) >> width);
                },
                [&](u64) { return wanted; }, sub, upto, unused_total, unused_goal);
            before += upto;
            const uint32_t top = khi - ((uint32_t)sub << width);
            const uint32_t span = (1u << width) - 1;
            klo = top - klo > span ? top - span : klo;
            khi = top;
        }
        // equal keys: the first so many by index
        const u64 value = weight(klo);
        u64 ties = value > 0 ? (goal - before + value - 1) / value : 1;
        // over the index likewise: the step of 2048 in which the last of them lies, then smaller ones
        uint32_t ilo = 0, ihi = 0xffffffffu;
        {
            u64 first = ~0ull, last = 0;
            each([&](uint32_t i, uint32_t key) {
                if (key != klo || !member(i, key)) return;
                first = i < first ? i : first;
                last = i > last ? i : last;
            });
            ilo = (uint32_t)reduce(first, [](u64 a, u64 b) { return a < b ? a : b; });
            ihi = (uint32_t)reduce(last, [](u64 a, u64 b) { return a > b ? a : b; });
        }
        for (int round = 0; ilo < ihi && round < 4; ++round) {
            int width = 0;
            while (((ihi - ilo) >> width) >= BINS) ++width;
            int sub;
            u64 upto, unused_total, unused_goal;
            crossing(
                [&](uint32_t i, uint32_t key, u64& one) {
                    if (key != klo || !member(i, key) || i < ilo || i > ihi) return -1;
                    one = 1;
                    return (int)((i - ilo) >> width);
                },
                [&](u64 n_ties) { return ties < n_ties ? ties : n_ties; }, sub, upto, unused_total, unused_goal);
            ties -= upto;
            ilo += (uint32_t)sub << width;
            const uint32_t span = (1u << width) - 1;
            ihi = ihi - ilo > span ? ilo + span : ihi;
        }
        out.key = klo;
        out.last = ilo;
        return true;
    }
};

template <typename T>
__global__ void __launch_bounds__(THREADS)
sample_kernel(const T* __restrict__ logits, const __grid_constant__ Job job, int ranks) {
    extern __shared__ __align__(16) unsigned char dynamic_shared[];
    Shared& sh = *reinterpret_cast<Shared*>(dynamic_shared);
    const int64_t row = blockIdx.x / ranks;
    const int rank = (int)(blockIdx.x % ranks), tid = threadIdx.x;
    const uint32_t V = (uint32_t)job.V, slice = (V + ranks - 1) / ranks;
    const uint32_t from = rank * slice < V ? rank * slice : V, to = from + slice < V ? from + slice : V;
    Row<T> r{logits + row * job.pitch, from, to, sh, cg::this_cluster(), rank, ranks, tid, tid & 31, tid >> 5, 0};
    const Rule rule(job, row);
    fill_table(sh.table, job.shift, tid, THREADS);

    // the largest key, and the lowest index that has it
    u64 best = 0;
    r.each([&](uint32_t i, uint32_t key) {
        const u64 c = (u64)key << 32 | (uint32_t)~i;
        best = key != 0u && c > best ? c : best;
    });
    best = r.reduce(best, [](u64 a, u64 b) { return a > b ? a : b; });
    const uint32_t most = (uint32_t)(best >> 32);
    if (most == 0u || rule.greedy) {
        if (rank == 0 && tid == 0) job.out[row] = most == 0u ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
        r.barrier();  // nobody leaves while others read its numbers
        return;
    }
    const Weigher weigh(sh.table, most, rule.inverse_T, job.shift);
    const float top = logit_of(most), steps_per_unit = 32.0f * (float)rule.inverse_T;
    // 2048 steps of 1/32 down from the largest logit, in fp32: monotone, and weights below 2^-50 are in the last one
    const auto coarse = [&](uint32_t key) {
        const float d = (top - logit_of(key)) * steps_per_unit;  // NaN for inf - inf: the first step
        return d < (float)(BINS - 1) ? (int)d : (d >= 0.0f ? BINS - 1 : 0);
    };
    Cut cut{1u, FULL};  // everything but key 0
    if (rule.top_k > 0) {
        const u64 k = (u64)rule.top_k;
        Cut c;
        if (r.cut([](uint32_t, uint32_t key) { return key != 0u; }, [](uint32_t) { return (u64)1; }, coarse,
                  [k](u64) { return k; }, c))
            cut = c;
    }
    if (rule.top_p < 1.0) {
        const Cut held = cut;
        const double p = rule.top_p;
        Cut c;
        if (r.cut([held](uint32_t i, uint32_t key) { return held.holds(key, i); }, weigh, coarse,
                  [p](u64 total) { return share_of(p, total); }, c))
            cut = c;
    }
    // the draw: every warp sums a run of the slice, the run that holds the point is cut up again
    const u64 least = rule.least;
    const auto kept = [&](uint32_t i) {
        const uint32_t key = key_of(dl_to_float(r.logits[i]));
        if (!cut.holds(key, i)) return (u64)0;
        const u64 w = weigh(key);
        return w < least ? (u64)0 : w;
    };
    uint32_t lo = from, hi = to;
    u64 point = 0;
    __syncthreads();
    for (int level = 0;; ++level) {
        const uint32_t run = (hi - lo + WARPS - 1) / WARPS;
        const uint32_t begin = lo + r.warp * run < hi ? lo + r.warp * run : hi, end = begin + run < hi ? begin + run : hi;
        u64 sum = 0;
#pragma unroll 4
        for (uint32_t i = begin + r.lane; i < end; i += 32) sum += kept(i);
        sum = warp_sum(sum);
        if (r.lane == 0) sh.warp_value[r.warp] = sum;
        __syncthreads();
        if (level == 0) {
            u64 mine = 0;
            for (int k = 0; k < WARPS; ++k) mine += sh.warp_value[k];
            u64 before = 0, total = mine;
            if (ranks > 1) {
                if (tid == 0) sh.published[r.turn][0] = mine;
                r.cluster.sync();
                total = 0;
                for (int q = 0; q < ranks; ++q) {
                    const u64 v = *r.cluster.map_shared_rank(&sh.published[r.turn][0], q);
                    if (q < rank) before += v;
                    total += v;
                }
            }
            point = point_of(rule.u, total);
            if (point < before || point >= before + mine) break;  // another block has it
            point -= before;
        }
        int at = 0;
        u64 before = 0;
        while (at < WARPS - 1 && before + sh.warp_value[at] <= point) before += sh.warp_value[at++];
        point -= before;
        lo = lo + at * run;
        hi = lo + run < hi ? lo + run : hi;
        __syncthreads();
        if (hi - lo <= 32) {
            if (r.warp == 0) {
                const u64 upto = warp_inclusive(lo + r.lane < hi ? kept(lo + r.lane) : 0ull, r.lane);
                const uint32_t hit = __ballot_sync(FULL, upto > point);
                if (r.lane == 0) job.out[row] = (int64_t)lo + __ffs(hit) - 1;
            }
            break;
        }
    }
    r.barrier();  // nobody leaves while others read its numbers
}

// ------------------------------------------------------------------------------------------ host
template <typename T>
int launch_sample(const void* logits, const Job& job, cudaStream_t s) {
    const T* src = static_cast<const T*>(logits);
    if (job.V <= SMALL_V) {
        const int64_t blocks = dl_ceil_div(job.R, 4);
        if (blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
        if (job.V <= 64) sample_small_kernel<T, 2><<<(unsigned)blocks, 128, 0, s>>>(src, job);
        else if (job.V <= 256) sample_small_kernel<T, 8><<<(unsigned)blocks, 128, 0, s>>>(src, job);
        else sample_small_kernel<T, 16><<<(unsigned)blocks, 128, 0, s>>>(src, job);
        return dl_launch_status();
    }
    // more blocks per row while they have 4096 classes each and the rows alone do not fill the SMs four times
    int ranks = 1;
    while (ranks < MAX_CLUSTER && job.V >= (int64_t)8192 * ranks && job.R * ranks < (int64_t)DL_NUM_SMS * 4) ranks *= 2;
    if (job.R * ranks > 0x7fffffff) return DL_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(job.R * ranks));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const auto kernel = sample_kernel<T>;
    static DlKernelLimits limits;
    if (!dl_allow(reinterpret_cast<const void*>(kernel), limits, sizeof(Shared), false)) return DL_ERR_LAUNCH;
    return cudaLaunchKernelEx(&cfg, kernel, src, job, ranks) == cudaSuccess ? dl_launch_status() : DL_ERR_LAUNCH;
}

}  // namespace

DL_EXPORT int dl_sample_rows(const void* logits, int64_t pitch, const void* u, int64_t u_double, const float* temperature,
                             double temperature_all, const int32_t* top_k, int64_t top_k_all, const float* top_p,
                             double top_p_all, const float* min_p, double min_p_all, int64_t* out, int64_t R, int64_t V,
                             int64_t dtype, dl_stream_t stream) {
    DL_REQUIRE(R >= 0 && V > 0 && dl_dtype_known(dtype));
    DL_REQUIRE(temperature_all >= 0.0 && top_k_all >= 0 && top_p_all > 0.0 && min_p_all >= 0.0 && min_p_all <= 1.0);
    if (V >= ((int64_t)1 << 30)) return DL_ERR_TOO_LARGE;  // a weight keeps 32 fractional bits at least
    if (R == 0) return DL_OK;
    DL_REQUIRE(logits && u && out && (R == 1 || pitch >= 0));
    DL_REQUIRE_ALIGNED(logits, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(u, u_double ? 8 : 4);
    Job job;
    job.u = u;
    job.u_double = u_double != 0;
    job.out = out;
    job.R = R;
    job.V = V;
    job.pitch = pitch;
    int log2V = 0;
    while (((int64_t)1 << log2V) < V) ++log2V;
    job.shift = 62 - log2V < 50 ? 62 - log2V : 50;
    job.set.temperature = temperature;
    job.set.top_k = top_k;
    job.set.top_p = top_p;
    job.set.min_p = min_p;
    job.set.temperature_all = temperature_all;
    job.set.top_k_all = top_k_all;
    job.set.top_p_all = top_p_all;
    job.set.min_p_all = min_p_all;
    cudaStream_t s = dl_cast(stream);
    if (dtype == DL_DTYPE_F32) return launch_sample<float>(logits, job, s);
    if (dtype == DL_DTYPE_BF16) return launch_sample<__nv_bfloat16>(logits, job, s);
    return launch_sample<__half>(logits, job, s);
}
