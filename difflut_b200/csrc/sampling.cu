// Sampling a class per row of logits with temperature, top-k, top-p and min-p from given random numbers.
//
//   w_i = exp((l_i - max) / T);  top-k keeps the k largest (equal logits: lowest index first);  top-p keeps, of those in
//   descending order, the ones with less than p * (their total) before them;  min-p keeps w_i >= min_p;
//   the class is the first i, in ascending order, whose running sum of kept weights exceeds u * (total kept weight).
//
// Both cuts are one question: down to which (logit, index) does a running sum, of ones or of weights, stay below a
// target?  It is answered without sorting the row: a histogram over (max - l) / T in 2048 steps of 1/32 finds the step in
// which the target falls.  The logits in that step and above it are collected in lists in shared memory, and only those of
// that one step are sorted.  The draw is a histogram as well, of the listed weights over the index, and the 1/2048 of
// the row in which the point falls is read once more.  (Sorting the whole list by key and then by index took 34 of 48 us
// for 1900 logits.)  For top-k the list is short: it is sorted, and cuts and draw are prefix sums.  Should the lists not
// hold them, the logits of the step are told apart by histograms over the bits of their keys and, for equal ones, over
// their index, and the draw goes over the row.
//
// A class next to a border must not depend on the order of additions, so weights are whole numbers: exp in double
// precision, as fixed point with up to 50 fractional bits, chosen so that the sum of a row fits 62 bits.  Integer sums are
// exact in any order, so shared-memory atomics are harmless here.  V classes that weigh less than (1 - p) / V of the
// largest each cannot hold the border of top-p: they go to a register instead.
//
// Rows of up to 512 classes take one warp and registers; longer ones a block of 512 threads, or a cluster of up to
// eight when there are few rows.  Each pass reads the logits again: after the first they come from L2.
//
// Measured: 64 rows of 32000 bf16 logits, T .8: 5.8 us for the largest, 19 us to draw from all, 20 us with top-k 50 and
// top-p .95, 34 us with top-p .95 alone (8 rows: 30).  Of the latter the histogram of the weights takes 7 us, the two
// searches in histograms 3 to 4 us each, collecting 4, the cut 5: latency of passes with few rounds of loads per thread,
// not bandwidth (the 4 MB are read in a microsecond).  256 rows of 65536 fp32 logits with top-p .9 and min-p .01: 88 us, 43 of them the
// histogram: no unit is at its limit (issue slots 51 % over all SMs, of which 108 hold two rows and 40 one, the data pipe of
// shared memory 40 %, double precision 12 %); what a logit costs is an exponential and two atomics, also below the reach of
// min-p, where they are not needed.  Reading the 67 MB once takes 10.
#include <cooperative_groups.h>

#include "elements.cuh"

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int BINS = 2048;
constexpr int LIST = 2048;  // most logits that a block collects, and that are sorted
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
        if (top_p < 0.0) top_p = 0.0;  // NaN stays and keeps all
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

// exp(-(top - l) / T) as fixed point.  With t = 128 (top - l) / (T ln 2), j = round(t) and f = t - j, it is
// 2^(-j / 128) 2^(-f / 128): a table for the fraction of the first power, its whole part as an exponent, and four terms of
// the series of e^(-f ln 2 / 128) (|f| <= 1/2: the fifth is below 2^-49).  Ten double-precision operations, which are
// what a pass of exponentials costs (about three cycles each for a warp); no branches, so that the steps of several logits
// overlap.
struct Weigher {
    const double* table;  // 2^(shift - i / 128)
    double top, scale;    // scale: 128 / (T ln 2)
    float least;          // logits below weigh less than half the last bit
    bool infinite;        // the largest logit is +inf: only such logits weigh something
    u64 one;
    __device__ __forceinline__ Weigher(const double* table, uint32_t top_key, double inverse_T, int shift)
        : table(table) {
        const float t = logit_of(top_key);
        infinite = t == INFINITY;
        top = infinite ? 0.0 : (double)t;
        scale = fmin(inverse_T * 184.6649652337873, 1e300);
        // no more than 2^-(shift + 2), so far away that fp32 rounding does not bring it back
        least = (float)fmax(top - (shift + 3) * 128.0 / scale, -3.4028234663852886e38);  // the lowest finite value
        one = 1ull << shift;
    }
    // 0 for NaN and -inf
    __device__ __forceinline__ u64 of(float l) const {
        const double d = top - (double)fmaxf(l, least);
        const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
        const double shifted = fma(d, scale, magic);
        const int j = __double2loint(shifted);
        const double f = fma(d, scale, magic - shifted);
        // (ln 2 / 128)^n / n!
        const double e = fma(f, fma(f, fma(f, fma(f, 3.583032305400251e-11, -2.6466421444330967e-08),
                                           1.4662262387640423e-05), -0.0054152123481245725), 1.0);
        double w = table[j & (TABLE - 1)] * e;
        w = __hiloint2double(__double2hiint(w) - ((j >> 7) << 20), __double2loint(w));
        const u64 fixed = (u64)__double_as_longlong(w + 4503599627370496.0) - 0x4330000000000000ull;  // w < 2^52, rounded
        return infinite ? (l == INFINITY ? one : 0ull) : (l >= least ? fixed : 0ull);
    }
    __device__ __forceinline__ u64 operator()(uint32_t key) const { return of(logit_of(key)); }
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
// Element j * 32 + lane sits in register j: index order is register, then lane.  The borders of top-k and top-p are found bit
// by bit of the key: counting 256 keys takes 8 comparisons and one reduction.  What top-k leaves is moved together, since
// every register of exponentials costs a row eighty double-precision issue slots.  Measured, 8192 rows of 256 fp32 logits,
// top-k 40: 15.6 us (17.9 before moving; reading the logits takes 1.3), 56 % of the issue slots: about 16 rounds of counting
// that follow one another.
template <typename T, int PER>
__global__ void __launch_bounds__(128)
sample_small_kernel(const T* __restrict__ logits, const __grid_constant__ Job job) {
    __shared__ double table[TABLE];
    __shared__ uint2 moved[4][PER * 32];
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
    uint32_t index[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) index[j] = j * 32 + lane;
    int rounds = PER;  // registers that hold members
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
                n = __reduce_add_sync(FULL, n);
                if (n >= rule.top_k) t = at;
                if (n == rule.top_k) break;  // exactly these
            }
            int above = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) above += key[j] > t;
            int ties = (int)rule.top_k - __reduce_add_sync(FULL, above);  // of the keys equal to t these are in
            // the members move up to the first registers, still in order of their indexes: they are few mostly
            int kept = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint32_t equal = __ballot_sync(FULL, key[j] == t);
                const bool in = key[j] > t || (key[j] == t && __popc(equal & ((1u << lane) - 1)) < ties);
                ties -= __popc(equal);
                const uint32_t all = __ballot_sync(FULL, in);
                if (in) moved[threadIdx.x >> 5][kept + __popc(all & ((1u << lane) - 1))] = make_uint2(key[j], j * 32 + lane);
                kept += __popc(all);
            }
            __syncwarp();
            rounds = (kept + 31) / 32;
            member = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = j * 32 + lane;
                const uint2 m = i < kept ? moved[threadIdx.x >> 5][i] : make_uint2(0u, 0u);
                key[j] = m.x;
                index[j] = m.y;
                member |= (uint32_t)(i < kept) << j;
            }
        }
    }
    const Weigher weigh(table, most, rule.inverse_T, job.shift);
    u64 w[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        w[j] = 0ull;
        if (j < rounds) w[j] = member >> j & 1 ? weigh(key[j]) : 0ull;
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
            if (lane == __ffs(hit) - 1) job.out[row] = index[j];
            return;
        }
        run = __shfl_sync(FULL, upto, 31);
    }
}

// ------------------------------------------------------------------------------------------ a block or cluster per row
struct __align__(16) Shared {
    double table[TABLE];
    uint32_t low[BINS], high[BINS];  // the two words of every step's sum
    u64 list[LIST];    // collected by this block: key, then the index inverted
    u64 part[LIST];    // those of the list that share a step
    u64 sorted[LIST];  // of the whole row, in the first block
    u64 warp_value[WARPS];
    u64 tail;
    u64 found[4];
    u64 published[2][4];  // for the other blocks, two turns
    uint32_t list_count, part_count;
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
    bool vectors;

    __device__ __forceinline__ void barrier() {
        if (ranks > 1) cluster.sync();
        else __syncthreads();
    }
    // f(index, stride, four logits) over the slice, element e at index + e * stride; NaN where there is none.  The lanes of a
    // warp call f together.  By vectors when every row starts on 16 bytes (slices do then).
    template <typename F>
    __device__ __forceinline__ void each4(F f) const {
        constexpr int N = 16 / sizeof(T), AHEAD = 16 / N;
        uint32_t i = from;
        if (vectors) {
            constexpr uint32_t STEP = THREADS * N;
            const uint32_t whole = from + (to - from) / STEP * STEP;
            for (i = from + tid * N; i < whole; i += AHEAD * STEP) {
                DlVec<T, N> v[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (i + k * STEP < whole) v[k] = *reinterpret_cast<const DlVec<T, N>*>(logits + i + k * STEP);
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (i + k * STEP >= whole) break;
                    float l[N];
                    dl_unpack(v[k], l);
#pragma unroll
                    for (int q = 0; q < N; q += 4) {
                        const float four[4] = {l[q], l[q + 1], l[q + 2], l[q + 3]};
                        f(i + k * STEP + q, 1u, four);
                    }
                }
            }
            i = whole;
        }
        for (; i < to; i += 4 * THREADS) {  // all lanes together
            float l[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t at = i + tid + k * THREADS;
                l[k] = at < to ? dl_to_float(logits[at]) : NAN;
            }
            f(i + tid, (uint32_t)THREADS, l);
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each4([&](uint32_t i, uint32_t stride, const float (&l)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f(i + e * stride, l[e]);
        });
    }
    template <typename F>
    __device__ __forceinline__ void each_key(F f) const {
        each([&](uint32_t i, float l) { f(i, key_of(l)); });
    }
    // over the whole row: `combine` of every thread's value
    template <typename F>
    __device__ __forceinline__ u64 reduce(u64 v, F combine) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) v = combine(v, __shfl_xor_sync(FULL, v, s));
        __syncthreads();
        if (lane == 0) sh.warp_value[warp] = v;
        __syncthreads();
        v = sh.warp_value[lane % WARPS];
#pragma unroll
        for (int s = WARPS / 2; s > 0; s >>= 1) v = combine(v, __shfl_xor_sync(FULL, v, s));
        if (ranks == 1) return v;
        if (tid == 0) sh.published[turn][0] = v;
        cluster.sync();
        v = *cluster.map_shared_rank(&sh.published[turn][0], 0);
        for (int r = 1; r < ranks; ++r) v = combine(v, *cluster.map_shared_rank(&sh.published[turn][0], r));
        turn ^= 1;
        return v;
    }
    void __device__ __forceinline__ clear_histogram() {
        __syncthreads();
        for (int b = tid; b < BINS; b += THREADS) sh.low[b] = sh.high[b] = 0;
        if (tid == 0) {
            sh.found[0] = BINS;
            sh.tail = 0;
        }
        __syncthreads();
    }
    __device__ __forceinline__ void add_weight(int b, u64 value) {
        const uint32_t lo = (uint32_t)value, old = atomicAdd(&sh.low[b], lo);
        const uint32_t hi = (uint32_t)(value >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&sh.high[b], hi);
    }
    // four at once, so that their round trips overlap
    __device__ __forceinline__ void add_weights(const int (&b)[4], const u64 (&value)[4]) {
        uint32_t old[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (value[e]) old[e] = atomicAdd(&sh.low[b[e]], (uint32_t)value[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!value[e]) continue;
            const uint32_t lo = (uint32_t)value[e], hi = (uint32_t)(value[e] >> 32) + (old[e] + lo < old[e] ? 1u : 0u);
            if (hi) atomicAdd(&sh.high[b[e]], hi);
        }
    }
    // The step at which the row's sum over the histogram reaches target(total); total includes the tails.  False: it never
    // does.
    template <typename G>
    __device__ __forceinline__ bool find_step(G target, int& at, u64& before, u64& total, u64& goal) {
        barrier();
        constexpr int PER = BINS / THREADS;
        u64 v[PER], sum = 0;
        total = 0;
        if (ranks > 1)
            for (int r = 0; r < ranks; ++r) total += *cluster.map_shared_rank(&sh.tail, r);
        else
            total = sh.tail;
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = 0;
        for (int r = 0; r < ranks; ++r) {
            const Shared* other = ranks > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
            static_assert(PER == 4, "one access per array");
            const uint4 lo = *reinterpret_cast<const uint4*>(&other->low[tid * PER]);
            const uint4 hi = *reinterpret_cast<const uint4*>(&other->high[tid * PER]);
            v[0] += (u64)lo.x | (u64)hi.x << 32;
            v[1] += (u64)lo.y | (u64)hi.y << 32;
            v[2] += (u64)lo.z | (u64)hi.z << 32;
            v[3] += (u64)lo.w | (u64)hi.w << 32;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) sum += v[k];
        const u64 inclusive = warp_inclusive(sum, lane);
        if (lane == 31) sh.warp_value[warp] = inclusive;
        __syncthreads();
        u64 run = inclusive - sum;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
            const u64 w = sh.warp_value[k];
            if (k < warp) run += w;
            total += w;
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
        __syncthreads();  // the other blocks may still read this one's histogram
        at = (int)sh.found[0];
        before = sh.found[1];
        return at < BINS;
    }
    // adds value(i, key) at step(i, key) wherever that is not negative, and finds the step of target(total)
    template <typename S, typename G>
    __device__ __forceinline__ bool crossing(S step, G target, int& at, u64& before, u64& total, u64& goal) {
        barrier();  // nobody reads the last histogram any more
        clear_histogram();
        each_key([&](uint32_t i, uint32_t key) {
            u64 value;
            const int b = step(i, key, value);
            if (b >= 0) add_weight(b, value);
        });
        return find_step(target, at, before, total, goal);
    }
    // Collects the logits that wanted(index, logit) accepts in the blocks' lists.  False: a list was too short for them.
    // Between one call and the next there is a barrier.
    template <typename F>
    __device__ __forceinline__ bool collect(F wanted) {
        __syncthreads();
        if (tid == 0) sh.list_count = 0;
        __syncthreads();
        each4([&](uint32_t i, uint32_t stride, const float (&l)[4]) {
            bool want[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) want[e] = wanted(i + e * stride, l[e]);
            // one atomic per warp: on one address they follow one another
            uint32_t mask[4], all = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mask[e] = __ballot_sync(FULL, want[e]);
                all += __popc(mask[e]);
            }
            if (all == 0) return;
            uint32_t at = lane == 0 ? atomicAdd(&sh.list_count, all) : 0u;
            at = __shfl_sync(FULL, at, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t n = at + __popc(mask[e] & ((1u << lane) - 1));
                if (want[e] && n < LIST) sh.list[n] = (u64)key_of(l[e]) << 32 | (uint32_t)~(i + e * stride);
                at += __popc(mask[e]);
            }
        });
        barrier();
        bool fits = true;
        for (int r = 0; r < ranks; ++r)
            fits &= (ranks > 1 ? *cluster.map_shared_rank(&sh.list_count, r) : sh.list_count) <= LIST;
        if (!fits) barrier();
        return fits;
    }
    // Brings the entries of the blocks' lists (`part`: of their parts) to the first block and sorts them there, if there
    // are no more than LIST, largest first, equal ones by index.  Returns how many there are.  After a barrier.
    __device__ __forceinline__ uint32_t gather(bool part) {
        uint32_t n = 0;
        for (int r = 0; r < ranks; ++r) {
            const Shared* other = ranks > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
            n += part ? other->part_count : other->list_count;
        }
        if (rank == 0 && n <= LIST) {
            uint32_t start = 0;
            for (int r = 0; r < ranks; ++r) {
                const Shared* other = ranks > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
                const uint32_t here = part ? other->part_count : other->list_count;
                for (uint32_t i = tid; i < here; i += THREADS) sh.sorted[start + i] = (part ? other->part : other->list)[i];
                start += here;
            }
            sort(sh, n, tid);
        }
        return n;
    }
    // Sorts `sorted` descending: by counting, or by a bitonic network.  There a thread holds four neighbours: partners
    // one and two apart are its own, up to 64 apart other lanes', farther ones come through shared memory (10 of 66 steps
    // for 2048).  (Out of line, like the two functions below: they run once. Whatever
    // they take by reference would live in memory for the whole kernel, so they take copies.)
    __device__ __noinline__ static void sort(Shared& sh, uint32_t n, int tid) {
        static_assert(LIST == 4 * THREADS, "four entries per thread");
        __syncthreads();
        if (n <= THREADS) {
            // few: the place of an entry is the number of larger ones; all are different.  Several lanes share the counting.
            uint32_t lanes = 32;
            while (lanes * n > THREADS) lanes /= 2;
            const uint32_t i = tid / lanes;
            const u64 mine = i < n ? sh.sorted[i] : 0ull;
            uint32_t place = 0;
            if (i < n)
                for (uint32_t j = tid % lanes; j < n; j += lanes) place += sh.sorted[j] > mine;
            for (uint32_t s = lanes / 2; s > 0; s /= 2) place += __shfl_xor_sync(FULL, place, s);
            __syncthreads();
            if (i < n && tid % lanes == 0) sh.sorted[place] = mine;
            __syncthreads();
            return;
        }
        uint32_t size = 2 * THREADS;
        while (size < n) size *= 2;
        const uint32_t first = 4 * tid;
        const bool active = first < size;
        u64 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = first + e < n ? sh.sorted[first + e] : 0ull;
        const auto order = [](u64& a, u64& b, bool descending) {
            if ((a < b) == descending) {
                const u64 c = a;
                a = b;
                b = c;
            }
        };
        for (uint32_t run = 2; run <= size; run *= 2) {
            for (uint32_t s = run / 2; s > 0; s /= 2) {
                if (s >= 128) {
                    __syncthreads();
                    if (active) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) sh.sorted[first + e] = v[e];
                    }
                    __syncthreads();
                }
                if (!active) continue;
                if (s == 1) {
                    order(v[0], v[1], (first & run) == 0);
                    order(v[2], v[3], ((first + 2) & run) == 0);
                } else if (s == 2) {
                    order(v[0], v[2], (first & run) == 0);
                    order(v[1], v[3], (first & run) == 0);
                } else {
                    const bool larger = ((first & s) == 0) == ((first & run) == 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const u64 o = s >= 128 ? sh.sorted[(first + e) ^ s] : __shfl_xor_sync(FULL, v[e], s / 4);
                        if ((v[e] < o) == larger) v[e] = o;
                    }
                }
            }
        }
        __syncthreads();
        if (active) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sh.sorted[first + e] = v[e];
        }
        __syncthreads();
    }
    // Running sums of two values per thread in list order: a, b become the sums up to and including them.  Returns the
    // total.
    __device__ __forceinline__ u64 scan_pairs(u64& a, u64& b) const {
        const u64 sum = a + b, inclusive = warp_inclusive(sum, lane);
        __syncthreads();
        if (lane == 31) sh.warp_value[warp] = inclusive;
        __syncthreads();
        u64 run = inclusive - sum, total = 0;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
            const u64 v = sh.warp_value[k];
            if (k < warp) run += v;
            total += v;
        }
        a += run;
        b = run + sum;
        return total;
    }
    // Cuts and draw among the n sorted logits, the row's largest, of which top-k keeps k; by the first block.  What is kept
    // is a prefix of them.
    template <typename W>
    __device__ __noinline__ static int64_t finish(Row r, uint32_t n, uint32_t k, Rule rule, W weigh) {
        Shared& sh = r.sh;
        const int tid = r.tid;
        constexpr uint32_t ROUND = 2 * THREADS;  // two entries per thread at a time
        if (k < n) n = k;
        const auto weight = [&](uint32_t i, int word) {  // word: where the key is
            return i < n ? weigh((uint32_t)(sh.sorted[i] >> (32 * word))) : 0ull;
        };
        u64 total = 0;
        if (rule.top_p < 1.0)
            for (uint32_t base = 0; base < n; base += ROUND) {
                u64 a = weight(base + 2 * tid, 1), b = weight(base + 2 * tid + 1, 1);
                total += r.scan_pairs(a, b);
            }
        const u64 goal = rule.top_p < 1.0 ? share_of(rule.top_p, total) : ~0ull;
        // by index from here on: the largest inverted index first
        const auto by_index = [](u64 e) { return e << 32 | e >> 32; };
        uint32_t kept = 0;
        u64 before = 0;
        for (uint32_t base = 0; base < n; base += ROUND) {
            const uint32_t i = base + 2 * tid;
            const u64 w0 = weight(i, 1), w1 = weight(i + 1, 1);
            u64 upto0 = w0, upto1 = w1;
            const u64 round = r.scan_pairs(upto0, upto1);
            const bool keep0 = i < n && before + upto0 - w0 < goal && w0 >= rule.least;
            const bool keep1 = i + 1 < n && before + upto1 - w1 < goal && w1 >= rule.least;
            if (keep0) {
                sh.sorted[i] = by_index(sh.sorted[i]);
                if (!keep1) sh.found[2] = before + upto0;  // the last one, unless a later thread has another
            }
            if (keep1) sh.sorted[i + 1] = by_index(sh.sorted[i + 1]);
            const uint32_t here = __syncthreads_count(keep0) + __syncthreads_count(keep1);
            if (keep1 && here == (uint32_t)(2 * tid + 2)) sh.found[2] = before + upto1;
            kept += here;
            before += round;
            __syncthreads();
            if (here < ROUND) break;
        }
        const u64 sum = sh.found[2], point = point_of(rule.u, sum);
        sort(sh, kept, tid);
        n = kept;
        before = 0;
        for (uint32_t base = 0; base < n; base += ROUND) {
            const uint32_t i = base + 2 * tid;
            const u64 w0 = weight(i, 0), w1 = weight(i + 1, 0);
            u64 upto0 = w0, upto1 = w1;
            const u64 round = r.scan_pairs(upto0, upto1);
            // one entry's weight spans the point
            if (w0 > 0 && before + upto0 > point && before + upto0 - w0 <= point)
                sh.found[3] = (uint32_t)~(uint32_t)(sh.sorted[i] >> 32);
            if (w1 > 0 && before + upto1 > point && before + upto1 - w1 <= point)
                sh.found[3] = (uint32_t)~(uint32_t)(sh.sorted[i + 1] >> 32);
            before += round;
        }
        __syncthreads();
        return (int64_t)sh.found[3];
    }
    // The cut among the n sorted logits: down to where their running sum, which starts with `before`, stays below `goal`.
    // At least one does, unless the logits change meanwhile.
    template <typename W>
    __device__ __forceinline__ Cut cut_sorted(uint32_t n, u64 before, u64 goal, W weight) {
        if (rank == 0) {
            uint32_t kept = 0;
            for (uint32_t base = 0; base < n; base += 2 * THREADS) {
                const uint32_t i = base + 2 * tid;
                const u64 w0 = i < n ? weight((uint32_t)(sh.sorted[i] >> 32)) : 0ull;
                const u64 w1 = i + 1 < n ? weight((uint32_t)(sh.sorted[i + 1] >> 32)) : 0ull;
                u64 upto0 = w0, upto1 = w1;
                const u64 round = scan_pairs(upto0, upto1);
                kept += __syncthreads_count(i < n && before + upto0 - w0 < goal) +
                        __syncthreads_count(i + 1 < n && before + upto1 - w1 < goal);
                before += round;
            }
            if (tid == 0) sh.found[3] = sh.sorted[kept > 0 ? kept - 1 : 0];
        }
        barrier();
        const u64 last = ranks > 1 ? *cluster.map_shared_rank(&sh.found[3], 0) : sh.found[3];
        return Cut{(uint32_t)(last >> 32), ~(uint32_t)last};
    }
    // cut_in among the logits in the blocks' lists, which hold step `at` and all above.  Key 0 when too many share the step.
    template <typename W, typename S>
    __device__ __noinline__ static Cut cut_in_list(Row r, int at, u64 before, u64 goal, W weight, S coarse) {
        Shared& sh = r.sh;
        if (r.tid == 0) sh.part_count = 0;
        __syncthreads();
        for (uint32_t i = r.tid; i < sh.list_count; i += THREADS) {
            const u64 entry = sh.list[i];
            if (coarse((uint32_t)(entry >> 32)) == at) sh.part[atomicAdd(&sh.part_count, 1u)] = entry;
        }
        r.barrier();
        const uint32_t n = r.gather(true);
        return n <= LIST ? r.cut_sorted(n, before, goal, weight) : Cut{0u, 0u};
    }
    // The draw among the logits in the blocks' lists that `cut` holds and that weigh no less than `least`: the run of
    // indexes, one of 2048 at most, in which the running sum first exceeds the point for u.
    struct Drawn {
        uint32_t from, to;
        u64 point;  // what is left of it there
    };
    template <typename W>
    __device__ __noinline__ static Drawn draw_in_list(Row r, uint32_t V, Cut cut, u64 least, double u, W weigh) {
        Shared& sh = r.sh;
        int width = 0;
        while (((V - 1) >> width) >= BINS) ++width;
        r.clear_histogram();
        for (uint32_t i = r.tid; i < sh.list_count; i += THREADS) {
            const u64 entry = sh.list[i];
            const uint32_t key = (uint32_t)(entry >> 32), index = ~(uint32_t)entry;
            const u64 w = weigh(key);
            if (cut.holds(key, index) && w >= least) r.add_weight((int)(index >> width), w);
        }
        int at;
        u64 before, total, goal;
        r.find_step([u](u64 all) { return point_of(u, all) + 1; }, at, before, total, goal);
        const uint32_t most = (V - 1) >> width;
        const uint32_t from = ((uint32_t)at < most ? (uint32_t)at : most) << width, last = from + ((1u << width) - 1);
        return Drawn{from, last < V ? last + 1 : V, goal - 1 - before};
    }
    // The cut in step `at`, before which the members weigh `before`, at which the sum of weight(key) over the members, in
    // descending order, stays below `goal`.
    template <typename M, typename W, typename S>
    __device__ __noinline__ static Cut cut_in(Row r, int at, u64 before, u64 goal, M member, W weight, S coarse) {
        return r.cut_here(at, before, goal, member, weight, coarse);
    }
    template <typename M, typename W, typename S>
    __device__ __forceinline__ Cut cut_here(int at, u64 before, u64 goal, M member, W weight, S coarse) {
        const bool fits = collect([=](uint32_t i, float l) {
            const uint32_t key = key_of(l);
            return member(i, key) && coarse(key) == at;
        });
        if (fits) {
            const uint32_t n = gather(false);
            if (n <= LIST) return cut_sorted(n, before, goal, weight);
        }
        Cut out;
        // very many in one step: narrow their keys down to one
        u64 least = ~0ull, most = 0;
        each_key([&](uint32_t i, uint32_t key) {
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
            each_key([&](uint32_t i, uint32_t key) {
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
        return out;
    }
    // the same with the step still to be found; goal_of: the target from the members' total.  False: no cut.
    template <typename M, typename W, typename S, typename G>
    __device__ __forceinline__ bool cut(M member, W weight, S coarse, G goal_of, Cut& out) {
        int at;
        u64 before, total, goal;
        if (!crossing(
                [&](uint32_t i, uint32_t key, u64& value) {
                    if (!member(i, key)) return -1;
                    value = weight(key);
                    return coarse(key);
                },
                goal_of, at, before, total, goal))
            return false;
        out = cut_in(*this, at, before, goal, member, weight, coarse);
        return true;
    }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 2)
sample_kernel(const T* __restrict__ logits, const __grid_constant__ Job job, int ranks, uint32_t slice, int vectors) {
    extern __shared__ __align__(16) unsigned char dynamic_shared[];
    Shared& sh = *reinterpret_cast<Shared*>(dynamic_shared);
    const int64_t row = blockIdx.x / ranks;
    const int rank = (int)(blockIdx.x % ranks), tid = threadIdx.x;
    const uint32_t V = (uint32_t)job.V;
    const uint32_t from = rank * slice < V ? rank * slice : V, to = from + slice < V ? from + slice : V;
    Row<T> r{logits + row * job.pitch, from, to, sh, cg::this_cluster(), rank, ranks, tid, tid & 31, tid >> 5, 0,
             vectors != 0};
    const Rule rule(job, row);
    fill_table(sh.table, job.shift, tid, THREADS);

    uint32_t most;
    if (rule.greedy) {  // the largest key, and the lowest index that has it
        u64 best = 0;
        r.each_key([&](uint32_t i, uint32_t key) {
            const u64 c = (u64)key << 32 | (uint32_t)~i;
            best = key != 0u && c > best ? c : best;
        });
        best = r.reduce(best, [](u64 a, u64 b) { return a > b ? a : b; });
        if (rank == 0 && tid == 0) job.out[row] = best == 0 ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
        r.barrier();  // nobody leaves while others read its numbers
        return;
    }
    float largest = -INFINITY;
    r.each([&](uint32_t, float l) { largest = fmaxf(largest, l); });  // NaN loses
    most = (uint32_t)r.reduce(key_of(largest), [](u64 a, u64 b) { return a > b ? a : b; });
    if (most == 0u) {
        if (rank == 0 && tid == 0) job.out[row] = -1;
        r.barrier();
        return;
    }
    const Weigher weigh(sh.table, most, rule.inverse_T, job.shift);
    // halves, so that no difference of finite logits overflows
    const float half_top = 0.5f * logit_of(most), steps_per_half = (float)fmin(64.0 * rule.inverse_T, 3e38);
    // 2048 steps of 1/32 down from the largest logit, in fp32: monotone, and weights below 2^-50 are in the last one.
    // It is not below any `behind` for NaN and -inf, nor for logits so far away that they weigh nothing; +inf, whose
    // distance is not a number either, is told apart.
    const auto distance = [half_top, steps_per_half](float l) { return fmaf(l, -0.5f, half_top) * steps_per_half; };
    const auto step_of = [distance](float l) { return l == INFINITY ? 0 : (int)fminf(distance(l), (float)(BINS - 1)); };
    const auto coarse = [step_of](uint32_t key) { return step_of(logit_of(key)); };
    const auto within = [distance](float l, float behind) { return distance(l) < behind || l == INFINITY; };
    // min-p keeps nothing behind this step; one step more for the rounding of the distance
    const double ratio = (double)rule.least / (double)(1ull << job.shift);
    const int last_step = rule.least > 0 && !weigh.infinite ? (int)fmin(-log(ratio) * 32.0 + 2.0, BINS - 1.0) : BINS - 1;
    Cut cut{1u, FULL};  // everything but key 0
    bool cut_found = false;
    bool listed = false;  // the blocks' lists hold all that can be drawn
    if (rule.top_k > 0 && rule.top_k <= LIST) {
        int at;
        u64 before, total, goal;
        r.clear_histogram();
        r.each([&](uint32_t, float l) {
            if (l > -INFINITY) atomicAdd(&sh.low[step_of(l)], 1u);
        });
        const u64 k = (u64)rule.top_k;
        const bool cuts = r.find_step([k](u64) { return k; }, at, before, total, goal);
        const float behind = cuts && at < BINS - 1 ? (float)(at + 1) : INFINITY;
        if (r.collect([within, behind](uint32_t, float l) { return within(l, behind); })) {
            const uint32_t n = r.gather(false);
            if (n <= LIST) {
                if (rank == 0) {
                    const int64_t id = Row<T>::finish(r, n, (uint32_t)rule.top_k, rule, weigh);
                    if (tid == 0) job.out[row] = id;
                }
                r.barrier();  // nobody leaves while others read its numbers
                return;
            }
        }
    } else if (rule.top_k == 0 && rule.top_p < 1.0) {
        int at;
        u64 before, total, goal;
        r.clear_histogram();
        // lighter than (1 - p) / V of the largest: together no more than 1 - p of the total, so the border lies above them
        const float light = (float)fmin(log((double)job.V / (1.0 - rule.top_p)) * 32.0 + 2.0, (double)(BINS - 1));
        u64 tail = 0;
        r.each4([&](uint32_t, uint32_t, const float (&l)[4]) {
            u64 w[4];
            int b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = weigh.of(l[e]);
                b[e] = 0;
                if (within(l[e], light)) b[e] = step_of(l[e]);
                else {
                    tail += w[e];
                    w[e] = 0;
                }
            }
            r.add_weights(b, w);
        });
        tail = warp_sum(tail);
        if (r.lane == 0 && tail > 0) atomicAdd(&sh.tail, tail);
        const double share = rule.top_p;
        if (r.find_step([share](u64 all) { return share_of(share, all); }, at, before, total, goal)) {
            const int end = at < last_step ? at + 1 : last_step + 1;
            const float behind = end < BINS ? (float)end : INFINITY;
            listed = r.collect([within, behind](uint32_t, float l) { return within(l, behind); });
            if (listed && at <= last_step) {
                cut = Row<T>::cut_in_list(r, at, before, goal, weigh, coarse);
                listed = cut.key != 0u;
            }
            if (!listed)
                cut = Row<T>::cut_in(r, at, before, goal, [](uint32_t, uint32_t key) { return key != 0u; }, weigh, coarse);
            cut_found = true;
        }
    } else if (rule.top_k == 0 && rule.least > 0) {
        const float behind = last_step + 1 < BINS ? (float)(last_step + 1) : INFINITY;
        listed = r.collect([within, behind](uint32_t, float l) { return within(l, behind); });
    }
    // many candidates: the cuts one after the other, then the draw over the row
    if (rule.top_k > 0) {
        const u64 k = (u64)rule.top_k;
        Cut c;
        if (r.cut([](uint32_t, uint32_t key) { return key != 0u; }, [](uint32_t) { return (u64)1; }, coarse,
                  [k](u64) { return k; }, c))
            cut = c;
    }
    if (rule.top_p < 1.0 && !cut_found) {
        const Cut held = cut;
        const double p = rule.top_p;
        Cut c;
        if (r.cut([held](uint32_t i, uint32_t key) { return held.holds(key, i); }, weigh, coarse,
                  [p](u64 total) { return share_of(p, total); }, c))
            cut = c;
    }
    // the draw: from the lists, if they hold all; else every warp sums a run of the slice, and the run that holds the point
    // is cut up again
    const u64 least = rule.least;
    const float border = cut.last == FULL ? -INFINITY : logit_of(cut.key);  // most logits are told by one comparison
    const auto kept = [&](uint32_t i, float l) {
        const u64 w = weigh.of(l);
        return cut.holds(key_of(l), i) && w >= least ? w : 0ull;
    };
    uint32_t lo = from, hi = to;
    u64 point = 0;
    if (listed) {
        const auto drawn = Row<T>::draw_in_list(r, V, cut, least, rule.u, weigh);
        lo = drawn.from;
        hi = drawn.to;
        point = drawn.point;
    }
    __syncthreads();
    const bool here = !listed || rank == 0;
    for (int level = listed ? 1 : 0; here; ++level) {
        if (level > 0 && hi - lo <= 32) {
            if (r.warp == 0) {
                const u64 mine = lo + r.lane < hi ? kept(lo + r.lane, dl_to_float(r.logits[lo + r.lane])) : 0ull;
                const u64 upto = warp_inclusive(mine, r.lane);
                const uint32_t hit = __ballot_sync(FULL, upto > point);
                if (r.lane == 0) job.out[row] = (int64_t)lo + __ffs(hit) - 1;
            }
            break;
        }
        const uint32_t run = (hi - lo + WARPS - 1) / WARPS;
        const uint32_t begin = lo + r.warp * run < hi ? lo + r.warp * run : hi, end = begin + run < hi ? begin + run : hi;
        u64 sum = 0;
        for (uint32_t i = begin + r.lane; i < end; i += 128) {
            float l[4];
            bool any = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                l[k] = i + 32 * k < end ? dl_to_float(r.logits[i + 32 * k]) : NAN;
                any |= l[k] >= border;
            }
            if (!any) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (l[k] >= border) sum += kept(i + 32 * k, l[k]);
        }
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
    // twice as many blocks per row while they keep 6144 classes each and there is an SM for every one: each has its own
    // histograms, lists and barriers to go through (top-p .95, 8 x 32000: 31 us with four blocks a row, 35 with two or eight;
    // 64 x 32000: 34 us with two, 41 with four; 1 x 8192: 18 with one, 23 with two)
    int ranks = 1;
    while (ranks < MAX_CLUSTER && job.V >= (int64_t)12288 * ranks && job.R * ranks * 2 <= DL_NUM_SMS) ranks *= 2;
    if (job.R * ranks > 0x7fffffff) return DL_ERR_TOO_LARGE;
    const int vectors = dl_address(logits) % 16 == 0 && (job.R == 1 || job.pitch * (int64_t)sizeof(T) % 16 == 0);
    const uint32_t slice = (uint32_t)(dl_ceil_div(dl_ceil_div(job.V, ranks), 8) * 8);  // whole vectors
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
    if (!dl_allow(reinterpret_cast<const void*>(kernel), limits, sizeof(Shared))) return DL_ERR_LAUNCH;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, src, job, ranks, slice, vectors);
    return e == cudaSuccess ? dl_launch_status() : DL_ERR_LAUNCH;
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
    DL_REQUIRE_ALIGNED(temperature, 4);
    DL_REQUIRE_ALIGNED(top_k, 4);
    DL_REQUIRE_ALIGNED(top_p, 4);
    DL_REQUIRE_ALIGNED(min_p, 4);
    DL_REQUIRE_ALIGNED(out, 8);
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
