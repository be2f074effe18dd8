// Dropout whose mask is a function of (seed, offset, element index) and is never stored: the backward pass
// calls the same kernel on the gradient.
//
// Element i takes word i % 4 of the block Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers:
// as easy as 1, 2, 3", 2011) computes for the counter (i / 4, offset) under the key `seed`, and is dropped when that
// word is below p * 2^32: the mask depends neither on the type nor on the launch.
#include "elements.cuh"

namespace {

struct Philox {
    uint32_t k0, k1, c2, c3;
    // the four words of block q
    __device__ __forceinline__ void block(uint64_t q, uint32_t (&w)[4]) const {
        uint32_t a = (uint32_t)q, b = (uint32_t)(q >> 32), c = c2, d = c3, key0 = k0, key1 = k1;
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const uint64_t first = (uint64_t)a * 0xD2511F53u, second = (uint64_t)c * 0xCD9E8D57u;
            a = (uint32_t)(second >> 32) ^ b ^ key0;
            b = (uint32_t)second;
            c = (uint32_t)(first >> 32) ^ d ^ key1;
            d = (uint32_t)first;
            key0 += 0x9E3779B9u;
            key1 += 0xBB67AE85u;
        }
        w[0] = a;
        w[1] = b;
        w[2] = c;
        w[3] = d;
    }
};

struct DropoutRule {
    uint64_t seed, offset;
    uint32_t highest_dropped;  // words up to and including this one drop their element
    int drops;                 // 0: nothing is dropped
    float scale;
};

template <typename T>
__device__ __forceinline__ T drop(const DropoutRule& rule, uint32_t word, T x) {
    const bool gone = rule.drops && word <= rule.highest_dropped;
    return gone ? dl_from_float<T>(0.0f) : dl_from_float<T>(dl_to_float(x) * rule.scale);
}

// W elements per access, ITEMS accesses in flight per thread; W is a multiple of 4, or 1 (no common alignment)
template <typename T, int W, int ITEMS>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* x, T* out, int64_t count, DropoutRule rule, const int64_t* counter) {
    constexpr int STEP = W == 1 ? 4 : W;  // a thread's elements always are whole Philox blocks
    if (counter != nullptr) rule.offset += (uint64_t)*counter;
    const Philox rng{(uint32_t)rule.seed, (uint32_t)(rule.seed >> 32), (uint32_t)rule.offset,
                     (uint32_t)(rule.offset >> 32)};
    const int64_t first = ((int64_t)blockIdx.x * ITEMS * 256 + threadIdx.x) * STEP;
    DlVec<T, STEP> in[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = first + (int64_t)k * 256 * STEP;
        if (W > 1 && i + STEP <= count) {
            in[k] = *reinterpret_cast<const DlVec<T, STEP>*>(x + i);
        } else {
#pragma unroll
            for (int e = 0; e < STEP; ++e)
                if (i + e < count) in[k].v[e] = x[i + e];
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = first + (int64_t)k * 256 * STEP;
        if (i >= count) break;
#pragma unroll
        for (int b = 0; b < STEP / 4; ++b) {
            uint32_t w[4];
            rng.block((uint64_t)i / 4 + b, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) in[k].v[4 * b + e] = drop(rule, w[e], in[k].v[4 * b + e]);
        }
        if (W > 1 && i + STEP <= count) {
            *reinterpret_cast<DlVec<T, STEP>*>(out + i) = in[k];
        } else {
#pragma unroll
            for (int e = 0; e < STEP; ++e)
                if (i + e < count) out[i + e] = in[k].v[e];
        }
    }
}

__global__ void counter_draw_kernel(int64_t* counter, int64_t* drawn) {
    *drawn = (int64_t)atomicAdd(reinterpret_cast<unsigned long long*>(counter), 1ull);
}

template <typename T>
int launch_dropout(const void* x, void* out, int64_t count, const DropoutRule& rule, const int64_t* counter,
                   cudaStream_t s) {
    constexpr int W = 16 / sizeof(T), ITEMS = 2;
    const T* src = static_cast<const T*>(x);
    T* dst = static_cast<T*>(out);
    if ((dl_address(x) | dl_address(out)) % 16 == 0) {
        const int64_t blocks = dl_ceil_div(count, (int64_t)256 * ITEMS * W);
        if (blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
        dropout_kernel<T, W, ITEMS><<<(unsigned)blocks, 256, 0, s>>>(src, dst, count, rule, counter);
    } else {
        const int64_t blocks = dl_ceil_div(count, (int64_t)256 * ITEMS * 4);
        if (blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
        dropout_kernel<T, 1, ITEMS><<<(unsigned)blocks, 256, 0, s>>>(src, dst, count, rule, counter);
    }
    return dl_launch_status();
}

}  // namespace

DL_EXPORT int dl_dropout(const void* x, void* out, int64_t count, int64_t dtype, double p, int64_t seed, int64_t offset,
                         const int64_t* counter, dl_stream_t stream) {
    DL_REQUIRE(count >= 0 && dl_dtype_known(dtype) && p >= 0.0 && p <= 1.0);
    if (count == 0) return DL_OK;
    DL_REQUIRE(x && out);
    DL_REQUIRE_ALIGNED(x, dl_dtype_size(dtype));
    DL_REQUIRE_ALIGNED(out, dl_dtype_size(dtype));
    const uint64_t threshold = (uint64_t)(p * 4294967296.0 + 0.5);  // 0 .. 2^32
    DropoutRule rule;
    rule.seed = (uint64_t)seed;
    rule.offset = (uint64_t)offset;
    rule.drops = threshold > 0;
    rule.highest_dropped = (uint32_t)(threshold - 1);
    rule.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    cudaStream_t s = dl_cast(stream);
    if (dtype == DL_DTYPE_F32) return launch_dropout<float>(x, out, count, rule, counter, s);
    if (dtype == DL_DTYPE_BF16) return launch_dropout<__nv_bfloat16>(x, out, count, rule, counter, s);
    return launch_dropout<__half>(x, out, count, rule, counter, s);
}

DL_EXPORT int dl_counter_draw(int64_t* counter, int64_t* drawn, dl_stream_t stream) {
    DL_REQUIRE(counter && drawn && counter != drawn);
    counter_draw_kernel<<<1, 1, 0, dl_cast(stream)>>>(counter, drawn);
    return dl_launch_status();
}
