// Dropout whose mask is a function of (seed, offset, element index) and is never stored: the backward pass
// calls the same kernel on the gradient.
//
// Element i takes word i % 4 of the block Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers:
// as easy as 1, 2, 3", 2011) computes for the counter (i / 4, offset) under the key `seed`, and is dropped when that
// word is below p * 2^32: the mask depends neither on the type nor on the launch.
//
// Every element is read and written once.  16-bit types wait for the generator: 18 wide products per four elements keep the
// pipe that multiplies wide 65 % busy, DRAM 45 %, and a thread loads, computes and stores once, so that the two overlap only
// across blocks: 65.5 M bf16 elements, 262 MB, take 63 us or 4.2 TB/s.  The fp32 kernel moves twice the bytes per product and
// runs at the copy rate of 6.5 TB/s.  A thread takes whole Philox blocks: two accesses of 16 bytes, so that the loads of the
// second are under way during the rounds of the first.
#include "elements.cuh"

namespace {

constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u;

struct DropoutRule {
    uint32_t key[20];  // the two round keys of every round, on their way to the threads as constants
    uint64_t offset;
    uint32_t threshold;  // words below it drop their element
    float scale;
};

__device__ __forceinline__ uint32_t high(uint64_t x) { return (uint32_t)(x >> 32); }
__device__ __forceinline__ uint64_t wide(uint32_t a, uint32_t b) { return (uint64_t)a * b; }

// What the first two rounds compute for every block of one CTA alike: the counter words 1 to 3 are the same there,
// which saves 2 of the 20 wide products per block.
struct PhiloxStart {
    uint32_t b1, c2_high, d2;
    uint32_t offset_high;
    __device__ __forceinline__ PhiloxStart(const DropoutRule& r, uint64_t offset, uint32_t q_high) {
        const uint64_t s = wide((uint32_t)offset, M1);
        offset_high = high(offset);
        b1 = (uint32_t)s;
        const uint64_t f = wide(high(s) ^ q_high ^ r.key[0], M0);
        c2_high = high(f);
        d2 = (uint32_t)f;
    }
};

// the four words of the block whose low counter word is q
__device__ __forceinline__ void philox_block(const DropoutRule& r, const PhiloxStart& u, uint32_t q, uint32_t (&w)[4]) {
    uint64_t f = wide(q, M0);
    const uint32_t c1 = high(f) ^ u.offset_high ^ r.key[1];
    uint64_t s = wide(c1, M1);
    uint32_t a = high(s) ^ u.b1 ^ r.key[2], b = (uint32_t)s, c = u.c2_high ^ (uint32_t)f ^ r.key[3], d = u.d2;
#pragma unroll
    for (int k = 4; k < 20; k += 2) {
        f = wide(a, M0);
        s = wide(c, M1);
        a = high(s) ^ b ^ r.key[k];
        b = (uint32_t)s;
        c = high(f) ^ d ^ r.key[k + 1];
        d = (uint32_t)f;
    }
    w[0] = a;
    w[1] = b;
    w[2] = c;
    w[3] = d;
}

// STEP elements (whole Philox blocks) per item, ITEMS items in flight per thread; VECTOR: x and out are aligned for
// one access per item.  A CTA covers 256 * ITEMS * STEP / 4 blocks, a power of two: their high counter word is one.
template <typename T, int STEP, int ITEMS, bool VECTOR>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* x, T* out, int64_t count, const __grid_constant__ DropoutRule rule, const int64_t* counter) {
    constexpr int CHUNK = 256 * ITEMS * STEP;
    const int64_t base = (int64_t)blockIdx.x * CHUNK;
    const uint64_t offset = rule.offset + (counter != nullptr ? (uint64_t)*counter : 0);
    const PhiloxStart start(rule, offset, high((uint64_t)base / 4));
    const uint32_t q0 = (uint32_t)((uint64_t)base / 4);
    const bool whole = VECTOR && base + CHUNK <= count;  // uniform: only the last CTA of a ragged tensor is not
    DlVec<T, STEP> in[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = base + (k * 256 + threadIdx.x) * STEP;
        if (whole) {
            in[k] = *reinterpret_cast<const DlVec<T, STEP>*>(x + i);
        } else {
#pragma unroll
            for (int e = 0; e < STEP; ++e)
                if (i + e < count) in[k].v[e] = x[i + e];
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const uint32_t at = (uint32_t)(k * 256 + threadIdx.x) * STEP;
        float f[STEP];
        dl_unpack(in[k], f);
#pragma unroll
        for (int b = 0; b < STEP / 4; ++b) {
            uint32_t w[4];
            philox_block(rule, start, q0 + at / 4 + b, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[4 * b + e] = w[e] < rule.threshold ? 0.0f : f[4 * b + e] * rule.scale;
        }
        dl_pack(f, in[k]);
        if (whole) {
            *reinterpret_cast<DlVec<T, STEP>*>(out + base + at) = in[k];
        } else {
#pragma unroll
            for (int e = 0; e < STEP; ++e)
                if (base + at + e < count) out[base + at + e] = in[k].v[e];
        }
    }
}

__global__ void counter_draw_kernel(int64_t* counter, int64_t* drawn) {
    *drawn = (int64_t)atomicAdd(reinterpret_cast<unsigned long long*>(counter), 1ull);
}

template <typename T>
int launch_dropout(const void* x, void* out, int64_t count, const DropoutRule& rule, const int64_t* counter,
                   cudaStream_t s) {
    constexpr int STEP = 16 / sizeof(T), ITEMS = 2;
    const int64_t blocks = dl_ceil_div(count, (int64_t)256 * ITEMS * STEP);
    if (blocks > 0x7fffffff) return DL_ERR_TOO_LARGE;
    const T* src = static_cast<const T*>(x);
    T* dst = static_cast<T*>(out);
    if ((dl_address(x) | dl_address(out)) % 16 == 0)
        dropout_kernel<T, STEP, ITEMS, true><<<(unsigned)blocks, 256, 0, s>>>(src, dst, count, rule, counter);
    else
        dropout_kernel<T, STEP, ITEMS, false><<<(unsigned)blocks, 256, 0, s>>>(src, dst, count, rule, counter);
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
    DL_REQUIRE_ALIGNED(counter, 8);
    cudaStream_t s = dl_cast(stream);
    const uint64_t threshold = (uint64_t)(p * 4294967296.0 + 0.5);  // 0 .. 2^32
    if (threshold > 0xFFFFFFFFull)  // everything is dropped; 0.0 is all zero bits in every type
        return cudaMemsetAsync(out, 0, (size_t)(count * dl_dtype_size(dtype)), s) == cudaSuccess ? DL_OK : DL_ERR_LAUNCH;
    DropoutRule rule;
    rule.offset = (uint64_t)offset;
    rule.threshold = (uint32_t)threshold;
    rule.scale = (float)(1.0 / (1.0 - p));
    uint32_t k0 = (uint32_t)(uint64_t)seed, k1 = (uint32_t)((uint64_t)seed >> 32);
    for (int r = 0; r < 10; ++r) {
        rule.key[2 * r] = k0;
        rule.key[2 * r + 1] = k1;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    if (dtype == DL_DTYPE_F32) return launch_dropout<float>(x, out, count, rule, counter, s);
    if (dtype == DL_DTYPE_BF16) return launch_dropout<__nv_bfloat16>(x, out, count, rule, counter, s);
    return launch_dropout<__half>(x, out, count, rule, counter, s);
}

DL_EXPORT int dl_counter_draw(int64_t* counter, int64_t* drawn, dl_stream_t stream) {
    DL_REQUIRE(counter && drawn && counter != drawn);
    DL_REQUIRE_ALIGNED(counter, 8);
    DL_REQUIRE_ALIGNED(drawn, 8);
    counter_draw_kernel<<<1, 1, 0, dl_cast(stream)>>>(counter, drawn);
    return dl_launch_status();
}
