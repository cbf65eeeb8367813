// Dropout from a counter-based generator, forward and backward:
//
//   y = residual + (kept ? x * 2^16 / (2^16 - drop) : 0),  kept: draw >= drop
//   dx = kept ? dy * 2^16 / (2^16 - drop) : 0
//
// An element's draw is 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw:
// Parallel random numbers, as easy as 1, 2, 3; 2011), keyed by the seed, whose counter
// is the element's number / 8 and the call's `site`: eight draws a counter. No mask
// is stored; the backward pass draws again. The probability is held in steps of
// 2^-16 and the gain is that step's own, so the mean is kept.
//
// Memory bounds it: eight draws a block make some 20 vector instructions an element
// (with the whole 32 bits for each it would be the generator). 65280 x 1024 bfloat16 onto a
// float32 residual 121 us (5.5 TB/s), and dx from its float32 gradient 69 (5.8). Two and
// four counters a thread: 2 and 9% more; 64 x 256 float32: 2.6, the launch.
#include "mg_types.h"

namespace mg {

constexpr int kDropThreads = 256;
constexpr int kDropEach = 8;                      // elements a counter, and a thread
constexpr int64_t kDropStreamBytes = 32 << 20;    // the L2 caches' together

struct DropArgs {
    const void *x, *residual;
    void *out;
    int64_t n;
    const int64_t *seed_at;                       // NULL: seed
    uint64_t seed, site;
    uint32_t drop;
    float gain;
    int32_t stream;
};

struct U32x4 {
    uint32_t v[4];
};

// One Philox4x32-10 block.
__device__ __forceinline__ U32x4 philox4x32(uint64_t index, uint64_t site, uint64_t seed) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32);
    uint32_t c2 = (uint32_t)site, c3 = (uint32_t)(site >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {c0, c1, c2, c3};
}

// In and Out: the types of x and of the result, which the residual shares.
template <typename In, typename Out, bool kResidual>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(DropArgs a) {
    const In *x = static_cast<const In *>(a.x);
    const Out *residual = static_cast<const Out *>(a.residual);
    Out *out = static_cast<Out *>(a.out);
    const uint64_t seed = a.seed_at ? (uint64_t)*a.seed_at : a.seed;
    const int64_t index = (int64_t)blockIdx.x * kDropThreads + threadIdx.x, at = index * kDropEach;
    if (at >= a.n) return;
    float f[kDropEach] = {}, r[kDropEach] = {};
    const bool whole = at + kDropEach <= a.n;
    if (whole) {
        load_vec<In, kDropEach>(x + at, f);
        if constexpr (kResidual) load_vec<Out, kDropEach>(residual + at, r);
    } else {
#pragma unroll
        for (int i = 0; i < kDropEach; ++i) {
            if (at + i >= a.n) continue;
            f[i] = (float)x[at + i];
            if constexpr (kResidual) r[i] = (float)residual[at + i];
        }
    }
    const U32x4 word = philox4x32((uint64_t)index, a.site, seed);
#pragma unroll
    for (int i = 0; i < kDropEach; ++i) {
        const uint32_t draw = i % 2 ? word.v[i / 2] >> 16 : word.v[i / 2] & 0xffffu;
        // Selected: an infinity or NaN that is dropped is gone.
        const float y = draw >= a.drop ? f[i] * a.gain : 0.f;
        f[i] = kResidual ? r[i] + y : y;
    }
    if (!whole) {
#pragma unroll
        for (int i = 0; i < kDropEach; ++i)
            if (at + i < a.n) out[at + i] = (Out)f[i];
    } else if (a.stream) {
        store_vec<Out, kDropEach, true>(out + at, f);
    } else {
        store_vec<Out, kDropEach>(out + at, f);
    }
}

template <typename In, typename Out>
static void dropout_go(const DropArgs &a, unsigned grid, hipStream_t st) {
    if constexpr (std::is_same<In, Out>::value || std::is_same<Out, float>::value) {
        if (a.residual) {
            dropout_kernel<In, Out, true><<<grid, kDropThreads, 0, st>>>(a);
            return;
        }
    }
    dropout_kernel<In, Out, false><<<grid, kDropThreads, 0, st>>>(a);
}

}  // namespace mg

extern "C" int32_t mg_dropout(int64_t n, int32_t dtype, const void *x, int32_t out_dtype,
                              const void *residual, void *out, int32_t drop, uint64_t seed,
                              const int64_t *seed_at, uint64_t site, mg_stream_t stream) {
    using namespace mg;
    MG_REQUIRE(type_known(dtype) && type_known(out_dtype), "mg_dropout: type codes %d and %d",
               dtype, out_dtype);
    MG_REQUIRE(dtype == out_dtype || out_dtype == MG_F32 || dtype == MG_F32,
               "mg_dropout: one of two types must be float32");
    MG_REQUIRE(!residual || dtype == out_dtype || out_dtype == MG_F32,
               "mg_dropout: a residual is float32 or of the input's type");
    MG_REQUIRE(drop >= 0 && drop <= 65536, "mg_dropout: %d of 65536 elements dropped", drop);
    MG_REQUIRE(n >= 0, "mg_dropout: %lld elements", (long long)n);
    const int64_t grid = ceil_div(n, kDropThreads * kDropEach);
    MG_REQUIRE(grid_fits(grid, kDropThreads), "mg_dropout: %lld elements are too many for one call",
               (long long)n);
    if (n == 0) return MG_OK;
    MG_REQUIRE(x && out, "mg_dropout: a pointer is NULL");
    DropArgs a{};
    a.x = x, a.residual = residual, a.out = out, a.n = n;
    a.seed_at = seed_at, a.seed = seed, a.site = site;
    a.drop = (uint32_t)drop;
    a.gain = drop == 65536 ? 0.f : (float)(65536.0 / (65536 - drop));
    a.stream = n * (out_dtype == MG_F32 ? 4 : 2) > kDropStreamBytes;
    hipStream_t st = as_stream(stream);
    TimedScope ts("dropout", st);
    const unsigned g = (unsigned)grid;
    if (dtype == MG_F32) {
        if (out_dtype == MG_F32)
            dropout_go<float, float>(a, g, st);
        else if (out_dtype == MG_BF16)
            dropout_go<float, bf16_t>(a, g, st);
        else
            dropout_go<float, f16_t>(a, g, st);
    } else if (dtype == MG_BF16) {
        if (out_dtype == MG_F32)
            dropout_go<bf16_t, float>(a, g, st);
        else
            dropout_go<bf16_t, bf16_t>(a, g, st);
    } else {
        if (out_dtype == MG_F32)
            dropout_go<f16_t, float>(a, g, st);
        else
            dropout_go<f16_t, f16_t>(a, g, st);
    }
    MG_LAUNCHED("dropout_kernel");
    return MG_OK;
}
