// Rotary positions: pair i of a head's first 2 P elements is turned by the
// angle position * frequency_i,
//
//   a' = a cos t - b sin t,  b' = b cos t + a sin t,
//
// the pair being elements (i, P + i) ("half") or (2i, 2i + 1) ("interleaved");
// the rest of the head is copied. The adjoint turns by -t, so the backward pass
// is the same kernel on the gradients.
//
// The angle's whole turns leave it in float64 (position * frequency / 2 pi,
// exact to 2^-53 of itself), so a token at position 10^6 is turned as exactly
// as one at 10; sine and cosine are then float32, formed once per token and
// pair and shared by all heads through LDS. What is left is memory: queries and
// keys are read once and written once, in one launch. A thread asks for all its
// elements before it forms its cosines, whose chain (position, float64 product,
// polynomial) is as long as a trip to memory: 10000 tokens of 32 heads of 64
// bfloat16 16 us (5.1 TB/s; 23 us with the cosines first), 32640 of 20 heads of
// 128 float32, a quarter of them elsewhere in their rows, 125 us (5.3 TB/s).
#include "mg_types.h"

namespace mg {

constexpr int kRotThreads = 256;
constexpr int kRotUnits = 4;               // units a thread
constexpr int kRotMaxPairs = 512;          // heads of up to 1024 elements
constexpr int kRotTable = 1024;            // cosines and sines held by a workgroup
constexpr int64_t kRotStreamBytes = 32 << 20;     // the L2 caches' together

struct RotArgs {
    const void *x[2];
    void *out[2];
    int64_t tok_stride[2], head_stride[2], out_tok_stride[2];
    int32_t heads[2];                      // heads[1] may be 0
    int64_t tokens;
    int32_t dim, pairs, axes;
    const void *positions;
    const double *freq;
    // A workgroup has tokens_at_once tokens, or one of `runs` runs of one token's
    // units.
    int32_t tokens_at_once, runs;
    float sign;
};

// kStream: results larger than the L2 caches pass by them (32640 tokens of 20
// heads of 128 float32, forward and backward: 268 us, with streaming stores 258;
// streaming loads gained nothing there and cost a third on smaller inputs).
template <bool kStream, typename T, int V>
__device__ __forceinline__ void copy_out(T *to, const T (&from)[V]) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if constexpr (kStream && V > 1) {
        vec t;
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = from[i];
        __builtin_nontemporal_store(t, reinterpret_cast<vec *>(to));
    } else {
        __builtin_memcpy(to, from, sizeof(from));
    }
}

// A unit is V neighbouring elements of a head's rotated part together with
// their partners (kHalf), V / 2 whole pairs (interleaved), or V elements that
// are copied. V = 16 bytes' worth where units do not straddle the parts'
// borders, else 1 (2 interleaved).
template <typename T, typename P, int V, bool kHalf, bool kStream>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a) {
    __shared__ float2 s_cs[kRotTable];
    const int run = a.runs > 1 ? blockIdx.x % a.runs : 0;
    const int64_t tok0 = (int64_t)(blockIdx.x / a.runs) * a.tokens_at_once;
    const int n_tok = (int)min((int64_t)a.tokens_at_once, a.tokens - tok0);
    const int rot_units = (kHalf ? a.pairs : 2 * a.pairs) / V;
    const int units = rot_units + (a.dim - 2 * a.pairs) / V;
    const int per_tok = (a.heads[0] + a.heads[1]) * units;
    struct Unit {
        const T *x;
        T *out;
        int pair;      // of the workgroup's table; -1: copied, -2: none
    };
    Unit unit[kRotUnits];
    T v[kRotUnits][V], w[kHalf ? kRotUnits : 1][V];
#pragma unroll
    for (int j = 0; j < kRotUnits; ++j) {
        const int i = (run * kRotUnits + j) * kRotThreads + (int)threadIdx.x;
        unit[j].pair = -2;
        if (i >= n_tok * per_tok) continue;
        const int tok = i / per_tok, r = i - tok * per_tok;
        int h = r / units;
        const int u = r - h * units;
        const int which = h >= a.heads[0];
        h -= which ? a.heads[0] : 0;
        const bool turned = u < rot_units;
        const int at = turned ? u * V : 2 * a.pairs + (u - rot_units) * V;
        unit[j].pair = turned ? tok * a.pairs + (kHalf ? at : at / 2) : -1;
        unit[j].x = static_cast<const T *>(a.x[which]) + (tok0 + tok) * a.tok_stride[which] +
                    h * a.head_stride[which] + at;
        unit[j].out = static_cast<T *>(a.out[which]) + (tok0 + tok) * a.out_tok_stride[which] +
                      (int64_t)h * a.dim + at;
        __builtin_memcpy(v[j], unit[j].x, sizeof(v[j]));
        if (kHalf && turned) __builtin_memcpy(w[j], unit[j].x + a.pairs, sizeof(w[j]));
    }
    const P *pos = static_cast<const P *>(a.positions);
    const int per_axis = a.pairs / a.axes;
    for (int i = threadIdx.x; i < n_tok * a.pairs; i += kRotThreads) {
        const int tok = i / a.pairs, pair = i - tok * a.pairs;
        const double turns = (double)pos[(tok0 + tok) * a.axes + pair / per_axis] * a.freq[pair] *
                             0.15915494309189533577;
        float sn, cs;
        // turns - rint(turns) in [-1/2, 1/2]; sincospi takes half turns.
        sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
        s_cs[i] = make_float2(cs, a.sign * sn);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRotUnits; ++j) {
        const Unit &m = unit[j];
        if (m.pair == -2) continue;
        if (m.pair >= 0) {
            if constexpr (kHalf) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float2 c = s_cs[m.pair + k];
                    const float p = (float)v[j][k], q = (float)w[j][k];
                    v[j][k] = (T)(p * c.x - q * c.y);
                    w[j][k] = (T)(q * c.x + p * c.y);
                }
                copy_out<kStream>(m.out + a.pairs, w[j]);
            } else {
#pragma unroll
                for (int k = 0; k + 1 < V; k += 2) {
                    const float2 c = s_cs[m.pair + k / 2];
                    const float p = (float)v[j][k], q = (float)v[j][k + 1];
                    v[j][k] = (T)(p * c.x - q * c.y);
                    v[j][k + 1] = (T)(q * c.x + p * c.y);
                }
            }
        }
        copy_out<kStream>(m.out, v[j]);
    }
}

// Cuts the tokens among workgroups for units of V elements, and launches.
template <typename T, typename P, int V, bool kHalf>
static bool rotary_go(RotArgs a, hipStream_t st) {
    const int units = ((kHalf ? a.pairs : 2 * a.pairs) + a.dim - 2 * a.pairs) / V;
    const int64_t per_tok = (int64_t)(a.heads[0] + a.heads[1]) * units;
    constexpr int64_t kAll = kRotUnits * kRotThreads;
    int64_t at_once = kAll / per_tok;
    if (at_once > kRotTable / a.pairs) at_once = kRotTable / a.pairs;
    // A few tokens are spread over the GPU.
    if (at_once > ceil_div(a.tokens, 512)) at_once = ceil_div(a.tokens, 512);
    a.tokens_at_once = (int32_t)(at_once < 1 ? 1 : at_once);
    a.runs = (int32_t)ceil_div(a.tokens_at_once * per_tok, kAll);
    const int64_t grid = ceil_div(a.tokens, a.tokens_at_once) * a.runs;
    if (!grid_fits(grid, kRotThreads)) return false;
    const int64_t bytes = a.tokens * (a.heads[0] + a.heads[1]) * a.dim * (int64_t)sizeof(T);
    if (bytes > kRotStreamBytes)
        rotary_kernel<T, P, V, kHalf, true><<<(unsigned)grid, kRotThreads, 0, st>>>(a);
    else
        rotary_kernel<T, P, V, kHalf, false><<<(unsigned)grid, kRotThreads, 0, st>>>(a);
    return true;
}

template <typename T, typename P>
static bool rotary_launch(const RotArgs &a, bool half, hipStream_t st) {
    constexpr int V = kVec<T>;
    const int rest = a.dim - 2 * a.pairs;
    const bool wide = (half ? a.pairs : 2 * a.pairs) % V == 0 && rest % V == 0;
    if (half) return wide ? rotary_go<T, P, V, true>(a, st) : rotary_go<T, P, 1, true>(a, st);
    return wide ? rotary_go<T, P, V, false>(a, st) : rotary_go<T, P, 2, false>(a, st);
}

}  // namespace mg

extern "C" int32_t mg_rotary(int64_t tokens, int32_t dtype, const void *q, int64_t q_token_stride,
                             int64_t q_head_stride, int32_t q_heads, const void *k,
                             int64_t k_token_stride, int64_t k_head_stride, int32_t k_heads,
                             int32_t dim, const void *positions, int32_t positions_64,
                             int32_t axes, const double *frequencies, int32_t pairs,
                             int32_t interleaved, int32_t inverse, void *q_out, void *k_out,
                             mg_stream_t stream) {
    using namespace mg;
    MG_REQUIRE(type_known(dtype), "mg_rotary: type code %d", dtype);
    MG_REQUIRE(tokens >= 0 && tokens < (int64_t(1) << 31), "mg_rotary: %lld tokens",
               (long long)tokens);
    MG_REQUIRE(q_heads >= 1 && k_heads >= 0 && q_heads <= 65536 && k_heads <= 65536,
               "mg_rotary: %d and %d heads", q_heads, k_heads);
    MG_REQUIRE(pairs >= 1 && 2 * pairs <= dim && pairs <= kRotMaxPairs && dim <= 65536,
               "mg_rotary: %d frequencies turn %d elements; heads have %d, and at most %d "
               "frequencies are taken", pairs, 2 * pairs, dim, kRotMaxPairs);
    MG_REQUIRE(interleaved == 0 || dim % 2 == 0,
               "mg_rotary: interleaved pairs need an even head dimension, got %d", dim);
    MG_REQUIRE(axes >= 1 && pairs % axes == 0,
               "mg_rotary: %d frequencies do not divide among %d axes", pairs, axes);
    // A workgroup's units are numbered in 32 bits.
    MG_REQUIRE((int64_t)(q_heads + k_heads) * dim <= (int64_t(1) << 30),
               "mg_rotary: tokens of %d heads of %d elements are too long", q_heads + k_heads,
               dim);
    if (tokens == 0) return MG_OK;
    MG_REQUIRE(q && q_out && positions && frequencies && (k_heads == 0 || (k && k_out)),
               "mg_rotary: a pointer is NULL");
    RotArgs a{};
    a.x[0] = q, a.x[1] = k, a.out[0] = q_out, a.out[1] = k_out;
    a.tok_stride[0] = q_token_stride, a.tok_stride[1] = k_token_stride;
    a.head_stride[0] = q_head_stride, a.head_stride[1] = k_head_stride;
    a.out_tok_stride[0] = (int64_t)q_heads * dim, a.out_tok_stride[1] = (int64_t)k_heads * dim;
    a.heads[0] = q_heads, a.heads[1] = k_heads;
    a.tokens = tokens, a.dim = dim, a.pairs = pairs, a.axes = axes;
    a.positions = positions, a.freq = frequencies;
    a.sign = inverse ? -1.f : 1.f;
    hipStream_t st = as_stream(stream);
    TimedScope ts("rotary", st);
    const bool half = interleaved == 0;
    const auto go = [&](auto t) {
        using T = decltype(t);
        return positions_64 ? rotary_launch<T, int64_t>(a, half, st)
                            : rotary_launch<T, int32_t>(a, half, st);
    };
    const bool fits = dtype == MG_F32    ? go(float{})
                      : dtype == MG_BF16 ? go(bf16_t{})
                                         : go(f16_t{});
    MG_REQUIRE(fits, "mg_rotary: %lld tokens of %d elements are too many for one call",
               (long long)tokens, (q_heads + k_heads) * dim);
    MG_LAUNCHED("rotary_kernel");
    return MG_OK;
}
