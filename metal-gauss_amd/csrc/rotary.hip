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
// keys are read once and written once, in one launch.
#include "mg_types.h"

namespace mg {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 512;          // heads of up to 1024 elements
constexpr int kRotTable = 1024;            // cosines and sines held by a workgroup

struct RotArgs {
    const void *x[2];
    void *out[2];
    int64_t tok_stride[2], head_stride[2], out_tok_stride[2];
    int32_t heads[2];                      // heads[1] may be 0
    int64_t tokens;
    int32_t dim, pairs, axes;
    const void *positions;
    const double *freq;
    int32_t tokens_at_once;
    float sign;
};

// A unit is V neighbouring elements of a head's rotated part together with
// their partners (kHalf), V / 2 whole pairs (interleaved), or V elements that
// are copied. V = 16 bytes' worth where units do not straddle the parts'
// borders, else 1 (2 interleaved).
template <typename T, typename P, int V, bool kHalf>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a) {
    __shared__ float2 s_cs[kRotTable];
    const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_at_once;
    const int n_tok = (int)min((int64_t)a.tokens_at_once, a.tokens - tok0);
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
    const int rot_units = (kHalf ? a.pairs : 2 * a.pairs) / V;
    const int units = rot_units + (a.dim - 2 * a.pairs) / V;
    const int heads = a.heads[0] + a.heads[1];
    const int per_tok = heads * units;
    for (int i = threadIdx.x; i < n_tok * per_tok; i += kRotThreads) {
        const int tok = i / per_tok, r = i - tok * per_tok;
        int h = r / units;
        const int u = r - h * units;
        const int which = h >= a.heads[0];
        h -= which ? a.heads[0] : 0;
        const T *x = static_cast<const T *>(a.x[which]) + (tok0 + tok) * a.tok_stride[which] +
                     h * a.head_stride[which];
        T *out = static_cast<T *>(a.out[which]) + (tok0 + tok) * a.out_tok_stride[which] +
                 (int64_t)h * a.dim;
        const float2 *cs = s_cs + tok * a.pairs;
        float v[V];
        if (u >= rot_units) {
            const int at = 2 * a.pairs + (u - rot_units) * V;
            load_vec<T, V>(x + at, v);
            store_vec<T, V>(out + at, v);
        } else if constexpr (kHalf) {
            float w[V];
            load_vec<T, V>(x + u * V, v);
            load_vec<T, V>(x + a.pairs + u * V, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float2 c = cs[u * V + k];
                const float p = v[k], q = w[k];
                v[k] = p * c.x - q * c.y;
                w[k] = q * c.x + p * c.y;
            }
            store_vec<T, V>(out + u * V, v);
            store_vec<T, V>(out + a.pairs + u * V, w);
        } else {
            load_vec<T, V>(x + u * V, v);
#pragma unroll
            for (int k = 0; k + 1 < V; k += 2) {
                const float2 c = cs[(u * V + k) / 2];
                const float p = v[k], q = v[k + 1];
                v[k] = p * c.x - q * c.y;
                v[k + 1] = q * c.x + p * c.y;
            }
            store_vec<T, V>(out + u * V, v);
        }
    }
}

template <typename T, typename P>
static void rotary_launch(const RotArgs &a, bool half, hipStream_t st) {
    constexpr int V = kVec<T>;
    const unsigned grid = (unsigned)ceil_div(a.tokens, a.tokens_at_once);
    const int rest = a.dim - 2 * a.pairs;
    const bool wide = (half ? a.pairs : 2 * a.pairs) % V == 0 && rest % V == 0;
    if (half) {
        if (wide)
            rotary_kernel<T, P, V, true><<<grid, kRotThreads, 0, st>>>(a);
        else
            rotary_kernel<T, P, 1, true><<<grid, kRotThreads, 0, st>>>(a);
    } else {
        if (wide)
            rotary_kernel<T, P, V, false><<<grid, kRotThreads, 0, st>>>(a);
        else
            rotary_kernel<T, P, 2, false><<<grid, kRotThreads, 0, st>>>(a);
    }
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
    // Tokens of a workgroup: about 32 KB of heads, as many as the table holds.
    const int64_t bytes = (int64_t)(q_heads + k_heads) * dim * type_bytes(dtype);
    int64_t at_once = 32768 / bytes;
    if (at_once > kRotTable / pairs) at_once = kRotTable / pairs;
    if (at_once * 1024 > tokens) at_once = tokens / 1024;
    a.tokens_at_once = (int32_t)(at_once < 1 ? 1 : at_once);
    hipStream_t st = as_stream(stream);
    TimedScope ts("rotary", st);
    const bool half = interleaved == 0;
    auto go = [&](auto t) {
        using T = decltype(t);
        if (positions_64)
            rotary_launch<T, int64_t>(a, half, st);
        else
            rotary_launch<T, int32_t>(a, half, st);
    };
    if (dtype == MG_F32)
        go(float{});
    else if (dtype == MG_BF16)
        go(bf16_t{});
    else
        go(f16_t{});
    MG_LAUNCHED("rotary_kernel");
    return MG_OK;
}
