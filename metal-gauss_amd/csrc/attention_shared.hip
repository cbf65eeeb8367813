// Attention of sequences over memories that several of them share, and over their
// own keys, one softmax over both:
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i)
//
// over all keys j of the memory that query i's group shares and those keys of its own
// sequence that it sees. Sums of both are formed apart, {top, sum, unscaled sum of
// values} a chunk of keys, and joined: sum 2^(top_c - top) o_c over sum 2^(top_c - top)
// sum_c.
//
// The queries of a group's sequences lie one after the other, so that over the
// shared memory they are one sequence of many rows, whose tiles read each key once
// for 128 rows where a sequence by itself would read it for its own few; over their
// own keys they are the packed sequences that they are. Both are the work items of
// attention_fwd.h, in two launches, whose partial results lie by rows, so that the
// third finds a row's without a search.
#include "attention_fwd.h"

namespace mg {

template <typename T, int DK, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 1 ? 1 : 2) void attn_part_kernel(AttnArgs a) {
    for (int work = blockIdx.x; attn_fwd_item<T, DK, kWaves, kByRow, false>(a, work);
         work += gridDim.x)
        tiles_ready();
}

// A wave has four columns of 32 rows in each of its halves: columns 8 j + 4 half ..
template <typename T, int DK>
__global__ __launch_bounds__(256) void attn_join_parts_kernel(AttnArgs shared, AttnArgs alone) {
    const AttnArgs *const sets[2] = {&shared, &alone};
    const int lane = lane_id(), half = lane / 32, G = alone.group, kh = blockIdx.y, j = blockIdx.z;
    const int64_t rows = (int64_t)alone.q_tokens * G;
    const int64_t row = ((int64_t)blockIdx.x * 4 + threadIdx.x / 64) * 32 + lane % 32;
    const int at = 8 * j + 4 * half;
    if (row >= rows || at >= alone.dim) return;
    float top = -INFINITY, sum = 0.f;
    f32x4 o = {};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 *st = row_stats(*sets[k], kh, row, 0);
#pragma unroll 8
        for (int c = 0; c < sets[k]->row_chunks; ++c) top = fmaxf(top, st[c * 32].x);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 *st = row_stats(*sets[k], kh, row, 0);
        const f32x4 *from = row_values<DK>(*sets[k], kh, row, 0, half) + 64 * j;
#pragma unroll 8
        for (int c = 0; c < sets[k]->row_chunks; ++c) {
            const float2 s = st[c * 32];
            const f32x4 x = from[c * (32 * DK / 4)];
            const float by = s.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s.x - top);
            // A NaN sum of a chunk without a finite score goes on; a place that no
            // chunk has filled holds anything.
            const bool used = s.x != -INFINITY || s.y != 0.f;
            sum = fmaf(s.y, by, sum);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = used ? fmaf(x[i], by, o[i]) : o[i];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    vec4<T> w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (T)(o[i] * inv);
    const int64_t token = row / G, head = kh * G + row % G;
    *reinterpret_cast<vec4<T> *>(static_cast<T *>(alone.out) +
                                 (token * (alone.k_heads * G) + head) * alone.dim + at) = w;
}

// -------------------------------------------------------------------- host
// How one set of items is cut (see fwd_plan, whose limits these are).
struct PartPlan {
    int waves, split_keys, row_chunks;
    int64_t items;              // of a key head, at most
    int64_t stats_bytes, bytes;
};

constexpr int64_t kPartWideSlots = 512, kPartNarrowSlots = 1536;
constexpr int64_t kPartSplitLeast = 768, kPartChunkLeast = 256, kPartMostChunks = 64;

static PartPlan part_plan(int64_t q_tokens, int64_t k_tokens, int64_t k_heads, int64_t group,
                          int dim, int64_t n_seq) {
    PartPlan p{};
    const int64_t rows = q_tokens * group;
    p.waves = rows <= 64 * n_seq ? kNarrowWaves : kWideWaves;
    const int64_t tile_rows = 32 * p.waves;
    const int64_t slots = p.waves == kNarrowWaves ? kPartNarrowSlots
                          : n_seq == 1            ? kPartWideSlots
                                                  : kPartWideSlots / 2;
    const int64_t likely = (ceil_div(rows, tile_rows) + n_seq - 1) * k_heads;
    const int64_t mean_keys = k_tokens / n_seq;
    p.split_keys = (int)kPartChunkLeast;
    p.row_chunks = 1;
    if (2 * likely <= slots && mean_keys >= kPartSplitLeast) {
        int64_t chunks = slots / likely;
        if (chunks > ceil_div(mean_keys, kPartChunkLeast))
            chunks = ceil_div(mean_keys, kPartChunkLeast);
        p.row_chunks = (int)(chunks < kPartMostChunks ? chunks : kPartMostChunks);
    }
    // The tokens before the first and past the last offset make tiles too, of one
    // chunk each.
    p.items = (rows / tile_rows + n_seq + 2) * p.row_chunks;
    const int64_t dk = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
    const int64_t places = k_heads * ceil_div(rows, 32) * 32 * p.row_chunks;
    p.stats_bytes = align256(places * 8);
    p.bytes = p.stats_bytes + align256(places * dk * 4);
    return p;
}

}  // namespace mg

extern "C" {

int64_t mg_shared_attention_workspace_bytes(int64_t q_tokens, int64_t k_tokens,
                                            int64_t shared_tokens, int32_t q_heads,
                                            int32_t k_heads, int32_t dim, int32_t sequences,
                                            int32_t groups) {
    if (q_tokens <= 0 || k_tokens < 0 || shared_tokens < 0 || k_heads < 1 || q_heads < k_heads ||
        sequences < 1 || groups < 1)
        return 0;
    const int group = q_heads / k_heads;
    return mg::part_plan(q_tokens, shared_tokens, k_heads, group, dim, groups).bytes +
           mg::part_plan(q_tokens, k_tokens, k_heads, group, dim, sequences).bytes;
}

int32_t mg_shared_attention(
    int32_t dtype, int64_t q_tokens, int64_t k_tokens, int64_t shared_tokens, int32_t q_heads,
    int32_t k_heads, int32_t dim, const void *q, int64_t q_token_stride, int64_t q_head_stride,
    const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
    int64_t v_token_stride, int64_t v_head_stride, const void *shared_k,
    int64_t shared_k_token_stride, int64_t shared_k_head_stride, const void *shared_v,
    int64_t shared_v_token_stride, int64_t shared_v_head_stride, const int32_t *q_offsets,
    const int32_t *k_offsets, int32_t sequences, const int32_t *group_offsets,
    const int32_t *shared_offsets, int32_t groups, int32_t causal, float scale, void *out,
    void *workspace, int64_t workspace_bytes, mg_stream_t stream) {
    using namespace mg;
    const char *who = "mg_shared_attention";
    MG_REQUIRE(k_heads >= 1 && q_heads >= 1 && q_heads % k_heads == 0,
               "%s: %d query heads are no multiple of %d key heads", who, q_heads, k_heads);
    const int group = q_heads / k_heads;
    constexpr int64_t kMost = int64_t(1) << 30;
    MG_REQUIRE(q_tokens >= 0 && k_tokens >= 0 && shared_tokens >= 0 && q_tokens * group < kMost &&
                   k_tokens < kMost && shared_tokens < kMost,
               "%s: %lld query, %lld key and %lld shared tokens", who, (long long)q_tokens,
               (long long)k_tokens, (long long)shared_tokens);
    AttnArgs sets[2] = {};                        // over the shared memories, and alone
    for (int i = 0; i < 2; ++i) {
        AttnArgs &a = sets[i];
        a.q = {q, q_token_stride, q_head_stride};
        a.k_heads = k_heads, a.group = group, a.dim = dim;
        a.q_tokens = (int32_t)q_tokens;
        a.scale = scale, a.scale_log2 = scale_to_log2(scale);
        a.out = out;
        a.span_most = INT32_MAX;
        if (i == 0) {
            a.k = {shared_k, shared_k_token_stride, shared_k_head_stride};
            a.v = {shared_v, shared_v_token_stride, shared_v_head_stride};
            a.q_off = group_offsets, a.k_off = shared_offsets, a.n_seq = groups;
            a.k_tokens = (int32_t)shared_tokens;
        } else {
            a.k = {k, k_token_stride, k_head_stride};
            a.v = {v, v_token_stride, v_head_stride};
            a.q_off = q_offsets, a.k_off = k_offsets, a.n_seq = sequences;
            a.k_tokens = (int32_t)k_tokens, a.causal = causal != 0;
        }
        const int32_t rc = attn_check(who, a, dtype);
        if (rc != MG_OK) return rc;
    }
    if (q_tokens == 0) return MG_OK;
    MG_REQUIRE(q && out && (k_tokens == 0 || (k && v)) &&
                   (shared_tokens == 0 || (shared_k && shared_v)),
               "%s: a pointer is NULL", who);
    const PartPlan plans[2] = {
        part_plan(q_tokens, shared_tokens, k_heads, group, dim, groups),
        part_plan(q_tokens, k_tokens, k_heads, group, dim, sequences)};
    const int64_t row_blocks = ceil_div(q_tokens * group, 4 * 32);
    for (const PartPlan &p : plans)
        MG_REQUIRE(grid_fits(p.items * k_heads, 64 * p.waves) && k_heads < 65536,
                   "%s: too many work items", who);
    MG_REQUIRE(workspace && workspace_bytes >= plans[0].bytes + plans[1].bytes,
               "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
               (long long)(plans[0].bytes + plans[1].bytes));
    hipStream_t st = as_stream(stream);
    char *ws = static_cast<char *>(workspace);
    for (int i = 0; i < 2; ++i) {
        AttnArgs &a = sets[i];
        const PartPlan &p = plans[i];
        a.split_keys = p.split_keys, a.row_chunks = p.row_chunks;
        a.part_stats = reinterpret_cast<float2 *>(ws);
        a.part_o = reinterpret_cast<float *>(ws + p.stats_bytes);
        ws += p.bytes;
        const int64_t items = p.items * k_heads;
        const int64_t most = 2 * (p.waves == kWideWaves ? kPartWideSlots : kPartNarrowSlots);
        const unsigned grid = (unsigned)(items > most ? most : items);
        TimedScope ts(i == 0 ? "attention_shared" : "attention_alone", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            if (p.waves == kWideWaves)
                attn_part_kernel<T, DK, kWideWaves><<<grid, 64 * kWideWaves, 0, st>>>(a);
            else
                attn_part_kernel<T, DK, kNarrowWaves><<<grid, 64 * kNarrowWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_part_kernel");
    }
    {
        TimedScope ts("attention_join_parts", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            const dim3 grid((unsigned)row_blocks, (unsigned)k_heads, DK / 8);
            attn_join_parts_kernel<T, DK><<<grid, 256, 0, st>>>(sets[0], sets[1]);
        });
        MG_LAUNCHED("attn_join_parts_kernel");
    }
    return MG_OK;
}

}  // extern "C"
