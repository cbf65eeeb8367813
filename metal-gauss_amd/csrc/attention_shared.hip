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
// attention_fwd.h, in one launch, those over the memory first (their own after them
// in a launch of narrow items: 128 streams of 16 heads on 4 of 128, 30 and 22 us).
// Partial results lie by rows, so that joining finds a row's without a search.
//
// Those streams over 16320 tokens and up to 500 of their own: 49 us and 6 to join (100 MB
// at 1.9 TB/s, 17 GFLOP: the items' starts weigh); eight streams over 2375: 10 and 7;
// 1957 tokens of frames over 10000 and 2500, 12 heads of 64: 85 and 10.
#include "attention_fwd.h"

namespace mg {

// Items over the shared memories come first, then those over the sequences' own
// keys, of which there are `most` in all at most: how many, the device alone knows.
template <typename T, int DK, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves == 1 ? 1 : 2) void attn_part_kernel(
    AttnArgs shared, AttnArgs alone, int most) {
    for (int work = blockIdx.x; work < most; work += gridDim.x) {
        SeqItem s = find_row_item<kWaves>(shared, work / shared.k_heads);
        const bool of_shared = s.found;
        if (!of_shared) s = find_row_item<kWaves>(alone, work / alone.k_heads - s.within);
        if (!s.found) return;
        attn_fwd_item<T, DK, kWaves, kByRow, false>(of_shared ? shared : alone, work, s);
        tiles_ready();
    }
}

// What a lane has joined so far: four columns of a row.
struct Joined {
    float top = -INFINITY, sum = 0.f;
    f32x4 o = {};

    // N chunks' results; those from n on are none.
    template <int N>
    __device__ __forceinline__ void add(const float2 (&st)[N], const f32x4 (&x)[N], int n) {
        float next = top;
#pragma unroll
        for (int i = 0; i < N; ++i) next = i < n ? fmaxf(next, st[i].x) : next;
        const float shrink = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - next);
        top = next;
        sum *= shrink;
        o *= shrink;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float by = st[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[i].x - top);
            // A NaN sum of a chunk without a finite score goes on; a place that no
            // chunk has filled holds anything.
            const bool used = i < n && (st[i].x != -INFINITY || st[i].y != 0.f);
            sum = used ? fmaf(st[i].y, by, sum) : sum;
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = used ? fmaf(x[i][k], by, o[k]) : o[k];
        }
    }
};

// Chunks c .. c + N - 1 of a row (past the last, the last's).
template <int DK, int N>
__device__ __forceinline__ void ask_chunks(const AttnArgs &a, const float2 *st, const f32x4 *from,
                                           int c, float2 (&s)[N], f32x4 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = min(c + i, a.row_chunks - 1);
        s[i] = st[at * 32];
        x[i] = from[at * (32 * DK / 4)];
    }
}

// A wave has four columns of 32 rows in each of its halves: columns 8 j + 4 half ..
// Stats and values are asked for together, the first chunks of both sets at once.
// kFirst and kFew are of the numbers of chunks, which are one mostly where rows are
// many.
template <typename T, int DK, int kFirst, int kFew>
__global__ __launch_bounds__(256) void attn_join_parts_kernel(AttnArgs shared, AttnArgs alone) {
    const int lane = lane_id(), half = lane / 32, G = alone.group, kh = blockIdx.y, j = blockIdx.z;
    const int64_t rows = (int64_t)alone.q_tokens * G;
    const int64_t row = ((int64_t)blockIdx.x * 4 + threadIdx.x / 64) * 32 + lane % 32;
    const int at = 8 * j + 4 * half;
    if (row >= rows || at >= alone.dim) return;
    const float2 *st[2] = {row_stats(shared, kh, row, 0), row_stats(alone, kh, row, 0)};
    const f32x4 *from[2] = {row_values<DK>(shared, kh, row, 0, half) + 64 * j,
                            row_values<DK>(alone, kh, row, 0, half) + 64 * j};
    Joined r;
    float2 s0[kFirst], s1[kFew];
    f32x4 x0[kFirst], x1[kFew];
    ask_chunks<DK>(shared, st[0], from[0], 0, s0, x0);
    ask_chunks<DK>(alone, st[1], from[1], 0, s1, x1);
    r.add(s0, x0, shared.row_chunks);
    r.add(s1, x1, alone.row_chunks);
    for (int c = kFirst; c < shared.row_chunks; c += kFirst) {
        ask_chunks<DK>(shared, st[0], from[0], c, s0, x0);
        r.add(s0, x0, shared.row_chunks - c);
    }
    for (int c = kFew; c < alone.row_chunks; c += kFirst) {
        ask_chunks<DK>(alone, st[1], from[1], c, s0, x0);
        r.add(s0, x0, alone.row_chunks - c);
    }
    const float inv = r.sum == 0.f ? 0.f : 1.f / r.sum;
    vec4<T> w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (T)(r.o[i] * inv);
    const int64_t token = row / G, head = kh * G + row % G;
    *reinterpret_cast<vec4<T> *>(static_cast<T *>(alone.out) +
                                 (token * (alone.k_heads * G) + head) * alone.dim + at) = w;
}

// -------------------------------------------------------------------- host
// How one set of items is cut.
struct PartPlan {
    int waves, split_keys, row_chunks;
    int64_t items;              // of a key head, at most
    int64_t stats_bytes, bytes;
};

// Items that run at once.
static int64_t part_slots(int waves) { return waves == kNarrowWaves ? 1536 : 512; }

constexpr int64_t kPartMostChunks = 64;
// Keys of a chunk, at least: wide items, narrow ones; and long ones, whose start and
// partial results cost little beside them.
constexpr int64_t kPartWideLeast = 256, kPartNarrowLeast = 64, kPartLong = 2048;

// Both sets take the items of one width: wide ones, unless the rows of both fill half
// of one at most.
static int part_waves(int64_t rows, int64_t groups, int64_t sequences) {
    return rows <= 64 * groups && rows <= 64 * sequences ? kNarrowWaves : kWideWaves;
}

// Items of a set whose keys are not cut.
static int64_t part_whole(int64_t rows, int64_t n_seq, int64_t k_heads, int waves) {
    return (ceil_div(rows, 32 * waves) + n_seq - 1) * k_heads;
}

// `beside`: the other set's items, which run beside these from the start. Those of the
// shared memories leave them up to half of the slots (128 streams over 16320 tokens
// and their own: 54 us and 9 to join with all slots taken by the first, 50 and 6 so).
static PartPlan part_plan(int64_t q_tokens, int64_t k_tokens, int64_t k_heads, int64_t group,
                          int dim, int64_t n_seq, int waves, int64_t beside) {
    PartPlan p{};
    const int64_t rows = q_tokens * group;
    p.waves = waves;
    const int64_t tile_rows = 32 * p.waves;
    int64_t slots = part_slots(waves);
    slots -= beside < slots / 2 ? beside : slots / 2;
    const int64_t likely = part_whole(rows, n_seq, k_heads, waves);
    const int64_t mean_keys = k_tokens / n_seq;
    // As many chunks as make items for all slots, of `least` keys at least; and where
    // chunks stay long, as make several rounds of items, which even out.
    const int64_t least = waves == kNarrowWaves ? kPartNarrowLeast : kPartWideLeast;
    int64_t chunks = slots / likely, longer = ceil_div(3 * slots, likely);
    if (chunks > ceil_div(mean_keys, least)) chunks = ceil_div(mean_keys, least);
    if (longer > mean_keys / kPartLong) longer = mean_keys / kPartLong;
    if (chunks < longer) chunks = longer;
    p.row_chunks = (int)(chunks < 1 ? 1 : chunks < kPartMostChunks ? chunks : kPartMostChunks);
    p.split_keys = (int)least;
    // The tokens before the first and past the last offset make tiles too, of one
    // chunk each.
    p.items = (rows / tile_rows + n_seq + 2) * p.row_chunks;
    const int64_t dk = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
    const int64_t places = k_heads * ceil_div(rows, 32) * 32 * p.row_chunks;
    p.stats_bytes = align256(places * 8);
    p.bytes = p.stats_bytes + align256(places * dk * 4);
    return p;
}

struct PartPlans {
    PartPlan of[2];             // over the shared memories, and alone
};
static PartPlans part_plans(int64_t q_tokens, int64_t k_tokens, int64_t shared_tokens,
                            int64_t k_heads, int64_t group, int dim, int64_t sequences,
                            int64_t groups) {
    const int64_t rows = q_tokens * group;
    const int waves = part_waves(rows, groups, sequences);
    return {{part_plan(q_tokens, shared_tokens, k_heads, group, dim, groups, waves,
                       part_whole(rows, sequences, k_heads, waves)),
             part_plan(q_tokens, k_tokens, k_heads, group, dim, sequences, waves, 0)}};
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
    const mg::PartPlans p = mg::part_plans(q_tokens, k_tokens, shared_tokens, k_heads, group, dim,
                                           sequences, groups);
    return p.of[0].bytes + p.of[1].bytes;
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
    const PartPlans all =
        part_plans(q_tokens, k_tokens, shared_tokens, k_heads, group, dim, sequences, groups);
    const PartPlan(&plans)[2] = all.of;
    const int waves = plans[0].waves;
    const int64_t items = (plans[0].items + plans[1].items) * k_heads;
    MG_REQUIRE(grid_fits(items, 64 * waves) && items < INT32_MAX && k_heads < 65536,
               "%s: too many work items", who);
    MG_REQUIRE(workspace && workspace_bytes >= plans[0].bytes + plans[1].bytes,
               "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
               (long long)(plans[0].bytes + plans[1].bytes));
    char *ws = static_cast<char *>(workspace);
    for (int i = 0; i < 2; ++i) {
        sets[i].split_keys = plans[i].split_keys, sets[i].row_chunks = plans[i].row_chunks;
        sets[i].part_stats = reinterpret_cast<float2 *>(ws);
        sets[i].part_o = reinterpret_cast<float *>(ws + plans[i].stats_bytes);
        ws += plans[i].bytes;
    }
    hipStream_t st = as_stream(stream);
    {
        // Items are taken in turn by twice as many workgroups as run at once.
        const int64_t most = 2 * part_slots(waves);
        const unsigned grid = (unsigned)(items > most ? most : items);
        TimedScope ts("attention_parts", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            if (waves == kWideWaves)
                attn_part_kernel<T, DK, kWideWaves>
                    <<<grid, 64 * kWideWaves, 0, st>>>(sets[0], sets[1], (int)items);
            else
                attn_part_kernel<T, DK, kNarrowWaves>
                    <<<grid, 64 * kNarrowWaves, 0, st>>>(sets[0], sets[1], (int)items);
        });
        MG_LAUNCHED("attn_part_kernel");
    }
    {
        TimedScope ts("attention_join_parts", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            const dim3 grid((unsigned)ceil_div(q_tokens * group, 4 * 32), (unsigned)k_heads,
                            DK / 8);
            if (plans[0].row_chunks == 1 && plans[1].row_chunks == 1)
                attn_join_parts_kernel<T, DK, 1, 1><<<grid, 256, 0, st>>>(sets[0], sets[1]);
            else
                attn_join_parts_kernel<T, DK, 12, 4><<<grid, 256, 0, st>>>(sets[0], sets[1]);
        });
        MG_LAUNCHED("attn_join_parts_kernel");
    }
    return MG_OK;
}

}  // extern "C"
