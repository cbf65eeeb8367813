// Attention over packed sequences, forward: the kernels that give out the work items
// of attention_fwd.h, those that join rows cut over their keys, and the entries.
#include "attention_fwd.h"

namespace mg {

// How many items the chunks make is known on the device alone: as many
// workgroups as fill the GPU take them in turn.
template <typename T, int DK, int kWaves, Cut kCut, bool kWin>
__global__ __launch_bounds__(64 * kWaves, kWaves == 1 ? 1 : 2) void attn_fwd_kernel(AttnArgs a) {
    if constexpr (kCut == kWhole) {
        attn_fwd_item<T, DK, kWaves, kCut, kWin>(a, blockIdx.x);
    } else {
        for (int work = blockIdx.x; attn_fwd_item<T, DK, kWaves, kCut, kWin>(a, work);
             work += gridDim.x)
            tiles_ready();
    }
}

// Joining the chunks of a row: o = sum 2^(top_c - top) o_c / sum of the same of
// sum_c.
//
// Wide items: a workgroup has 32 columns of a tile of one key head, its threads
// the elements that the item's had.
template <typename T, int DK>
__global__ __launch_bounds__(64 * kWideWaves) void attn_join_tile_kernel(AttnArgs a) {
    constexpr int kRows = 32 * kWideWaves;
    const int lane = lane_id(), half = lane / 32, G = a.group, block = blockIdx.y;
    const int wave = uniform(threadIdx.x / 64);
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads;
    const auto tiles_of = [&](int ql, int) { return (ql * G + kRows - 1) / kRows; };
    const SeqItem s = find_item<false>(a, item, tiles_of, [&](int ql, int kl) {
        const int tiles = tiles_of(ql, kl);
        return tiles * chunks_of(a, tiles, kl);
    });
    if (!s.found) return;
    const int tiles = tiles_of(s.q_len, 0), chunks = chunks_of(a, tiles, s.k_len);
    const int item0 = s.before + s.within * chunks;
    const int row = (tiles - 1 - s.within) * kRows + wave * 32 + lane % 32;
    const int token = row / G, head = kh * G + row % G;
    if (token >= s.q_len) return;
    const int64_t work0 = (int64_t)item0 * a.k_heads + kh;
    const float2 *stats = a.part_stats + work0 * kRows + wave * 32 + lane % 32;
    const float *po =
        a.part_o + work0 * kRows * DK + wave * 32 * DK + 4 * lane + 4 * block * 4 * 64;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) top = fmaxf(top, stats[(int64_t)c * a.k_heads * kRows].x);
    f32x16 o[1] = {};
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) {
        const float2 st = stats[(int64_t)c * a.k_heads * kRows];
        const float *p = po + (int64_t)c * a.k_heads * kRows * DK;
        const float by = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - top);
        // A NaN sum of a chunk without a finite score goes on.
        sum = fmaf(st.y, by, sum);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(p + e * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[0][e + i] = fmaf(x[i], by, o[0][e + i]);
        }
    }
    store_row_result<T, 32>(a, s.q_lo + token, head, half, block, top, sum, o);
}

// Narrow items: kJoin waves a row (four where rows have many chunks), wave w with
// every kJoin-th chunk from w; a lane first holds a chunk's weight, then DK / 64
// columns.
template <typename T, int DK, int kJoin>
__global__ __launch_bounds__(256) void attn_join_row_kernel(AttnArgs a) {
    constexpr int kRows = 32 * kNarrowWaves, kCols = DK <= 64 ? 1 : 2;
    __shared__ float s_o[kJoin > 1 ? kJoin : 1][64 * kCols], s_top[kJoin], s_sum[kJoin];
    const int lane = lane_id(), G = a.group, heads = a.k_heads * G;
    const int wave = uniform(threadIdx.x / 64);
    const int64_t row_head = kJoin > 1 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    const int at_token = (int)(row_head / heads), head = (int)(row_head % heads);
    if (at_token >= a.q_tokens) return;
    const int kh = head / G, first = kJoin > 1 ? wave : 0;
    const auto tiles_of = [&](int ql) { return (ql * G + kRows - 1) / kRows; };
    const SeqItem s = find_item<false>(
        a, at_token, [](int ql, int) { return ql; },
        [&](int ql, int kl) {
            const int tiles = tiles_of(ql);
            return tiles * chunks_of(a, tiles, kl);
        });
    if (!s.found) return;
    const int row = s.within * G + head % G, tile = row / kRows, tiles = tiles_of(s.q_len);
    const int chunks = chunks_of(a, tiles, s.k_len), item0 = s.before + (tiles - 1 - tile) * chunks;
    const auto slot = [&](int c) {
        return ((int64_t)(item0 + c) * a.k_heads + kh) * kRows + row % kRows;
    };
    float top = -INFINITY, sum = 0.f, o[kCols] = {};
    for (int c0 = first; c0 < chunks; c0 += 64 * kJoin) {
        const int n = min((chunks - c0 + kJoin - 1) / kJoin, 64);
        const float2 st =
            lane < n ? a.part_stats[slot(c0 + kJoin * lane)] : make_float2(-INFINITY, 0.f);
        const float next = fmaxf(top, wave_max(st.x));
        const float shrink = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - next);
        const float w = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - next);
        top = next;
        // A NaN sum of a chunk without a finite score goes on.
        sum = sum * shrink + wave_sum_all(st.y * w);
#pragma unroll
        for (int k = 0; k < kCols; ++k) o[k] *= shrink;
        const auto add = [&](int c) {
            const float wc = __builtin_bit_cast(
                float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), c));
            const float *p = a.part_o + slot(c0 + kJoin * c) * DK + lane * kCols;
            float f[kCols];
            if (lane * kCols < DK) {
                __builtin_memcpy(f, p, sizeof(f));
#pragma unroll
                for (int k = 0; k < kCols; ++k) o[k] = fmaf(f[k], wc, o[k]);
            }
        };
        int c = 0;
        for (; c + 8 <= n; c += 8)
#pragma unroll
            for (int k = 0; k < 8; ++k) add(c + k);
        for (; c < n; ++c) add(c);
    }
    if constexpr (kJoin > 1) {
#pragma unroll
        for (int k = 0; k < kCols; ++k) s_o[wave][lane * kCols + k] = o[k];
        if (lane == 0) {
            s_top[wave] = top;
            s_sum[wave] = sum;
        }
        __syncthreads();
        if (wave != 0) return;
        top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < kCols; ++k) o[k] = 0.f;
#pragma unroll
        for (int w = 0; w < kJoin; ++w) {
            const float by = s_top[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_top[w] - top);
            sum = fmaf(s_sum[w], by, sum);
#pragma unroll
            for (int k = 0; k < kCols; ++k) o[k] = fmaf(s_o[w][lane * kCols + k], by, o[k]);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t at = ((int64_t)(s.q_lo + s.within) * heads + head) * a.dim + lane * kCols;
    T w[kCols], x[kCols];
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
        w[k] = (T)(o[k] * inv);
        x[k] = (T)(o[k] * inv - (float)w[k]);
    }
    if (lane * kCols < a.dim) {
        __builtin_memcpy(static_cast<T *>(a.out) + at, w, sizeof(w));
        if (a.out_rest) __builtin_memcpy(static_cast<T *>(a.out_rest) + at, x, sizeof(x));
    }
    if (a.lse && lane == 0)
        a.lse[(int64_t)head * a.q_tokens + s.q_lo + s.within] =
            sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
}

// -------------------------------------------------------------------- host
int32_t attn_check(const char *who, const AttnArgs &a, int32_t dtype) {
    MG_REQUIRE(dtype == MG_BF16 || dtype == MG_F16, "%s: bfloat16 or float16 needed", who);
    MG_REQUIRE(a.dim >= 8 && a.dim <= 128 && a.dim % 8 == 0,
               "%s: heads of %d elements; multiples of 8 up to 128 are taken", who, a.dim);
    MG_REQUIRE(a.k_heads >= 1 && a.group >= 1 && (int64_t)a.k_heads * a.group <= 65536,
               "%s: the query heads must be a multiple of the key heads", who);
    MG_REQUIRE(a.n_seq >= 1 && a.n_seq < (1 << 30), "%s: %d sequences", who, a.n_seq);
    MG_REQUIRE(a.q_off || a.k_off || a.n_seq == 1, "%s: %d sequences without offsets", who,
               a.n_seq);
    MG_REQUIRE((a.q_off == nullptr) == (a.k_off == nullptr),
               "%s: offsets of queries and keys go together", who);
    MG_REQUIRE(a.scale >= 0.f && a.scale < INFINITY, "%s: scale %g", who, (double)a.scale);
    MG_REQUIRE(a.window >= 0 && a.sinks >= 0 && (a.window > 0 || a.sinks == 0),
               "%s: a window of %d keys and %d first ones", who, a.window, a.sinks);
    MG_REQUIRE(a.window == 0 || a.causal, "%s: a window is for causal attention", who);
    for (const AttnTensor *t : {&a.q, &a.k, &a.v, &a.dout}) {
        MG_REQUIRE(((uintptr_t)t->p & 15) == 0 && t->tok_stride % 8 == 0 &&
                       t->head_stride % 8 == 0,
                   "%s: rows must be 16-byte aligned", who);
        MG_REQUIRE(t->tok_stride >= 0 && t->tok_stride < (1 << 24) && t->head_stride >= 0,
                   "%s: token strides of 0 to 2^24 elements are taken", who);
    }
    return MG_OK;
}

// How the work is cut. Narrow items where rows fill half a wide item at most (on
// the average of the sequences); chunks of keys where the items alone leave the
// GPU idle and a row has keys enough to be worth the second launch. The host
// knows the average alone: one long memory among many short ones is not cut (40
// tokens, 16 heads on 4 of 64, over 16320 keys and 39 times 64: 358 us, over 40
// times 470: 16).
struct FwdPlan {
    int waves;
    int split_keys;             // 0: whole rows
    int64_t chunk_tiles;        // see chunk_keys
    int64_t tiles, items;       // a key head's, at most
    int32_t span_extra, span_most;
    int64_t stats_bytes, bytes; // of partial results
};

// Items that run at once. Of several sequences the longer ones have more chunks
// than the average says, so half as many are aimed at (chunks of 475, 256, 1 and
// 64 queries over up to 16320 keys: 106 us, aimed at 512 it is 109 and 384 124;
// one sequence of 2500, 8 heads of 64: 40 aimed at 256, 26 at 512).
constexpr int64_t kWideSlots = 512, kNarrowSlots = 1536;
constexpr int64_t kSplitLeast = 768, kChunkLeast = 256;
// Single tokens with a window have few keys each: shorter chunks (16 tokens of 16
// heads on 4 of 64, window 2000: 11 us, in chunks of 256 14).
constexpr int64_t kWindowSplitLeast = 256, kWindowChunkLeast = 128;

static FwdPlan fwd_plan(int64_t q_tokens, int64_t k_tokens, int k_heads, int group, int dim,
                        int n_seq, int window, int sinks) {
    FwdPlan p{};
    const int64_t rows = q_tokens * group;
    p.waves = rows <= 64 * (int64_t)n_seq ? kNarrowWaves : kWideWaves;
    const int64_t tile_rows = 32 * p.waves, tile = p.waves == kNarrowWaves ? 32 : kTileRows;
    const int64_t slots = p.waves == kNarrowWaves ? kNarrowSlots
                          : n_seq == 1            ? kWideSlots
                                                  : kWideSlots / 2;
    // The tokens before the first and past the last offset make tiles too.
    p.items = p.tiles = rows / tile_rows + n_seq + 2;
    const int64_t likely = (ceil_div(rows, tile_rows) + n_seq - 1) * k_heads;
    // A window bounds the keys that an item goes through: its queries', and the
    // sinks' in whole tiles, which may pass the sequence's own by a tile.
    p.span_most = INT32_MAX;
    if (window > 0) {
        p.span_extra = sinks > 0 ? (int)tile : 0;
        const int64_t most = ceil_div(sinks, tile) * tile + window + (tile_rows - 1) / group + 2;
        if (most < INT32_MAX) p.span_most = (int)most;
        k_tokens += (int64_t)n_seq * p.span_extra;
        if (k_tokens > n_seq * most) k_tokens = n_seq * most;
    }
    const int64_t mean_keys = k_tokens / n_seq;
    const bool short_chunks = window > 0 && p.waves == kNarrowWaves;
    if (2 * likely <= slots && mean_keys >= (short_chunks ? kWindowSplitLeast : kSplitLeast)) {
        int64_t keys = ceil_div(ceil_div(mean_keys * likely, slots), tile) * tile;
        const int64_t least = short_chunks ? kWindowChunkLeast : kChunkLeast;
        if (keys < least) keys = least;
        p.split_keys = (int)keys;
        // Sum of tiles * (1 + keys / chunk) over the sequences, which have each
        // token once whatever the offsets hold (seq_bounds): the partial results
        // of every item have room, without a check on the device. No sequence has
        // more tiles than all rows make; of many sequences those that have over
        // four times the average take longer chunks, as room for any would be
        // gigabytes (384 tokens of 32 heads on one of 128, 1000 keys each: 4.8,
        // now 0.11).
        const int64_t most = rows / tile_rows + 1;
        p.chunk_tiles = 4 * ceil_div(rows / tile_rows + n_seq, n_seq);
        p.items += most <= p.chunk_tiles ? most * (k_tokens / keys)
                                         : p.chunk_tiles * k_tokens / keys;
        const int dk = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
        const int64_t part_rows = p.items * k_heads * tile_rows;
        p.stats_bytes = align256(part_rows * 8);
        p.bytes = p.stats_bytes + part_rows * dk * 4;
    }
    return p;
}

static int64_t forward_workspace(int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                                 int32_t k_heads, int32_t dim, int32_t sequences, int32_t window,
                                 int32_t sinks) {
    if (q_tokens <= 0 || k_tokens < 0 || k_heads < 1 || q_heads < k_heads || sequences < 1)
        return 0;
    AttnArgs a{};
    a.k_tokens = (int32_t)k_tokens, a.window = window, a.sinks = sinks;
    hold_window(a);
    return fwd_plan(q_tokens, k_tokens, k_heads, q_heads / k_heads, dim, sequences, a.window,
                    a.sinks)
        .bytes;
}

static int32_t attention_forward(const char *who, int32_t dtype, int64_t q_tokens,
                                 int64_t k_tokens, int32_t q_heads, int32_t k_heads, int32_t dim,
                                 const void *q, int64_t q_token_stride, int64_t q_head_stride,
                                 const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                 const void *v, int64_t v_token_stride, int64_t v_head_stride,
                                 const int32_t *q_offsets, const int32_t *k_offsets,
                                 int32_t sequences, int32_t causal, int32_t window, int32_t sinks,
                                 float scale, void *out, void *out_rest, float *lse,
                                 void *workspace, int64_t workspace_bytes, mg_stream_t stream) {
    MG_REQUIRE(k_heads >= 1 && q_heads >= 1 && q_heads % k_heads == 0,
               "%s: %d query heads are no multiple of %d key heads", who, q_heads, k_heads);
    const int group = q_heads / k_heads;
    MG_REQUIRE(q_tokens >= 0 && k_tokens >= 0 && q_tokens * group < (int64_t(1) << 30) &&
                   k_tokens < (int64_t(1) << 30),
               "%s: %lld query and %lld key tokens", who, (long long)q_tokens,
               (long long)k_tokens);
    AttnArgs a{};
    a.q = {q, q_token_stride, q_head_stride};
    a.k = {k, k_token_stride, k_head_stride};
    a.v = {v, v_token_stride, v_head_stride};
    a.q_off = q_offsets, a.k_off = k_offsets, a.n_seq = sequences;
    a.q_tokens = (int32_t)q_tokens, a.k_tokens = (int32_t)k_tokens;
    a.k_heads = k_heads, a.group = group, a.dim = dim, a.causal = causal != 0;
    a.window = window, a.sinks = sinks;
    a.scale = scale, a.scale_log2 = scale_to_log2(scale);
    a.out = out, a.out_rest = out_rest, a.lse = lse;
    int32_t rc = attn_check(who, a, dtype);
    if (rc != MG_OK) return rc;
    if (q_tokens == 0) return MG_OK;
    MG_REQUIRE(q && out && (k_tokens == 0 || (k && v)), "%s: a pointer is NULL", who);
    hold_window(a);
    const FwdPlan p =
        fwd_plan(q_tokens, k_tokens, k_heads, group, dim, sequences, a.window, a.sinks);
    MG_REQUIRE(grid_fits(p.items * k_heads, 64 * p.waves), "%s: too many work items", who);
    MG_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes),
               "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
               (long long)p.bytes);
    a.split_keys = p.split_keys, a.chunk_tiles = (int32_t)p.chunk_tiles;
    a.span_extra = p.span_extra, a.span_most = p.span_most;
    a.part_stats = static_cast<float2 *>(workspace);
    a.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + p.stats_bytes);
    hipStream_t st = as_stream(stream);
    const int64_t items = p.items * k_heads;
    // Chunks are taken in turn by twice as many workgroups as run at once.
    const int64_t most = 2 * (p.waves == kWideWaves ? kWideSlots : kNarrowSlots);
    const unsigned grid = (unsigned)(p.split_keys && items > most ? most : items);
    {
        TimedScope ts("attention_fwd", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            using std::bool_constant;
            using std::integral_constant;
            const auto go = [&](auto waves, auto split, auto win) {
                constexpr int kWaves = decltype(waves)::value;
                attn_fwd_kernel<T, DK, kWaves, decltype(split)::value, decltype(win)::value>
                    <<<grid, 64 * kWaves, 0, st>>>(a);
            };
            const auto with = [&](auto waves, auto split) {
                if (a.window)
                    go(waves, split, bool_constant<true>{});
                else
                    go(waves, split, bool_constant<false>{});
            };
            const auto cut = [&](auto waves) {
                if (p.split_keys)
                    with(waves, integral_constant<Cut, kByItem>{});
                else
                    with(waves, integral_constant<Cut, kWhole>{});
            };
            if (p.waves == kWideWaves)
                cut(integral_constant<int, kWideWaves>{});
            else
                cut(integral_constant<int, kNarrowWaves>{});
        });
        MG_LAUNCHED("attn_fwd_kernel");
    }
    if (p.split_keys) {
        TimedScope ts("attention_join", st);
        // Four waves a row where rows have more chunks than one wave asks for
        // at once, on the average.
        const int64_t mean = k_tokens / sequences;
        const bool many = (mean < p.span_most ? mean : p.span_most) > 8 * (int64_t)p.split_keys;
        const int64_t rows = q_tokens * q_heads;
        const unsigned tiles = (unsigned)(p.tiles * k_heads);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            if (p.waves == kWideWaves)
                attn_join_tile_kernel<T, DK>
                    <<<dim3(tiles, DK / 32), 64 * kWideWaves, 0, st>>>(a);
            else if (many)
                attn_join_row_kernel<T, DK, 4><<<(unsigned)rows, 256, 0, st>>>(a);
            else
                attn_join_row_kernel<T, DK, 1><<<(unsigned)ceil_div(rows, 4), 256, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_join kernels");
    }
    return MG_OK;
}

}  // namespace mg

extern "C" {

int64_t mg_attention_forward_workspace_bytes(int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                                             int32_t k_heads, int32_t dim, int32_t sequences) {
    return mg::forward_workspace(q_tokens, k_tokens, q_heads, k_heads, dim, sequences, 0, 0);
}

int32_t mg_attention_forward(int32_t dtype, int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                             int32_t k_heads, int32_t dim, const void *q, int64_t q_token_stride,
                             int64_t q_head_stride, const void *k, int64_t k_token_stride,
                             int64_t k_head_stride, const void *v, int64_t v_token_stride,
                             int64_t v_head_stride, const int32_t *q_offsets,
                             const int32_t *k_offsets, int32_t sequences, int32_t causal,
                             float scale, void *out, void *out_rest, float *lse,
                             void *workspace, int64_t workspace_bytes, mg_stream_t stream) {
    return mg::attention_forward("mg_attention_forward", dtype, q_tokens, k_tokens, q_heads,
                                 k_heads, dim, q, q_token_stride, q_head_stride, k, k_token_stride,
                                 k_head_stride, v, v_token_stride, v_head_stride, q_offsets,
                                 k_offsets, sequences, causal, 0, 0, scale, out, out_rest, lse,
                                 workspace, workspace_bytes, stream);
}

int64_t mg_attention_window_forward_workspace_bytes(int64_t q_tokens, int64_t k_tokens,
                                                    int32_t q_heads, int32_t k_heads, int32_t dim,
                                                    int32_t sequences, int32_t window,
                                                    int32_t sinks) {
    if (window < 1 || sinks < 0) return 0;
    return mg::forward_workspace(q_tokens, k_tokens, q_heads, k_heads, dim, sequences, window,
                                 sinks);
}

int32_t mg_attention_window_forward(
    int32_t dtype, int64_t q_tokens, int64_t k_tokens, int32_t q_heads, int32_t k_heads,
    int32_t dim, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
    int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
    int64_t v_head_stride, const int32_t *q_offsets, const int32_t *k_offsets, int32_t sequences,
    int32_t window, int32_t sinks, float scale, void *out, void *out_rest, float *lse,
    void *workspace, int64_t workspace_bytes, mg_stream_t stream) {
    const char *who = "mg_attention_window_forward";
    MG_REQUIRE(window >= 1, "%s: a window of %d keys", who, window);
    return mg::attention_forward(who, dtype, q_tokens, k_tokens, q_heads, k_heads, dim, q,
                                 q_token_stride, q_head_stride, k, k_token_stride, k_head_stride,
                                 v, v_token_stride, v_head_stride, q_offsets, k_offsets, sequences,
                                 1, window, sinks, scale, out, out_rest, lse, workspace,
                                 workspace_bytes, stream);
}

}  // extern "C"
