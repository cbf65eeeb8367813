// A work item of attention over packed sequences, forward:
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i)
//
// over the keys j of query i's own sequence, causal: those that stand at or
// before it, a sequence's last query standing at its last key; with a window, the
// last `window` of these and the sequence's first `sinks`. Queries that see no key
// give zeros.
//
// A work item is a tile of rows of one key head, a row being a query token
// together with one of the `group` query heads that share the head: a single
// token's heads fill a tile together, and keys and values are read once for
// all of them. Its waves hold 32 rows each; keys and values pass through LDS in
// tiles of 64, double buffered. With S^T = K Q^T a lane of the product holds
// scores of one row only, so the running maximum and sum of its softmax are a
// lane's own registers (and its partner's, 32 lanes on), and the scores are
// already where the product O^T = V^T P^T wants them.
//
// With 128 columns a tile's products take as long as its softmax, with 64 the
// softmax (exponentials) is the bound; two to four waves a SIMD take turns at
// both. 16320 tokens, causal, 16 heads on 4 of 128: 950 to 1050 us (1150 to 1040
// TFLOP/s, as the GPU's clock holds); 10000 tokens, 16 heads of 64: 440 us (930), of 80
// 620 (830) and of 96 627 (980): 80 columns take the form of 96. With a window of 1900
// and 16 sinks the 16320 tokens take 274 us (880 TFLOP/s of what is seen: 34 tiles an
// item, of which the first, the last and the sinks' are masked).
//
// The running maximum lags: the accumulators are rescaled only when a score
// passes the maximum they go by by more than kMaxLag, which leaves every sum exact
// to its 24 bits and skips nearly all rescaling.
//
// float16: p is kept 2^kRise times as large, sum and all, for the product. As they
// are, keys of less than 2^-14 of the largest would lose digits and those of less
// than 2^-25 everything, which many of them add up to (16000 keys at 2^-22 beside
// one whose value is zero: a result 9% off); so it is 2^-25 and 2^-36. Lag and
// rise together stay below float16's 2^16. bfloat16 has float32's range.
#pragma once

#include "attention.h"

namespace mg {

template <typename T>                             // powers of 2
constexpr float kMaxLag = std::is_same<T, f16_t>::value ? 4.f : 8.f;
template <typename T>
constexpr float kRise = std::is_same<T, f16_t>::value ? 11.f : 0.f;

// Work items come in two widths. Wide: 128 rows by four waves, tiles of 64
// keys that all four read. Narrow, where a sequence's rows would leave most of
// that empty (single tokens): 32 rows by one wave, tiles of 32 keys; memory
// bounds it, and of those cut over their keys ten waves a CU (64 columns; with a
// window eight) or four (128) each have a tile's loads under way. 16 tokens of 16 heads on 4 of 64 over 75000 keys: 16.5 us
// and 8 to join (tiles of 64 keys: 19, half as many waves), 75 MB of keys and
// values at 7 TB/s once the loop runs.
constexpr int kWideWaves = 4, kNarrowWaves = 1;
template <int kWaves>
constexpr int kKeyTile = kWaves == kNarrowWaves ? 32 : kTileRows;

// Keys that the last row of a tile sees bound its loop.
__device__ __forceinline__ int keys_seen(const SeqItem &s, int token, int causal) {
    if (!causal) return s.k_len;
    return clamp_to(token + 1 + s.k_len - s.q_len, 0, s.k_len);
}

// Infinities and NaN among values that a mask leaves out for some rows: 0 times
// one would reach rows that do not see it. Tiles that some row of the item does
// not see whole are cleared of them before their products, and they are added
// after the last tile to the rows that see them (add_seen_values).

// Bits of the halves of a word that are not finite: their exponents are all ones.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t lo = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u, hi = lo << 16;
    return ((w & lo) == lo ? 0xffffu : 0u) | ((w & hi) == hi ? 0xffff0000u : 0u);
}

// Clears wave `wave`'s part of a tile; whether anything was there.
template <typename T, int DK, int kTile, int kWaves>
__device__ __forceinline__ bool clear_not_finite(char *tile, int wave) {
    constexpr int kPart = kTileBytes<DK, kTile> / kWaves;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kPart / 1024; ++i) {
        i32x4 *at = reinterpret_cast<i32x4 *>(tile + wave * kPart + 1024 * i + 16 * lane_id());
        i32x4 w = *at;
        uint32_t bad[4], any = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) any |= bad[k] = not_finite<T>(w[k]);
        if (any) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] &= ~bad[k];
            *at = w;
            found = true;
        }
    }
    return ballot(found) != 0;
}

// Adds what is not finite of the run's keys from .. to - 1 to the rows that see
// them.
template <typename T, int DK, bool kWin>
__device__ __forceinline__ void add_seen_values(const char *head, int64_t tok_stride, int dim,
                                                const KeyRun &run, int from, int to, int low,
                                                int see, int half, f32x16 (&o)[DK / 32]) {
#pragma unroll 1
    for (int number = from; number < to; ++number) {
        if (kWin && number >= run.sink && number < run.sink_up) continue;
        const int key = key_at<kWin>(run, number);
        const bool sees = key < see && (!kWin || number < run.sink_up || key >= low);
        const T *row = reinterpret_cast<const T *>(head) + (int64_t)key * tok_stride;
        // No branches: a row that does not see the key adds 0.
#pragma unroll
        for (int b = 0; b < DK / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int at = 32 * b + c_row(e, half);
                const vec4<T> v = *reinterpret_cast<const vec4<T> *>(row + min(at, dim - 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float f = (float)v[k];
                    o[b][e + k] += sees && f - f != 0.f ? f : 0.f;
                }
            }
    }
}

// The result of a lane's row in columns 32 block0 .. of DK, its sums of values o
// unscaled.
template <typename T, int DK>
__device__ __forceinline__ void store_row_result(const AttnArgs &a, int token, int head, int half,
                                                 int block0, float top, float sum,
                                                 const f32x16 (&o)[DK / 32]) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t at_row = ((int64_t)token * (a.k_heads * a.group) + head) * a.dim;
    T *out = static_cast<T *>(a.out) + at_row, *rest = static_cast<T *>(a.out_rest) + at_row;
#pragma unroll
    for (int b = 0; b < DK / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int at = 32 * (block0 + b) + c_row(e, half);
            vec4<T> w, x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = o[b][e + i] * inv;
                w[i] = (T)f;
                x[i] = (T)(f - (float)w[i]);
            }
            if (at >= a.dim) continue;
            *reinterpret_cast<vec4<T> *>(out + at) = w;
            if (a.out_rest) *reinterpret_cast<vec4<T> *>(rest + at) = x;
        }
    if (a.lse && half == 0 && block0 == 0)
        a.lse[(int64_t)head * a.q_tokens + token] =
            sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
}

// Keys of the chunks of a sequence of so many tiles. One of many more tiles than
// most have longer chunks by as much, so that tiles * (keys / chunk) adds up to
// chunk_tiles * (all keys / split_keys) at most.
__device__ __forceinline__ int chunk_keys(const AttnArgs &a, int tiles) {
    if (tiles <= a.chunk_tiles) return a.split_keys;
    return a.split_keys * ((tiles + a.chunk_tiles - 1) / a.chunk_tiles);
}
// Keys that an item goes through at most: with a window, its own and the sinks'
// tiles, whatever the sequence has.
__device__ __forceinline__ int span_keys(const AttnArgs &a, int keys) {
    return min(keys + a.span_extra, a.span_most);
}
__device__ __forceinline__ int chunks_of(const AttnArgs &a, int tiles, int keys) {
    const int each = chunk_keys(a, tiles);
    return max(1, (span_keys(a, keys) + each - 1) / each);
}

// How an item's keys are cut: not at all; into chunks, whose partial results lie one
// item after the other; or into chunks whose partial results lie by their rows, for
// two sets of items over the same rows (attention_shared.hip).
enum Cut { kWhole, kByItem, kByRow };

// By rows: at most row_chunks chunks of a sequence, of split_keys at least.
template <int kTile>
__device__ __forceinline__ int row_chunk_keys(const AttnArgs &a, int keys) {
    const int even = (keys + a.row_chunks - 1) / a.row_chunks;
    return max(a.split_keys, (even + kTile - 1) / kTile * kTile);
}
template <int kTile>
__device__ __forceinline__ int row_chunks_of(const AttnArgs &a, int keys) {
    const int each = row_chunk_keys<kTile>(a, keys);
    return max(1, (keys + each - 1) / each);
}

// Row `row` (token * group + head within the group) of key head kh has its partial
// results in groups of 32 rows, a chunk's one after the other: stats (32), and
// values in the order a wave holds them, four columns 8 j + 4 half .. at a time.
__device__ __forceinline__ int64_t row_group(const AttnArgs &a, int kh, int64_t row) {
    const int64_t groups = ((int64_t)a.q_tokens * a.group + 31) / 32;
    return kh * groups + row / 32;
}
__device__ __forceinline__ float2 *row_stats(const AttnArgs &a, int kh, int64_t row, int chunk) {
    return a.part_stats + (row_group(a, kh, row) * a.row_chunks + chunk) * 32 + row % 32;
}
template <int DK>
__device__ __forceinline__ f32x4 *row_values(const AttnArgs &a, int kh, int64_t row, int chunk,
                                             int half) {
    return reinterpret_cast<f32x4 *>(a.part_o) +
           (row_group(a, kh, row) * a.row_chunks + chunk) * (32 * DK / 4) + 32 * half + row % 32;
}

// The item of a number among those cut into chunks by rows.
template <int kWaves>
__device__ __forceinline__ SeqItem find_row_item(const AttnArgs &a, int item) {
    constexpr int kRows = 32 * kWaves;
    return find_item<false>(
        a, item,
        [&](int ql, int kl) {
            return (ql * a.group + kRows - 1) / kRows * row_chunks_of<kKeyTile<kWaves>>(a, kl);
        },
        [](int, int) { return 0; });
}

// One work item: false if there is none of this number. By rows, the caller has
// found it.
template <typename T, int DK, int kWaves, Cut kCut, bool kWin>
__device__ __forceinline__ bool attn_fwd_item(const AttnArgs &a, int work, SeqItem s = {}) {
    constexpr int kRows = 32 * kWaves, kSteps = DK / 16, kBlocks = DK / 32;
    constexpr bool kInterleave = kWaves == kWideWaves;
    constexpr int kTile = kKeyTile<kWaves>, kParts = kTile / 32;
    __shared__ __align__(16) char s_tile[2][2][kTileBytes<DK, kTile>];
    // The first key of a tile that was cleared: a register of the only wave, or in
    // LDS.
    __shared__ int s_not_finite;
    int not_finite_from = 0;
    const int lane = lane_id(), half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kh = work % a.k_heads, item = work / a.k_heads, G = a.group;
    const auto tiles_of = [&](int ql, int) { return (ql * G + kRows - 1) / kRows; };
    int tile, chunk = 0, split_keys = 0;
    if constexpr (kCut == kByRow) {
        const int chunks = row_chunks_of<kTile>(a, s.k_len);
        split_keys = row_chunk_keys<kTile>(a, s.k_len);
        tile = tiles_of(s.q_len, 0) - 1 - s.within / chunks;
        chunk = s.within % chunks;
    } else if constexpr (kCut == kByItem) {
        s = find_item<false>(
            a, item,
            [&](int ql, int kl) {
                const int tiles = tiles_of(ql, kl);
                return tiles * chunks_of(a, tiles, kl);
            },
            [](int, int) { return 0; });
        if (!s.found) return false;
        const int tiles = tiles_of(s.q_len, 0), chunks = chunks_of(a, tiles, s.k_len);
        split_keys = chunk_keys(a, tiles);
        tile = tiles - 1 - s.within / chunks;
        chunk = s.within % chunks;
    } else if constexpr (kWin) {
        // Most tiles have a window's keys: no order would even them out.
        s = find_item<false>(a, item, tiles_of, [](int, int) { return 0; });
        if (!s.found) return false;
        tile = tiles_of(s.q_len, 0) - 1 - s.within;
    } else {
        s = find_longest<false>(a, item, kRows);
        if (!s.found) return false;
        tile = s.within;
    }

    // This lane's row.
    const int row0 = tile * kRows + wave * 32;
    const int row = row0 + lane % 32;
    const int token = row / G, head = kh * G + row % G;
    const bool row_ok = token < s.q_len;
    const int see = row_ok ? keys_seen(s, token, a.causal) : 0;
    // The keys of its wave's first and last row, and of the tile's.
    const int see_least = keys_seen(s, min(tile * kRows / G, s.q_len - 1), a.causal);
    const int last_token = min((tile * kRows + kRows - 1) / G, s.q_len - 1);
    const int see_first = keys_seen(s, min(row0 / G, s.q_len - 1), a.causal);
    const int see_last = keys_seen(s, min((row0 + 31) / G, s.q_len - 1), a.causal);
    const int low = kWin ? key_low(a, s, token) : 0;
    const int low_first = kWin ? key_low(a, s, min(row0 / G, s.q_len - 1)) : 0;
    const int low_last = kWin ? key_low(a, s, min((row0 + 31) / G, s.q_len - 1)) : 0;
    const int low_most = kWin ? key_low(a, s, last_token) : 0;
    const KeyRun run = key_run<kWin, kTile>(a, s, min(tile * kRows / G, s.q_len - 1),
                                            keys_seen(s, last_token, a.causal));
    int k_from = 0, k_to = run.end;               // numbers in the run
    if (kCut != kWhole) {
        k_from = min(chunk * split_keys, k_to);
        k_to = min(k_from + split_keys, k_to);
    }

    vec8<T> q[kSteps];
    {
        const T *qr = static_cast<const T *>(a.q.p) + (int64_t)(s.q_lo + token) * a.q.tok_stride +
                      (int64_t)head * a.q.head_stride;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int at = 16 * i + 8 * half;
            q[i] = memory_operand<T>(qr, at, row_ok && at < a.dim);
        }
    }
    const char *kp = reinterpret_cast<const char *>(static_cast<const T *>(a.k.p) +
                                                    (int64_t)s.k_lo * a.k.tok_stride +
                                                    (int64_t)kh * a.k.head_stride);
    const char *vp = reinterpret_cast<const char *>(static_cast<const T *>(a.v.p) +
                                                    (int64_t)s.k_lo * a.v.tok_stride +
                                                    (int64_t)kh * a.v.head_stride);
    TileFill<DK, kWaves, kTile> fill_k, fill_v;
    fill_k.init(a.k.tok_stride, a.dim, wave);
    fill_v.init(a.v.tok_stride, a.dim, wave);
    const auto ask = [&](int key0, int buf) {
        fill_k.ask(kp, a.k.tok_stride, a.dim, key0, s.k_len, wave, lds_address(s_tile[buf][0]));
        fill_v.ask(vp, a.v.tok_stride, a.dim, key0, s.k_len, wave, lds_address(s_tile[buf][1]));
    };

    f32x16 o[kBlocks] = {};
    // top: in powers of 2, what p goes by: kRise below a maximum seen.
    float top = -INFINITY, sum = 0.f;
    if constexpr (kWaves == 1)
        not_finite_from = k_to;
    else if (threadIdx.x == 0)
        s_not_finite = k_to;
    TileLane<T, DK> lane_at;
    int buf = 0;
    if (k_from < k_to) ask(key_at<kWin>(run, k_from), 0);
    loads_done();
    for (int number = k_from; number < k_to; number += kTile, buf ^= 1) {
        const int key0 = key_at<kWin>(run, number);
        const TileSees sees = tile_sees<kWin>(run, number);
        tiles_ready();
        lane_at.fresh();
        if (key0 + kTile > sees.to(see_least) || (kWin && key0 < sees.from(low_most))) {
            const bool found = clear_not_finite<T, DK, kTile, kWaves>(s_tile[buf][1], wave);
            if constexpr (kWaves == 1) {
                if (found) not_finite_from = min(not_finite_from, number);
            } else {
                if (found && lane == 0 && number < s_not_finite) s_not_finite = number;
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        const char *kt = s_tile[buf][0], *vt = s_tile[buf][1];
        f32x16 sc[kParts] = {};
        const bool more = number + kTile < k_to;
        const int next0 = key_at<kWin>(run, number + kTile);
        // The wave's rows see none of these keys.
        const bool none = key0 >= sees.to(see_last) ||
                          (kWin && key0 + kTile <= sees.from(low_first)) ||
                          (kCut == kByRow && row0 >= s.q_len * G);
        constexpr int kEach = decltype(fill_k)::kLoads;
        if (kInterleave && next0 + kTile <= s.k_len && more && !none) {
            // The next tile's loads one by one between the products: all at once
            // they queue before the wave's first product (2.4% of a prompt of
            // 16320 with 128 columns, 1% with 64).
            const auto ok = fill_k.order(kp, a.k.tok_stride, a.dim, next0, s.k_len, wave,
                                         lds_address(s_tile[buf ^ 1][0]));
            const auto ov = fill_v.order(vp, a.v.tok_stride, a.dim, next0, s.k_len, wave,
                                         lds_address(s_tile[buf ^ 1][1]));
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                for (int b = 0; b < kParts; ++b)
                    sc[b] = mfma32(lane_at.rows(kt, 32 * b, i), q[i], sc[b]);
#pragma unroll
                for (int l = i * 2 * kEach / kSteps; l < (i + 1) * 2 * kEach / kSteps; ++l)
                    if (l < kEach)
                        fill_k.load(l, ok);
                    else
                        fill_v.load(l - kEach, ov);
            }
        } else {
            if (more) ask(next0, buf ^ 1);
            if (none) continue;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int b = 0; b < kParts; ++b)
                    sc[b] = mfma32(lane_at.rows(kt, 32 * b, i), q[i], sc[b]);
        }
        if (key0 + kTile > sees.to(see_first) || (kWin && key0 < sees.from(low_last))) {
            // Selected, not added to: a NaN of a key that is not seen goes too.
            const int to = sees.to(see), from = sees.from(low);
#pragma unroll
            for (int b = 0; b < kParts; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = key0 + 32 * b + c_row(e, half);
                    if (key >= to || (kWin && key < from)) sc[b][e] = -INFINITY;
                }
        }
        float most = sc[0][0];
#pragma unroll
        for (int b = 0; b < kParts; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) most = fmaxf(most, sc[b][e]);
        most = fmaf(halves_max(most), a.scale_log2, -kRise<T>);
        if (ballot(most > top + kMaxLag<T>)) {
            const float next = fmaxf(top, most);
            // A row that has seen no finite score yet keeps zeros.
            const float shrink = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - next);
            top = next;
            sum *= shrink;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) o[b] *= shrink;
        }
        const float by = top == -INFINITY ? 0.f : top;
        vec8<T> p[2 * kParts];
#pragma unroll
        for (int b = 0; b < kParts; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(sc[b][e], a.scale_log2, -by));
                sum += x;
                // Rounded to the type of the values for the product, after
                // the sum has its full digits: half an ulp of each p (in float16
                // below 2^-25 of the largest: of 2^-25).
                p[2 * b + e / 8][e % 8] = (T)x;
            }
#pragma unroll
        for (int i = 0; i < 2 * kParts; ++i)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                o[b] = mfma32(lane_at.columns(vt, 16 * i, b), p[i], o[b]);
    }
    lds_reads_done();
    if (k_from < k_to) {
        if constexpr (kWaves > 1) not_finite_from = uniform(s_not_finite);
        if (not_finite_from < k_to)
            add_seen_values<T, DK, kWin>(vp, a.v.tok_stride, a.dim, run, not_finite_from,
                                         kWin ? k_to : min(see_last, k_to), low, see, half, o);
    }
    sum = halves_sum(sum);

    if constexpr (kCut == kByRow) {
        if (!row_ok) return true;
        const int64_t at = (int64_t)s.q_lo * G + row;
        f32x4 *po = row_values<DK>(a, kh, at, chunk, half);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                po[(4 * b + e / 4) * 64] = f32x4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]};
        if (half == 0) {
            *row_stats(a, kh, at, chunk) = make_float2(top, sum);
            // The places of chunks that this sequence has not.
            const int chunks = row_chunks_of<kTile>(a, s.k_len);
            if (chunk == chunks - 1)
                for (int c = chunks; c < a.row_chunks; ++c)
                    *row_stats(a, kh, at, c) = make_float2(-INFINITY, 0.f);
        }
        return true;
    } else if constexpr (kCut == kByItem) {
        const int64_t slot = (int64_t)work * kRows + wave * 32 + lane % 32;
        if (!row_ok) return true;
        // Narrow items hold few rows, and keep them one after the other; wide
        // ones are kept as their waves hold them, 1024 bytes a store.
        float *po = kWaves == kNarrowWaves
                        ? a.part_o + slot * DK + 4 * half
                        : a.part_o + (int64_t)work * kRows * DK + wave * 32 * DK + 4 * lane;
        constexpr int kApart = kWaves == kNarrowWaves ? 8 : 4 * 64;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<f32x4 *>(po + (4 * b + e / 4) * kApart) =
                    f32x4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]};
        if (half == 0) a.part_stats[slot] = make_float2(top, sum);
        return true;
    }
    static_assert(kWaves * kRowBytes<DK> <= (int)sizeof(s_tile), "rows in the tiles' memory");
    tiles_ready();
    const RowStore<T, DK> store{&s_tile[0][0][0] + wave * kRowBytes<DK>};
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int at_token = s.q_lo + token;
    const int64_t at_row = ((int64_t)at_token * (a.k_heads * G) + head) * a.dim;
    store(static_cast<T *>(a.out), at_row, row_ok, a.dim,
          [&](int b, int e) { return (T)(o[b][e] * inv); });
    if (a.out_rest)
        store(static_cast<T *>(a.out_rest), at_row, row_ok, a.dim, [&](int b, int e) {
            const float f = o[b][e] * inv;
            return (T)(f - (float)(T)f);
        });
    if (a.lse && half == 0 && row_ok)
        a.lse[(int64_t)head * a.q_tokens + at_token] =
            sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
    return true;
}

}  // namespace mg
