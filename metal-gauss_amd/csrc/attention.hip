// Attention over packed sequences, forward:
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
// 620 (830) and of 96 627 (980): 80 columns take the form of 96.
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
#include "attention.h"

namespace mg {

template <typename T>                             // powers of 2
constexpr float kMaxLag = std::is_same<T, f16_t>::value ? 4.f : 8.f;
template <typename T>
constexpr float kRise = std::is_same<T, f16_t>::value ? 11.f : 0.f;

// Work items come in two widths. Wide: 128 rows by four waves, tiles of 64
// keys that all four read. Narrow, where a sequence's rows would leave most of
// that empty (single tokens): 32 rows by one wave, tiles of 32 keys; memory
// bounds it, and ten waves (64 columns) or five (128) of a CU each have a
// tile's loads under way. 16 tokens of 16 heads on 4 of 64 over 75000 keys: 16.5 us
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

// One work item: false if there is none of this number.
template <typename T, int DK, int kWaves, bool kSplit, bool kWin>
__device__ __forceinline__ bool attn_fwd_item(const AttnArgs &a, int work) {
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
    SeqItem s;
    int tile, chunk = 0, split_keys = 0;
    if constexpr (kSplit) {
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
    if (kSplit) {
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
        const bool none =
            key0 >= sees.to(see_last) || (kWin && key0 + kTile <= sees.from(low_first));
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

    if constexpr (kSplit) {
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
    if (row_ok) store_row_result<T, DK>(a, s.q_lo + token, head, half, 0, top, sum, o);
    return true;
}

// How many items the chunks make is known on the device alone: as many
// workgroups as fill the GPU take them in turn.
template <typename T, int DK, int kWaves, bool kSplit, bool kWin>
__global__ __launch_bounds__(64 * kWaves, kWaves == 1 ? 1 : 2) void attn_fwd_kernel(AttnArgs a) {
    if constexpr (!kSplit) {
        attn_fwd_item<T, DK, kWaves, kSplit, kWin>(a, blockIdx.x);
    } else {
        for (int work = blockIdx.x; attn_fwd_item<T, DK, kWaves, kSplit, kWin>(a, work);
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
    if (2 * likely <= slots && mean_keys >= kSplitLeast) {
        int64_t keys = ceil_div(ceil_div(mean_keys * likely, slots), tile) * tile;
        if (keys < kChunkLeast) keys = kChunkLeast;
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
                    with(waves, bool_constant<true>{});
                else
                    with(waves, bool_constant<false>{});
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
