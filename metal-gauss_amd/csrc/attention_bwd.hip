// Attention's backward pass, from the rows' lse of the forward:
//
//   p_ij = exp(scale q_i k_j - lse_i)
//   dv_j = sum_i p_ij do_i
//   ds_ij = p_ij (do_i v_j - delta_i),  delta_i = do_i o_i
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// delta takes o with what rounding took from it (out_rest), where the forward
// kept that: delta's error enters every ds of a row with the same sign.
//
// Two kernels form the scores once each: the queries' gradient goes over the
// keys and keeps its sums in registers, the keys' and values' goes over the
// queries of all heads that share them. Seven products in place of the five of
// a single pass, but no gradient is added to memory by several workgroups: no
// atomics, no float32 copy of dq, and the same bits from call to call.
//
// float16: p and ds of a long row lie where float16 has few digits or none left
// (p of 16000 equal keys is 6e-5), so p enters its product 2^15 times as large,
// and ds by a power of two that takes the largest ds there can be,
// 2 max|do| max|v|, to about 2^14; the results are scaled back in float32. The
// maxima are those of the item's own sequence and key head (in the queries'
// gradient, whose sums are a row's own, of the row's do), so that neither a
// sequence packed with it nor tokens of none take digits from it. bfloat16 has
// float32's range and needs neither.
//
// 8192 tokens, 16 heads of 128 bfloat16: queries 800 us, keys 1092 (1030 and 1010 TFLOP/s);
// of 64: 487 and 635 (850 and 870). The queries' kernel is never cut over its keys:
// 64 queries over 16000 of them, 16 heads on 4 of 128, take 417 us. With a window of 475
// and 4 sinks 7033 packed tokens (16 heads on 4 of 128) take 94 and 106. As the
// forward, both need two waves a SIMD to keep products and exponentials going side by
// side: the keys' kernel with one (256 columns of sums and operands in 472 registers)
// took 1970.
#include "attention.h"

namespace mg {

constexpr int kBwdWaves = 4;
constexpr int kBwdTile = 32 * kBwdWaves;         // rows, or keys, of a work item

template <typename T>
constexpr float kPowerP = sizeof(T) == 2 && std::is_same<T, f16_t>::value ? 15.f : 0.f;

// A sequence's tokens in tiles of 64 have a place each in an array of this many:
// tile t of sequence seq, whose tokens begin at lo, is at lo / 64 + seq + t.
__host__ __device__ constexpr int64_t norm_places(int64_t tokens, int64_t n_seq) {
    return tokens / kTileRows + n_seq + 2;
}

// The largest |row|^2 of a tile's tokens in do (blockIdx.y 0: over the query heads
// that share the key head) and in v (1). Tokens of no sequence are not looked at.
// A NaN counts as nothing.
constexpr int kLargestThreads = 256;

template <typename T>
__global__ __launch_bounds__(kLargestThreads) void attn_largest_kernel(AttnArgs a) {
    __shared__ float s_most[kLargestThreads / 64];
    const bool of_v = blockIdx.y != 0;
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads;
    const auto tiles_of = [&](int ql, int kl) {
        return ((of_v ? kl : ql) + kTileRows - 1) / kTileRows;
    };
    const auto none = [](int, int) { return 0; };
    const SeqItem s = of_v ? find_item<true>(a, item, tiles_of, none)
                           : find_item<false>(a, item, tiles_of, none);
    if (!s.found || s.seq == 0 || s.seq > a.n_seq) return;
    const AttnTensor &x = of_v ? a.v : a.dout;
    const int heads = of_v ? 1 : a.group, lo = of_v ? s.k_lo : s.q_lo;
    const int tokens = min((of_v ? s.k_len : s.q_len) - s.within * kTileRows, kTileRows);
    const T *from = static_cast<const T *>(x.p) +
                    (int64_t)(lo + s.within * kTileRows) * x.tok_stride +
                    (int64_t)(kh * heads) * x.head_stride;
    // 16 lanes a row, eight elements each, four rows asked for at once.
    const int at = threadIdx.x % 16 * 8, rows = tokens * heads;
    float most = 0.f;
    for (int row = threadIdx.x / 16; row < rows; row += 4 * 16) {
        float f[4][8] = {};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = row + k * 16, token = r / heads, head = r % heads;
            if (r < rows && at < a.dim)
                load_vec<T, 8>(from + token * x.tok_stride + head * x.head_stride + at, f[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sq = fmaf(f[k][i], f[k][i], sq);
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) sq += __shfl_xor(sq, o, 16);
            most = fmaxf(most, sq);
        }
    }
    most = wave_max(most);
    if (lane_id() == 0) s_most[threadIdx.x / 64] = most;
    __syncthreads();
    if (threadIdx.x == 0)
        (of_v ? a.largest_v : a.largest_do)[
            kh * norm_places(of_v ? a.k_tokens : a.q_tokens, a.n_seq) + lo / kTileRows + s.seq +
            s.within] = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
}

// The largest of a sequence, whose `len` tokens of `tokens` begin at lo.
__device__ __forceinline__ float seq_largest(const AttnArgs &a, const float *largest, int kh,
                                             int tokens, int seq, int lo, int len) {
    const float *p = largest + kh * norm_places(tokens, a.n_seq) + lo / kTileRows + seq;
    float most = 0.f;
    for (int t = lane_id(); t * kTileRows < len; t += 64) most = fmaxf(most, p[t]);
    return wave_max(most);
}

// The power of two that ds is taken by, from the largest |do|^2 and |v|^2 it can
// be of.
__device__ __forceinline__ float ds_power(float do_sq, float v_sq) {
    const float l = 13.f - 0.5f * (__builtin_amdgcn_logf(do_sq) + __builtin_amdgcn_logf(v_sq));
    return l > -100.f && l < 100.f ? floorf(l) : 0.f;
}

// ------------------------------------------------------- the queries' gradient
// With a window results leave by whole rows, by way of LDS, as the few keys of an item
// leave its rows most of the time; without one the stores' code weighs more in the loop
// than it gains behind it: seven sequences of 7033 tokens, 16 heads on 4 of 128
// bfloat16, unmasked, 254 us so and 230 by fours (causal 134 and 128; of 64 columns, where it
// took registers past the 128 of four waves a SIMD, 86 and 82). Of 32 columns it is no
// slower, float16's 213 and 205.
template <typename T, int DK, bool kWin>
__global__ __launch_bounds__(64 * kBwdWaves, 2) void attn_dq_kernel(AttnArgs a) {
    constexpr int kSteps = DK / 16, kBlocks = DK / 32;
    __shared__ __align__(16) char s_tile[2][2][kTileBytes<DK>];
    const int lane = lane_id(), half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads, G = a.group;
    const auto tiles_of = [&](int ql, int) { return (ql * G + kBwdTile - 1) / kBwdTile; };
    const SeqItem s = kWin ? find_item<false>(a, item, tiles_of, [](int, int) { return 0; })
                           : find_longest<false>(a, item, kBwdTile);
    if (!s.found) return;
    const int tile = kWin ? tiles_of(s.q_len, 0) - 1 - s.within : s.within;
    const auto sees = [&](int token) {
        return a.causal ? clamp_to(token + 1 + s.k_len - s.q_len, 0, s.k_len) : s.k_len;
    };
    const int row0 = tile * kBwdTile + wave * 32;
    const int row = row0 + lane % 32;
    const int token = row / G, head = kh * G + row % G;
    const bool row_ok = token < s.q_len;
    const int see = row_ok ? sees(token) : 0;
    const int see_first = sees(min(row0 / G, s.q_len - 1));
    const int see_last = sees(min((row0 + 31) / G, s.q_len - 1));
    const int low = kWin ? key_low(a, s, token) : 0;
    const int low_first = kWin ? key_low(a, s, min(row0 / G, s.q_len - 1)) : 0;
    const int low_last = kWin ? key_low(a, s, min((row0 + 31) / G, s.q_len - 1)) : 0;
    const KeyRun run = key_run<kWin, kTileRows>(
        a, s, min(tile * kBwdTile / G, s.q_len - 1),
        sees(min((tile * kBwdTile + kBwdTile - 1) / G, s.q_len - 1)));

    vec8<T> q[kSteps], dout[kSteps];
    float lse = INFINITY, delta = 0.f, do_sq = 0.f;
    {
        const T *qr = static_cast<const T *>(a.q.p) + (int64_t)(s.q_lo + token) * a.q.tok_stride +
                      (int64_t)head * a.q.head_stride;
        const T *dor = static_cast<const T *>(a.dout.p) +
                       (int64_t)(s.q_lo + token) * a.dout.tok_stride +
                       (int64_t)head * a.dout.head_stride;
        const int64_t at_row = ((int64_t)(s.q_lo + token) * (a.k_heads * G) + head) * a.dim;
        const T *outr = static_cast<const T *>(a.out) + at_row;
        const T *restr = static_cast<const T *>(a.out_rest) + at_row;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int at = 16 * i + 8 * half;
            const bool ok = row_ok && at < a.dim;
            q[i] = memory_operand<T>(qr, at, ok);
            dout[i] = memory_operand<T>(dor, at, ok);
            const vec8<T> out = memory_operand<T>(outr, at, ok);
            const vec8<T> rest = memory_operand<T>(restr, at, ok && a.out_rest);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                delta = fmaf((float)dout[i][k], (float)out[k] + (float)rest[k], delta);
                if constexpr (kPowerP<T> != 0.f)
                    do_sq = fmaf((float)dout[i][k], (float)dout[i][k], do_sq);
            }
        }
        delta = halves_sum(delta);
        if (row_ok) {
            const int64_t at = (int64_t)head * a.q_tokens + s.q_lo + token;
            lse = a.lse[at];
            if (half == 0) const_cast<float *>(a.delta)[at] = delta;
        }
    }
    const char *kp = reinterpret_cast<const char *>(static_cast<const T *>(a.k.p) +
                                                    (int64_t)s.k_lo * a.k.tok_stride +
                                                    (int64_t)kh * a.k.head_stride);
    const char *vp = reinterpret_cast<const char *>(static_cast<const T *>(a.v.p) +
                                                    (int64_t)s.k_lo * a.v.tok_stride +
                                                    (int64_t)kh * a.v.head_stride);
    TileFill<DK, kBwdWaves> fill_k, fill_v;
    fill_k.init(a.k.tok_stride, a.dim, wave);
    fill_v.init(a.v.tok_stride, a.dim, wave);
    const auto ask = [&](int key0, int buf) {
        fill_k.ask(kp, a.k.tok_stride, a.dim, key0, s.k_len, wave, lds_address(s_tile[buf][0]));
        fill_v.ask(vp, a.v.tok_stride, a.dim, key0, s.k_len, wave, lds_address(s_tile[buf][1]));
    };
    float power = 0.f;                   // this lane's row's
    if constexpr (kPowerP<T> != 0.f)
        power = ds_power(halves_sum(do_sq), seq_largest(a, a.largest_v, kh, a.k_tokens, s.seq,
                                                        s.k_lo, s.k_len));
    const float up = __builtin_amdgcn_exp2f(power);
    const float delta_up = delta * up;

    f32x16 dq[kBlocks] = {};
    TileLane<T, DK> lane_at;
    int buf = 0;
    if (run.end > 0) ask(key_at<kWin>(run, 0), 0);
    loads_done();
    for (int number = 0; number < run.end; number += kTileRows, buf ^= 1) {
        const int key0 = key_at<kWin>(run, number);
        const TileSees in = tile_sees<kWin>(run, number);
        tiles_ready();
        lane_at.fresh();
        if (number + kTileRows < run.end) ask(key_at<kWin>(run, number + kTileRows), buf ^ 1);
        if (key0 >= in.to(see_last) || (kWin && key0 + kTileRows <= in.from(low_first))) continue;
        const char *kt = s_tile[buf][0], *vt = s_tile[buf][1];
        const bool masked =
            key0 + kTileRows > in.to(see_first) || (kWin && key0 < in.from(low_last));
        const int to = in.to(see), from = in.from(low);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                sc = mfma32(lane_at.rows(kt, 32 * b, i), q[i], sc);
                dp = mfma32(lane_at.rows(vt, 32 * b, i), dout[i], dp);
            }
            vec8<T> ds[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(fmaf(sc[e], a.scale_log2, -lse));
                float d = p * fmaf(dp[e], up, -delta_up);
                // Selected: what is not seen may be anything.
                const int key = key0 + 32 * b + c_row(e, half);
                if (masked && (key >= to || (kWin && key < from))) d = 0.f;
                ds[e / 8][e % 8] = (T)d;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < kBlocks; ++c)
                    dq[c] = mfma32(lane_at.columns(kt, 32 * b + 16 * i, c), ds[i], dq[c]);
        }
    }
    lds_reads_done();
    const float down = a.scale * __builtin_amdgcn_exp2f(-power);
    const int64_t at_row = ((int64_t)(s.q_lo + token) * (a.k_heads * G) + head) * a.dim;
    T *out = static_cast<T *>(a.dq);
    if constexpr (kWin || DK == 32) {
        static_assert(kBwdWaves * kRowBytes<DK> <= (int)sizeof(s_tile), "rows in the tiles' memory");
        tiles_ready();
        const RowStore<T, DK> store{&s_tile[0][0][0] + wave * kRowBytes<DK>};
        store(out, at_row, row_ok, a.dim, [&](int b, int e) { return (T)(dq[b][e] * down); });
    } else {
        if (!row_ok) return;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int at = 32 * b + c_row(e, half);
                vec4<T> w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (T)(dq[b][e + i] * down);
                if (at < a.dim) *reinterpret_cast<vec4<T> *>(out + at_row + at) = w;
            }
    }
}

// ------------------------------------------- the keys' and values' gradients
// Asks for 64 rows' lse and delta (past the last row, the last row's again).
__device__ __forceinline__ void ask_row_values(const float *at, int rows, uint32_t lds) {
    const uint32_t off = 4 * min(lane_id(), rows - 1);
    const i32x4 rsrc = buffer_of(at, 4 * rows);
    asm volatile("s_mov_b32 m0, %0\n\t"
                 "s_nop 4\n\t"
                 "buffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(uniform((int)lds)), "v"(off), "s"(rsrc)
                 : "m0", "memory");
}

// A run's sums for one key tile, in the order the waves hold them (a store is
// 1024 bytes in a row): dk, then dv, a wave's blocks one after the other.
template <int DK>
constexpr int kPartFours = 2 * kBwdTile * DK / 4;

template <int DK>
__device__ __forceinline__ f32x4 *part_of(const AttnArgs &a, int item, int kh, int split) {
    return reinterpret_cast<f32x4 *>(a.part) +
           (((int64_t)item * a.k_heads + kh) * a.splits + split) * kPartFours<DK>;
}

// With a window, the queries that see a key tile are few, but those further on all
// see the sinks. Where these are many (sink_cut), their sums for the sinks are work items
// of their own, which come last, being short ones (first, those of 7033 packed tokens,
// window 475, took 17% longer): one tile of kBwdTile keys and a run of query tiles each.
// Their sums, of sink_rows keys, have a place each in sink_part, and so have those of the
// window items of key tiles that have sinks; attn_sink_sum_kernel adds them up, in
// order. A sequence's places follow one another, a key tile's far items' and then
// its window items'. A sequence with few far queries has its window items go on for them
// (512 of 64 tokens, 16 heads on 4 of 128, window 16 and 4 sinks, both gradients: 914 us
// with items and places of their own, so 476).
static_assert(kSinkTokens == kTileRows && kSinkKeys == kBwdTile, "tiles of the items");

struct SinkItems : SinkCut {
    __device__ __forceinline__ SinkItems(const AttnArgs &a, int q_len, int k_len)
        : SinkCut(sink_cut(q_len, k_len, a.window, a.sinks, a.group, a.sink_steps,
                           a.sink_near)) {}
    // Places of a key tile, and of a sequence; items of a sequence.
    __device__ __forceinline__ int places(const AttnArgs &a) const { return runs + a.splits; }
    __device__ __forceinline__ int all(const AttnArgs &a) const { return key_tiles * places(a); }
    __device__ __forceinline__ int items() const { return key_tiles * runs; }
};

template <int DK>
__device__ __forceinline__ f32x4 *sink_part_of(const AttnArgs &a, int place, int kh) {
    return reinterpret_cast<f32x4 *>(a.sink_part) +
           ((int64_t)place * a.k_heads + kh) * (2 * a.sink_rows * DK / 4);
}

// The query tiles that see a key tile (tiles of each of the group's heads, from
// q_from), and the runs they are cut into: whole heads, or `parts` of each head
// where there are more runs than heads. Key tiles that run at the same time then
// read the same heads' queries, which stay in their XCD's L2. `on`: the tile has sinks
// that no other items have the later queries of.
struct KeySteps {
    int q_from, tiles, runs, parts;
};

template <bool kWin>
__device__ __forceinline__ KeySteps key_steps(const AttnArgs &a, const SeqItem &s, int first_key,
                                             bool on) {
    const int ahead = s.k_len - s.q_len, G = a.group;
    int from = a.causal ? max(0, first_key - ahead) / kTileRows * kTileRows : 0, to = s.q_len;
    if constexpr (kWin) {
        from = max(0, first_key - ahead);
        const int last = min(first_key + kBwdTile, s.k_len) - 1;
        to = (int)min((int64_t)s.q_len, max((int64_t)0, (int64_t)last + a.window - ahead));
        if (on) to = s.q_len;
    }
    const int tiles = from < to ? (to - from + kTileRows - 1) / kTileRows : 0;
    int runs = (int)(((int64_t)tiles * G + a.split_steps - 1) / a.split_steps);
    runs = even_runs(clamp_to(runs, 1, a.splits), G, a.splits);
    return {from, tiles, runs, runs > G ? runs / G : 1};
}

template <typename T, int DK, bool kWin>
__global__ __launch_bounds__(64 * kBwdWaves, 2) void attn_dkv_kernel(AttnArgs a) {
    constexpr int kSteps = DK / 16, kBlocks = DK / 32;
    __shared__ __align__(16) char s_tile[2][2][kTileBytes<DK>];
    __shared__ __align__(16) float s_row[2][2][kTileRows];     // lse, delta
    const int lane = lane_id(), half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kh = blockIdx.x % a.k_heads, at_item = blockIdx.x / a.k_heads;
    // Queries past the window, for the sinks.
    const bool far = kWin && at_item >= a.key_runs;
    const auto sink_count = [&](int ql, int kl) { return SinkItems(a, ql, kl).all(a); };
    const auto key_tiles = [&](int, int kl) { return (kl + kBwdTile - 1) / kBwdTile; };
    const auto far_items = [&](int ql, int kl) { return SinkItems(a, ql, kl).items(); };
    const int item = at_item / a.splits, split = at_item % a.splits;
    SeqItem s;
    if constexpr (kWin)
        s = far ? find_item<true>(a, at_item - a.key_runs, far_items, sink_count)
                : find_item<true>(a, item, key_tiles, sink_count);
    else
        s = find_longest<true>(a, item, kBwdTile);
    if (!s.found) return;
    KeySteps steps_of;
    int first_key = s.within * kBwdTile, sink_run = 0, sink_runs = 0, sink_place = 0;
    int sinks_to = 0;            // keys below it count as sinks in this item
    if (kWin && a.sinks > 0) {
        const SinkItems of(a, s.q_len, s.k_len);
        sink_runs = of.runs;
        if (far || sink_runs == 0) sinks_to = a.sinks;
        if (far) {
            const int tile = s.within / sink_runs;
            first_key = tile * kBwdTile;
            sink_run = s.within % sink_runs;
            sink_place = s.before + tile * of.places(a) + sink_run;
            steps_of = {of.from, of.tiles, sink_runs,
                        sink_runs > a.group ? sink_runs / a.group : 1};
        } else {
            sink_place = s.before + s.within * of.places(a) + sink_runs + split;
        }
    }
    if (!far) {
        steps_of = key_steps<kWin>(a, s, first_key, first_key < sinks_to);
        if (split >= steps_of.runs) return;
    }
    const int key0 = first_key + wave * 32, key = key0 + lane % 32;
    const bool key_ok = key < s.k_len;
    const int ahead = s.k_len - s.q_len;       // query i sees keys up to i + ahead
    // This run's heads, and its query tiles of each.
    const int parts = steps_of.parts, runs = steps_of.runs / parts;
    const int nth = far ? sink_run : split, run = nth / parts, piece = nth % parts;
    const int g_from = run * a.group / runs, heads = (run + 1) * a.group / runs - g_from;
    const int t_from = (int)((int64_t)steps_of.tiles * piece / parts);
    const int tiles = (int)((int64_t)steps_of.tiles * (piece + 1) / parts) - t_from;
    const int q_from = steps_of.q_from + t_from * kTileRows;
    const int q_to = q_from + tiles * kTileRows;

    vec8<T> k[kSteps], v[kSteps];
    {
        const T *kr = static_cast<const T *>(a.k.p) + (int64_t)(s.k_lo + key) * a.k.tok_stride +
                      (int64_t)kh * a.k.head_stride;
        const T *vr = static_cast<const T *>(a.v.p) + (int64_t)(s.k_lo + key) * a.v.tok_stride +
                      (int64_t)kh * a.v.head_stride;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int at = 16 * i + 8 * half;
            const bool ok = key_ok && at < a.dim;
            k[i] = memory_operand<T>(kr, at, ok);
            v[i] = memory_operand<T>(vr, at, ok);
        }
    }
    TileFill<DK, kBwdWaves> fill_q, fill_do;
    fill_q.init(a.q.tok_stride, a.dim, wave);
    fill_do.init(a.dout.tok_stride, a.dim, wave);
    const auto ask = [&](int g, int row0, int buf) {
        const int head = kh * a.group + g;
        const char *qp = reinterpret_cast<const char *>(static_cast<const T *>(a.q.p) +
                                                        (int64_t)s.q_lo * a.q.tok_stride +
                                                        (int64_t)head * a.q.head_stride);
        const char *dop = reinterpret_cast<const char *>(
            static_cast<const T *>(a.dout.p) + (int64_t)s.q_lo * a.dout.tok_stride +
            (int64_t)head * a.dout.head_stride);
        fill_q.ask(qp, a.q.tok_stride, a.dim, row0, s.q_len, wave, lds_address(s_tile[buf][0]));
        fill_do.ask(dop, a.dout.tok_stride, a.dim, row0, s.q_len, wave,
                    lds_address(s_tile[buf][1]));
        if (wave < 2) {
            const float *from = wave == 0 ? a.lse : a.delta;
            ask_row_values(from + (int64_t)head * a.q_tokens + s.q_lo + row0,
                           min(s.q_len - row0, kTileRows),
                           lds_address(reinterpret_cast<const char *>(s_row[buf][wave])));
        }
    };
    float power = 0.f;
    if constexpr (kPowerP<T> != 0.f)
        power = ds_power(
            seq_largest(a, a.largest_do, kh, a.q_tokens, s.seq, s.q_lo, s.q_len),
            seq_largest(a, a.largest_v, kh, a.k_tokens, s.seq, s.k_lo, s.k_len));
    const float ds_up = __builtin_amdgcn_exp2f(power - kPowerP<T>);

    // With a window: the queries that see this lane's key, `sees` from sees_from on, of
    // those that are this item's.
    int sees_from = 0;
    uint32_t sees = 0;
    if constexpr (kWin) {
        const int past = max(0, key - ahead + a.window);
        sees_from = far ? past : max(0, key - ahead);
        const int to = far || key < sinks_to ? s.q_len : min(s.q_len, past);
        if (key_ok && (!far || key < sinks_to)) sees = max(0, to - sees_from);
    }

    f32x16 dk[kBlocks] = {}, dv[kBlocks] = {};
    const int steps = tiles * heads;
    TileLane<T, DK> lane_at;
    int g = g_from, row0 = q_from, buf = 0;
    if (steps > 0) ask(g, row0, 0);
    loads_done();
    for (int step = 0; step < steps; ++step, buf ^= 1) {
        tiles_ready();
        lane_at.fresh();
        const int at_row0 = row0;
        row0 += kTileRows;
        if (row0 >= q_to) {
            row0 = q_from;
            ++g;
        }
        if (step + 1 < steps) ask(g, row0, buf ^ 1);
        const char *qt = s_tile[buf][0], *dot = s_tile[buf][1];
        // Every row of the tile sees every key of the wave?
        bool masked = at_row0 + kTileRows > s.q_len || key0 + 32 > s.k_len ||
                      (a.causal && at_row0 + ahead < key0 + 31);
        if (a.causal && at_row0 + kTileRows - 1 + ahead < key0) continue;    // none sees any
        if constexpr (kWin) {
            // How far on the tile's rows stand, of the wave's keys.
            const int least = at_row0 + ahead - (key0 + 31);
            const int most = at_row0 + kTileRows - 1 + ahead - key0;
            if (far ? key0 >= sinks_to || most < a.window : key0 >= sinks_to && least >= a.window)
                continue;
            masked |= far ? key0 + 32 > sinks_to || least < a.window : most >= a.window;
        }
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
            f32x16 sc = {}, dp = {};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                sc = mfma32(lane_at.rows(qt, 32 * b, i), k[i], sc);
                dp = mfma32(lane_at.rows(dot, 32 * b, i), v[i], dp);
            }
            vec8<T> p[2], ds[2];
#pragma unroll
            for (int e4 = 0; e4 < 16; e4 += 4) {
                const int r = 32 * b + c_row(e4, half);
                const f32x4 lse = *reinterpret_cast<const f32x4 *>(&s_row[buf][0][r]);
                const f32x4 delta = *reinterpret_cast<const f32x4 *>(&s_row[buf][1][r]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = e4 + i;
                    float x = __builtin_amdgcn_exp2f(
                        fmaf(sc[e], a.scale_log2, kPowerP<T> - lse[i]));
                    float d = x * ((dp[e] - delta[i]) * ds_up);
                    if (masked) {
                        const int token = at_row0 + r + i;
                        bool seen;
                        if constexpr (kWin) {
                            // Keeps this a branch: as selects it costs every tile (16320
                            // tokens, window 1900: 1229 us with the queries', so 1075).
                            asm volatile("");
                            seen = (uint32_t)(token - sees_from) < sees;
                        } else {
                            seen = token < s.q_len && key_ok && (!a.causal || key <= token + ahead);
                        }
                        x = seen ? x : 0.f;
                        d = seen ? d : 0.f;
                    }
                    p[e / 8][e % 8] = (T)x;
                    ds[e / 8][e % 8] = (T)d;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < kBlocks; ++c) {
                    dv[c] = mfma32(lane_at.columns(dot, 32 * b + 16 * i, c), p[i], dv[c]);
                    dk[c] = mfma32(lane_at.columns(qt, 32 * b + 16 * i, c), ds[i], dk[c]);
                }
        }
    }
    lds_reads_done();
    const float down = a.scale * __builtin_amdgcn_exp2f(-power);
    const float down_v = __builtin_amdgcn_exp2f(-kPowerP<T>);
    const bool sinks_apart = kWin && sink_runs > 0 && key < a.sinks;
    if (sinks_apart) {
        f32x4 *part = sink_part_of<DK>(a, sink_place, kh) + wave * kBlocks * 4 * 64 + lane;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                f32x4 w, x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = dk[b][e + i] * down;
                    x[i] = dv[b][e + i] * down_v;
                }
                part[(b * 4 + e / 4) * 64] = w;
                part[(b * 4 + e / 4) * 64 + a.sink_rows * DK / 4] = x;
            }
    }
    if (kWin && far) return;
    if (steps_of.runs > 1) {
        if (sinks_apart) return;
        f32x4 *part = part_of<DK>(a, item, kh, split) + wave * kBlocks * 4 * 64 + lane;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                f32x4 w, x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = dk[b][e + i] * down;
                    x[i] = dv[b][e + i] * down_v;
                }
                part[(b * 4 + e / 4) * 64] = w;
                part[(b * 4 + e / 4) * 64 + kPartFours<DK> / 2] = x;
            }
        return;
    }
    if (!key_ok || sinks_apart) return;
    const int64_t at_row = ((int64_t)(s.k_lo + key) * a.k_heads + kh) * a.dim;
    T *dkr = static_cast<T *>(a.dk) + at_row, *dvr = static_cast<T *>(a.dv) + at_row;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int at = 32 * b + c_row(e, half);
            vec4<T> w, x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = (T)(dk[b][e + i] * down);
                x[i] = (T)(dv[b][e + i] * down_v);
            }
            if (at < a.dim) {
                *reinterpret_cast<vec4<T> *>(dkr + at) = w;
                *reinterpret_cast<vec4<T> *>(dvr + at) = x;
            }
        }
}

// The sums of the keys' tiles that were cut into runs, in order. A workgroup has
// 32 columns of dk or dv of one tile of one key head, its threads the elements
// that attn_dkv_kernel's have.
template <typename T, int DK, bool kWin>
__global__ __launch_bounds__(64 * kBwdWaves) void attn_sum_kernel(AttnArgs a) {
    constexpr int kBlocks = DK / 32;
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads;
    const auto key_tiles = [](int, int kl) { return (kl + kBwdTile - 1) / kBwdTile; };
    const SeqItem s = kWin ? find_item<true>(a, item, key_tiles, [](int, int) { return 0; })
                           : find_longest<true>(a, item, kBwdTile);
    if (!s.found) return;
    const int first_key = s.within * kBwdTile;
    // attn_sink_sum_kernel has the sinks that have items of their own.
    const bool sinks_apart =
        kWin && first_key < a.sinks && SinkItems(a, s.q_len, s.k_len).runs > 0;
    const int runs = key_steps<kWin>(a, s, first_key, first_key < a.sinks && !sinks_apart).runs;
    if (runs == 1) return;
    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / 64);
    const int key = first_key + wave * 32 + lane % 32;
    const int64_t at_row = ((int64_t)(s.k_lo + key) * a.k_heads + kh) * a.dim;
    const f32x4 *part = part_of<DK>(a, item, kh, 0) + wave * kBlocks * 4 * 64 + lane;
    const int which = blockIdx.y % 2, block = blockIdx.y / 2;
    if (sinks_apart && key < a.sinks) return;
#pragma unroll
    for (int i = 4 * block; i < 4 * block + 4; ++i) {
        const f32x4 *p = part + i * 64 + which * kPartFours<DK> / 2;
        f32x4 sum = *p;
        for (int k = 1; k < runs; ++k) sum += p[k * kPartFours<DK>];
        const int at = 32 * block + c_row(i % 4 * 4, half);
        if (key < s.k_len && at < a.dim)
            *reinterpret_cast<vec4<T> *>(static_cast<T *>(which ? a.dv : a.dk) + at_row + at) =
                __builtin_convertvector(sum, vec4<T>);
    }
}

// The sinks' sums: a workgroup has four columns in each half of a wave, of 32 sinks,
// of dk or dv, and its waves every kSinkWaves-th place (16 waves: both gradients
// of 7033 packed tokens 207 us in place of 196). How many key tiles have sums, of `tiles` at most, the device
// alone knows: as many workgroups as run at once take them in turn (512 sequences of 64
// tokens that have none: 14 us, with a workgroup for each there might be 74).
constexpr int kSinkWaves = 4;
constexpr int64_t kSinkSlots = 2048;
template <typename T, int DK>
__global__ __launch_bounds__(64 * kSinkWaves) void attn_sink_sum_kernel(AttnArgs a, int tiles) {
    constexpr int kBlocks = DK / 32;
    __shared__ f32x4 s_sum[kSinkWaves][64];
    const int kh = blockIdx.x % a.k_heads;
    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / 64);
    const int i = blockIdx.y % (kBlocks * 4), rows = blockIdx.y / (kBlocks * 4) / 2 * 32;
    const int which = blockIdx.y / (kBlocks * 4) % 2;
    for (int item = blockIdx.x / a.k_heads; item < tiles; item += gridDim.x / a.k_heads) {
        const SeqItem s = find_item<true>(
            a, item, [&](int ql, int kl) { return SinkItems(a, ql, kl).key_tiles; },
            [&](int ql, int kl) { return SinkItems(a, ql, kl).all(a); });
        if (!s.found) return;
        const SinkItems of(a, s.q_len, s.k_len);
        const int first_key = s.within * kBwdTile;
        const int places = of.runs + key_steps<true>(a, s, first_key, false).runs;
        const int key = first_key + rows + lane % 32, at = 32 * (i / 4) + c_row(i % 4 * 4, half);
        const f32x4 *from = sink_part_of<DK>(a, s.before + s.within * of.places(a), kh) +
                            (rows / 32 * kBlocks * 4 + i) * 64 + lane +
                            which * (a.sink_rows * DK / 4);
        const int64_t step = (int64_t)a.k_heads * (2 * a.sink_rows * DK / 4);
        f32x4 sum = {};
        if (key < a.sinks) {
#pragma unroll 8
            for (int p = wave; p < places; p += kSinkWaves) sum += from[p * step];
        }
        s_sum[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && key < min(a.sinks, s.k_len) && at < a.dim) {
            for (int w = 1; w < kSinkWaves; ++w) sum += s_sum[w][lane];
            *reinterpret_cast<vec4<T> *>(static_cast<T *>(which ? a.dv : a.dk) +
                                         ((int64_t)(s.k_lo + key) * a.k_heads + kh) * a.dim + at) =
                __builtin_convertvector(sum, vec4<T>);
        }
        __syncthreads();
    }
}

// Bytes of the backward's scratch: delta, the largest norms, and the runs' sums.
// The keys' gradients are cut into runs where their tiles are fewer than fill
// the GPU twice over, of eight query tiles at least (7033 packed tokens, 62 tiles
// on 4 key heads: 528 us uncut, 187 and 27 to add the runs in four).
struct BwdPlan {
    int64_t k_items, largest_at, part_at, sink_at, bytes;
    int splits, split_steps;
    int64_t sink_items, sink_places, sink_tiles;
    int sink_steps, sink_rows;
};

constexpr int64_t kBwdRuns = 1024, kBwdRunLeast = 8, kBwdMostSplits = 8;
// With a window: as many as fill the GPU, as partial results weigh more beside fewer
// queries (both gradients of 7033 packed tokens, window 475, take 196 us, 226 with twice as
// many and 237 with half), of four query tiles at least (nine sequences of 3 to 1210
// tokens, 6 heads on 3 of 128: 84 us, of eight 92). As many runs of far items, of
// sink_steps = kSinkStepsLeast tiles at least (of eight: the nine sequences 105 us).
constexpr int64_t kBwdWindowRuns = 512, kBwdWindowRunLeast = 4, kSinkItems = 512, kSinkStepsLeast = 4;

static BwdPlan bwd_plan(int64_t q_tokens, int64_t k_tokens, int64_t k_heads, int64_t group,
                        int64_t dim, int64_t n_seq, int64_t window, int64_t sinks) {
    BwdPlan p{};
    p.k_items = k_tokens / kBwdTile + n_seq + 2;
    const int64_t tiles = (ceil_div(k_tokens, kBwdTile) + n_seq - 1) * k_heads;
    int64_t queries = ceil_div(q_tokens, n_seq * kTileRows);
    // The most that any key tile has, not the average: of unequal sequences the longer
    // ones are cut, the shorter ones' items have steps for one run and stay whole (12
    // sequences of 5 to 1461 tokens, 4 heads on 2 of 128: 31 us and 8 to add the runs, by
    // the average 43 and 6; 32 equal ones of 100: 26 and 4, by the average 23).
    if (window > 0) {
        const int64_t seen = ceil_div(window + kBwdTile, kTileRows);
        queries = ceil_div(q_tokens, kTileRows);
        if (queries > seen) queries = seen;
    }
    const int64_t steps = queries * group;
    int64_t splits = (window > 0 ? kBwdWindowRuns : kBwdRuns) / (tiles > 0 ? tiles : 1);
    const int64_t least = window > 0 ? kBwdWindowRunLeast : kBwdRunLeast;
    if (splits > steps / least) splits = steps / least;
    splits = splits < 1 ? 1 : splits > kBwdMostSplits ? kBwdMostSplits : splits;
    p.splits = even_runs((int)splits, (int)group, (int)kBwdMostSplits);
    p.split_steps = (int)least;
    p.largest_at = align256(q_tokens * k_heads * group * 4);
    p.part_at = align256(p.largest_at + k_heads * 4 * (norm_places(q_tokens, n_seq) +
                                                       norm_places(k_tokens, n_seq)));
    p.bytes = p.part_at;
    const int64_t dk = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
    if (p.splits > 1) p.bytes += p.k_items * k_heads * p.splits * 2 * kBwdTile * dk * 4;
    p.sink_at = p.bytes;
    p.sink_steps = 1;
    if (sinks > 0) {
        int64_t most = ceil_div(q_tokens, kTileRows) * group * k_heads *
                       ceil_div(sinks, kBwdTile) / kSinkItems;
        most = most < kSinkStepsLeast ? kSinkStepsLeast : most < (1 << 30) ? most : 1 << 30;
        p.sink_steps = (int)most;
        p.sink_rows = (int)(sinks < kBwdTile ? ceil_div(sinks, 32) * 32 : kBwdTile);
        const SinkRoom room = sink_room(q_tokens, k_tokens, n_seq, window, sinks, group, most);
        p.sink_items = room.runs;
        p.sink_tiles = room.key_tiles;
        p.sink_places = room.runs + room.key_tiles * p.splits;
        p.bytes += p.sink_places * k_heads * 2 * p.sink_rows * dk * 4;
    }
    return p;
}

static int64_t backward_workspace(int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                                  int32_t k_heads, int32_t dim, int32_t sequences, int32_t window,
                                  int32_t sinks) {
    if (q_tokens < 0 || k_tokens < 0 || k_heads < 1 || q_heads < k_heads || sequences < 1) return 0;
    AttnArgs a{};
    a.k_tokens = (int32_t)k_tokens, a.window = window, a.sinks = sinks;
    hold_window(a);
    return bwd_plan(q_tokens, k_tokens, k_heads, q_heads / k_heads, dim, sequences, a.window,
                    a.sinks)
        .bytes;
}

static int32_t attention_backward(const char *who, int32_t dtype, int64_t q_tokens,
                                  int64_t k_tokens, int32_t q_heads, int32_t k_heads, int32_t dim,
                                  const void *q, int64_t q_token_stride, int64_t q_head_stride,
                                  const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                  const void *v, int64_t v_token_stride, int64_t v_head_stride,
                                  const int32_t *q_offsets, const int32_t *k_offsets,
                                  int32_t sequences, int32_t causal, int32_t window, int32_t sinks,
                                  float scale, const void *out, const void *out_rest,
                                  const float *lse, const void *dout, int64_t dout_token_stride,
                                  int64_t dout_head_stride, void *dq, void *dk, void *dv,
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
    a.dout = {dout, dout_token_stride, dout_head_stride};
    a.q_off = q_offsets, a.k_off = k_offsets, a.n_seq = sequences;
    a.q_tokens = (int32_t)q_tokens, a.k_tokens = (int32_t)k_tokens;
    a.k_heads = k_heads, a.group = group, a.dim = dim, a.causal = causal != 0;
    a.window = window, a.sinks = sinks;
    a.scale = scale, a.scale_log2 = scale_to_log2(scale);
    a.out = const_cast<void *>(out), a.out_rest = const_cast<void *>(out_rest), a.lse = const_cast<float *>(lse);
    a.dq = dq, a.dk = dk, a.dv = dv;
    int32_t rc = attn_check(who, a, dtype);
    if (rc != MG_OK) return rc;
    MG_REQUIRE(q_tokens == 0 || (q && out && lse && dout && dq), "%s: a pointer is NULL", who);
    MG_REQUIRE(k_tokens == 0 || (k && v), "%s: a pointer is NULL", who);
    MG_REQUIRE((dk == nullptr) == (dv == nullptr), "%s: dk and dv go together", who);
    hold_window(a);
    const BwdPlan p =
        bwd_plan(q_tokens, k_tokens, k_heads, group, dim, sequences, a.window, a.sinks);
    const int64_t q_items = (q_tokens * group / kBwdTile + sequences + 2) * k_heads;
    const int64_t k_items = (p.k_items * p.splits + p.sink_items) * k_heads;
    const int64_t places =
        k_heads * norm_places(q_tokens > k_tokens ? q_tokens : k_tokens, sequences);
    MG_REQUIRE(grid_fits(q_items, 64 * kBwdWaves) && grid_fits(k_items, 64 * kBwdWaves) &&
                   p.sink_places < INT32_MAX &&
                   (dtype != MG_F16 || grid_fits(places, kLargestThreads)),
               "%s: too many work items", who);
    MG_REQUIRE(workspace && workspace_bytes >= p.bytes, "%s: workspace of %lld bytes, %lld needed",
               who, (long long)workspace_bytes, (long long)p.bytes);
    char *ws = static_cast<char *>(workspace);
    a.delta = reinterpret_cast<float *>(ws);
    a.largest_do = reinterpret_cast<float *>(ws + p.largest_at);
    a.largest_v = a.largest_do + k_heads * norm_places(q_tokens, sequences);
    a.splits = p.splits, a.split_steps = p.split_steps;
    a.part = reinterpret_cast<float *>(ws + p.part_at);
    a.key_runs = (int32_t)(p.k_items * p.splits), a.sink_steps = p.sink_steps;
    a.sink_near = (int32_t)sink_near(group, p.sink_steps), a.sink_rows = p.sink_rows;
    a.sink_part = reinterpret_cast<float *>(ws + p.sink_at);
    hipStream_t st = as_stream(stream);
    if (dtype == MG_F16) {
        TimedScope ts("attention_largest", st);
        attn_largest_kernel<f16_t><<<dim3((unsigned)places, 2), kLargestThreads, 0, st>>>(a);
        MG_LAUNCHED("attn_largest_kernel");
    }
    if (q_tokens > 0) {
        TimedScope ts("attention_dq", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            if (a.window)
                attn_dq_kernel<T, DK, true><<<(unsigned)q_items, 64 * kBwdWaves, 0, st>>>(a);
            else
                attn_dq_kernel<T, DK, false><<<(unsigned)q_items, 64 * kBwdWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_dq_kernel");
    }
    if (k_tokens > 0 && dk) {
        TimedScope ts("attention_dkv", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int DK = decltype(d)::value;
            if (a.window)
                attn_dkv_kernel<T, DK, true><<<(unsigned)k_items, 64 * kBwdWaves, 0, st>>>(a);
            else
                attn_dkv_kernel<T, DK, false><<<(unsigned)k_items, 64 * kBwdWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_dkv_kernel");
    }
    if (dk && p.sink_tiles > 0) {
        TimedScope ts("attention_sinks", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            constexpr int DK = decltype(d)::value;
            const int64_t parts = p.sink_rows / 32 * 2 * DK / 8;
            const int64_t most = ceil_div(kSinkSlots, k_heads * parts);
            const dim3 grid((unsigned)((p.sink_tiles < most ? p.sink_tiles : most) * k_heads),
                            (unsigned)parts);
            attn_sink_sum_kernel<decltype(t), DK>
                <<<grid, 64 * kSinkWaves, 0, st>>>(a, (int)p.sink_tiles);
        });
        MG_LAUNCHED("attn_sink_sum_kernel");
    }
    if (k_tokens > 0 && dk && p.splits > 1) {
        TimedScope ts("attention_sum", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            constexpr int DK = decltype(d)::value;
            const dim3 grid((unsigned)(p.k_items * k_heads), 2 * DK / 32);
            if (a.window)
                attn_sum_kernel<decltype(t), DK, true><<<grid, 64 * kBwdWaves, 0, st>>>(a);
            else
                attn_sum_kernel<decltype(t), DK, false><<<grid, 64 * kBwdWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_sum_kernel");
    }
    return MG_OK;
}

}  // namespace mg

extern "C" {

int64_t mg_attention_backward_workspace_bytes(int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                                              int32_t k_heads, int32_t dim, int32_t sequences) {
    return mg::backward_workspace(q_tokens, k_tokens, q_heads, k_heads, dim, sequences, 0, 0);
}

int32_t mg_attention_backward(int32_t dtype, int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                              int32_t k_heads, int32_t dim, const void *q, int64_t q_token_stride,
                              int64_t q_head_stride, const void *k, int64_t k_token_stride,
                              int64_t k_head_stride, const void *v, int64_t v_token_stride,
                              int64_t v_head_stride, const int32_t *q_offsets,
                              const int32_t *k_offsets, int32_t sequences, int32_t causal,
                              float scale, const void *out, const void *out_rest,
                              const float *lse, const void *dout,
                              int64_t dout_token_stride, int64_t dout_head_stride, void *dq,
                              void *dk, void *dv, void *workspace, int64_t workspace_bytes,
                              mg_stream_t stream) {
    return mg::attention_backward("mg_attention_backward", dtype, q_tokens, k_tokens, q_heads,
                                  k_heads, dim, q, q_token_stride, q_head_stride, k,
                                  k_token_stride, k_head_stride, v, v_token_stride, v_head_stride,
                                  q_offsets, k_offsets, sequences, causal, 0, 0, scale, out,
                                  out_rest, lse, dout, dout_token_stride, dout_head_stride, dq, dk,
                                  dv, workspace, workspace_bytes, stream);
}

int64_t mg_attention_window_backward_workspace_bytes(int64_t q_tokens, int64_t k_tokens,
                                                     int32_t q_heads, int32_t k_heads, int32_t dim,
                                                     int32_t sequences, int32_t window,
                                                     int32_t sinks) {
    if (window < 1 || sinks < 0) return 0;
    return mg::backward_workspace(q_tokens, k_tokens, q_heads, k_heads, dim, sequences, window,
                                  sinks);
}

int32_t mg_attention_window_backward(
    int32_t dtype, int64_t q_tokens, int64_t k_tokens, int32_t q_heads, int32_t k_heads,
    int32_t dim, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
    int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
    int64_t v_head_stride, const int32_t *q_offsets, const int32_t *k_offsets, int32_t sequences,
    int32_t window, int32_t sinks, float scale, const void *out, const void *out_rest,
    const float *lse, const void *dout, int64_t dout_token_stride, int64_t dout_head_stride,
    void *dq, void *dk, void *dv, void *workspace, int64_t workspace_bytes, mg_stream_t stream) {
    const char *who = "mg_attention_window_backward";
    MG_REQUIRE(window >= 1, "%s: a window of %d keys", who, window);
    return mg::attention_backward(who, dtype, q_tokens, k_tokens, q_heads, k_heads, dim, q,
                                  q_token_stride, q_head_stride, k, k_token_stride, k_head_stride,
                                  v, v_token_stride, v_head_stride, q_offsets, k_offsets,
                                  sequences, 1, window, sinks, scale, out, out_rest, lse, dout,
                                  dout_token_stride, dout_head_stride, dq, dk, dv, workspace,
                                  workspace_bytes, stream);
}

}  // extern "C"
