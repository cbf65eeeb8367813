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
// 8192 tokens, 16 heads of 128: queries 748 us, keys 1047 (1100 and 1050 TFLOP/s);
// of 64: 462 and 623 (890 and 880). The queries' kernel is never cut over its keys:
// 64 queries over 16000 of them, 16 heads on 4 of 128, take 417 us. As the forward, both need two waves a SIMD to
// keep products and exponentials going side by side: the keys' kernel with one
// (256 columns of sums and operands in 472 registers) took 1970.
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
template <typename T, int DK>
__global__ __launch_bounds__(64 * kBwdWaves, 2) void attn_dq_kernel(AttnArgs a) {
    constexpr int kSteps = DK / 16, kBlocks = DK / 32;
    __shared__ __align__(16) char s_tile[2][2][kTileBytes<DK>];
    const int lane = lane_id(), half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads, G = a.group;
    const SeqItem s = find_longest<false>(a, item, kBwdTile);
    if (!s.found) return;
    const int tile = s.within;
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
    const int k_to = sees(min((tile * kBwdTile + kBwdTile - 1) / G, s.q_len - 1));

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
    if (k_to > 0) ask(0, 0);
    loads_done();
    for (int key0 = 0; key0 < k_to; key0 += kTileRows, buf ^= 1) {
        tiles_ready();
        lane_at.fresh();
        if (key0 + kTileRows < k_to) ask(key0 + kTileRows, buf ^ 1);
        if (key0 >= see_last) continue;
        const char *kt = s_tile[buf][0], *vt = s_tile[buf][1];
        const bool masked = key0 + kTileRows > see_first;
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
                if (masked && key0 + 32 * b + c_row(e, half) >= see) d = 0.f;
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
    if (!row_ok) return;
    const float down = a.scale * __builtin_amdgcn_exp2f(-power);
    T *out = static_cast<T *>(a.dq) +
             ((int64_t)(s.q_lo + token) * (a.k_heads * G) + head) * a.dim;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int at = 32 * b + c_row(e, half);
            vec4<T> w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (T)(dq[b][e + i] * down);
            if (at < a.dim) *reinterpret_cast<vec4<T> *>(out + at) = w;
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

// The query tiles that see a key tile (tiles of each of the group's heads, from
// q_from), and the runs they are cut into: whole heads, or `parts` of each head
// where there are more runs than heads. Key tiles that run at the same time then
// read the same heads' queries, which stay in their XCD's L2.
struct KeySteps {
    int q_from, tiles, runs, parts;
};

__device__ __forceinline__ KeySteps key_steps(const AttnArgs &a, const SeqItem &s, int first_key) {
    const int ahead = s.k_len - s.q_len, G = a.group;
    const int from = a.causal ? max(0, first_key - ahead) / kTileRows * kTileRows : 0;
    const int tiles = from < s.q_len ? (s.q_len - from + kTileRows - 1) / kTileRows : 0;
    int runs = (int)(((int64_t)tiles * G + a.split_steps - 1) / a.split_steps);
    runs = even_runs(clamp_to(runs, 1, a.splits), G, a.splits);
    return {from, tiles, runs, runs > G ? runs / G : 1};
}

template <typename T, int DK>
__global__ __launch_bounds__(64 * kBwdWaves, 2) void attn_dkv_kernel(AttnArgs a) {
    constexpr int kSteps = DK / 16, kBlocks = DK / 32;
    __shared__ __align__(16) char s_tile[2][2][kTileBytes<DK>];
    __shared__ __align__(16) float s_row[2][2][kTileRows];     // lse, delta
    const int lane = lane_id(), half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads / a.splits;
    const int split = blockIdx.x / a.k_heads % a.splits;
    const SeqItem s = find_longest<true>(a, item, kBwdTile);
    if (!s.found) return;
    const int first_key = s.within * kBwdTile;
    const KeySteps steps_of = key_steps(a, s, first_key);
    if (split >= steps_of.runs) return;
    const int key0 = first_key + wave * 32, key = key0 + lane % 32;
    const bool key_ok = key < s.k_len;
    const int ahead = s.k_len - s.q_len;       // query i sees keys up to i + ahead
    // This run's heads, and its query tiles of each.
    const int parts = steps_of.parts, runs = steps_of.runs / parts, run = split / parts;
    const int g_from = run * a.group / runs, heads = (run + 1) * a.group / runs - g_from;
    const int t_from = steps_of.tiles * (split % parts) / parts;
    const int tiles = steps_of.tiles * (split % parts + 1) / parts - t_from;
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
        const bool masked = at_row0 + kTileRows > s.q_len || key0 + 32 > s.k_len ||
                            (a.causal && at_row0 + ahead < key0 + 31);
        if (a.causal && at_row0 + kTileRows - 1 + ahead < key0) continue;    // none sees any
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
                        const bool seen = token < s.q_len && key_ok &&
                                          (!a.causal || key <= token + ahead);
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
    if (steps_of.runs > 1) {
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
    if (!key_ok) return;
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
template <typename T, int DK>
__global__ __launch_bounds__(64 * kBwdWaves) void attn_sum_kernel(AttnArgs a) {
    constexpr int kBlocks = DK / 32;
    const int kh = blockIdx.x % a.k_heads, item = blockIdx.x / a.k_heads;
    const SeqItem s = find_longest<true>(a, item, kBwdTile);
    if (!s.found) return;
    const int first_key = s.within * kBwdTile;
    const int runs = key_steps(a, s, first_key).runs;
    if (runs == 1) return;
    const int lane = lane_id(), half = lane / 32, wave = uniform(threadIdx.x / 64);
    const int key = first_key + wave * 32 + lane % 32;
    const int64_t at_row = ((int64_t)(s.k_lo + key) * a.k_heads + kh) * a.dim;
    const f32x4 *part = part_of<DK>(a, item, kh, 0) + wave * kBlocks * 4 * 64 + lane;
    const int which = blockIdx.y % 2, block = blockIdx.y / 2;
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

// Bytes of the backward's scratch: delta, the largest norms, and the runs' sums.
// The keys' gradients are cut into runs where their tiles are fewer than fill
// the GPU twice over, of eight query tiles at least (7033 packed tokens, 62 tiles
// on 4 key heads: 528 us uncut, 187 and 27 to add the runs in four).
struct BwdPlan {
    int64_t k_items, largest_at, part_at, bytes;
    int splits, split_steps;
};

constexpr int64_t kBwdRuns = 1024, kBwdRunLeast = 8, kBwdMostSplits = 8;

static BwdPlan bwd_plan(int64_t q_tokens, int64_t k_tokens, int64_t k_heads, int64_t group,
                        int64_t dim, int64_t n_seq) {
    BwdPlan p{};
    p.k_items = k_tokens / kBwdTile + n_seq + 2;
    const int64_t tiles = (ceil_div(k_tokens, kBwdTile) + n_seq - 1) * k_heads;
    const int64_t steps = ceil_div(q_tokens, n_seq * kTileRows) * group;
    int64_t splits = kBwdRuns / (tiles > 0 ? tiles : 1);
    if (splits > steps / kBwdRunLeast) splits = steps / kBwdRunLeast;
    splits = splits < 1 ? 1 : splits > kBwdMostSplits ? kBwdMostSplits : splits;
    p.splits = even_runs((int)splits, (int)group, (int)kBwdMostSplits);
    p.split_steps = (int)kBwdRunLeast;
    p.largest_at = align256(q_tokens * k_heads * group * 4);
    p.part_at = align256(p.largest_at + k_heads * 4 * (norm_places(q_tokens, n_seq) +
                                                       norm_places(k_tokens, n_seq)));
    p.bytes = p.part_at;
    const int64_t dk = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
    if (p.splits > 1) p.bytes += p.k_items * k_heads * p.splits * 2 * kBwdTile * dk * 4;
    return p;
}

}  // namespace mg

extern "C" {

int64_t mg_attention_backward_workspace_bytes(int64_t q_tokens, int64_t k_tokens, int32_t q_heads,
                                              int32_t k_heads, int32_t dim, int32_t sequences) {
    if (q_tokens < 0 || k_tokens < 0 || k_heads < 1 || q_heads < k_heads || sequences < 1) return 0;
    return mg::bwd_plan(q_tokens, k_tokens, k_heads, q_heads / k_heads, dim, sequences).bytes;
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
    using namespace mg;
    const char *who = "mg_attention_backward";
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
    a.scale = scale, a.scale_log2 = scale_to_log2(scale);
    a.out = const_cast<void *>(out), a.out_rest = const_cast<void *>(out_rest), a.lse = const_cast<float *>(lse);
    a.dq = dq, a.dk = dk, a.dv = dv;
    int32_t rc = attn_check(who, a, dtype);
    if (rc != MG_OK) return rc;
    MG_REQUIRE(q_tokens == 0 || (q && out && lse && dout && dq), "%s: a pointer is NULL", who);
    MG_REQUIRE(k_tokens == 0 || (k && v), "%s: a pointer is NULL", who);
    MG_REQUIRE((dk == nullptr) == (dv == nullptr), "%s: dk and dv go together", who);
    const BwdPlan p = bwd_plan(q_tokens, k_tokens, k_heads, group, dim, sequences);
    MG_REQUIRE(workspace && workspace_bytes >= p.bytes, "%s: workspace of %lld bytes, %lld needed",
               who, (long long)workspace_bytes, (long long)p.bytes);
    char *ws = static_cast<char *>(workspace);
    a.delta = reinterpret_cast<float *>(ws);
    a.largest_do = reinterpret_cast<float *>(ws + p.largest_at);
    a.largest_v = a.largest_do + k_heads * norm_places(q_tokens, sequences);
    a.splits = p.splits, a.split_steps = p.split_steps;
    a.part = reinterpret_cast<float *>(ws + p.part_at);
    hipStream_t st = as_stream(stream);
    const int64_t q_items = (q_tokens * group / kBwdTile + sequences + 2) * k_heads;
    const int64_t k_items = p.k_items * p.splits * k_heads;
    const int64_t places =
        k_heads * norm_places(q_tokens > k_tokens ? q_tokens : k_tokens, sequences);
    MG_REQUIRE(grid_fits(q_items, 64 * kBwdWaves) && grid_fits(k_items, 64 * kBwdWaves) &&
                   (dtype != MG_F16 || grid_fits(places, kLargestThreads)),
               "%s: too many work items", who);
    if (dtype == MG_F16) {
        TimedScope ts("attention_largest", st);
        attn_largest_kernel<f16_t><<<dim3((unsigned)places, 2), kLargestThreads, 0, st>>>(a);
        MG_LAUNCHED("attn_largest_kernel");
    }
    if (q_tokens > 0) {
        TimedScope ts("attention_dq", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            attn_dq_kernel<decltype(t), decltype(d)::value>
                <<<(unsigned)q_items, 64 * kBwdWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_dq_kernel");
    }
    if (k_tokens > 0 && dk) {
        TimedScope ts("attention_dkv", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            attn_dkv_kernel<decltype(t), decltype(d)::value>
                <<<(unsigned)k_items, 64 * kBwdWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_dkv_kernel");
    }
    if (k_tokens > 0 && dk && p.splits > 1) {
        TimedScope ts("attention_sum", st);
        attn_form(dtype, dim, [&](auto t, auto d) {
            constexpr int DK = decltype(d)::value;
            const dim3 grid((unsigned)(p.k_items * k_heads), 2 * DK / 32);
            attn_sum_kernel<decltype(t), DK><<<grid, 64 * kBwdWaves, 0, st>>>(a);
        });
        MG_LAUNCHED("attn_sum_kernel");
    }
    return MG_OK;
}

}  // extern "C"
