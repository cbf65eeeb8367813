// Heads normed by their root mean square and turned by their token's position, in
// one pass, forward and backward. Per head x of n elements, with weights w and
// the rotation R of rotary.hip (pairs of the first 2 P elements, the rest kept):
//
//   s = 1 / sqrt(mean(x^2) + eps), u = x s, y = R (u w)
//   g = R^-1 dy, dw = sum over heads and tokens of g u
//   h = g w, dx = s (h - u mean(h u))
//
// Memory bounds it: a head is read once into registers and written once; the
// backward reads x and dy, forms s again from x and writes dx. All arithmetic is
// float32 and each result is rounded once.
//
// A head is held by L lanes (a power of two), each with one unit: V neighbouring
// elements and V others P further on, so that a pair's elements are in one lane
// in either layout, and 64 / L heads share a wave. A workgroup takes whole
// tokens of q or of k, and forms its tokens' cosines and sines once for all heads
// in LDS, after it has asked for its heads.
#include "rotary.h"

namespace mg {

constexpr int kHeadThreads = 256;
constexpr int kHeadTable = 2048;                  // cosines and sines a workgroup holds
constexpr int kHeadMaxDim = 512;
constexpr int64_t kHeadStreamBytes = 32 << 20;    // the L2 caches' together

// Heads a thread has at a time.
constexpr int kHeadsFwd = 4, kHeadsBwd = 2;

struct HeadTensor {
    const void *x, *dy;                           // (tokens, heads, dim)
    int64_t tok_stride, head_stride, dy_tok_stride, dy_head_stride;
    const void *weight;                           // NULL: ones
    void *out;                                    // y, or dx (NULL: not wanted); contiguous
    int32_t heads;
    // Its tokens' batches: `at_once` tokens, or `runs` runs of one token's heads.
    int32_t at_once, runs;
    int64_t batches;
    // Workgroups (backward), and where their sums for dw begin in `partial`.
    int32_t groups, first_part;
};

struct HeadArgs {
    HeadTensor t[2];                              // q, k
    int64_t tokens;
    int32_t dim, pairs, axes, lanes;              // lanes a head
    float eps;
    const void *positions;
    const double *freq;
    int32_t positions_64, weight_f32, interleaved, stream;
    float *partial;                               // (groups of q and k, dim); NULL: no dw
    AxisTable axis;
};

// Sum over aligned groups of `lanes` lanes, in all of them.
__device__ __forceinline__ float group_sum(float v, int lanes) {
    if (lanes > 1) v += dpp_f<0xb1>(v);           // quad_perm 1 0 3 2
    if (lanes > 2) v += dpp_f<0x4e>(v);           // quad_perm 2 3 0 1
    if (lanes > 4) v += dpp_f<0x141>(v);          // row_half_mirror
    if (lanes > 8) v += dpp_f<0x140>(v);          // row_mirror
    if (lanes > 16) v += __shfl_xor(v, 16, 64);
    if (lanes > 32) v += __shfl_xor(v, 32, 64);
    return v;
}

// A lane's units: elements a .. a + V - 1 and b .. b + V - 1 of a head.
struct HeadUnit {
    int a, b;              // -1: none
    int pair, pair_b;      // first pair of each; -1: kept as they are
};

// kHalf: pairs are (i, P + i), the unit's two runs being partners (of one element
// each, V = 1, in either layout); else they are neighbours within each run.
template <int V, bool kHalf>
__device__ __forceinline__ HeadUnit head_unit(const HeadArgs &p, int u) {
    const int turned = p.pairs / V, rest = (p.dim - 2 * p.pairs) / V, units = (rest + 1) / 2;
    if (u < turned) {
        if (V == 1 && p.interleaved) return {2 * u, 2 * u + 1, u, u};
        if (kHalf) return {u * V, p.pairs + u * V, u * V, u * V};
        return {u * V, p.pairs + u * V, u * V / 2, (p.pairs + u * V) / 2};
    }
    u -= turned;
    if (u >= units) return {-1, -1, -1, -1};
    return {2 * p.pairs + u * V, u + units < rest ? 2 * p.pairs + (units + u) * V : -1, -1, -1};
}

template <int V>
__device__ __forceinline__ void load_weight(const HeadArgs &p, const void *w, int code_bf16, int at,
                                            float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = at < 0 ? 0.f : 1.f;
    if (!w || at < 0) return;
    if (p.weight_f32)
        load_vec<float, V>(static_cast<const float *>(w) + at, f);
    else if (code_bf16)
        load_vec<bf16_t, V>(static_cast<const bf16_t *>(w) + at, f);
    else
        load_vec<f16_t, V>(static_cast<const f16_t *>(w) + at, f);
}

template <typename T, int V>
__device__ __forceinline__ void put(T *to, const float (&f)[V], int stream) {
    if (stream)
        store_vec<T, V, true>(to, f);
    else
        store_vec<T, V>(to, f);
}

// Turns a unit's elements; sn may be of the other sign (the adjoint).
template <int V, bool kHalf>
__device__ __forceinline__ void turn_unit(const float2 *cs, const HeadUnit &m, float sign,
                                          float (&a)[V], float (&b)[V]) {
    if constexpr (kHalf) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 c = cs[m.pair + i];
            const float sn = sign * c.y, p = a[i], q = b[i];
            a[i] = p * c.x - q * sn;
            b[i] = q * c.x + p * sn;
        }
    } else {
#pragma unroll
        for (int i = 0; i + 1 < V; i += 2) {
            const float2 c = cs[m.pair + i / 2], d = cs[m.pair_b + i / 2];
            float p = a[i], q = a[i + 1], sn = sign * c.y;
            a[i] = p * c.x - q * sn;
            a[i + 1] = q * c.x + p * sn;
            p = b[i], q = b[i + 1], sn = sign * d.y;
            b[i] = p * d.x - q * sn;
            b[i + 1] = q * d.x + p * sn;
        }
    }
}

// The batch's tokens and heads.
struct HeadBatch {
    int64_t tok0;
    int n_tok, head0, heads;
};
__device__ __forceinline__ HeadBatch head_batch(const HeadArgs &p, const HeadTensor &t, int64_t b,
                                                int rows) {
    const int run = t.runs > 1 ? (int)(b % t.runs) : 0;
    const int64_t tok0 = (t.runs > 1 ? b / t.runs : b) * t.at_once;
    const int n_tok = (int)min((int64_t)t.at_once, p.tokens - tok0);
    const int head0 = run * rows;
    return {tok0, n_tok, head0, t.runs > 1 ? min(t.heads - head0, rows) : t.heads};
}

__device__ __forceinline__ void head_angles(const HeadArgs &p, const HeadBatch &b, float2 *cs) {
    for (int i = threadIdx.x; i < b.n_tok * p.pairs; i += kHeadThreads) {
        const int tok = i / p.pairs, pair = i - tok * p.pairs;
        const int64_t at = (b.tok0 + tok) * p.axes + p.axis.axis[pair];
        const double pos = p.positions_64
                               ? (double)static_cast<const int64_t *>(p.positions)[at]
                               : (double)static_cast<const int32_t *>(p.positions)[at];
        cs[i] = turn_of(pos, p.freq[pair], 1.f);
    }
}

// C units a lane: heads of more than 64 units have them 64 apart.
template <typename T, int V, int C, bool kHalf>
__global__ __launch_bounds__(kHeadThreads) void norm_rotary_fwd_kernel(HeadArgs p) {
    constexpr int R = C == 1 ? kHeadsFwd : 1;
    __shared__ float2 s_cs[kHeadTable];
    const int which = blockIdx.x >= p.t[0].batches;
    const HeadTensor &t = p.t[which];
    const int64_t at_batch = blockIdx.x - (which ? p.t[0].batches : 0);
    const int L = p.lanes, each = kHeadThreads / L;
    const HeadBatch b = head_batch(p, t, at_batch, each * R);
    const int rows = b.n_tok * b.heads;
    HeadUnit unit[C];
    float wa[C][V], wb[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) unit[c] = head_unit<V, kHalf>(p, threadIdx.x % L + 64 * c);
    T xa[R][C][V] = {}, xb[R][C][V] = {};
    int tok[R], head[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = r * each + threadIdx.x / L;
        tok[r] = row / b.heads, head[r] = b.head0 + row % b.heads;
        if (row >= rows) {
            tok[r] = -1;
            continue;
        }
        const T *x = static_cast<const T *>(t.x) + (b.tok0 + tok[r]) * t.tok_stride +
                     head[r] * t.head_stride;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (unit[c].a >= 0) __builtin_memcpy(xa[r][c], x + unit[c].a, sizeof(xa[r][c]));
            if (unit[c].b >= 0) __builtin_memcpy(xb[r][c], x + unit[c].b, sizeof(xb[r][c]));
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        load_weight<V>(p, t.weight, std::is_same<T, bf16_t>::value, unit[c].a, wa[c]);
        load_weight<V>(p, t.weight, std::is_same<T, bf16_t>::value, unit[c].b, wb[c]);
    }
    head_angles(p, b, s_cs);
    __syncthreads();
    const float per = 1.f / (float)p.dim;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                ss = fmaf((float)xa[r][c][i], (float)xa[r][c][i], ss);
                ss = fmaf((float)xb[r][c][i], (float)xb[r][c][i], ss);
            }
        ss = group_sum(ss, L);
        if (tok[r] < 0) continue;
        const float s = 1.f / sqrtf(ss * per + p.eps);
        T *out = static_cast<T *>(t.out) +
                 ((b.tok0 + tok[r]) * t.heads + head[r]) * (int64_t)p.dim;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const HeadUnit &m = unit[c];
            float a[V], bb[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[i] = (float)xa[r][c][i] * s * wa[c][i];
                bb[i] = (float)xb[r][c][i] * s * wb[c][i];
            }
            if (m.pair >= 0) turn_unit<V, kHalf>(s_cs + tok[r] * p.pairs, m, 1.f, a, bb);
            if (m.a >= 0) put<T, V>(out + m.a, a, p.stream);
            if (m.b >= 0) put<T, V>(out + m.b, bb, p.stream);
        }
    }
}

// A workgroup takes every groups-th batch and keeps its sums for dw in registers,
// joined by norm_rotary_join_kernel in a fixed order.
template <typename T, int V, int C, bool kHalf>
__global__ __launch_bounds__(kHeadThreads) void norm_rotary_bwd_kernel(HeadArgs p) {
    constexpr int R = C == 1 ? kHeadsBwd : 1;
    __shared__ float2 s_cs[2][kHeadTable / 2];
    __shared__ float s_dw[kHeadMaxDim];
    const int which = (int)blockIdx.x >= p.t[0].groups;
    const HeadTensor &t = p.t[which];
    const int group = blockIdx.x - (which ? p.t[0].groups : 0);
    const int L = p.lanes, each = kHeadThreads / L;
    HeadUnit unit[C];
    float wa[C][V], wb[C][V], da[C][V] = {}, db[C][V] = {};
#pragma unroll
    for (int c = 0; c < C; ++c) {
        unit[c] = head_unit<V, kHalf>(p, threadIdx.x % L + 64 * c);
        load_weight<V>(p, t.weight, std::is_same<T, bf16_t>::value, unit[c].a, wa[c]);
        load_weight<V>(p, t.weight, std::is_same<T, bf16_t>::value, unit[c].b, wb[c]);
    }
    const float per = 1.f / (float)p.dim;
    int buf = 0;
    for (int64_t at = group; at < t.batches; at += t.groups, buf ^= 1) {
        const HeadBatch b = head_batch(p, t, at, each * R);
        const int rows = b.n_tok * b.heads;
        T xa[R][C][V] = {}, xb[R][C][V] = {}, ga[R][C][V] = {}, gb[R][C][V] = {};
        int tok[R], head[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = r * each + threadIdx.x / L;
            tok[r] = row / b.heads, head[r] = b.head0 + row % b.heads;
            if (row >= rows) {
                tok[r] = -1;
                continue;
            }
            const T *x = static_cast<const T *>(t.x) + (b.tok0 + tok[r]) * t.tok_stride +
                         head[r] * t.head_stride;
            const T *dy = static_cast<const T *>(t.dy) + (b.tok0 + tok[r]) * t.dy_tok_stride +
                          head[r] * t.dy_head_stride;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const HeadUnit &m = unit[c];
                if (m.a >= 0) {
                    __builtin_memcpy(xa[r][c], x + m.a, sizeof(xa[r][c]));
                    __builtin_memcpy(ga[r][c], dy + m.a, sizeof(ga[r][c]));
                }
                if (m.b >= 0) {
                    __builtin_memcpy(xb[r][c], x + m.b, sizeof(xb[r][c]));
                    __builtin_memcpy(gb[r][c], dy + m.b, sizeof(gb[r][c]));
                }
            }
        }
        head_angles(p, b, s_cs[buf]);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float ss = 0.f, hx = 0.f, a[C][V], c2[C][V];
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    a[c][i] = (float)ga[r][c][i];
                    c2[c][i] = (float)gb[r][c][i];
                }
                if (unit[c].pair >= 0)
                    turn_unit<V, kHalf>(s_cs[buf] + max(tok[r], 0) * p.pairs, unit[c], -1.f, a[c],
                                        c2[c]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x = (float)xa[r][c][i], y = (float)xb[r][c][i];
                    ss = fmaf(x, x, ss);
                    ss = fmaf(y, y, ss);
                    hx = fmaf(a[c][i] * wa[c][i], x, hx);
                    hx = fmaf(c2[c][i] * wb[c][i], y, hx);
                }
            }
            ss = group_sum(ss, L);
            hx = group_sum(hx, L);
            if (tok[r] < 0) continue;
            const float s = 1.f / sqrtf(ss * per + p.eps);
            const float along = hx * s * per;          // mean(h u)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float u = (float)xa[r][c][i] * s, v = (float)xb[r][c][i] * s;
                    da[c][i] = fmaf(a[c][i], u, da[c][i]);
                    db[c][i] = fmaf(c2[c][i], v, db[c][i]);
                    a[c][i] = s * (a[c][i] * wa[c][i] - u * along);
                    c2[c][i] = s * (c2[c][i] * wb[c][i] - v * along);
                }
            if (!t.out) continue;
            T *out = static_cast<T *>(t.out) +
                     ((b.tok0 + tok[r]) * t.heads + head[r]) * (int64_t)p.dim;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (unit[c].a >= 0) put<T, V>(out + unit[c].a, a[c], p.stream);
                if (unit[c].b >= 0) put<T, V>(out + unit[c].b, c2[c], p.stream);
            }
        }
        lds_reads_done();
    }
    if (!p.partial) return;
    // The lanes of one unit, then the waves, one after the other.
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i)
            for (int o = L; o < 64; o <<= 1) {
                da[c][i] += __shfl_xor(da[c][i], o, 64);
                db[c][i] += __shfl_xor(db[c][i], o, 64);
            }
    const int wave = threadIdx.x / 64;
    for (int from = 0; from < kHeadThreads / 64; ++from) {
        if (wave == from && lane_id() < L) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const HeadUnit &m = unit[c];
                    if (m.a >= 0) s_dw[m.a + i] = da[c][i] + (from ? s_dw[m.a + i] : 0.f);
                    if (m.b >= 0) s_dw[m.b + i] = db[c][i] + (from ? s_dw[m.b + i] : 0.f);
                }
        }
        lds_reads_done();
        __syncthreads();
    }
    float *out = p.partial + (int64_t)(t.first_part + group) * p.dim;
    for (int i = threadIdx.x; i < p.dim; i += kHeadThreads) out[i] = s_dw[i];
}

// dw of q (blockIdx.y 0) and k (1), 32 columns: 32 threads a column, each over
// every 32nd workgroup's sums.
constexpr int kHeadJoinCols = 32, kHeadJoinThreads = 1024;
template <typename W>
__global__ __launch_bounds__(kHeadJoinThreads) void norm_rotary_join_kernel(HeadArgs p, W *dq,
                                                                           W *dk) {
    constexpr int kGroups = kHeadJoinThreads / kHeadJoinCols;
    __shared__ float s[kGroups][kHeadJoinCols + 1];
    const HeadTensor &t = p.t[blockIdx.y];
    W *out = blockIdx.y ? dk : dq;
    const int col = threadIdx.x % kHeadJoinCols, group = threadIdx.x / kHeadJoinCols;
    const int at = blockIdx.x * kHeadJoinCols + col;
    float sum = 0.f;
    if (at < p.dim) {
        const float *from = p.partial + (int64_t)t.first_part * p.dim + at;
#pragma unroll 8
        for (int i = group; i < t.groups; i += kGroups) sum += from[(int64_t)i * p.dim];
    }
    s[group][col] = sum;
    __syncthreads();
    if (group == 0 && at < p.dim && out) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) total += s[i][col];
        out[at] = (W)total;
    }
}

// -------------------------------------------------------------------- host
constexpr int64_t kHeadGroups = 1024;             // workgroups of a backward pass, at most

// Units of V elements: how many lanes a head takes, 0 where they do not fit.
static int head_lanes(int dim, int pairs, int V, int C) {
    if (pairs % V || (dim - 2 * pairs) % V) return 0;
    const int units = pairs / V + ((dim - 2 * pairs) / V + 1) / 2;
    if (C > 1) return units <= 64 * C ? 64 : 0;
    int lanes = 1;
    while (lanes < units) lanes *= 2;
    return lanes <= 64 ? lanes : 0;
}

// Cuts the tokens into batches that R heads a thread hold.
static void head_cut(HeadTensor &t, int64_t tokens, int pairs, int lanes, int R, int table) {
    if (t.heads == 0) {
        t.at_once = t.runs = 1;
        t.batches = 0;
        return;
    }
    const int rows = R * kHeadThreads / lanes;
    int64_t at_once = rows / t.heads;
    if (at_once > table / pairs) at_once = table / pairs;
    // A few tokens are spread over the GPU.
    if (at_once > ceil_div(tokens, 512)) at_once = ceil_div(tokens, 512);
    t.at_once = (int32_t)(at_once < 1 ? 1 : at_once);
    t.runs = t.at_once == 1 ? (int32_t)ceil_div(t.heads, rows) : 1;
    t.batches = ceil_div(tokens, t.at_once) * t.runs;
}

// Calls f<V, C, kHalf>(lanes) for the widest units that heads are made of.
template <typename T, typename F>
static void head_form(const HeadArgs &p, F f) {
    using std::bool_constant;
    using std::integral_constant;
    constexpr int kWide = kVec<T>, kMid = kVec<T> / 2;
    const auto with = [&](auto v, int lanes) {
        if (p.interleaved)
            f(v, integral_constant<int, 1>{}, bool_constant<false>{}, lanes);
        else
            f(v, integral_constant<int, 1>{}, bool_constant<true>{}, lanes);
    };
    if (int lanes = head_lanes(p.dim, p.pairs, kWide, 1))
        with(integral_constant<int, kWide>{}, lanes);
    else if (int mid = head_lanes(p.dim, p.pairs, kMid, 1))
        with(integral_constant<int, kMid>{}, mid);
    else if (int one = head_lanes(p.dim, p.pairs, 1, 1))
        f(integral_constant<int, 1>{}, integral_constant<int, 1>{}, bool_constant<true>{}, one);
    else
        f(integral_constant<int, 1>{}, integral_constant<int, 4>{}, bool_constant<true>{}, 64);
}

template <typename F>
static void head_types(int32_t dtype, F f) {
    if (dtype == MG_F32)
        f(float{});
    else if (dtype == MG_BF16)
        f(bf16_t{});
    else
        f(f16_t{});
}

static int32_t head_check(const char *who, HeadArgs &p, int32_t dtype, int32_t weight_dtype,
                          const uint8_t *axis_of) {
    MG_REQUIRE(type_known(dtype), "%s: type code %d", who, dtype);
    MG_REQUIRE(weight_dtype == MG_F32 || weight_dtype == dtype,
               "%s: the weights must be float32 or of the input's type", who);
    MG_REQUIRE(p.tokens >= 0 && p.tokens < (int64_t(1) << 31), "%s: %lld tokens", who,
               (long long)p.tokens);
    MG_REQUIRE(p.t[0].heads >= 0 && p.t[1].heads >= 0 && p.t[0].heads <= 65536 &&
                   p.t[1].heads <= 65536 && p.t[0].heads + p.t[1].heads > 0,
               "%s: %d and %d heads", who, p.t[0].heads, p.t[1].heads);
    MG_REQUIRE(p.dim >= 2 && p.dim <= kHeadMaxDim, "%s: heads of %d elements; 2 to %d are taken",
               who, p.dim, kHeadMaxDim);
    MG_REQUIRE(p.pairs >= 1 && 2 * p.pairs <= p.dim,
               "%s: %d frequencies turn %d elements; heads have %d", who, p.pairs, 2 * p.pairs,
               p.dim);
    MG_REQUIRE(p.axes >= 1 && p.axes <= 256 && (axis_of || p.pairs % p.axes == 0),
               "%s: %d frequencies do not divide among %d axes", who, p.pairs, p.axes);
    MG_REQUIRE(fill_axes(p.axis, axis_of, p.pairs, p.axes),
               "%s: a pair's axis is not among the %d of the positions", who, p.axes);
    MG_REQUIRE(p.eps >= 0.f && p.eps < INFINITY, "%s: eps %g", who, (double)p.eps);
    return MG_OK;
}

// Shared by the backward pass and its workspace.
static void head_groups(HeadArgs &p) {
    const int64_t all = p.t[0].batches + p.t[1].batches;
    int first = 0;
    for (HeadTensor &t : p.t) {
        int64_t groups = t.batches;
        if (all > kHeadGroups) groups = ceil_div(t.batches * kHeadGroups, all);
        t.groups = (int32_t)groups, t.first_part = first;
        first += t.groups;
    }
}

static HeadArgs head_args(int64_t tokens, const void *q, int64_t q_token_stride,
                          int64_t q_head_stride, int32_t q_heads, const void *k,
                          int64_t k_token_stride, int64_t k_head_stride, int32_t k_heads,
                          int32_t dim, int32_t weight_dtype, const void *q_weight,
                          const void *k_weight, float eps, const void *positions,
                          int32_t positions_64, int32_t axes, const double *frequencies,
                          int32_t pairs, int32_t interleaved) {
    HeadArgs p{};
    p.t[0].x = q, p.t[0].tok_stride = q_token_stride, p.t[0].head_stride = q_head_stride;
    p.t[1].x = k, p.t[1].tok_stride = k_token_stride, p.t[1].head_stride = k_head_stride;
    p.t[0].heads = q_heads, p.t[1].heads = k_heads;
    p.t[0].weight = q_weight, p.t[1].weight = k_weight;
    p.tokens = tokens, p.dim = dim, p.pairs = pairs, p.axes = axes, p.eps = eps;
    p.positions = positions, p.positions_64 = positions_64 != 0, p.freq = frequencies;
    p.weight_f32 = weight_dtype == MG_F32, p.interleaved = interleaved != 0;
    return p;
}

}  // namespace mg

extern "C" {

int32_t mg_norm_rotary_forward(int64_t tokens, int32_t dtype, const void *q,
                               int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads,
                               const void *k, int64_t k_token_stride, int64_t k_head_stride,
                               int32_t k_heads, int32_t dim, int32_t weight_dtype,
                               const void *q_weight, const void *k_weight, float eps,
                               const void *positions, int32_t positions_64, int32_t axes,
                               const uint8_t *axis_of, const double *frequencies, int32_t pairs,
                               int32_t interleaved, void *q_out, void *k_out,
                               mg_stream_t stream) {
    using namespace mg;
    const char *who = "mg_norm_rotary_forward";
    HeadArgs p = head_args(tokens, q, q_token_stride, q_head_stride, q_heads, k, k_token_stride,
                           k_head_stride, k_heads, dim, weight_dtype, q_weight, k_weight, eps,
                           positions, positions_64, axes, frequencies, pairs, interleaved);
    const int32_t rc = head_check(who, p, dtype, weight_dtype, axis_of);
    if (rc != MG_OK) return rc;
    if (tokens == 0) return MG_OK;
    MG_REQUIRE(positions && frequencies && (q_heads == 0 || (q && q_out)) &&
                   (k_heads == 0 || (k && k_out)),
               "%s: a pointer is NULL", who);
    p.t[0].out = q_out, p.t[1].out = k_out;
    const int size = dtype == MG_F32 ? 4 : 2;
    p.stream = tokens * (q_heads + k_heads) * dim * size > kHeadStreamBytes;
    hipStream_t st = as_stream(stream);
    TimedScope ts("norm_rotary_fwd", st);
    bool fits = true;
    head_types(dtype, [&](auto type) {
        using T = decltype(type);
        head_form<T>(p, [&](auto v, auto c, auto half, int lanes) {
            constexpr int V = decltype(v)::value, C = decltype(c)::value;
            p.lanes = lanes;
            for (HeadTensor &t : p.t)
                head_cut(t, tokens, pairs, lanes, C == 1 ? kHeadsFwd : 1, kHeadTable);
            const int64_t grid = p.t[0].batches + p.t[1].batches;
            fits = grid_fits(grid, kHeadThreads);
            if (fits)
                norm_rotary_fwd_kernel<T, V, C, decltype(half)::value>
                    <<<(unsigned)grid, kHeadThreads, 0, st>>>(p);
        });
    });
    MG_REQUIRE(fits, "%s: %lld tokens of %d heads are too many for one call", who,
               (long long)tokens, q_heads + k_heads);
    MG_LAUNCHED("norm_rotary_fwd_kernel");
    return MG_OK;
}

int64_t mg_norm_rotary_backward_workspace_bytes(int32_t dim) {
    // One row of sums a workgroup; each tensor's share of them is rounded up.
    return dim > 0 ? (mg::kHeadGroups + 2) * (int64_t)dim * 4 : 0;
}

int32_t mg_norm_rotary_backward(
    int64_t tokens, int32_t dtype, const void *q, int64_t q_token_stride, int64_t q_head_stride,
    int32_t q_heads, const void *k, int64_t k_token_stride, int64_t k_head_stride, int32_t k_heads,
    int32_t dim, int32_t weight_dtype, const void *q_weight, const void *k_weight, float eps,
    const void *positions, int32_t positions_64, int32_t axes, const uint8_t *axis_of,
    const double *frequencies, int32_t pairs, int32_t interleaved, const void *dq_out,
    int64_t dq_token_stride, int64_t dq_head_stride, const void *dk_out, int64_t dk_token_stride,
    int64_t dk_head_stride, void *dq, void *dk, void *dq_weight, void *dk_weight, void *workspace,
    int64_t workspace_bytes, mg_stream_t stream) {
    using namespace mg;
    const char *who = "mg_norm_rotary_backward";
    HeadArgs p = head_args(tokens, q, q_token_stride, q_head_stride, q_heads, k, k_token_stride,
                           k_head_stride, k_heads, dim, weight_dtype, q_weight, k_weight, eps,
                           positions, positions_64, axes, frequencies, pairs, interleaved);
    const int32_t rc = head_check(who, p, dtype, weight_dtype, axis_of);
    if (rc != MG_OK) return rc;
    const bool sums = dq_weight || dk_weight;
    MG_REQUIRE(tokens > 0 || !sums, "%s: the weights' gradients of no tokens are zeros", who);
    if (tokens == 0 || (!dq && !dk && !sums)) return MG_OK;
    MG_REQUIRE(positions && frequencies && (q_heads == 0 || (q && dq_out)) &&
                   (k_heads == 0 || (k && dk_out)),
               "%s: a pointer is NULL", who);
    MG_REQUIRE((q_heads > 0 || (!dq && !dq_weight)) && (k_heads > 0 || (!dk && !dk_weight)),
               "%s: gradients of no heads", who);
    const int64_t need = mg_norm_rotary_backward_workspace_bytes(dim);
    MG_REQUIRE(!sums || (workspace && workspace_bytes >= need),
               "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
               (long long)need);
    p.t[0].dy = dq_out, p.t[0].dy_tok_stride = dq_token_stride;
    p.t[0].dy_head_stride = dq_head_stride;
    p.t[1].dy = dk_out, p.t[1].dy_tok_stride = dk_token_stride;
    p.t[1].dy_head_stride = dk_head_stride;
    p.t[0].out = dq, p.t[1].out = dk;
    p.partial = sums ? static_cast<float *>(workspace) : nullptr;
    const int size = dtype == MG_F32 ? 4 : 2;
    p.stream = tokens * (q_heads + k_heads) * dim * size > kHeadStreamBytes;
    hipStream_t st = as_stream(stream);
    {
        TimedScope ts("norm_rotary_bwd", st);
        head_types(dtype, [&](auto type) {
            using T = decltype(type);
            head_form<T>(p, [&](auto v, auto c, auto half, int lanes) {
                constexpr int V = decltype(v)::value, C = decltype(c)::value;
                p.lanes = lanes;
                for (HeadTensor &t : p.t)
                    head_cut(t, tokens, pairs, lanes, C == 1 ? kHeadsBwd : 1, kHeadTable / 2);
                head_groups(p);
                norm_rotary_bwd_kernel<T, V, C, decltype(half)::value>
                    <<<(unsigned)(p.t[0].groups + p.t[1].groups), kHeadThreads, 0, st>>>(p);
            });
        });
        MG_LAUNCHED("norm_rotary_bwd_kernel");
    }
    if (sums) {
        TimedScope ts("norm_rotary_join", st);
        const dim3 grid((unsigned)ceil_div(dim, kHeadJoinCols), 2);
        const auto go = [&](auto w) {
            using W = decltype(w);
            norm_rotary_join_kernel<W><<<grid, kHeadJoinThreads, 0, st>>>(
                p, static_cast<W *>(dq_weight), static_cast<W *>(dk_weight));
        };
        head_types(weight_dtype, go);
        MG_LAUNCHED("norm_rotary_join_kernel");
    }
    return MG_OK;
}

}  // extern "C"
