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
// in either layout, and 64 / L heads share a wave. A lane has up to R heads of one
// token: their cosines and sines are registers then, as are the weights. A
// workgroup takes whole tokens, q's heads and k's, and forms its tokens' cosines and
// sines, once for all heads, in LDS while its heads are on their way: positions are
// asked for first, as loads return in order, and what is loaded is taken apart
// only where it is used.
//
// 32640 tokens of 20 heads of 128 bfloat16, a sixth of their rows between them: forward
// 57 us (5.9 TB/s), backward 98 (5.1) and 4 to join dw; with loads made as they were
// needed 77 and 120. 9975 tokens of 32 heads of 64: 18 (4.5 TB/s); 16 tokens: 5.9.
#include "rotary.h"

namespace mg {

constexpr int kHeadThreads = 256;
constexpr int kHeadTable = 2048;                  // cosines and sines a workgroup holds
constexpr int kHeadMaxDim = 512;
constexpr int64_t kHeadStreamBytes = 32 << 20;    // the L2 caches' together
constexpr int kHeadsFwd = 4, kHeadsBwd = 2;        // heads a lane has, at most

struct HeadTensor {
    const void *x, *dy;                           // (tokens, heads, dim)
    int64_t tok_stride, head_stride, dy_tok_stride, dy_head_stride;
    const void *weight;                           // NULL: ones
    void *out;                                    // y, or dx (NULL: not wanted); contiguous
    int32_t heads;
    int32_t blocks, each;                         // lanes' shares: blocks of `each` heads
};

struct HeadArgs {
    HeadTensor t[2];                              // q, k
    int64_t tokens;
    int32_t dim, pairs, axes, lanes;              // lanes a head
    // A workgroup takes at_once tokens, or one of `runs` runs of a token's blocks.
    int32_t at_once, runs;
    int64_t batches;
    float eps;
    const void *positions;
    const double *freq;
    int32_t positions_64, weight_f32, interleaved, stream;
    int32_t whole;                                // every lane's unit is
    float *partial;                               // (workgroups, 2, dim); NULL: no dw
    AxisTable axis;
};

// The first or the second of two values of the arguments, both in scalar registers:
// the compiler makes such a selection a load from one of two places otherwise, which
// each lane waits for.
template <typename V>
__device__ __forceinline__ V pick(int which, V first, V second) {
    asm("" : "+s"(first), "+s"(second));
    return which ? second : first;
}
// A pointer picked so has lost its address space.
template <typename T>
using Global = __attribute__((address_space(1))) T;

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

// A lane's unit: elements a .. a + V - 1 and b .. b + V - 1 of a head.
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

// V elements as they are loaded, from any address an element may have: whole, so
// that nothing waits for them before they are taken apart.
template <typename T, int V>
using HeadVec = T __attribute__((ext_vector_type(V), aligned(sizeof(T))));

// A unit's 2 V values as V pairs: run a with run b, or neighbours, a's first.
template <int V, bool kHalf>
struct HeadPairs {
    float p[V], q[V];

    template <typename A>
    __device__ __forceinline__ void set(const A &a, const A &b) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (kHalf) {
                p[i] = (float)a[i], q[i] = (float)b[i];
            } else {
                constexpr int H = V / 2;
                p[i] = (float)(i < H ? a[2 * i % V] : b[2 * i % V]);
                q[i] = (float)(i < H ? a[2 * i % V + 1] : b[2 * i % V + 1]);
            }
        }
    }
    __device__ __forceinline__ void get(float (&a)[V], float (&b)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (kHalf) {
                a[i] = p[i], b[i] = q[i];
            } else {
                constexpr int H = V / 2;
                float(&to)[V] = i < H ? a : b;
                to[2 * i % V] = p[i], to[2 * i % V + 1] = q[i];
            }
        }
    }
};

// The weights as float32 in LDS, q's, then k's. A thread's first is asked for ahead:
// by halves, so that no load depends on a branch.
struct HeadWeights {
    uint16_t lo, hi;

    static __device__ __forceinline__ const Global<uint16_t> *at(const HeadArgs &p, int i) {
        const bool second = i >= p.dim;
        // Without weights, some memory that is there.
        const void *none = p.freq;
        const void *w = pick(second, p.t[0].weight ? p.t[0].weight : none,
                             p.t[1].weight ? p.t[1].weight : none);
        const bool any = second ? p.t[1].weight != nullptr : p.t[0].weight != nullptr;
        return (const Global<uint16_t> *)w + (any ? (second ? i - p.dim : i) << p.weight_f32 : 0);
    }
    __device__ __forceinline__ void ask(const HeadArgs &p, int i) {
        const Global<uint16_t> *from = at(p, min(i, 2 * p.dim - 1));
        lo = from[0], hi = from[p.weight_f32];
    }
    __device__ __forceinline__ float value(const HeadArgs &p, bool bf16, int i) const {
        const uint32_t wide = (uint32_t)hi << 16 | lo;
        const float f = p.weight_f32 ? __builtin_bit_cast(float, wide)
                        : bf16       ? __builtin_bit_cast(float, (uint32_t)lo << 16)
                                     : (float)__builtin_bit_cast(f16_t, lo);
        return (i < p.dim ? p.t[0].weight : p.t[1].weight) ? f : 1.f;
    }
    // After ask(p, threadIdx.x).
    __device__ __forceinline__ void finish(const HeadArgs &p, bool bf16, float *to) {
        for (int i = threadIdx.x; i < 2 * p.dim; i += kHeadThreads) {
            if (i >= kHeadThreads) ask(p, i);
            to[i] = value(p, bf16, i);
        }
    }
};
template <int V, bool kHalf>
__device__ __forceinline__ HeadPairs<V, kHalf> unit_weights(const float *w, const HeadUnit &m) {
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        a[i] = m.a < 0 ? 0.f : w[m.a + i];
        b[i] = m.b < 0 ? 0.f : w[m.b + i];
    }
    HeadPairs<V, kHalf> x;
    x.set(a, b);
    return x;
}

// A unit of a head's row; a run that is none is cleared when it is looked at.
template <bool kStream, typename T, int V>
__device__ __forceinline__ void load_unit(const T *row, const HeadUnit &m, HeadVec<T, V> &a,
                                          HeadVec<T, V> &b) {
    auto *from_a = (const Global<HeadVec<T, V>> *)(row + max(m.a, 0));
    auto *from_b = (const Global<HeadVec<T, V>> *)(row + max(m.b, 0));
    if constexpr (kStream) {
        a = __builtin_nontemporal_load(from_a);
        b = __builtin_nontemporal_load(from_b);
    } else {
        a = *from_a;
        b = *from_b;
    }
}
template <typename A>
__device__ __forceinline__ void clear_none(const HeadArgs &p, const HeadUnit &m, A &a, A &b) {
    if (p.whole) return;
    if (m.a < 0) a = A{};
    if (m.b < 0) b = A{};
}
template <typename T, int V, bool kHalf>
__device__ __forceinline__ void store_unit(T *row, const HeadUnit &m, const HeadPairs<V, kHalf> &x,
                                           int stream) {
    float f[2][V];
    x.get(f[0], f[1]);
    HeadVec<T, V> a, b;
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = (T)f[0][i], b[i] = (T)f[1][i];
    auto *to_a = (Global<HeadVec<T, V>> *)(row + m.a), *to_b = (Global<HeadVec<T, V>> *)(row + m.b);
    if (stream) {
        if (m.a >= 0) __builtin_nontemporal_store(a, to_a);
        if (m.b >= 0) __builtin_nontemporal_store(b, to_b);
    } else {
        if (m.a >= 0) *to_a = a;
        if (m.b >= 0) *to_b = b;
    }
}

// What a thread has: heads h0 .. h0 + n - 1 of tensor `which` in its token of each
// batch, the slot-th; a thread without any has n = 0 and looks at the first. (Every
// blocks-th head in place of neighbours: a fifth slower backward.)
struct HeadShare {
    int which, slot, h0, n;
};
__device__ __forceinline__ HeadShare head_share(const HeadArgs &p, int run) {
    const int groups = kHeadThreads / p.lanes, g = threadIdx.x / p.lanes;
    const int first = p.t[0].blocks, all = first + p.t[1].blocks;
    int block = p.runs > 1 ? run * groups + g : g % all;
    int slot = p.runs > 1 ? 0 : g / all;
    const bool ok = block < all && slot < p.at_once;
    if (!ok) block = slot = 0;
    const int which = block >= first;
    const int each = pick(which, p.t[0].each, p.t[1].each);
    const int heads = pick(which, p.t[0].heads, p.t[1].heads);
    const int h0 = (block - (which ? first : 0)) * each;
    const bool any = ok && h0 < heads;
    return {which, slot, any ? h0 : 0, any ? min(each, heads - h0) : 0};
}

__device__ __forceinline__ HeadTensor head_tensor(const HeadArgs &p, int which) {
    const HeadTensor &q = p.t[0], &k = p.t[1];
    HeadTensor t{};
    t.x = pick(which, q.x, k.x), t.dy = pick(which, q.dy, k.dy);
    t.out = pick(which, q.out, k.out), t.heads = pick(which, q.heads, k.heads);
    t.tok_stride = pick(which, q.tok_stride, k.tok_stride);
    t.head_stride = pick(which, q.head_stride, k.head_stride);
    t.dy_tok_stride = pick(which, q.dy_tok_stride, k.dy_tok_stride);
    t.dy_head_stride = pick(which, q.dy_head_stride, k.dy_head_stride);
    return t;
}

// The angles of a batch: entry i is pair i % pairs of token i / pairs. A thread's
// first ones have their axis and frequency in registers.
constexpr int kHeadAngles = 2;
struct HeadAngles {
    int tok[kHeadAngles], axis[kHeadAngles];
    double freq[kHeadAngles];
    uint32_t lo[kHeadAngles], hi[kHeadAngles];

    __device__ __forceinline__ void init(const HeadArgs &p) {
#pragma unroll
        for (int e = 0; e < kHeadAngles; ++e) {
            const int i = threadIdx.x + e * kHeadThreads, pair = i % p.pairs;
            tok[e] = i / p.pairs;
            axis[e] = p.axis.axis[pair];
            freq[e] = p.freq[pair];
        }
    }
    // Asks for the positions (of tokens past the batch, the last one's).
    __device__ __forceinline__ void ask(const HeadArgs &p, int64_t tok0, int n_tok) {
#pragma unroll
        for (int e = 0; e < kHeadAngles; ++e) {
            const int64_t at = (tok0 + min(tok[e], n_tok - 1)) * p.axes + axis[e];
            const uint32_t *word = static_cast<const uint32_t *>(p.positions);
            lo[e] = word[at << p.positions_64];
            hi[e] = word[(at << p.positions_64) + p.positions_64];
        }
    }
    __device__ __forceinline__ void finish(const HeadArgs &p, int64_t tok0, int n_tok,
                                           float2 *cs) const {
#pragma unroll
        for (int e = 0; e < kHeadAngles; ++e) {
            const int64_t wide = (int64_t)((uint64_t)hi[e] << 32 | lo[e]);
            const double pos = p.positions_64 ? (double)wide : (double)(int32_t)lo[e];
            if (tok[e] < n_tok)
                cs[threadIdx.x + e * kHeadThreads] = turn_of(pos, freq[e], 1.f);
        }
        for (int i = threadIdx.x + kHeadAngles * kHeadThreads; i < n_tok * p.pairs;
             i += kHeadThreads) {
            const int t = i / p.pairs, pair = i - t * p.pairs;
            const int64_t at = (tok0 + t) * p.axes + p.axis.axis[pair];
            const double pos = p.positions_64
                                   ? (double)static_cast<const int64_t *>(p.positions)[at]
                                   : (double)static_cast<const int32_t *>(p.positions)[at];
            cs[i] = turn_of(pos, p.freq[pair], 1.f);
        }
    }
};

// A unit's cosines and sines of one token.
template <int V, bool kHalf>
__device__ __forceinline__ void unit_angles(const float2 *cs, const HeadUnit &m, float2 (&c)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = kHalf || i < V / 2 ? m.pair + i : m.pair_b + i - V / 2;
        c[i] = m.pair < 0 ? make_float2(1.f, 0.f) : cs[at];
    }
}

// C units a lane, 64 apart, of heads of more than 64.
template <typename T, int V, int C, bool kHalf>
__global__ __launch_bounds__(kHeadThreads) void norm_rotary_fwd_kernel(HeadArgs p) {
    constexpr int R = C == 1 ? kHeadsFwd : 1;
    __shared__ float2 s_cs[kHeadTable];
    __shared__ float s_w[2 * kHeadMaxDim];
    const int run = p.runs > 1 ? blockIdx.x % p.runs : 0;
    const int64_t tok0 = (int64_t)(blockIdx.x / p.runs) * p.at_once;
    const int n_tok = (int)min((int64_t)p.at_once, p.tokens - tok0);
    HeadAngles angles;
    angles.init(p);
    angles.ask(p, tok0, n_tok);
    HeadWeights weights;
    weights.ask(p, threadIdx.x);
    const HeadShare mine = head_share(p, run);
    const HeadTensor t = head_tensor(p, mine.which);
    const int slot = min(mine.slot, n_tok - 1), n = mine.slot < n_tok ? mine.n : 0;
    HeadUnit unit[C];
#pragma unroll
    for (int c = 0; c < C; ++c)
        unit[c] = head_unit<V, kHalf>(p, threadIdx.x % p.lanes + 64 * c);
    HeadVec<T, V> xa[R][C], xb[R][C];
    const T *x = static_cast<const T *>(t.x) + (tok0 + slot) * t.tok_stride +
                 mine.h0 * t.head_stride;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T *row = x + min(r, max(n - 1, 0)) * t.head_stride;
#pragma unroll
        for (int c = 0; c < C; ++c) load_unit<false, T, V>(row, unit[c], xa[r][c], xb[r][c]);
    }
    angles.finish(p, tok0, n_tok, s_cs);
    weights.finish(p, std::is_same<T, bf16_t>::value, s_w);
    __syncthreads();
    // y = s R (x w): the weights and the rotation are a token's.
    float pc[C][V], ps[C][V], qc[C][V], qs[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float2 cs[V];
        unit_angles<V, kHalf>(s_cs + slot * p.pairs, unit[c], cs);
        const HeadPairs<V, kHalf> w = unit_weights<V, kHalf>(s_w + mine.which * p.dim, unit[c]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            pc[c][i] = w.p[i] * cs[i].x, ps[c][i] = w.p[i] * cs[i].y;
            qc[c][i] = w.q[i] * cs[i].x, qs[c][i] = w.q[i] * cs[i].y;
        }
    }
    const float per = 1.f / (float)p.dim;
    T *out = static_cast<T *>(t.out) + ((tok0 + slot) * t.heads + mine.h0) * (int64_t)p.dim;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float ss = 0.f;
        HeadPairs<V, kHalf> h[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            clear_none(p, unit[c], xa[r][c], xb[r][c]);
            h[c].set(xa[r][c], xb[r][c]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                ss = fmaf(h[c].p[i], h[c].p[i], ss);
                ss = fmaf(h[c].q[i], h[c].q[i], ss);
            }
        }
        const float s = rsqrtf(group_sum(ss, p.lanes) * per + p.eps);
        if (r >= n) continue;
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float a = h[c].p[i] * s, b = h[c].q[i] * s;
                h[c].p[i] = a * pc[c][i] - b * qs[c][i];
                h[c].q[i] = b * qc[c][i] + a * ps[c][i];
            }
            store_unit<T, V, kHalf>(out + r * p.dim, unit[c], h[c], p.stream);
        }
    }
}

// A workgroup takes every so many batches and keeps its sums for dw in registers,
// joined by norm_rotary_join_kernel in a fixed order.
template <typename T, int V, int C, bool kHalf, bool kStream>
__global__ __launch_bounds__(kHeadThreads) void norm_rotary_bwd_kernel(HeadArgs p) {
    constexpr int R = C == 1 ? kHeadsBwd : 1;
    constexpr int kSums = 2 * V * C * kHeadThreads;
    // The angles of two batches in turn, then the threads' sums for dw.
    __shared__ float2 s_cs[kSums > 2 * kHeadTable ? kSums / 2 : kHeadTable];
    __shared__ float s_w[2 * kHeadMaxDim];
    const int run = p.runs > 1 ? blockIdx.x % p.runs : 0;
    HeadAngles angles;
    angles.init(p);
    const HeadShare mine = head_share(p, run);
    const HeadTensor t = head_tensor(p, mine.which);
    HeadUnit unit[C];
    HeadPairs<V, kHalf> w[C], dw[C] = {};
    HeadWeights weights;
    weights.ask(p, threadIdx.x);
    weights.finish(p, std::is_same<T, bf16_t>::value, s_w);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c) {
        unit[c] = head_unit<V, kHalf>(p, threadIdx.x % p.lanes + 64 * c);
        w[c] = unit_weights<V, kHalf>(s_w + mine.which * p.dim, unit[c]);
    }
    lds_reads_done();
    const float per = 1.f / (float)p.dim;
    int buf = 0;
    for (int64_t at = blockIdx.x / p.runs; at < p.batches; at += gridDim.x / p.runs, buf ^= 1) {
        const int64_t tok0 = at * p.at_once;
        const int n_tok = (int)min((int64_t)p.at_once, p.tokens - tok0);
        const int slot = min(mine.slot, n_tok - 1), n = mine.slot < n_tok ? mine.n : 0;
        angles.ask(p, tok0, n_tok);
        HeadVec<T, V> xa[R][C], xb[R][C], ga[R][C], gb[R][C];
        const T *x = static_cast<const T *>(t.x) + (tok0 + slot) * t.tok_stride +
                     mine.h0 * t.head_stride;
        const T *dy = static_cast<const T *>(t.dy) + (tok0 + slot) * t.dy_tok_stride +
                      mine.h0 * t.dy_head_stride;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int at_r = min(r, max(n - 1, 0));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                load_unit<kStream, T, V>(x + at_r * t.head_stride, unit[c], xa[r][c], xb[r][c]);
                load_unit<kStream, T, V>(dy + at_r * t.dy_head_stride, unit[c], ga[r][c], gb[r][c]);
            }
        }
        float2 *table = s_cs + buf * (kHeadTable / 2);
        angles.finish(p, tok0, n_tok, table);
        __syncthreads();
        float2 cs[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c)
            unit_angles<V, kHalf>(table + slot * p.pairs, unit[c], cs[c]);
        lds_reads_done();
        T *out = static_cast<T *>(t.out) + ((tok0 + slot) * t.heads + mine.h0) * (int64_t)p.dim;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float ss = 0.f, hx = 0.f;
            HeadPairs<V, kHalf> h[C], g[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                clear_none(p, unit[c], xa[r][c], xb[r][c]);
                clear_none(p, unit[c], ga[r][c], gb[r][c]);
                h[c].set(xa[r][c], xb[r][c]);
                g[c].set(ga[r][c], gb[r][c]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float a = g[c].p[i], b = g[c].q[i];
                    g[c].p[i] = a * cs[c][i].x + b * cs[c][i].y;
                    g[c].q[i] = b * cs[c][i].x - a * cs[c][i].y;
                    ss = fmaf(h[c].p[i], h[c].p[i], ss);
                    ss = fmaf(h[c].q[i], h[c].q[i], ss);
                    hx = fmaf(g[c].p[i] * h[c].p[i], w[c].p[i], hx);
                    hx = fmaf(g[c].q[i] * h[c].q[i], w[c].q[i], hx);
                }
            }
            const float s = rsqrtf(group_sum(ss, p.lanes) * per + p.eps);
            // By u, never by powers of s, which pass float32's range before dx does.
            const float along = group_sum(hx, p.lanes) * per * s;            // mean(h u)
            if (r >= n) continue;
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float a = h[c].p[i] * s, b = h[c].q[i] * s;
                    dw[c].p[i] = fmaf(g[c].p[i], a, dw[c].p[i]);
                    dw[c].q[i] = fmaf(g[c].q[i], b, dw[c].q[i]);
                    h[c].p[i] = (g[c].p[i] * w[c].p[i] - a * along) * s;
                    h[c].q[i] = (g[c].q[i] * w[c].q[i] - b * along) * s;
                }
                if (t.out) store_unit<T, V, kHalf>(out + r * p.dim, unit[c], h[c], p.stream);
            }
        }
    }
    if (!p.partial) return;
    // All threads' sums, (group, dim) of a group's lanes, added up group by group.
    lds_reads_done();
    __syncthreads();
    float *sums = reinterpret_cast<float *>(s_cs);
    const int groups = kHeadThreads / p.lanes, group = threadIdx.x / p.lanes;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float a[V], b[V];
        dw[c].get(a, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (unit[c].a >= 0) sums[group * p.dim + unit[c].a + i] = a[i];
            if (unit[c].b >= 0) sums[group * p.dim + unit[c].b + i] = b[i];
        }
    }
    __syncthreads();
    const int all = p.t[0].blocks + p.t[1].blocks;
    for (int i = threadIdx.x; i < 2 * p.dim; i += kHeadThreads) {
        const int which = i >= p.dim, at = which ? i - p.dim : i;
        float sum = 0.f;
        for (int g = 0; g < groups; ++g) {
            const int block = p.runs > 1 ? run * groups + g : g % all;
            if (block < all && (block >= p.t[0].blocks) == which) sum += sums[g * p.dim + at];
        }
        p.partial[(int64_t)blockIdx.x * 2 * p.dim + i] = sum;
    }
}

// dw of q (blockIdx.y 0) and k (1), 32 columns: 32 threads a column, each over
// every 32nd workgroup's sums.
constexpr int kHeadJoinCols = 32, kHeadJoinThreads = 1024;
template <typename W>
__global__ __launch_bounds__(kHeadJoinThreads) void norm_rotary_join_kernel(
    const float *__restrict__ partial, int parts, int dim, W *dq, W *dk) {
    constexpr int kGroups = kHeadJoinThreads / kHeadJoinCols;
    __shared__ float s[kGroups][kHeadJoinCols + 1];
    W *out = blockIdx.y ? dk : dq;
    const int col = threadIdx.x % kHeadJoinCols, group = threadIdx.x / kHeadJoinCols;
    const int at = blockIdx.x * kHeadJoinCols + col;
    float sum = 0.f;
    if (at < dim) {
        const float *from = partial + (int64_t)blockIdx.y * dim + at;
#pragma unroll 8
        for (int i = group; i < parts; i += kGroups) sum += from[(int64_t)i * 2 * dim];
    }
    s[group][col] = sum;
    __syncthreads();
    if (group == 0 && at < dim && out) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) total += s[i][col];
        out[at] = (W)total;
    }
}

// -------------------------------------------------------------------- host
constexpr int64_t kHeadGroups = 1024;             // workgroups of a backward pass

// Units of V elements: how many lanes a head takes, 0 where they do not fit.
static int head_lanes(int dim, int pairs, int V, int C) {
    if (pairs % V || (dim - 2 * pairs) % V) return 0;
    const int units = pairs / V + ((dim - 2 * pairs) / V + 1) / 2;
    if (C > 1) return units <= 64 * C ? 64 : 0;
    int lanes = 1;
    while (lanes < units) lanes *= 2;
    return lanes <= 64 ? lanes : 0;
}

// Cuts the tokens' heads into blocks of up to R, a lane's, and the tokens into
// batches of as many as a workgroup has lanes for.
static void head_cut(HeadArgs &p, int lanes, int V, int C, int R, int table) {
    p.lanes = lanes, p.whole = p.dim == 2 * V * C * lanes;
    int blocks = 0;
    for (HeadTensor &t : p.t) {
        t.blocks = (int32_t)ceil_div(t.heads, R);
        t.each = t.blocks ? (int32_t)ceil_div(t.heads, t.blocks) : 1;
        blocks += t.blocks;
    }
    const int groups = kHeadThreads / lanes;
    p.runs = (int32_t)ceil_div(blocks, groups);
    int64_t at_once = p.runs > 1 ? 1 : groups / blocks;
    if (at_once > table / p.pairs) at_once = table / p.pairs;
    // A few tokens are spread over the GPU.
    if (at_once > ceil_div(p.tokens, 512)) at_once = ceil_div(p.tokens, 512);
    p.at_once = (int32_t)(at_once < 1 ? 1 : at_once);
    p.batches = ceil_div(p.tokens, p.at_once);
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
            head_cut(p, lanes, V, C, C == 1 ? kHeadsFwd : 1, kHeadTable);
            const int64_t grid = p.batches * p.runs;
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

int64_t mg_norm_rotary_backward_workspace_bytes(int32_t q_heads, int32_t k_heads, int32_t dim) {
    // Two rows of sums a workgroup: kHeadGroups of them, or one for each run of a
    // token's heads (a workgroup has four heads at least).
    if (dim <= 0 || q_heads < 0 || k_heads < 0) return 0;
    const int64_t runs = ((int64_t)q_heads + k_heads) / 4 + 1;
    return (runs > mg::kHeadGroups ? runs : mg::kHeadGroups) * 2 * dim * 4;
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
    const int64_t need = mg_norm_rotary_backward_workspace_bytes(q_heads, k_heads, dim);
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
    int64_t grid = 0;
    {
        TimedScope ts("norm_rotary_bwd", st);
        head_types(dtype, [&](auto type) {
            using T = decltype(type);
            head_form<T>(p, [&](auto v, auto c, auto half, int lanes) {
                constexpr int V = decltype(v)::value, C = decltype(c)::value;
                head_cut(p, lanes, V, C, C == 1 ? kHeadsBwd : 1, kHeadTable / 2);
                const int64_t turns = p.runs > kHeadGroups ? 1 : kHeadGroups / p.runs;
                grid = (p.batches < turns ? p.batches : turns) * p.runs;
                constexpr bool kHalf = decltype(half)::value;
                if (p.stream)
                    norm_rotary_bwd_kernel<T, V, C, kHalf, true>
                        <<<(unsigned)grid, kHeadThreads, 0, st>>>(p);
                else
                    norm_rotary_bwd_kernel<T, V, C, kHalf, false>
                        <<<(unsigned)grid, kHeadThreads, 0, st>>>(p);
            });
        });
        MG_LAUNCHED("norm_rotary_bwd_kernel");
    }
    if (sums) {
        TimedScope ts("norm_rotary_join", st);
        const dim3 columns((unsigned)ceil_div(dim, kHeadJoinCols), 2);
        const auto go = [&](auto w) {
            using W = decltype(w);
            norm_rotary_join_kernel<W><<<columns, kHeadJoinThreads, 0, st>>>(
                p.partial, (int)grid, dim, static_cast<W *>(dq_weight),
                static_cast<W *>(dk_weight));
        };
        head_types(weight_dtype, go);
        MG_LAUNCHED("norm_rotary_join_kernel");
    }
    return MG_OK;
}

}  // extern "C"
