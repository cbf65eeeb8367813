// Shared by the attention kernels' files. Internal header.
#pragma once

#include "attention_tiles.h"
#include "mg_types.h"

namespace mg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mfma32(vec8<bf16_t> a, vec8<bf16_t> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(vec8<f16_t> a, vec8<f16_t> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Keys (or, in the keys' gradient, queries) of one LDS tile.
constexpr int kTileRows = 64;
template <int DK, int kTile = kTileRows>
constexpr int kTileBytes = kTile * tile_chunks<DK>() * 16;

struct AttnTensor {
    const void *p;
    int64_t tok_stride, head_stride;     // elements
};

struct AttnArgs {
    AttnTensor q, k, v, dout;            // dout: the backward pass only
    const int32_t *q_off, *k_off;        // NULL: one sequence of all tokens
    int32_t n_seq;
    int32_t q_tokens, k_tokens;
    int32_t k_heads, group, dim;         // q_heads = k_heads * group
    int32_t causal;
    // With a window (causal): a query sees the last `window` keys up to where it
    // stands, and the sequence's first `sinks`. 0: no window.
    int32_t window, sinks;
    float scale, scale_log2;             // scale, scale * log2(e)
    void *out;                           // (q_tokens, q_heads, dim)
    void *out_rest;                      // what rounding took from out, or NULL
    float *lse;                          // (q_heads, q_tokens), in powers of 2; NULL: not kept
    // Split over the keys: chunks of split_keys (more with over chunk_tiles tiles:
    // chunks_of), whose {top, sum} and unscaled sums of values are joined
    // afterwards.
    int32_t split_keys, chunk_tiles;
    int32_t span_extra, span_most;       // of the keys an item goes through: span_keys
    int32_t row_chunks;                  // see Cut
    float2 *part_stats;
    float *part_o;
    // Backward.
    const float *delta;                  // (q_heads, q_tokens)
    float *largest_do, *largest_v;       // float16: see attention_bwd.hip
    void *dq, *dk, *dv;
    // Keys' gradients over up to `splits` runs of query tiles, of split_steps at
    // least, each in float32 (part_of).
    int32_t splits, split_steps;
    float *part;
    // With sinks: the first keys' gradients from queries further on than the
    // window, in runs of about sink_steps query tiles of one head (sink_cut).
    int32_t key_runs, sink_steps, sink_near, sink_rows;
    float *sink_part;
};

// ---------------------------------------------------------------- sequences
// A work item's sequence. Tokens before the first offset and past the last
// belong to no sequence: they are given out as sequences of queries without
// keys (kByKeys: of keys without queries), so that their outputs and gradients
// are zeros and no row stays unwritten.
struct SeqItem {
    int q_lo, q_len, k_lo, k_len;
    int seq;           // 1 .. n; 0 and n + 1: the tokens of no sequence
    int within;        // the item's number within its sequence
    int before;        // sum of the second count over the sequences before
    bool found;
};

// A value that is the same in all lanes, where the compiler cannot tell.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int clamp_to(int v, int lo, int hi) { return min(max(v, lo), hi); }

template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ int dpp_i(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false);
}
__device__ __forceinline__ int wave_inclusive_sum(int v) {
    v += dpp_i<0x111>(v);        // row_shr:1
    v += dpp_i<0x112>(v);        // row_shr:2
    v += dpp_i<0x114>(v);        // row_shr:4
    v += dpp_i<0x118>(v);        // row_shr:8
    v += dpp_i<0x142, 0xa>(v);   // row_bcast:15
    v += dpp_i<0x143, 0xc>(v);   // row_bcast:31
    return v;
}
__device__ __forceinline__ int wave_inclusive_max(int v) {       // v >= 0
    v = max(v, dpp_i<0x111>(v));
    v = max(v, dpp_i<0x112>(v));
    v = max(v, dpp_i<0x114>(v));
    v = max(v, dpp_i<0x118>(v));
    v = max(v, dpp_i<0x142, 0xa>(v));
    v = max(v, dpp_i<0x143, 0xc>(v));
    return v;
}

// Tokens of pseudo sequences s0 + lane of n + 2 (0: before the first, n + 1: past
// the last), s0 a multiple of 64 and `end` where the one before s0 ends, which is
// carried on. Offsets are held to [0, tokens] and made to rise (an offset below
// one before it counts as that one), so that no value of theirs leads out of the
// tensors and every token is in one pseudo sequence. For all lanes of a wave.
__device__ __forceinline__ void seq_bounds(const int32_t *off, int n, int tokens, int s0, int &end,
                                           int &lo, int &len) {
    const int s = s0 + lane_id();
    int to = tokens;
    if (off) {
        if (s <= n) to = clamp_to(off[s], 0, tokens);
    } else if (s == 0) {
        to = 0;
    }
    to = max(end, wave_inclusive_max(to));
    lo = __builtin_amdgcn_update_dpp(end, to, 0x138, 0xf, 0xf, false);   // wave_shr:1
    len = to - lo;
    end = __builtin_amdgcn_readlane(to, 63);
}

// The sequence that has `item` when a sequence has count(q_len, k_len) items;
// `before` sums second(q_len, k_len). Every lane of a wave calls with the same
// item and gets the same answer; where no sequence has the item, found is false
// and within the number of all items.
template <bool kByKeys, typename Count, typename Second>
__device__ __forceinline__ SeqItem find_item(const AttnArgs &a, int item, Count count,
                                             Second second) {
    SeqItem r{};
    int base = 0, base2 = 0, q_end = 0, k_end = 0;
    for (int s0 = 0; s0 < a.n_seq + 2; s0 += 64) {
        const int s = s0 + lane_id();
        int q_lo, q_len, k_lo, k_len;
        seq_bounds(a.q_off, a.n_seq, a.q_tokens, s0, q_end, q_lo, q_len);
        seq_bounds(a.k_off, a.n_seq, a.k_tokens, s0, k_end, k_lo, k_len);
        if (s == 0 || s > a.n_seq) (kByKeys ? q_len : k_len) = 0;
        const int n = count(q_len, k_len), n2 = second(q_len, k_len);
        const int upto = wave_inclusive_sum(n), upto2 = wave_inclusive_sum(n2);
        const uint64_t past = ballot(base + upto > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            r.seq = s0 + l;
            const auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            r.q_lo = get(q_lo), r.q_len = get(q_len), r.k_lo = get(k_lo), r.k_len = get(k_len);
            r.within = clamp_to(item - (base + get(upto) - get(n)), 0, get(n) - 1);
            r.before = base2 + get(upto2) - get(n2);
            r.found = true;
            return r;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
        base2 += __builtin_amdgcn_readlane(upto2, 63);
    }
    r.within = base;
    return r;
}

// ------------------------------------------------------------------ windows
// The first key of a query's window.
__device__ __forceinline__ int key_low(const AttnArgs &a, const SeqItem &s, int token) {
    return max(0, token + 1 + s.k_len - s.q_len - a.window);
}

// The keys that the queries from `first` to `last` go through, numbered in the order
// they are: all from the first to the last seen, or, with a window, first the
// sinks in whole tiles, then those from the first query's window on that are
// none. A sink lies in a query's window or before it: it counts as a sink.
struct KeyRun {
    int sink, sink_up, start, end;
};
template <bool kWin, int kTile>
__device__ __forceinline__ KeyRun key_run(const AttnArgs &a, const SeqItem &s, int first,
                                          int seen_to) {
    if constexpr (!kWin) return {0, 0, 0, seen_to};
    const int sink = min(a.sinks, seen_to), start = max(key_low(a, s, first), sink);
    const int sink_up = (sink + kTile - 1) / kTile * kTile;
    return {sink, sink_up, start, sink_up + max(0, seen_to - start)};
}

// The key of a number in the run.
template <bool kWin>
__device__ __forceinline__ int key_at(const KeyRun &r, int number) {
    return !kWin ? number : number < r.sink_up ? number : number - r.sink_up + r.start;
}

// The bounds of what a query sees, within the tile of a number: among the sinks,
// they alone; past them, the window alone.
struct TileSees {
    bool sinks;
    int sink;
    __device__ __forceinline__ int to(int see) const { return sinks ? min(see, sink) : see; }
    __device__ __forceinline__ int from(int low) const { return sinks ? 0 : low; }
};
template <bool kWin>
__device__ __forceinline__ TileSees tile_sees(const KeyRun &r, int number) {
    return {kWin && number < r.sink_up, r.sink};
}

// ------------------------------------------------------------- longest first
// Tiles of R rows (tokens by `per`) of a sequence that have at least w >= 1 pairs a
// row to go through. By queries: the tile's last query's seen keys, rising with
// the tile. By keys: the queries that see the tile's first key, falling with it.
template <bool kByKeys>
__device__ __forceinline__ int tiles_with(const AttnArgs &a, int R, int q_len, int k_len, int w) {
    const int ahead = k_len - q_len;
    if constexpr (kByKeys) {
        const int tiles = (k_len + R - 1) / R;
        if (q_len < w) return 0;
        if (!a.causal) return tiles;
        const int last = q_len - w + ahead;       // the last first key that w see
        return last < 0 ? 0 : min(tiles, last / R + 1);
    } else {
        const int tiles = (q_len * a.group + R - 1) / R;
        if (k_len < w) return 0;
        if (!a.causal) return tiles;
        const int query = w - 1 - ahead;          // the first query that sees w
        if (query >= q_len) return 0;
        return tiles - max(0, query) * a.group / R;
    }
}

// Work item `item` of all sequences' tiles of R rows, in falling order of the
// pairs a row has, in steps of 64: workgroups start in order, so that the
// longest are not left for the end (packed sequences of 1 to 2500 tokens, causal:
// see attention_bwd.hip). s.within is the tile. Up to 62 sequences; with more
// the items come sequence by sequence.
template <bool kByKeys>
__device__ __forceinline__ SeqItem find_longest(const AttnArgs &a, int item, int R) {
    const auto tiles_of = [&](int ql, int kl) {
        return kByKeys ? (kl + R - 1) / R : (ql * a.group + R - 1) / R;
    };
    if (a.n_seq == 1 || a.n_seq + 2 > 64) {
        SeqItem s = find_item<kByKeys>(a, item, tiles_of, [](int, int) { return 0; });
        if (!kByKeys) s.within = tiles_of(s.q_len, 0) - 1 - s.within;
        return s;
    }
    const int seq = lane_id();
    int q_end = 0, k_end = 0, q_lo, q_len, k_lo, k_len;
    seq_bounds(a.q_off, a.n_seq, a.q_tokens, 0, q_end, q_lo, q_len);
    seq_bounds(a.k_off, a.n_seq, a.k_tokens, 0, k_end, k_lo, k_len);
    if (seq == 0 || seq > a.n_seq) (kByKeys ? q_len : k_len) = 0;
    const int tiles = tiles_of(q_len, k_len);
    const auto with = [&](int w) {                // this lane's sequence's
        return w == 0 ? tiles : tiles_with<kByKeys>(a, R, q_len, k_len, w * 64);
    };
    const auto all = [&](int w) {
        return __builtin_amdgcn_readlane(wave_inclusive_sum(with(w)), 63);
    };
    SeqItem r{};
    if (all(0) <= item) return r;
    int lo = 0, hi = uniform(wave_max_i(kByKeys ? q_len : k_len)) / 64 + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (all(mid) > item)
            lo = mid;
        else
            hi = mid;
    }
    // The item is among the tiles that lo has and lo + 1 has not.
    const int longer = with(lo + 1), here = with(lo) - longer;
    const int rank = item - all(lo + 1), upto = wave_inclusive_sum(here);
    const uint64_t past = ballot(upto > rank);
    const int l = past ? __builtin_ctzll(past) : 0;
    r.seq = l;
    const auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
    r.q_lo = get(q_lo), r.q_len = get(q_len), r.k_lo = get(k_lo), r.k_len = get(k_len);
    const int nth = get(longer) + rank - (get(upto) - get(here));
    r.within = clamp_to(kByKeys ? nth : get(tiles) - 1 - nth, 0, get(tiles) - 1);
    r.found = past != 0;
    return r;
}

// ------------------------------------------------------------- filling tiles
// Descriptor of `bytes` bytes from a wave-uniform address; accesses past them
// do not reach memory.
__device__ __forceinline__ i32x4 buffer_of(const void *base, uint32_t bytes) {
    const uint64_t at = (uintptr_t)base;
    return i32x4{uniform((int)(uint32_t)at), uniform((int)(uint32_t)(at >> 32) & 0xffff),
                 uniform((int)bytes), 0x00020000};
}

// Asks for rows row0 .. row0 + kTile - 1 (of n_rows; past the last, the last row again,
// whose products the masks leave out) of one head into an LDS tile, straight
// from memory: nothing passes through registers, and the wave goes on at once.
// tiles_ready() waits. Wave `wave` of kWaves makes every kWaves-th load.
//
// The loads are written in assembly because the compiler, which cannot tell
// one LDS buffer from the other, would wait for them before the next LDS read.
// Its hazard pass does not look into assembly: the five wait states between a
// vector instruction's scalar result (v_readfirstlane, in the descriptor) and a
// memory access that reads it stand before the first load, and m0's one before
// each.
template <int DK, int kWaves, int kTile = kTileRows>
struct TileFill {
    static constexpr int kAll = kTileBytes<DK, kTile> / 1024, kLoads = kAll / kWaves;
    static_assert(kAll % kWaves == 0, "whole loads a wave");
    uint32_t off[kLoads];          // bytes from row0's, of a whole tile

    __device__ __forceinline__ void init(int64_t tok_stride, int dim, int wave) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) off[i] = offset(i, tok_stride, dim, wave, kTile);
    }

    // Columns past the head's dimension read column 0 .. 7: the products beside
    // them are with zeros or are dropped.
    static __device__ __forceinline__ uint32_t offset(int i, int64_t tok_stride, int dim, int wave,
                                                      int rows) {
        const int lane = lane_id(), load = i * kWaves + wave;
        const int r = min(fill_row<DK>(load, lane), rows - 1), c = fill_chunk<DK>(load, lane);
        return (uint32_t)r * (uint32_t)(tok_stride * 2) + (c * 8 < dim ? c * 16 : 0);
    }

    // A tile to be asked for, load by load.
    struct Order {
        i32x4 rsrc;
        int to, rows;
    };

    __device__ __forceinline__ Order order(const char *head, int64_t tok_stride, int dim, int row0,
                                           int n_rows, int wave, uint32_t lds) const {
        const int rows = min(n_rows - row0, kTile);
        const char *base = head + (int64_t)row0 * tok_stride * 2;
        const uint32_t bytes = (uint32_t)(rows - 1) * (uint32_t)(tok_stride * 2) + dim * 2;
        return {buffer_of(base, bytes), uniform((int)lds + wave * 1024), rows};
    }

    // Load i of a whole tile.
    __device__ __forceinline__ void load(int i, const Order &o) const { load(i, o, off[i]); }

    // The compiler knows nothing of the LDS that this writes: it is ordered by
    // the barriers of tiles_ready() alone, and LDS reads may pass it.
    static __device__ __forceinline__ void load(int i, const Order &o, uint32_t at) {
        // The descriptor is the same for all of them: the first waits for it.
        if (i == 0)
            asm volatile("s_mov_b32 m0, %0\n\t"
                         "s_nop 4\n\t"
                         "buffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(o.to), "v"(at), "s"(o.rsrc)
                         : "m0");
        else
            asm volatile("s_mov_b32 m0, %0\n\t"
                         "s_nop 0\n\t"
                         "buffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(o.to + i * kWaves * 1024), "v"(at), "s"(o.rsrc)
                         : "m0");
    }

    __device__ __forceinline__ void ask(const char *head, int64_t tok_stride, int dim, int row0,
                                        int n_rows, int wave, uint32_t lds) const {
        const Order o = order(head, tok_stride, dim, row0, n_rows, wave, lds);
        if (o.rows == kTile) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(i, o);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                load(i, o, offset(i, tok_stride, dim, wave, o.rows));
        }
    }
};

// The tiles asked for are there, for every wave, and no wave reads from what is
// asked for next.
__device__ __forceinline__ void tiles_ready() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Ends the loads made so far, in a way that the compiler counts: a loop after it
// holds no wait for them, which would be one for the tiles asked for in between.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

__device__ __forceinline__ uint32_t lds_address(const char *p) {
    return (uint32_t)(uintptr_t)(const lds_char *)p;
}

// ------------------------------------------------------------------ operands
// A lane's places in any tile. fresh() keeps the compiler from holding an
// address for every step in registers of its own: each is one exclusive or.
template <typename T, int DK>
struct TileLane {
    int row, column;

    __device__ __forceinline__ TileLane()
        : row(row_lane_byte<DK>(lane_id())), column(column_lane_byte<DK>(lane_id())) {}

    __device__ __forceinline__ void fresh() {
        asm volatile("" : "+v"(row), "+v"(column));
    }

    __device__ __forceinline__ vec8<T> rows(const char *tile, int row0, int step) const {
        return *reinterpret_cast<const vec8<T> *>(tile + row_operand_byte<DK>(row, row0, step));
    }

    // Rows row0 .. row0 + 15 in the order a C leaves its rows, columns 32 block ...
    __device__ __forceinline__ vec8<T> columns(const char *tile, int row0, int block) const {
        const auto read = [&](int r) {
            return __builtin_bit_cast(
                vec4<T>, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                             (lds_s16x4 *)(tile + column_operand_byte<DK>(column, r, block))));
        };
        return __builtin_shufflevector(read(row0), read(row0 + 8), 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// ------------------------------------------------------------------- results
// A wave's 32 rows of results, by way of LDS: a lane of a product has four columns
// of its row at a time, and stores of those would be 16 bytes a row; from LDS each
// row goes out whole. (Stored by fours: 16384 tokens of 16 heads of 128 with a window
// of one key, result and what rounding took from it, 120 us.) Of the tiles'
// memory, which every wave has done with.
template <int DK>
constexpr int kRowPitch = DK * 2 + 16;           // bytes, rows spread over the banks
template <int DK>
constexpr int kRowBytes = 32 * kRowPitch<DK>;    // a wave's

template <typename T, int DK>
struct RowStore {
    char *lds;                                   // the wave's

    // value(b, e): element e of block b of this lane's row, in T. The row goes to
    // out + at_row (as lane l % 32 has it) where row_ok.
    template <typename F>
    __device__ __forceinline__ void operator()(T *out, int64_t at_row, bool row_ok, int dim,
                                               F value) const {
        const int lane = lane_id(), half = lane / 32;
#pragma unroll
        for (int b = 0; b < DK / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                vec4<T> w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = value(b, e + i);
                *reinterpret_cast<vec4<T> *>(lds + lane % 32 * kRowPitch<DK> +
                                             (32 * b + c_row(e, half)) * 2) = w;
            }
        lds_reads_done();
        constexpr int kLanes = DK <= 32 ? 4 : DK <= 64 ? 8 : 16, kRows = 64 / kLanes;
        const int chunk = lane % kLanes;
        const uint64_t to = row_ok ? (uint64_t)(out + at_row) : 0;
#pragma unroll
        for (int r = 0; r < 32; r += kRows) {
            const int row = r + lane / kLanes;
            // The address that the row's own lane has.
            const uint32_t lo = __shfl((uint32_t)to, row, 64);
            const uint32_t hi = __shfl((uint32_t)(to >> 32), row, 64);
            const uint64_t at = (uint64_t)hi << 32 | lo;
            const i32x4 w =
                *reinterpret_cast<const i32x4 *>(lds + row * kRowPitch<DK> + chunk * 16);
            if (at && chunk * 8 < dim)
                *(__attribute__((address_space(1))) i32x4 *)(at + chunk * 16) = w;
        }
        lds_reads_done();
    }
};

// Eight elements of row `row` from column `at` in memory, zeros if !ok.
template <typename T>
__device__ __forceinline__ vec8<T> memory_operand(const T *row, int at, bool ok) {
    vec8<T> v = {};
    if (ok) v = *reinterpret_cast<const vec8<T> *>(row + at);
    return v;
}

// Max and sum over the two halves of a wave, lane l and l + 32.
__device__ __forceinline__ float halves_max(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]),
                 __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Host: f<T, DK>() for the element type and the head dimension's tile.
template <typename F>
static void attn_form(int32_t dtype, int dim, F f) {
    const auto with = [&](auto t) {
        using std::integral_constant;
        if (dim <= 32)
            f(t, integral_constant<int, 32>{});
        else if (dim <= 64)
            f(t, integral_constant<int, 64>{});
        else if (dim <= 96)
            f(t, integral_constant<int, 96>{});
        else
            f(t, integral_constant<int, 128>{});
    };
    if (dtype == MG_BF16)
        with(bf16_t{});
    else
        with(f16_t{});
}

// scale * log2(e). A scale of 0 (all seen keys alike) keeps a trace, by which
// the -inf of an unseen key stays what it is.
inline float scale_to_log2(float scale) {
    const float s = scale * 1.44269504088896340736f;
    return s < 1e-30f ? 1e-30f : s;
}

// Window and sinks held to the keys: a window of all of them is none.
inline void hold_window(AttnArgs &a) {
    if (a.window >= a.k_tokens) a.window = a.sinks = 0;
    if (a.sinks > a.k_tokens) a.sinks = a.k_tokens;
}

int32_t attn_check(const char *who, const AttnArgs &a, int32_t dtype);

}  // namespace mg
