// Index rules of the attention kernels' tiles: plain constexpr functions, also
// compiled by the host compiler alone for the index tests. Internal header.
#pragma once

#include <stdint.h>

namespace mg {

// ------------------------------------------------- 32x32x16 matrix products
// C (32 x 32) += A (32 x 16) B (16 x 32), a wave's 64 lanes in two halves h:
//   A: lane l holds row l % 32, eight of its 16 columns;
//   B: lane l holds column l % 32, eight of its 16 rows;
//   C: lane l holds column l % 32, element e (of 16) is row c_row(e, h).
// The product sums over the 16 in any order as long as A and B agree on it.
// Operands read along memory rows take them in memory order (half h has
// 8h .. 8h + 7). An operand that is a C of an earlier product has its rows
// where that product left them, elements 8s .. 8s + 7 being the s-th B, and the
// A beside it is read in that order: 4h .. 4h + 3 and 8 + 4h .. 8 + 4h + 3.
constexpr int c_row(int e, int h) { return 8 * (e / 4) + 4 * h + e % 4; }

// --------------------------------------------------------------- LDS tiles
// Rows of DK elements of two bytes in chunks of 16 bytes, tile_chunks<DK>() to
// a row; chunk c of row r lies at place c ^ tile_swizzle<DK>(r) of its row. Both
// ways of reading then spread over the 64 banks (256 bytes): four neighbouring
// rows at four chunks (an operand across rows, the transposing read, 32 lanes at
// a time), and 16 neighbouring rows at one chunk (an operand along rows, 16 lanes
// at a time). The shorter rows take the latter in two turns: a swizzle that
// spared that needs twice the addresses, and cost 3% (forward, 64 columns) to 9%
// (keys' gradient) where the vector unit is the bound; of 128 columns a swizzle
// with conflicts in both (a third of the LDS cycles) was 1% slower.
template <int DK>
constexpr int tile_chunks() {
    return DK <= 32 ? 4 : DK <= 64 ? 8 : 16;
}

template <int DK>
constexpr int tile_swizzle(int r) {
    return tile_chunks<DK>() == 4   ? ((r >> 1 & 1) << 1 | (r >> 2 & 1))
           : tile_chunks<DK>() == 8 ? ((r & 3) << 1 | (r >> 2 & 1))
                                    : ((r & 3) << 2 | (r >> 2 & 3));
}

// Byte of chunk c of row r.
template <int DK>
constexpr int tile_byte(int r, int c) {
    return (r * tile_chunks<DK>() + (c ^ tile_swizzle<DK>(r))) * 16;
}

// An operand along rows, 32 rows from row0 (a multiple of 32), columns 16 step +
// 8 h .. of a k step: byte that lane l reads. The lane's own part stands apart:
// chunk 2 step + h differs from h in bits that the swizzle is added to without
// carry, so a step is one exclusive or away.
template <int DK>
constexpr int row_lane_byte(int lane) {
    return tile_byte<DK>(lane % 32, lane / 32);
}
template <int DK>
constexpr int row_operand_byte(int lane_byte, int row0, int step) {
    return (lane_byte ^ 32 * step) + row0 * tile_chunks<DK>() * 16;
}

// An operand across rows: byte that lane l points the transposing read at, for
// four rows row0 + 4 h .. (row0 a multiple of 8) and the 32 columns from 32 block.
// 16 lanes hand over four rows of 16 columns, and get a column's four rows each.
template <int DK>
constexpr int column_lane_byte(int lane) {
    const int r = 4 * (lane / 32) + lane % 16 / 4;
    const int col = 16 * (lane / 16 % 2) + 4 * (lane % 4);
    return tile_byte<DK>(r, col / 8) + col % 8 * 2;
}
template <int DK>
constexpr int column_operand_byte(int lane_byte, int row0, int block) {
    return (lane_byte ^ (64 * block ^ 16 * tile_swizzle<DK>(row0))) +
           row0 * tile_chunks<DK>() * 16;
}

// A tile is filled by loads of 64 chunks, in the order of their places: load i's
// lane l fills place 64 i + l, whose row and chunk are these.
template <int DK>
constexpr int fill_row(int i, int lane) {
    return (64 * i + lane) / tile_chunks<DK>();
}
template <int DK>
constexpr int fill_chunk(int i, int lane) {
    return (64 * i + lane) % tile_chunks<DK>() ^ tile_swizzle<DK>(fill_row<DK>(i, lane));
}

// ------------------------------------------------------------------ runs
// `runs` runs over the heads that share a key head, made even: the next number
// that divides them, where `most` allows it; more runs than heads cut each head
// into parts alike. Uneven runs leave the GPU to the longest (the backward pass
// of 7033 packed tokens, 128 columns, 4 key heads, in four runs or in as many as
// heads: 616 and 531 us with 5 heads each, 664 and 595 with 6, 716 and 682 with 7).
constexpr int even_runs(int runs, int group, int most) {
    if (runs >= group) return runs / group * group;
    int even = runs;
    while (group % even) ++even;
    return even <= most ? even : runs;
}

// ------------------------------------------------------------------ sinks
// The keys' gradients of a windowed sequence: the queries past the window of its key 0
// (tiles of kSinkTokens of them, of each of `group` heads) reach its sinks alone. They
// are work items of their own, over `key_tiles` tiles of kSinkKeys keys in `runs` runs
// each: about `steps` tiles of one head a run, a run having whole heads, or each
// head's being cut into runs / group alike. Where they are one run, or four tiles, the
// sequence's window items go on for them and it has no runs (both gradients of 7033
// packed tokens, window 475, and of 64 sequences of 255, window 50: 196 and 121 us; from
// two tiles on apart 204 and 142, from 13 on 262 and 116).
constexpr int kSinkTokens = 64, kSinkKeys = 128;
constexpr int64_t sink_near(int64_t group, int64_t steps) {
    return steps / group > 4 ? steps / group : 4;
}

struct SinkCut {
    int from, tiles;             // the first query past the window; tiles from it on
    int key_tiles, runs;
};
// near: sink_near(group, steps). Tokens by `group`, keys and the window are below 2^30.
constexpr SinkCut sink_cut(int q_len, int k_len, int window, int sinks, int group, int steps,
                           int near) {
    const int past = window + q_len - k_len;
    const int from = past < 0 ? 0 : past < q_len ? past : q_len;
    const int tiles = (q_len - from + kSinkTokens - 1) / kSinkTokens;
    if (tiles <= near || sinks == 0) return {from, tiles, 0, 0};
    const int keys = sinks < k_len ? sinks : k_len;
    const int runs = (tiles * group + steps - 1) / steps;
    return {from, tiles, (keys + kSinkKeys - 1) / kSinkKeys,
            runs > group ? runs / group * group : runs};
}

// Their sums over all of n_seq sequences, at most, with `sinks` no more than the keys.
// A sequence with runs has more queries than sink_near tiles, and as many keys past
// its window.
struct SinkRoom {
    int64_t key_tiles, runs;     // runs: over the key tiles
};
constexpr SinkRoom sink_room(int64_t q_tokens, int64_t k_tokens, int64_t n_seq, int64_t window,
                             int64_t sinks, int64_t group, int64_t steps) {
    const int64_t far = sink_near(group, steps) * kSinkTokens + 1;
    int64_t with = n_seq;        // sequences that have any
    if (with > q_tokens / far) with = q_tokens / far;
    if (with > k_tokens / (window + far)) with = k_tokens / (window + far);
    if (with == 0) return {0, 0};
    const int64_t each = (sinks + kSinkKeys - 1) / kSinkKeys;
    int64_t key_tiles = with * each;
    if (key_tiles > k_tokens / kSinkKeys + with) key_tiles = k_tokens / kSinkKeys + with;
    return {key_tiles, each * ((q_tokens / kSinkTokens + with) * group / steps) + key_tiles};
}

}  // namespace mg
