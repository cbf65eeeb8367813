"""Room and work items of the gradients of attention's first keys that stay visible, on
the CPU: what the device counts, sequence by sequence, against the bound that the
host reserves by, and the room itself for packs of many sequences."""

from __future__ import annotations

import pytest

from test_kernel_indexes import _run

# Random packs: sequences of a few lengths about the ones at which they get items of
# their own, and others; `steps` as few and as many as a plan may have.
PACKS = """
    uint64_t seed = %d;
    const auto below = [&](int64_t n) {
        seed = seed * 6364136223846793005ull + 1442695040888963407ull;
        return (int64_t)((seed >> 33) %% (uint64_t)n);
    };
    for (int pack = 0; pack < 4000; ++pack) {
        const int n = 1 + (int)below(pack %% 3 ? 12 : 300), group = 1 + (int)below(9);
        const int window = 1 + (int)below(pack %% 2 ? 900 : 20), steps = 4 + (int)below(pack %% 5 ? 60 : 900);
        const int64_t far = sink_near(group, steps) * kSinkTokens;
        int64_t q_sum = 0, k_sum = 0;
        int q[300], k[300];
        for (int s = 0; s < n; ++s) {
            const int kind = (int)below(4);
            q[s] = (int)(kind == 0 ? below(2000) : kind == 1 ? far + below(3) : kind == 2 ? below(70)
                                                 : window + far + below(3));
            k[s] = (int)(below(3) == 0 ? below(3000) : below(2) ? q[s] : window + far + below(3));
            q_sum += q[s], k_sum += k[s];
        }
        if (k_sum == 0) continue;
        int64_t sinks = 1 + below(pack %% 7 == 0 ? 4000 : 300);
        if (sinks > k_sum) sinks = k_sum;
        int64_t tiles = 0, runs = 0, most = 0;
        for (int s = 0; s < n; ++s) {
            const SinkCut c = sink_cut(q[s], k[s], window, (int)sinks, group, steps,
                                       (int)sink_near(group, steps));
            tiles += c.key_tiles, runs += (int64_t)c.key_tiles * c.runs;
            if (c.runs > most) most = c.runs;
            if (c.runs > 0 && c.runs != group && c.runs > group && c.runs %% group) return 1;
            // Either items of its own for all tiles, or none.
            if ((c.runs == 0) != (c.key_tiles == 0)) return 2;
            if (c.runs == 0 && c.tiles > sink_near(group, steps)) return 3;
            // No query before `from` is past the window of key 0, all later ones are.
            const int64_t ahead = k[s] - q[s];
            if (c.from > 0 && c.from - 1 + ahead - window >= 0) return 4;
            if (c.from < q[s] && c.from + ahead - window < 0) return 5;
        }
        const SinkRoom room = sink_room(q_sum, k_sum, n, window, sinks, group, steps);
        std::printf("%%lld %%lld %%lld %%lld %%lld\\n", (long long)tiles, (long long)room.key_tiles,
                    (long long)runs, (long long)room.runs, (long long)most);
    }"""


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_the_devices_counts_are_within_the_hosts_room(tmp_path, seed):
    rows = _run(tmp_path, "attention_tiles.h", PACKS % seed)
    assert len(rows) > 3000
    assert sum(tiles > 0 for tiles, *_ in rows) > 1000 and sum(tiles == 0 for tiles, *_ in rows) > 100
    for tiles, most_tiles, runs, most_runs, _ in rows:
        assert tiles <= most_tiles and runs <= most_runs
    # Tight enough to hold something: some packs fill what is reserved.
    assert any(tiles == most for tiles, most, *_ in rows if tiles)


def backward_room(tokens, heads, kv, dim, sequences, window, sinks):
    from metal_gauss_amd import _lib

    query = _lib.open_library().mg_attention_window_backward_workspace_bytes
    return query(tokens, tokens, heads, kv, dim, sequences, window, sinks)


@pytest.mark.parametrize("tokens,heads,kv,dim,sequences,window,sinks", [
    (65280, 16, 4, 128, 1024, 475, 4), (65280, 16, 4, 128, 1024, 475, 130),
    (65280, 16, 4, 128, 4096, 475, 130), (65280, 32, 32, 128, 1024, 475, 130),
    (65280, 32, 32, 64, 4096, 475, 1000), (16320, 16, 16, 128, 64, 475, 16320),
    (65280, 16, 4, 128, 4096, 1, 130), (65280, 32, 32, 128, 250, 1, 130),
    (65280, 16, 4, 128, 1, 16, 65279), (65280, 32, 1, 128, 65280, 1, 1)])
def test_room_of_sinks_does_not_go_by_the_sequences(tokens, heads, kv, dim, sequences, window,
                                                    sinks):
    none, some = (backward_room(tokens, heads, kv, dim, sequences, window, s) for s in (0, sinks))
    assert none <= some <= none + (256 << 20)


@pytest.mark.parametrize("sinks", [1, 130, 1000])
def test_sequences_within_the_window_take_no_room_for_sinks(sinks):
    """One query past the window is no item of its own."""
    assert backward_room(300, 16, 4, 128, 1, 299, sinks) == backward_room(300, 16, 4, 128, 1, 299, 0)


def backward_call(tokens, heads, kv, dim, sequences, window, sinks, dtype=1):
    """A call whose room is too small: refused before any launch."""
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    rows = (heads * dim, dim), (kv * dim, dim)
    rc = lib.mg_attention_window_backward(
        dtype, tokens, tokens, heads, kv, dim, 16, *rows[0], 16, *rows[1], 16, *rows[1], 16, 16,
        sequences, window, sinks, 1.0, 16, None, 16, 16, *rows[0], 16, 16, 16, 16, 8, None)
    assert rc == 1
    return lib.mg_last_error().decode()


@pytest.mark.parametrize("tokens,heads,kv,dim,sequences,window,sinks", [
    (32768, 32, 32, 64, 2048, 475, 130), (32768, 32, 32, 64, 512, 475, 1000),
    (16320, 32, 32, 32, 1024, 475, 500), (65280, 32, 32, 128, 4096, 1, 130),
    (90000, 512, 512, 8, 350, 1, 300), (65280, 16, 1, 128, 1, 16, 65279),
    (262144, 32, 4, 128, 8192, 30, 1000)])
def test_packs_that_forward_takes_are_taken_backward(tokens, heads, kv, dim, sequences, window,
                                                     sinks):
    for dtype in (1, 2):
        message = backward_call(tokens, heads, kv, dim, sequences, window, sinks, dtype)
        assert "workspace of 8 bytes" in message


def test_more_items_than_a_launch_has_are_refused():
    assert "too many work items" in backward_call(1 << 25, 2, 2, 64, 1 << 25, 5, 1)
