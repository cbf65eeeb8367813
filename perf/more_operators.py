"""What the speed of the operators of networks over frames is measured on: heads
normed and turned in one pass, attention with a window, attention over a memory
that streams share, and dropout. They stand next to the operators of
operators.py, in networks that predict splats from the frames of a camera path.

A case is a dict of plain values; ``kind`` names the entry point:

  norm_rotary  norm_rotary() on the queries and keys of one projection
  window       attention() with a window and first tokens that stay visible
  shared       shared_attention(): streams over memories that several share
  dropout      dropout(), onto a residual stream or by itself

``grad`` adds the backward pass to every differentiable input. Token counts are
those of frames in patches of 16 x 16 pixels, the renderer's tile: 64 for
128x128, 256 for 256x256, 475 for 400x300, 2500 for 800x800 and 8160 for
1920x1080.

The plain forms compute in 32 bits, rounded once at the end. ``exact`` restates
each operator in 64 bits from its definition.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-6
BASE = 10000.0


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One new token for each of 16 live streams: frame, row and column as
        # three axes of a head's pairs. Latency.
        dict(name="norm_rotary_streams_16", kind="norm_rotary", tokens=16, heads=16, kv_heads=4,
             dim=64, sections="8,12,12", order="runs", layout="half", dtype="bfloat16",
             weights="float32", reach=4096, grad=False),
        # 21 frames of 400x300, every head its own keys, pairs dealt to the
        # axes in turn.
        dict(name="norm_rotary_frames_9975", kind="norm_rotary", tokens=9975, heads=16,
             kv_heads=16, dim=64, sections="8,12,12", order="turns", layout="interleaved",
             dtype="bfloat16", weights="bfloat16", reach=475, grad=False),
        # Training on four 1920x1080 frames with shared keys.
        dict(name="norm_rotary_views_32640_grad", kind="norm_rotary", tokens=32640, heads=16,
             kv_heads=4, dim=128, sections="16,24,24", order="runs", layout="half",
             dtype="bfloat16", weights="float32", reach=32640, grad=True),
        # One new token for each of 16 streams over memories of every length,
        # of which the last 2000 tokens and the first four are seen.
        dict(name="window_streams_16", kind="window", q_lens=",".join(["1"] * 16),
             k_lens="8160,10000,1,475,2500,64,4056,7313,256,9001,16320,33,5000,2531,1200,6000",
             heads=16, kv_heads=4, dim=64, window=2000, sinks=4, dtype="bfloat16", grad=False),
        # A camera path of 16320 tokens at once, each seeing four frames of
        # 400x300 back and the path's first tokens.
        dict(name="window_path_16320", kind="window", q_lens="16320", k_lens="16320", heads=16,
             kv_heads=4, dim=128, window=1900, sinks=16, dtype="bfloat16", grad=False),
        # A training step on packed paths of every size, with shared key heads.
        dict(name="window_packed_7033_grad", kind="window", q_lens="2500,475,1,2500,256,64,1237",
             k_lens="2500,475,1,2500,256,64,1237", heads=16, kv_heads=4, dim=128, window=475,
             sinks=4, dtype="bfloat16", grad=True),
        # A training step on four paths, the first frame's 64 tokens always seen.
        dict(name="window_paths_6712_grad", kind="window", q_lens="2500,1237,475,2500",
             k_lens="2500,1237,475,2500", heads=12, kv_heads=12, dim=64, window=777, sinks=64,
             dtype="float16", grad=True),
        # Eight candidate cameras, a few tokens each, over one 400x300 scene.
        dict(name="shared_cameras_8", kind="shared", q_lens=",".join(["1"] * 8),
             k_lens="1,2,3,5,8,13,21,34", shared_lens="2375", members="8", heads=16, kv_heads=4,
             dim=64, causal=True, dtype="bfloat16", grad=False),
        # 128 streams over one scene of two 1920x1080 views.
        dict(name="shared_streams_128", kind="shared", q_lens=",".join(["1"] * 128),
             k_lens=",".join(str(1 + 37 * i % 500) for i in range(128)), shared_lens="16320",
             members="128", heads=16, kv_heads=4, dim=128, causal=True, dtype="bfloat16",
             grad=False),
        # Whole frames added over the memories of two scenes, five over one and
        # two over the other, without an order within a frame.
        dict(name="shared_frames_1957", kind="shared", q_lens="475,256,256,475,64,256,175",
             k_lens="475,256,256,475,64,256,175", shared_lens="10000,2500", members="5,2",
             heads=12, kv_heads=12, dim=64, causal=False, dtype="float16", grad=False),
        # A 128x128 preview's tokens in full precision.
        dict(name="dropout_preview_64", kind="dropout", rows=64, width=256, p=0.1,
             dtype="float32", residual="none", grad=False),
        # Training on eight 1920x1080 views: a bfloat16 branch onto the float32
        # residual stream.
        dict(name="dropout_views_65280_grad", kind="dropout", rows=65280, width=1024, p=0.1,
             dtype="bfloat16", residual="float32", grad=True),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_norm_rotary(rng):
    kv = rng.choice((1, 2, 3, 4, 8, 16))
    heads = kv * rng.choice((1, 1, 2, 4, 5))
    dim = rng.choice((32, 64, 64, 80, 96, 128, 128))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    pairs = rng.choice((dim, dim, dim // 2)) // 2
    axes = rng.choice((1, 2, 3, 3))
    parts = [pairs // axes] * axes
    if axes > 1:
        move = rng.randint(0, parts[0] - 1)
        parts[0] -= move
        parts[1] += move
    parts[-1] += pairs - sum(parts)
    # Two fifths of the largest case's elements where they take twice the bytes.
    most = 32640 * 20 * 128 * 2 // (5 * heads * dim)
    return dict(kind="norm_rotary", tokens=_log_between(rng, 1, max(2, min(65280, most))),
                heads=heads, kv_heads=kv, dim=dim, sections=",".join(map(str, parts)),
                order=rng.choice(("runs", "turns")), layout=rng.choice(("half", "interleaved")),
                dtype=dtype, weights=rng.choice(("float32", dtype)),
                reach=_log_between(rng, 50, 131072), grad=rng.random() < 0.5)


def _heads(rng):
    kv = rng.choice((1, 2, 3, 4, 8, 12))
    return kv, kv * rng.choice((1, 1, 2, 4, 5))


def _draw_window(rng):
    kv, heads = _heads(rng)
    shape = rng.choice(("one", "packed", "packed", "chunk", "token"))
    grad = shape in ("one", "packed") and rng.random() < 0.6
    if shape == "token":
        n = _log_between(rng, 1, 48)
        k_lens = [_log_between(rng, 1, 16320) for _ in range(n)]
        q_lens = [1] * n
    elif shape == "chunk":
        n = rng.randint(1, 6)
        q_lens = [_log_between(rng, 2, 700) for _ in range(n)]
        k_lens = [q + _log_between(rng, 1, 10000) for q in q_lens]
    else:
        n = 1 if shape == "one" else rng.randint(2, 12)
        q_lens = [_log_between(rng, 2, 8160 if n == 1 else 2500) for _ in range(n)]
        k_lens = list(q_lens)
    # The plain form holds every score of every pair of tokens.
    most = 2 ** 30 if grad else 2 ** 32
    while len(q_lens) > 1 and sum(q_lens) * sum(k_lens) * heads > most:
        q_lens.pop()
        k_lens.pop()
    while sum(q_lens) * sum(k_lens) * heads > most:
        q_lens, k_lens = [max(1, q_lens[0] // 2)], [max(1, k_lens[0] // 2)]
    return dict(kind="window", q_lens=",".join(map(str, q_lens)),
                k_lens=",".join(map(str, k_lens)), heads=heads, kv_heads=kv,
                dim=rng.choice((32, 64, 64, 80, 96, 128, 128)),
                window=_log_between(rng, 16, 4000), sinks=rng.choice((0, 1, 4, 16, 64, 130)),
                dtype=rng.choice(("bfloat16", "bfloat16", "float16")), grad=grad)


def _draw_shared(rng):
    kv, heads = _heads(rng)
    groups = rng.choice((1, 1, 2, 3))
    members = [_log_between(rng, 1, 128 // groups) for _ in range(groups)]
    n = sum(members)
    one = rng.random() < 0.6
    q_lens = [1 if one else _log_between(rng, 1, max(2, 1800 // n)) for _ in range(n)]
    k_lens = [q + _log_between(rng, 1, 500) - 1 for q in q_lens]
    shared = [_log_between(rng, 64, 16320) for _ in range(groups)]
    while sum(q_lens) * (sum(k_lens) + sum(shared)) * heads > 2 ** 30:
        shared = [max(1, s // 2) for s in shared]
        q_lens = [max(1, q // 2) for q in q_lens]
        k_lens = [max(q, k // 2) for q, k in zip(q_lens, k_lens)]
    return dict(kind="shared", q_lens=",".join(map(str, q_lens)),
                k_lens=",".join(map(str, k_lens)), shared_lens=",".join(map(str, shared)),
                members=",".join(map(str, members)), heads=heads, kv_heads=kv,
                dim=rng.choice((32, 64, 64, 80, 96, 128, 128)),
                causal=one or rng.random() < 0.5,
                dtype=rng.choice(("bfloat16", "bfloat16", "float16")), grad=False)


def _draw_dropout(rng):
    width = rng.choice((_log_between(rng, 64, 8192), 64 * rng.randint(2, 64)))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    rows = _log_between(rng, 1, 65280 * 1024 // width // (2 if dtype == "float32" else 1))
    return dict(kind="dropout", rows=rows, width=width,
                p=rng.choice((0.05, 0.1, 0.25, rng.uniform(0.01, 0.9))), dtype=dtype,
                residual=rng.choice(("none", "float32", dtype)), grad=rng.random() < 0.6)


def draw(rng):
    return rng.choices((_draw_norm_rotary, _draw_window, _draw_shared, _draw_dropout),
                       (3, 4, 3, 2))[0](rng)


# ------------------------------------------------------------------ inputs

def _ints(text):
    return [int(x) for x in text.split(",")]


def _bounds(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _on_gpu(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _leaf(t, grad):
    return t.detach().requires_grad_(grad)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, grad, kind = TYPES[case["dtype"]], case["grad"], case["kind"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    state = {"case": case}
    if kind == "dropout":
        shape = (case["rows"], case["width"])
        # A step's seed lies on the GPU, where a captured step counts it on.
        state.update(x=_leaf(randn(*shape).to(dtype), grad),
                     seed=torch.randint(0, 2 ** 62, (1,), generator=g, device=DEVICE),
                     residual=None)
        if case["residual"] != "none":
            state["residual"] = _leaf(randn(*shape).to(TYPES[case["residual"]]), grad)
        if grad:
            state["dy"] = randn(*shape).to((state["x"] if state["residual"] is None
                                            else state["residual"]).dtype)
        return state

    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "norm_rotary":
        n, sections = case["tokens"], _ints(case["sections"])
        pairs = sum(sections)
        # One projection holds queries, keys and values side by side.
        qkv = (randn(n, heads + 2 * kv, dim) * (0.5 + randn(dim).abs())).to(dtype)
        weights = TYPES[case["weights"]]
        i = torch.arange(pairs, dtype=torch.float64, device=DEVICE)
        state.update(q=_leaf(qkv[:, :heads], grad), k=_leaf(qkv[:, heads:heads + kv], grad),
                     q_weight=_leaf((1.0 + 0.1 * randn(dim)).to(weights), grad),
                     k_weight=_leaf((1.0 + 0.1 * randn(dim)).to(weights), grad),
                     positions=torch.randint(0, case["reach"], (n, len(sections)), generator=g,
                                             device=DEVICE, dtype=torch.int32),
                     frequencies=BASE ** (-i / pairs), sections=tuple(sections))
        if grad:
            state.update(dq=randn(n, heads, dim).to(dtype), dk=randn(n, kv, dim).to(dtype))
        return state

    q_lens, k_lens = _ints(case["q_lens"]), _ints(case["k_lens"])
    if q_lens == k_lens:
        qkv = randn(sum(q_lens), heads + 2 * kv, dim).to(dtype)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q = randn(sum(q_lens), heads, dim).to(dtype)
        # A memory keeps a token's keys and values side by side.
        rows = randn(sum(k_lens), 2, kv, dim).to(dtype)
        k, v = rows[:, 0], rows[:, 1]
    state.update(q=_leaf(q, grad), k=_leaf(k, grad), v=_leaf(v, grad),
                 q_offsets=_on_gpu(_bounds(q_lens)), k_offsets=_on_gpu(_bounds(k_lens)))
    if kind == "shared":
        lens, members = _ints(case["shared_lens"]), _ints(case["members"])
        rows = randn(sum(lens), 2, kv, dim).to(dtype)
        at = _bounds(q_lens)
        state.update(shared_k=rows[:, 0], shared_v=rows[:, 1],
                     shared_offsets=_on_gpu(_bounds(lens)),
                     group_offsets=_on_gpu([at[m] for m in _bounds(members)]))
    if grad:
        state["do"] = randn(sum(q_lens), heads, dim).to(dtype)
    return state


# ------------------------------------------------------------- plain forms

def _axis_of(sections, order):
    """The axis of every pair."""
    if order == "runs":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    out, left = [], list(sections)
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def _plain_turn(x, cos, sin, part, layout):
    head, rest = x[..., :part], x[..., part:]
    if layout == "half":
        a, b = head[..., :part // 2], head[..., part // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_norm_rotary(s):
    case = s["case"]
    dtype, layout, part = s["q"].dtype, case["layout"], 2 * sum(s["sections"])
    axis = torch.tensor(_axis_of(s["sections"], case["order"]), device=DEVICE)
    # Whole turns leave the angle before it is held in 32 bits.
    turns = s["positions"][:, axis].double() * (s["frequencies"] / (2.0 * math.pi))
    angle = ((turns - turns.round()).float() * (2.0 * math.pi))[:, None]
    cos, sin = angle.cos(), angle.sin()
    out, grads = [], []
    with torch.no_grad():
        for n in ("q", "k"):
            x, w = s[n].float(), s[n + "_weight"].float()
            rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
            u = x * rstd
            out.append(_plain_turn(u * w, cos, sin, part, layout).to(dtype))
            if case["grad"]:
                # A rotation's adjoint turns back.
                d = _plain_turn(s["d" + n].float(), cos, -sin, part, layout)
                dw = (d * u).sum((0, 1)).to(s[n + "_weight"].dtype)
                d = d * w
                dx = rstd * (d - u * (d * u).mean(-1, keepdim=True))
                grads.append((dx.to(dtype), dw))
    if case["grad"]:
        out += [grads[0][0], grads[1][0], grads[0][1], grads[1][1]]
    return out


def _sequence_of(offsets, n):
    return torch.bucketize(torch.arange(n, device=DEVICE), offsets[1:], right=True)


def _plain_softmax(scores, allowed):
    p = scores.masked_fill_(~allowed, -math.inf)
    top = p.amax(2, keepdim=True)
    p = p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    return p.div_(p.sum(2, keepdim=True).clamp_min_(1e-38))


def _plain_in_order(s, nq, nk):
    """For causal sequences: (nq, nk) whether a key is the query's own sequence's
    and stands at or before it, the key each query stands at, and the first key
    of its sequence, all by key number."""
    sq, sk = _sequence_of(s["q_offsets"], nq), _sequence_of(s["k_offsets"], nk)
    at_k = torch.arange(nk, device=DEVICE)
    # A sequence's last query stands at its last key.
    stands = torch.arange(nq, device=DEVICE) - (s["q_offsets"][1:] - s["k_offsets"][1:])[sq]
    allowed = (sq[:, None] == sk[None, :]) & (at_k[None, :] <= stands[:, None])
    return allowed, stands, s["k_offsets"][:-1][sq]


def _plain_window(s):
    case = s["case"]
    dtype, group = s["q"].dtype, case["heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    with torch.no_grad():
        q = s["q"].float().transpose(0, 1).contiguous()
        k = s["k"].float().transpose(0, 1).repeat_interleave(group, 0)
        v = s["v"].float().transpose(0, 1).repeat_interleave(group, 0)
        allowed, stands, first = _plain_in_order(s, q.shape[1], k.shape[1])
        at_k = torch.arange(k.shape[1], device=DEVICE)
        allowed &= ((at_k[None, :] > stands[:, None] - case["window"])
                    | (at_k[None, :] < first[:, None] + case["sinks"]))
        p = _plain_softmax(torch.bmm(q, k.transpose(1, 2)).mul_(scale), allowed)
        o = torch.bmm(p, v)
        out = [o.transpose(0, 1).to(dtype)]
        if case["grad"]:
            do = s["do"].float().transpose(0, 1).contiguous()
            dv = torch.bmm(p.transpose(1, 2), do)
            dp = torch.bmm(do, v.transpose(1, 2))
            ds = dp.sub_((do * o).sum(2, keepdim=True)).mul_(p).mul_(scale)
            dq = torch.bmm(ds, k)
            dk = torch.bmm(ds.transpose(1, 2), q)
            shared = (case["kv_heads"], group, *dk.shape[1:])
            out += [dq.transpose(0, 1).to(dtype),
                    dk.reshape(shared).sum(1).transpose(0, 1).to(dtype),
                    dv.reshape(shared).sum(1).transpose(0, 1).to(dtype)]
    return [t.contiguous() for t in out]


def _plain_shared(s):
    case = s["case"]
    dtype, group = s["q"].dtype, case["heads"] // case["kv_heads"]
    with torch.no_grad():
        q = s["q"].float().transpose(0, 1).contiguous()
        k, v = (torch.cat([s["shared_" + n], s[n]]).float().transpose(0, 1)
                .repeat_interleave(group, 0) for n in ("k", "v"))
        nq, ns, nk = q.shape[1], s["shared_k"].shape[0], s["k"].shape[0]
        of_q = _sequence_of(s["group_offsets"], nq)
        shared = of_q[:, None] == _sequence_of(s["shared_offsets"], ns)[None, :]
        if case["causal"]:
            alone = _plain_in_order(s, nq, nk)[0]
        else:
            alone = (_sequence_of(s["q_offsets"], nq)[:, None]
                     == _sequence_of(s["k_offsets"], nk)[None, :])
        scores = torch.bmm(q, k.transpose(1, 2)).mul_(case["dim"] ** -0.5)
        p = _plain_softmax(scores, torch.cat([shared, alone], 1))
        return [torch.bmm(p, v).transpose(0, 1).to(dtype).contiguous()]


# Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as
# 1, 2, 3; 2011).
PHILOX_MUL = (0xD2511F53, 0xCD9E8D57)
PHILOX_KEY = (0x9E3779B9, 0xBB67AE85)
LOW = 0xFFFFFFFF


def _plain_draws(seed, n):
    """n numbers of 16 bits: eight of each counter."""
    c0 = torch.arange((n + 7) // 8, device=DEVICE)
    c = [c0 & LOW, c0 >> 32, torch.zeros_like(c0), torch.zeros_like(c0)]
    key = [seed & LOW, (seed >> 32) & LOW]

    def product(a, m):
        # The high half by parts of 16 bits: a product of 64 has no room.
        high = (a * (m >> 16) + ((a * (m & 0xFFFF)) >> 16)) >> 16
        return high, (a * m) & LOW

    for _ in range(10):
        (h0, l0), (h1, l1) = product(c[0], PHILOX_MUL[0]), product(c[2], PHILOX_MUL[1])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(k + step) & LOW for k, step in zip(key, PHILOX_KEY)]
    words = torch.stack(c, 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).flatten()[:n]


def _dropped(p):
    """Draws below this drop their element: p in steps of 2^-16."""
    return int(round(p * 65536))


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    least = _dropped(case["p"])
    scale = 65536.0 / (65536 - least)
    with torch.no_grad():
        keep = (_plain_draws(s["seed"], x.numel()) >= least).view(x.shape)
        y = (x.float() * scale).masked_fill(~keep, 0.0)
        if s["residual"] is None:
            out = [y.to(x.dtype)]
        else:
            out = [(s["residual"].float() + y).to(s["residual"].dtype)]
        if case["grad"]:
            out.append((s["dy"].float() * scale).masked_fill(~keep, 0.0).to(x.dtype))
            if s["residual"] is not None:
                out.append(s["dy"])
    return out


# --------------------------------------------------------------------- run

def _own_run(s):
    import metal_gauss_amd as mg

    case = s["case"]
    kind, grad = case["kind"], case["grad"]
    if kind == "dropout":
        y = mg.dropout(s["x"], case["p"], s["seed"], residual=s["residual"])
        if not grad:
            return [y]
        leaves = [s["x"]] + ([] if s["residual"] is None else [s["residual"]])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if kind == "norm_rotary":
        leaves = [s["q"], s["k"], s["q_weight"], s["k_weight"]]
        q, k = mg.norm_rotary(*leaves, s["positions"], s["frequencies"], eps=EPS,
                              layout=case["layout"], sections=s["sections"], order=case["order"])
        if not grad:
            return [q, k]
        return [q.detach(), k.detach(),
                *torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))]
    if kind == "shared":
        return [mg.shared_attention(s["q"], s["k"], s["v"], s["shared_k"], s["shared_v"],
                                    s["q_offsets"], s["k_offsets"], s["group_offsets"],
                                    s["shared_offsets"], causal=case["causal"])]
    o = mg.attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], causal=True,
                     window=case["window"], sinks=case["sinks"])
    if not grad:
        return [o]
    return [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]


def run(state):
    if own:
        return _own_run(state)
    return {"norm_rotary": _plain_norm_rotary, "window": _plain_window, "shared": _plain_shared,
            "dropout": _plain_dropout}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- work

def _window_pairs(case):
    """(query-key pairs seen, keys that some query sees), over all sequences."""
    pairs = keys = 0
    for nq, nk in zip(_ints(case["q_lens"]), _ints(case["k_lens"])):
        first = max(0, nk - nq)                       # the first query that sees any
        p = np.arange(first, nk, dtype=np.int64)
        pairs += int((np.minimum(p + 1, case["window"])
                      + np.minimum(case["sinks"],
                                   np.maximum(0, p + 1 - case["window"]))).sum())
        low = max(0, first - case["window"] + 1)
        keys += nk - low + min(case["sinks"], low)
    return pairs, keys


def _shared_pairs(case):
    q_lens, k_lens = _ints(case["q_lens"]), _ints(case["k_lens"])
    total = at = 0
    for n, m in zip(_ints(case["shared_lens"]), _ints(case["members"])):
        total += n * sum(q_lens[at:at + m])
        at += m
    for nq, nk in zip(q_lens, k_lens):
        n = min(nq, nk)
        total += n * (nk - n + 1 + nk) // 2 if case["causal"] else nq * nk
    return total


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "dropout":
        n = case["rows"] * case["width"]
        r = {"none": 0, "float32": 4}.get(case["residual"], size)
        result = r or size
        moved = size + r + result                        # x, residual, y
        if case["grad"]:
            moved += result + size                       # dy, dx; the residual's is dy itself
        return {"bytes": n * moved, "flops": (6 if case["grad"] else 3) * n}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "norm_rotary":
        n = case["tokens"] * (heads + kv) * dim
        weights = 2 * dim * (4 if case["weights"] == "float32" else 2)
        angles = 4 * case["tokens"] * len(_ints(case["sections"]))
        arrays = 4 if case["grad"] else 2                # x, y; dy, dx
        return {"bytes": arrays * n * size + angles + weights * (2 if case["grad"] else 1),
                "flops": (22 if case["grad"] else 8) * n}
    q_lens, k_lens = _ints(case["q_lens"]), _ints(case["k_lens"])
    nq = sum(q_lens) * heads * dim
    if case["kind"] == "shared":
        keys = (sum(k_lens) + sum(_ints(case["shared_lens"]))) * kv * dim
        return {"bytes": (2 * nq + 2 * keys) * size + 16 * (len(q_lens) + 1),
                "flops": 4 * _shared_pairs(case) * heads * dim}
    pairs, keys = _window_pairs(case)
    moved = 2 * nq + 2 * keys * kv * dim                 # q, o, the k and v that are seen
    if case["grad"]:
        moved += 2 * nq + 2 * sum(k_lens) * kv * dim     # do, dq, dk, dv
    products = 7 if case["grad"] else 2                  # two forward, five backward
    return {"bytes": moved * size + 8 * (len(q_lens) + 1),
            "flops": 2 * products * pairs * heads * dim}


# ------------------------------------------------------------------- exact

def _exact_norm_rotary(s, case):
    axes, sections = len(s["sections"]), s["sections"]
    if case["order"] == "runs":
        axis = np.repeat(np.arange(axes), sections)
    else:
        # The n-th pair of an axis stands before the next axis's n-th.
        axis = np.array(sorted((n, a) for a in range(axes) for n in range(sections[a])))[:, 1]
    pairs = len(axis)
    theta = torch.pow(torch.tensor(BASE, dtype=torch.float64, device=DEVICE),
                      -torch.arange(pairs, device=DEVICE).double() / pairs)
    where = s["positions"].double()[:, torch.as_tensor(axis, device=DEVICE)]
    z = torch.polar(torch.ones_like(where), where * theta)[:, None]
    if case["layout"] == "half":
        first, second = slice(0, pairs), slice(pairs, 2 * pairs)
    else:
        first, second = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)

    def turn(x, z):
        y = x.clone()
        w = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    results, dxs, dws = [], [], []
    for n in ("q", "k"):
        x, w = s[n].detach().double(), s[n + "_weight"].detach().double()
        size = ((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
        results.append(turn(x / size * w, z))
        if case["grad"]:
            back = turn(s["d" + n].double(), z.conj())
            dws.append((back * x / size).sum(0).sum(0))
            # The Jacobian (I - x x^T / (n size^2)) / size, applied to a head.
            d = back * w
            along = (d * x).sum(-1, keepdim=True) / (x.shape[-1] * size * size)
            dxs.append((d - x * along) / size)
    return results + dxs + dws


def _exact_head(q, k, v, seen, scale, do=None):
    """One head over a block of queries and the keys that they may see."""
    score = (q @ k.T * scale).masked_fill(~seen, -1e300)
    p = torch.softmax(score, 1) * seen.any(1, keepdim=True)
    o = p @ v
    if do is None:
        return o, None, None, None
    dp = do @ v.T
    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
    return o, ds @ k, ds.T @ q, p.T @ do


def _exact_window(s, case):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    do = s["do"].double() if case["grad"] else None
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    window, sinks, block = case["window"], case["sinks"], 1024
    o, dq, dk, dv = (torch.zeros_like(t, memory_format=torch.contiguous_format)
                     for t in (q, q, k, v))
    q0 = k0 = 0
    for nq, nk in zip(_ints(case["q_lens"]), _ints(case["k_lens"])):
        for r0 in range(0, nq, block):
            r1 = min(nq, r0 + block)
            at = torch.arange(r0, r1, device=DEVICE) + nk - nq
            low, high = max(0, r0 + nk - nq - window + 1), max(0, r1 + nk - nq)
            keys = torch.cat([torch.arange(0, min(sinks, low), device=DEVICE),
                              torch.arange(low, max(low, high), device=DEVICE)])
            if keys.numel() == 0:
                continue
            far = at[:, None] - keys[None, :]
            seen = (far >= 0) & ((far < window) | (keys[None, :] < sinks))
            rows, cols = slice(q0 + r0, q0 + r1), keys + k0
            for h in range(case["heads"]):
                kh = h // group
                got = _exact_head(q[rows, h], k[cols, kh], v[cols, kh], seen, scale,
                                  None if do is None else do[rows, h])
                o[rows, h] = got[0]
                if do is not None:
                    dq[rows, h] = got[1]
                    dk[cols, kh] += got[2]
                    dv[cols, kh] += got[3]
        q0, k0 = q0 + nq, k0 + nk
    return [o, dq, dk, dv] if case["grad"] else [o]


def _exact_shared(s, case):
    q, k, v, sk, sv = (s[n].detach().double() for n in ("q", "k", "v", "shared_k", "shared_v"))
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    o = torch.zeros_like(q, memory_format=torch.contiguous_format)
    q_lens, k_lens = _ints(case["q_lens"]), _ints(case["k_lens"])
    q0 = k0 = s0 = at = 0
    for ns, m in zip(_ints(case["shared_lens"]), _ints(case["members"])):
        for nq, nk in zip(q_lens[at:at + m], k_lens[at:at + m]):
            seen = torch.ones(nq, ns + nk, dtype=torch.bool, device=DEVICE)
            if case["causal"]:
                seen[:, ns:] = seen[:, ns:].tril(nk - nq)
            for h in range(case["heads"]):
                kh = h // group
                keys = torch.cat([sk[s0:s0 + ns, kh], k[k0:k0 + nk, kh]])
                values = torch.cat([sv[s0:s0 + ns, kh], v[k0:k0 + nk, kh]])
                o[q0:q0 + nq, h] = _exact_head(q[q0:q0 + nq, h], keys, values, seen, scale)[0]
            q0, k0 = q0 + nq, k0 + nk
        s0, at = s0 + ns, at + m
    return [o]


def _exact_keep(seed, n, least):
    """Truth values of n elements, by the generator's definition in 64 unsigned bits."""
    low, half = np.uint64(LOW), np.uint64(32)
    x = np.zeros((4, (n + 7) // 8), np.uint64)
    x[0] = np.arange(x.shape[1], dtype=np.uint64)
    x[1], x[0] = x[0] >> half, x[0] & low
    k0, k1 = seed & LOW, seed >> 32 & LOW
    for r in range(10):
        a, b = x[0] * np.uint64(PHILOX_MUL[0]), x[2] * np.uint64(PHILOX_MUL[1])
        x = np.stack([(b >> half) ^ x[1] ^ np.uint64((k0 + r * PHILOX_KEY[0]) & LOW), b & low,
                      (a >> half) ^ x[3] ^ np.uint64((k1 + r * PHILOX_KEY[1]) & LOW), a & low])
    halves = np.ascontiguousarray(x.T.astype("<u4")).view("<u2").reshape(-1)
    return halves[:n] >= least


def _exact_dropout(s, case):
    x = s["x"].detach().double()
    least = _dropped(case["p"])
    keep = _exact_keep(int(s["seed"]), x.numel(), least)
    gain = torch.from_numpy(keep).to(DEVICE).view(x.shape).double() * (65536 / (65536 - least))
    y = x * gain
    out = [y if s["residual"] is None else y + s["residual"].detach().double()]
    if case["grad"]:
        out.append(s["dy"].double() * gain)
        if s["residual"] is not None:
            out.append(s["dy"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rotary": _exact_norm_rotary, "window": _exact_window, "shared": _exact_shared,
            "dropout": _exact_dropout}[case["kind"]](s, case)
