"""What the speed of the token operators is measured on: rotary positions,
layer norm and attention over packed sequences, the three that a network
predicting or refining splats from image patches is built of, next to matrix
products.

A case is a dict of plain values; ``kind`` names the entry point:

  rotary     rotary() on the queries and keys of one projection
  norm       layer_norm()
  attention  attention() on packed sequences

``grad`` adds the backward pass to every differentiable input. Token counts are
those of frames in patches of 16 x 16 pixels, the renderer's tile: 64 for
128x128, 256 for 256x256, 475 for 400x300, 2500 for 800x800, 4056 for 1237x823
and 8160 for 1920x1080.

The plain forms compute in 32 bits, rounded once at the end. ``exact`` restates
each operator in 64 bits from its definition, one sequence and head at a time.
"""

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5
BASE = 10000.0


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One new token for each of 16 live streams (a camera path rendered
        # frame by frame), far into their contexts: latency.
        dict(name="rotary_streams_16", kind="rotary", tokens=16, heads=16, kv_heads=4, dim=64,
             part=64, axes=1, layout="half", dtype="bfloat16", reach=131072, grad=False),
        # Four 800x800 views, the patch's column and row as two axes.
        dict(name="rotary_scene_10000", kind="rotary", tokens=10000, heads=16, kv_heads=16,
             dim=64, part=64, axes=2, layout="interleaved", dtype="bfloat16", reach=50,
             grad=False),
        # Training on four 1920x1080 views, half of each head rotated.
        dict(name="rotary_part_32640_grad", kind="rotary", tokens=32640, heads=16, kv_heads=4,
             dim=128, part=64, axes=1, layout="half", dtype="float32", reach=32640, grad=True),
        # A 128x128 preview through a narrow network in full precision.
        dict(name="norm_preview_64", kind="norm", rows=64, width=256, dtype="float32",
             weights="float32", grad=False),
        # Training on an 800x800 view with 31 extra tokens, an odd width.
        dict(name="norm_odd_2531_grad", kind="norm", rows=2531, width=771, dtype="float32",
             weights="float32", grad=True),
        # Training on eight 1920x1080 views, weights kept in full precision.
        dict(name="norm_views_65280_grad", kind="norm", rows=65280, width=1024,
             dtype="bfloat16", weights="float32", grad=True),
        # One new token for each of 16 streams over memories of every length,
        # one of them still empty but for the token itself.
        dict(name="attend_streams_16", kind="attention", q_lens=",".join(["1"] * 16),
             k_lens="8160,10000,1,475,2500,64,4056,7313,256,9001,16320,33,5000,2531,1200,6000",
             heads=16, kv_heads=4, dim=64, dtype="bfloat16", causal=True, grad=False),
        # Four 800x800 views attending to one another: a whole scene.
        dict(name="attend_scene_10000", kind="attention", q_lens="10000", k_lens="10000",
             heads=16, kv_heads=16, dim=64, dtype="bfloat16", causal=False, grad=False),
        # New views' tokens over the memories of four scenes.
        dict(name="attend_chunk_796", kind="attention", q_lens="475,256,1,64",
             k_lens="16320,2500,8160,64", heads=16, kv_heads=4, dim=128, dtype="float16",
             causal=True, grad=False),
        # A training step on packed frames of every size, in order, with
        # shared key heads.
        dict(name="attend_packed_7033_grad", kind="attention",
             q_lens="2500,475,1,2500,256,64,1237", k_lens="2500,475,1,2500,256,64,1237",
             heads=16, kv_heads=4, dim=128, dtype="bfloat16", causal=True, grad=True),
        # A training step on four scenes without an order.
        dict(name="attend_views_6712_grad", kind="attention", q_lens="2500,1237,475,2500",
             k_lens="2500,1237,475,2500", heads=12, kv_heads=12, dim=64, dtype="float16",
             causal=False, grad=True),
        # Two 1920x1080 views as one ordered prompt.
        dict(name="attend_prompt_16320", kind="attention", q_lens="16320", k_lens="16320",
             heads=16, kv_heads=4, dim=128, dtype="bfloat16", causal=True, grad=False),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rotary(rng):
    kv = rng.choice((1, 2, 3, 4, 8, 16))
    heads = kv * rng.choice((1, 1, 2, 4, 5))
    dim = rng.choice((32, 64, 64, 80, 96, 128, 128))
    axes = rng.choice((1, 1, 2))
    part = rng.choice((dim, dim, dim // 2))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    most = 32640 * 20 * 128 // (heads * dim)
    return dict(kind="rotary", tokens=_log_between(rng, 1, max(2, min(65280, most // 2))),
                heads=heads, kv_heads=kv, dim=dim, part=part, axes=axes,
                layout=rng.choice(("half", "interleaved")), dtype=dtype,
                reach=_log_between(rng, 50, 131072), grad=rng.random() < 0.4)


def _draw_norm(rng):
    width = rng.choice((_log_between(rng, 64, 8192), 64 * rng.randint(2, 64)))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    rows = _log_between(rng, 1, 65280 * 1024 // width // (4 if dtype == "float32" else 2))
    return dict(kind="norm", rows=rows, width=width, dtype=dtype,
                weights=rng.choice(("float32", dtype)), grad=rng.random() < 0.6)


def _draw_attention(rng):
    dim = rng.choice((32, 64, 64, 80, 96, 128, 128))
    kv = rng.choice((1, 2, 3, 4, 8, 12))
    heads = kv * rng.choice((1, 1, 2, 4, 5))
    shape = rng.choice(("one", "packed", "packed", "chunk", "token"))
    grad = shape in ("one", "packed") and rng.random() < 0.5
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
        q_lens = [_log_between(rng, 1, 8160 if n == 1 else 2500) for _ in range(n)]
        k_lens = list(q_lens)
    case = dict(kind="attention", q_lens="", k_lens="", heads=heads, kv_heads=kv, dim=dim,
                dtype=rng.choice(("bfloat16", "bfloat16", "float16")),
                causal=shape in ("token", "chunk") or rng.random() < 0.6, grad=grad)
    # The plain form holds every score of every pair of tokens.
    while len(q_lens) > 1 and sum(q_lens) * sum(k_lens) * heads > (2 ** 30 if grad else 2 ** 32):
        q_lens.pop()
        k_lens.pop()
    while sum(q_lens) * sum(k_lens) * heads > (2 ** 30 if grad else 2 ** 32):
        q_lens, k_lens = [max(1, q_lens[0] // 2)], [max(1, k_lens[0] // 2)]
    case["q_lens"] = ",".join(map(str, q_lens))
    case["k_lens"] = ",".join(map(str, k_lens))
    return case


def draw(rng):
    return rng.choices((_draw_rotary, _draw_norm, _draw_attention), (2, 2, 4))[0](rng)


# ------------------------------------------------------------------ inputs

def _lens(case):
    return ([int(x) for x in case["q_lens"].split(",")],
            [int(x) for x in case["k_lens"].split(",")])


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _axis_frequencies(case):
    """Radians per position of every pair: BASE^(-i / pairs of an axis)."""
    pairs = case["part"] // 2
    per = pairs // case["axes"]
    return torch.tensor([BASE ** (-(i % per) / per) for i in range(pairs)], dtype=torch.float64)


def _leaf(t, grad):
    return t.detach().requires_grad_(grad)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    grad = case["grad"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    state = {"case": case}
    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        # The residual stream: channels with their own size and offset.
        x = randn(rows, width) * (0.5 + randn(width).abs()) + 0.5 * randn(width)
        weights = TYPES[case["weights"]]
        state.update(x=_leaf(x.to(dtype), grad),
                     weight=_leaf((1.0 + 0.1 * randn(width)).to(weights), grad),
                     bias=_leaf((0.1 * randn(width)).to(weights), grad))
        if grad:
            state["dy"] = randn(rows, width).to(dtype)
        return state

    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rotary":
        n = case["tokens"]
        # One projection holds queries, keys and values side by side.
        qkv = randn(n, heads + 2 * kv, dim).to(dtype)
        shape = (n,) if case["axes"] == 1 else (n, case["axes"])
        positions = torch.randint(0, case["reach"], shape, generator=g, device=DEVICE,
                                  dtype=torch.int32)
        state.update(q=_leaf(qkv[:, :heads], grad), k=_leaf(qkv[:, heads:heads + kv], grad),
                     positions=positions, frequencies=_axis_frequencies(case).to(DEVICE))
        if grad:
            state.update(dq=randn(n, heads, dim).to(dtype), dk=randn(n, kv, dim).to(dtype))
        return state

    q_lens, k_lens = _lens(case)
    if q_lens == k_lens:
        qkv = randn(sum(q_lens), heads + 2 * kv, dim).to(dtype)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q = randn(sum(q_lens), heads, dim).to(dtype)
        # A memory keeps a token's keys and values side by side.
        kv_rows = randn(sum(k_lens), 2, kv, dim).to(dtype)
        k, v = kv_rows[:, 0], kv_rows[:, 1]
    state.update(q=_leaf(q, grad), k=_leaf(k, grad), v=_leaf(v, grad),
                 q_offsets=torch.tensor(_offsets(q_lens), dtype=torch.int32, device=DEVICE),
                 k_offsets=torch.tensor(_offsets(k_lens), dtype=torch.int32, device=DEVICE))
    if grad:
        state["do"] = randn(sum(q_lens), heads, dim).to(dtype)
    return state


# ------------------------------------------------------------- plain forms

def _plain_rotate(x, cos, sin, part, layout):
    x = x.float()
    head, rest = x[..., :part], x[..., part:]
    if layout == "half":
        a, b = head[..., :part // 2], head[..., part // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    case = s["case"]
    part, axes, layout = case["part"], case["axes"], case["layout"]
    dtype = s["q"].dtype
    positions = s["positions"].reshape(-1, axes).repeat_interleave(part // 2 // axes, 1)
    # Whole turns leave the angle before it is held in 32 bits: at a position
    # of 100000 the product itself has only three decimals left there.
    turns = positions.double() * (s["frequencies"] / (2.0 * math.pi))
    angle = ((turns - turns.round()).float() * (2.0 * math.pi))[:, None]
    cos, sin = angle.cos(), angle.sin()
    with torch.no_grad():
        out = [_plain_rotate(s[n], cos, sin, part, layout).to(dtype) for n in ("q", "k")]
        if case["grad"]:
            # A rotation's adjoint turns back.
            out += [_plain_rotate(s[n], cos, -sin, part, layout).to(dtype) for n in ("dq", "dk")]
    return out


def _plain_norm(s):
    with torch.no_grad():
        x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
        centred = x - x.mean(1, keepdim=True)
        rstd = (centred.square().mean(1, keepdim=True) + EPS).rsqrt()
        xhat = centred * rstd
        out = [(xhat * w + b).to(s["x"].dtype)]
        if s["case"]["grad"]:
            dy = s["dy"].float()
            dxhat = dy * w
            dx = rstd * (dxhat - dxhat.mean(1, keepdim=True)
                         - xhat * (dxhat * xhat).mean(1, keepdim=True))
            out += [dx.to(s["x"].dtype), (dy * xhat).sum(0).to(s["weight"].dtype),
                    dy.sum(0).to(s["bias"].dtype)]
    return out


def _plain_allowed(q_offsets, k_offsets, nq, nk, causal):
    """(nq, nk) truth values: whether a query sees a key."""
    at_q = torch.arange(nq, device=DEVICE)
    at_k = torch.arange(nk, device=DEVICE)
    sq = torch.bucketize(at_q, q_offsets[1:], right=True)
    sk = torch.bucketize(at_k, k_offsets[1:], right=True)
    allowed = sq[:, None] == sk[None, :]
    if causal:
        # A sequence's last query stands at its last key.
        ahead = (q_offsets[1:] - k_offsets[1:])[sq]
        allowed &= (at_k[None, :] <= (at_q - ahead)[:, None])
    return allowed


def _plain_attention(s):
    case = s["case"]
    dtype, group = s["q"].dtype, case["heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    with torch.no_grad():
        q = s["q"].float().transpose(0, 1).contiguous()
        k = s["k"].float().transpose(0, 1).repeat_interleave(group, 0)
        v = s["v"].float().transpose(0, 1).repeat_interleave(group, 0)
        allowed = _plain_allowed(s["q_offsets"], s["k_offsets"], q.shape[1], k.shape[1],
                                 case["causal"])
        p = torch.bmm(q, k.transpose(1, 2)).mul_(scale).masked_fill_(~allowed, -math.inf)
        top = p.amax(2, keepdim=True)
        p = p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
        p = p.div_(p.sum(2, keepdim=True).clamp_min_(1e-38))
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


# --------------------------------------------------------------------- run

def _own_run(s):
    import metal_gauss_amd as mg

    case = s["case"]
    if case["kind"] == "norm":
        y = mg.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        if not case["grad"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])]
    if case["kind"] == "rotary":
        q, k = mg.rotary(s["q"], s["k"], s["positions"], s["frequencies"],
                         layout=case["layout"])
        if not case["grad"]:
            return [q, k]
        return [q.detach(), k.detach(),
                *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
    o = mg.attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"],
                     causal=case["causal"])
    if not case["grad"]:
        return [o]
    return [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]


def run(state):
    if own:
        return _own_run(state)
    return {"rotary": _plain_rotary, "norm": _plain_norm,
            "attention": _plain_attention}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- work

def _pairs(case):
    """Query-key pairs that the mask leaves, over all sequences."""
    total = 0
    for nq, nk in zip(*_lens(case)):
        if not case["causal"]:
            total += nq * nk
            continue
        # Query i sees keys 0 .. i + nk - nq: those queries that see any.
        n = min(nq, nk)
        total += n * (nk - n + 1 + nk) // 2
    return total


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "norm":
        n, weights = case["rows"] * case["width"], 4 if case["weights"] == "float32" else 2
        arrays = 4 if case["grad"] else 2            # x, y; dy, dx
        return {"bytes": arrays * n * size + (4 if case["grad"] else 2) * case["width"] * weights,
                "flops": (20 if case["grad"] else 8) * n}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rotary":
        n = case["tokens"] * (heads + kv)
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * dim * size + 4 * case["tokens"] * case["axes"]),
                "flops": passes * 3 * n * case["part"]}
    q_lens, k_lens = _lens(case)
    nq, nk = sum(q_lens) * heads * dim, sum(k_lens) * kv * dim
    moved = 2 * nq + 2 * nk                          # q, o, k, v
    if case["grad"]:
        moved += 2 * nq + 2 * nk                     # do, dq, dk, dv
    products = 7 if case["grad"] else 2              # two forward, five backward
    return {"bytes": moved * size + 8 * (len(q_lens) + 1),
            "flops": 2 * products * _pairs(case) * heads * dim}


# ------------------------------------------------------------------- exact

def _exact_rotary(s, case):
    pairs, axes = case["part"] // 2, case["axes"]
    per = pairs // axes
    i = torch.arange(pairs, device=DEVICE)
    theta = torch.pow(torch.tensor(BASE, dtype=torch.float64, device=DEVICE),
                      -(i % per).double() / per)
    where = s["positions"].reshape(-1, axes).double()[:, i // per]
    z = torch.polar(torch.ones_like(where), where * theta)[:, None]

    def turn(x, z):
        x = x.detach().double()
        y = x.clone()
        if case["layout"] == "half":
            first, second = slice(0, pairs), slice(pairs, 2 * pairs)
        else:
            first, second = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
        w = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    out = [turn(s["q"], z), turn(s["k"], z)]
    return out + [turn(s["dq"], z.conj()), turn(s["dk"], z.conj())] if case["grad"] else out


def _exact_norm(s, case):
    x = s["x"].detach().double()
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sd = (var + EPS).sqrt()
    out = [(x - mean) / sd * w + b]
    if case["grad"]:
        dy, n = s["dy"].double(), x.shape[1]
        u, d = (x - mean) / sd, dy * w
        # The Jacobian (I - 1/n - u u^T / n) / sd, applied to a row.
        out.append((d - d.sum(1, keepdim=True) / n
                    - u * ((d * u).sum(1, keepdim=True) / n)) / sd)
        out += [(dy * u).sum(0), dy.sum(0)]
    return out


def _exact_attention(s, case):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    o, dq, dk, dv = (torch.zeros_like(t, memory_format=torch.contiguous_format)
                     for t in (q, q, k, v))
    q_lens, k_lens = _lens(case)
    q0, k0 = 0, 0
    for nq, nk in zip(q_lens, k_lens):
        seen = torch.ones(nq, nk, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            seen = seen.tril(nk - nq)
        any_seen = seen.any(1, keepdim=True)
        rows, keys = slice(q0, q0 + nq), slice(k0, k0 + nk)
        for h in range(case["heads"]):
            kh, vh = k[keys, h // group], v[keys, h // group]
            score = (q[rows, h] @ kh.T * scale).masked_fill(~seen, -1e300)
            p = torch.softmax(score, 1) * any_seen
            o[rows, h] = p @ vh
            if case["grad"]:
                do = s["do"][rows, h].double()
                dv[keys, h // group] += p.T @ do
                dp = do @ vh.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[rows, h] = ds @ kh
                dk[keys, h // group] += ds.T @ q[rows, h]
        q0, k0 = q0 + nq, k0 + nk
    return [o, dq, dk, dv] if case["grad"] else [o]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "norm": _exact_norm,
            "attention": _exact_attention}[case["kind"]](s, case)
