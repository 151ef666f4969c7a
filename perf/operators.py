"""The operators of a trainable local block, as they are timed and compared: rotary positions, the attention over a
neighbour mask with its gradients, and the gated feed-forward block.

``own = False`` computes each in plain torch (products, exp, indexing; 32 bits, angles in 64), ``own = True`` by the
framework's entry points.  ``exact`` restates each in 64 bits.  ``listed`` holds sizes from the framework's own
configurations (QM9-like and GEOM-Drugs-like molecules, MOF cells, the trunk's widths) and a few wider ones; ``draw``
gives sizes from the ranges around them.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# -- the cases ---------------------------------------------------------------------------------------------------
def _rotary(**kw):
    case = dict(kind="rotary", base=10000.0, scaling="none", factor=1.0, original=0, offset=0)
    case.update(kw)
    return case


def listed():
    return [
        # q and k of one molecule's fp32 attention layer in sampling: the smallest call, where latency counts;
        # three coordinates as positions, 24 of 32 dimensions rotate
        _rotary(name="rotary_molecule", form="views", train=False, dtype="float32", batch=1, tokens=19, heads=8,
                kv_heads=8, head_dim=32, rotary_dim=24, axes=3, base=100.0, layout="half"),
        # a GEOM-Drugs batch padded to 181 atoms, straight from the in_proj rows, with the gradient of the rows
        _rotary(name="rotary_geom_train", form="rows", train=True, dtype="bfloat16", batch=64, tokens=181, heads=8,
                kv_heads=8, head_dim=64, rotary_dim=60, axes=3, base=100.0, layout="half"),
        # long sequences by their index, far past the trained length, fewer key heads than query heads
        _rotary(name="rotary_long", form="rows", train=False, dtype="float16", batch=2, tokens=32768, heads=12,
                kv_heads=4, head_dim=128, rotary_dim=128, axes=1, layout="interleaved", scaling="yarn", factor=8.0,
                original=4096, offset=100000),
        # QM9 molecules trained: 9 to 29 atoms, every atom's 16 nearest
        dict(name="local_qm9_train", kind="local", mask="knn", dtype="bfloat16", batch=128, tokens=29, mean=19, heads=8,
             head_dim=32, knn=16),
        # GEOM-Drugs molecules trained: about 44 atoms padded to 181, 32 nearest
        dict(name="local_geom_train", kind="local", mask="knn", dtype="bfloat16", batch=64, tokens=181, mean=44,
             heads=8, head_dim=64, knn=32),
        # periodic MOF cells trained: 512 atoms, 6 A cutoff, atoms in no order (every tile of the mask has entries)
        dict(name="local_cells_train", kind="local", mask="radius", dtype="bfloat16", batch=32, tokens=512, mean=512,
             heads=8, head_dim=64, box=22.5, cutoff=6.0, ordered=False),
        # large cells, atoms ordered along one axis (tiles without an entry), wide heads, an odd atom count
        dict(name="local_large_train", kind="local", mask="radius", dtype="float16", batch=4, tokens=1997, mean=1997,
             heads=8, head_dim=128, box=36.0, cutoff=6.0, ordered=True),
        # one token through the feed-forward block: the weights are read once
        dict(name="gated_token", kind="gated", train=False, dtype="bfloat16", tokens=1, width=512, hidden=2048,
             activation="silu", bias=False),
        # the valid atoms of a GEOM-Drugs batch, the hidden width of 8/3 that keeps an ungated block's weights (odd)
        dict(name="gated_trunk", kind="gated", train=False, dtype="bfloat16", tokens=2738, width=512, hidden=1365,
             activation="gelu_tanh", bias=True),
        # the same atoms trained
        dict(name="gated_trunk_train", kind="gated", train=True, dtype="bfloat16", tokens=2738, width=512, hidden=2048,
             activation="silu", bias=True),
        # a large training batch at the wider of the two model widths
        dict(name="gated_large_train", kind="gated", train=True, dtype="bfloat16", tokens=32768, width=768,
             hidden=2048, activation="silu", bias=True),
        # QM9 molecules trained in fp32
        dict(name="gated_qm9_fp32_train", kind="gated", train=True, dtype="float32", tokens=2432, width=384,
             hidden=1024, activation="gelu", bias=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(("rotary", "local", "gated"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    if kind == "rotary":
        head_dim = rng.choice((32, 64, 128))
        heads = rng.choice((4, 8, 12))
        kv_heads = rng.choice((heads, heads, heads // 4, 1))
        long = rng.random() < 0.5
        axes = 1 if long else rng.choice((2, 3))
        per = 2 * axes
        rotary_dim = per * rng.randint(max(1, head_dim // (2 * per)), head_dim // per)
        tokens = _log_int(rng, 100, 32768) if long else rng.randint(9, 512)
        size = 2 if dtype != "float32" else 4
        most = 2 * 32768 * 20 * 128 * 2 / (tokens * (heads + 2 * kv_heads) * head_dim * size)
        form = rng.choice(("rows", "views"))
        train = form == "rows" and rng.random() < 0.5
        batch = _log_int(rng, 1, max(1, min(256, int(most / (2 if train else 1)))))
        scaling = rng.choice(("none", "linear", "ntk", "yarn")) if long and rotary_dim > 2 else "none"
        return _rotary(form=form, train=train, dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads,
                       head_dim=head_dim, rotary_dim=rotary_dim, axes=axes, base=10000.0 if long else 100.0,
                       layout=rng.choice(("half", "interleaved")), scaling=scaling,
                       factor=1.0 if scaling == "none" else float(rng.choice((2, 4, 8))), original=4096,
                       offset=rng.choice((0, 1000, 100000)) if long else 0)
    if kind == "local":
        dtype = rng.choice(("bfloat16", "float16"))
        head_dim = rng.choice((32, 64, 128))
        heads = rng.choice((4, 8, 12))
        if rng.random() < 0.5:
            tokens = rng.randint(29, 181)
            most = 128 * 8 * 181 * 128 / (tokens * heads * head_dim)
            return dict(kind="local", mask="knn", dtype=dtype, batch=_log_int(rng, 1, max(1, min(256, int(most)))),
                        tokens=tokens, mean=max(9, tokens // 3), heads=heads, head_dim=head_dim,
                        knn=rng.choice((8, 16, 32)))
        tokens = _log_int(rng, 100, 1997)
        most = 4 * 8 * 1997 * 1997 * 128 / (tokens * tokens * heads * head_dim)
        return dict(kind="local", mask="radius", dtype=dtype, batch=_log_int(rng, 1, max(1, min(32, int(most / 3)))),
                    tokens=tokens, mean=tokens, heads=heads, head_dim=head_dim,
                    box=round(2.85 * tokens ** (1.0 / 3.0), 2), cutoff=round(rng.uniform(4.0, 7.0), 2),
                    ordered=rng.random() < 0.5)
    width = rng.choice((128, 256, 384, 512, 768, rng.randint(60, 768)))
    hidden = rng.choice((2 * width, 4 * width, (8 * width) // 3)) if width < 700 else rng.randint(700, 2048)
    train = rng.random() < 0.5
    most = 32768 * 768 * 2048 / (width * hidden)
    if dtype == "float32":
        most /= 16
    return dict(kind="gated", train=train, dtype=dtype, tokens=_log_int(rng, 1, min(32768, int(most))), width=width,
                hidden=hidden, activation=rng.choice(("silu", "gelu", "gelu_tanh", "relu", "sigmoid")),
                bias=rng.random() < 0.5)


# -- inputs ------------------------------------------------------------------------------------------------------
def _gen(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 7919 + 11)
    return gen


def _randn(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE) * std).to(dtype)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEVICE)


def _allowed(case, gen):
    """(B, N, N) bool: the neighbours of every atom, itself among them; padded atoms have and are none."""
    B, N = case["batch"], case["tokens"]
    if case["mask"] == "knn":
        spread = min(N - case["mean"], case["mean"] - 9) if N > case["mean"] else 0
        counts = (case["mean"] + (2.0 * _rand(gen, B) - 1.0) * spread).round().long().clamp(1, N)
        valid = torch.arange(N, device=DEVICE)[None] < counts[:, None]
        coords = torch.randn(B, N, 3, generator=gen, device=DEVICE) * math.sqrt(2.0)
        d2 = (coords[:, :, None] - coords[:, None]).square().sum(-1)
        both = valid[:, :, None] & valid[:, None]
        eye = torch.eye(N, dtype=torch.bool, device=DEVICE)[None]
        near = d2.masked_fill(~both | eye, float("inf")).topk(min(case["knn"], N), dim=-1, largest=False).indices
        hit = torch.zeros(B, N, N, dtype=torch.bool, device=DEVICE).scatter_(2, near, True)
        return (hit | eye) & both
    frac = _rand(gen, B, N, 3)
    if case["ordered"]:
        frac = frac.gather(1, frac[..., :1].argsort(dim=1).expand(B, N, 3))
    allowed = torch.empty(B, N, N, dtype=torch.bool, device=DEVICE)
    for b in range(B):
        d = frac[b, :, None] - frac[b, None]
        d = (d - d.round()) * case["box"]
        allowed[b] = d.square().sum(-1) <= case["cutoff"] ** 2
    return allowed


def _pack_bits(allowed):
    """int32 words: bit t of word w is column 32 w + t."""
    B, N, _ = allowed.shape
    W = (N + 31) // 32
    words = torch.empty(B, N, W, dtype=torch.int32, device=DEVICE)
    shift = torch.arange(32, device=DEVICE)
    for b in range(B):
        full = torch.zeros(N, W * 32, dtype=torch.int64, device=DEVICE)
        full[:, :N] = allowed[b]
        word = (full.view(N, W, 32) << shift).sum(-1)
        words[b] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)
    return words


def _block_flags(allowed):
    """uint8: whether a 64 by 64 block of the mask has an entry."""
    B, N, _ = allowed.shape
    NB = (N + 63) // 64
    flags = torch.empty(B, NB, NB, dtype=torch.uint8, device=DEVICE)
    for b in range(B):
        full = torch.zeros(NB * 64, NB * 64, dtype=torch.bool, device=DEVICE)
        full[:N, :N] = allowed[b]
        flags[b] = full.view(NB, 64, NB, 64).any(3).any(1)
    return flags


def prepare(case, seed):
    gen = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "rotary":
        B, N, D = case["batch"], case["tokens"], case["head_dim"]
        columns = (case["heads"] + 2 * case["kv_heads"]) * D
        state["rows"] = _randn(gen, B, N, columns, dtype=dtype)
        if case["axes"] == 1:
            start = torch.randint(0, case["offset"] + 1, (B, 1), generator=gen, device=DEVICE)
            state["positions"] = start + torch.arange(N, device=DEVICE)[None]
        else:
            state["positions"] = torch.randn(B, N, case["axes"], generator=gen, device=DEVICE) * 3.0
        if case["train"]:
            state["grads"] = [_randn(gen, B, h, N, D, dtype=dtype)
                              for h in (case["heads"], case["kv_heads"], case["kv_heads"])]
        if own:
            from matterformer_amd.rotary import rotary_frequencies

            state["frequencies"] = rotary_frequencies(
                case["rotary_dim"], axes=case["axes"], base=case["base"], scaling=case["scaling"],
                factor=case["factor"], original_length=case["original"] or None, device=DEVICE)
            state["rows"].requires_grad_(case["train"])
        else:
            state["frequencies"] = _table(case)
        return state
    if case["kind"] == "local":
        B, H, N, D = case["batch"], case["heads"], case["tokens"], case["head_dim"]
        allowed = _allowed(case, gen)
        state["bits"], state["blocks"] = _pack_bits(allowed), _block_flags(allowed)
        state["qkv"] = [_randn(gen, B, H, N, D, dtype=dtype) for _ in range(3)]
        state["grad"] = _randn(gen, B, H, N, D, dtype=dtype, std=0.1)
        if own:
            for t in state["qkv"]:
                t.requires_grad_(True)
        return state
    T, C, F = case["tokens"], case["width"], case["hidden"]
    state["x"] = _randn(gen, T, C, dtype=dtype)
    state["weight"] = ((2.0 * _rand(gen, 2 * F, C) - 1.0) * C ** -0.5).to(dtype)
    state["bias"] = ((2.0 * _rand(gen, 2 * F) - 1.0) * C ** -0.5).to(dtype) if case["bias"] else None
    if case["train"]:
        state["grad"] = _randn(gen, T, F, dtype=dtype, std=0.1)
        if own:
            for t in (state["x"], state["weight"], state["bias"]):
                if t is not None:
                    t.requires_grad_(True)
    return state


# -- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "local": _own_local, "gated": _own_gated}[kind](state)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "local": _plain_local, "gated": _plain_gated}[kind](state)


def _views(case, rows):
    """q (B, H, N, D), k and v (B, KV, N, D) inside the in_proj rows."""
    B, N, _ = rows.shape
    H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = rows.split((H * D, KV * D, KV * D), dim=-1)
    return (q.view(B, N, H, D).transpose(1, 2), k.view(B, N, KV, D).transpose(1, 2),
            v.view(B, N, KV, D).transpose(1, 2))


def _own_rotary(state):
    from matterformer_amd.rotary import apply_rotary, rotary_heads

    case = state["case"]
    if case["form"] == "views":
        q, k, _ = _views(case, state["rows"])
        return list(apply_rotary(q, k, state["positions"], state["frequencies"], layout=case["layout"]))
    out = rotary_heads(state["rows"], state["positions"], state["frequencies"], heads=case["heads"],
                       kv_heads=case["kv_heads"], layout=case["layout"])
    if not case["train"]:
        return list(out)
    return [*out, *torch.autograd.grad(out, state["rows"], state["grads"])]


def _own_local(state):
    from matterformer_amd.geometry_ops import radius_attention

    out = radius_attention(*state["qkv"], state["bits"], state["blocks"])
    return [out, *torch.autograd.grad(out, state["qkv"], state["grad"])]


def _own_gated(state):
    from matterformer_amd.gated_mlp import gated_linear

    case = state["case"]
    out = gated_linear(state["x"], state["weight"], state["bias"], activation=case["activation"])
    if not case["train"]:
        return [out]
    leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    return [out, *torch.autograd.grad(out, leaves, state["grad"])]


# -- the plain forms ---------------------------------------------------------------------------------------------
def _table(case):
    """Frequencies (pairs,) in 64 bits, the axis of each pair, and the factor of the rotated part."""
    per = case["rotary_dim"] // (2 * case["axes"])
    i = torch.arange(per, dtype=torch.float64, device=DEVICE)
    base, s = case["base"], case["factor"]
    gain = 1.0
    if case["scaling"] == "ntk" and per > 1:
        base = base * s ** (per / (per - 1))
    f = base ** (-i / per)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "yarn":
        turns = case["original"] * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / s * (1.0 - keep)
        gain = 0.1 * math.log(s) + 1.0
    return f.repeat(case["axes"]), torch.arange(case["axes"], device=DEVICE).repeat_interleave(per), gain


def _cos_sin(state):
    f, axis, gain = state["frequencies"]
    pos = state["positions"].double()
    if pos.ndim == 2:
        pos = pos[..., None]
    angle = pos[..., axis] * f
    return (angle.cos() * gain).float()[:, None], (angle.sin() * gain).float()[:, None]


def _turn(x, cos, sin, case):
    R = case["rotary_dim"]
    x32 = x.float()
    if case["layout"] == "half":
        a, b = x32[..., :R // 2], x32[..., R // 2:R]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos, x32[..., R:]], dim=-1)
    else:
        a, b = x32[..., 0:R:2], x32[..., 1:R:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        y = torch.cat([y, x32[..., R:]], dim=-1)
    return y.to(x.dtype)


def _plain_rotary(state):
    case = state["case"]
    q, k, v = _views(case, state["rows"])
    cos, sin = _cos_sin(state)
    out = [_turn(q, cos, sin, case), _turn(k, cos, sin, case)]
    if case["form"] == "views":
        return out
    out.append(v.contiguous())
    if case["train"]:
        gq, gk, gv = state["grads"]
        back = [_turn(gq, cos, -sin, case), _turn(gk, cos, -sin, case), gv]
        out.append(torch.cat([g.transpose(1, 2).flatten(2) for g in back], dim=-1))
    return out


def _unpack(bits, N):
    shift = torch.arange(32, device=bits.device, dtype=torch.int32)
    return ((bits[..., None] >> shift) & 1).flatten(-2)[..., :N].bool()


def _plain_local(state):
    q, k, v = (t.float() for t in state["qkv"])
    go = state["grad"].float()
    dtype = state["grad"].dtype
    N, D = q.shape[-2:]
    scale = D ** -0.5
    allowed = _unpack(state["bits"], N)[:, None]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(~allowed, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), go)
    dp = torch.matmul(go, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (go * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    return [t.to(dtype) for t in (out, dq, dk, dv)]


def _act(a, name):
    """The activation and its derivative."""
    if name == "relu":
        return a.clamp_min(0.0), (a > 0).to(a.dtype)
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(a * math.sqrt(0.5)))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) * (2.0 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (a + 0.044715 * a ** 3))
        return 0.5 * a * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * a * a)
    sig = 1.0 / (1.0 + torch.exp(-a))
    if name == "sigmoid":
        return sig, sig * (1.0 - sig)
    return a * sig, sig * (1.0 + a * (1.0 - sig))


def _plain_gated(state):
    case = state["case"]
    x, w = state["x"].float(), state["weight"].float()
    dtype = state["x"].dtype
    both = torch.matmul(x, w.t())
    if state["bias"] is not None:
        both = both + state["bias"].float()
    a, b = both.chunk(2, dim=-1)
    y, slope = _act(a, case["activation"])
    out = [(y * b).to(dtype)]
    if case["train"]:
        go = state["grad"].float()
        back = torch.cat([go * b * slope, go * y], dim=-1)
        out += [torch.matmul(back, w).to(dtype), torch.matmul(back.t(), x).to(dtype)]
        if state["bias"] is not None:
            out.append(back.sum(0).to(dtype))
    return out


# -- the work a pass cannot do without ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "rotary":
        tokens = case["batch"] * case["tokens"]
        parts = case["heads"] + case["kv_heads"] * (1 if case["form"] == "views" else 2)
        passes = 2 if case["train"] else 1
        moved = 2 * tokens * parts * case["head_dim"] * size
        turned = tokens * (case["heads"] + case["kv_heads"]) * case["rotary_dim"]
        positions = tokens * (8 if case["axes"] == 1 else 4 * case["axes"])
        return {"bytes": passes * moved + positions, "flops": passes * 3 * turned}
    if case["kind"] == "local":
        B, H, N, D = case["batch"], case["heads"], case["tokens"], case["head_dim"]
        if case["mask"] == "knn":
            pairs = B * case["mean"] * min(case["mean"], case["knn"] + 1)
        else:
            share = min(1.0, 4.0 / 3.0 * math.pi * (case["cutoff"] / case["box"]) ** 3)
            pairs = B * N * (1 + (N - 1) * share)
        return {"bytes": 8 * B * H * N * D * size + B * N * ((N + 31) // 32) * 4, "flops": 14 * D * H * pairs}
    T, C, F = case["tokens"], case["width"], case["hidden"]
    n = T * C + 2 * F * C + T * F + (2 * F if case["bias"] else 0)
    if not case["train"]:
        return {"bytes": n * size, "flops": 4 * T * C * F}
    return {"bytes": (2 * n) * size, "flops": 12 * T * C * F}


# -- from the definitions, in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "local": _exact_local, "gated": _exact_gated}[case["kind"]](case, state)


def _exact_rotary(case, state):
    """Every pair as a complex number times gain e^(i angle)."""
    R, axes = case["rotary_dim"], case["axes"]
    per = R // (2 * axes)
    s, gain, freqs = case["factor"], 1.0, []
    for i in range(per):
        f = math.pow(case["base"], -i / per)
        if case["scaling"] == "linear":
            f /= s
        elif case["scaling"] == "ntk" and per > 1:
            f *= math.pow(s, -i / (per - 1))
        elif case["scaling"] == "yarn":
            keep = min(1.0, max(0.0, (case["original"] * f / (2.0 * math.pi) - 1.0) / 31.0))
            f = keep * f + (1.0 - keep) * f / s
        freqs.append(f)
    if case["scaling"] == "yarn":
        gain = 1.0 + 0.1 * math.log(s)
    pos = state["positions"].double()
    pos = pos[..., None] if axes == 1 else pos
    f = torch.tensor(freqs, dtype=torch.float64, device=DEVICE)
    angle = (pos[..., None] * f).flatten(-2)[:, None]  # (B, 1, N, axes * per)
    turn = torch.polar(torch.full_like(angle, gain), angle)

    def rotate(x, turn):
        x = x.double()
        y = x.clone()
        a, b = (slice(0, R // 2), slice(R // 2, R)) if case["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
        y[..., a], y[..., b] = z.real, z.imag
        return y

    q, k, v = _views(case, state["rows"].detach())
    out = [rotate(q, turn), rotate(k, turn)]
    if case["form"] == "views":
        return out
    out.append(v.double())
    if case["train"]:
        gq, gk, gv = state["grads"]
        back = [rotate(gq, turn.conj()), rotate(gk, turn.conj()), gv.double()]
        out.append(torch.cat([g.permute(0, 2, 1, 3).flatten(2) for g in back], dim=-1))
    return out


def _exact_local(case, state):
    B, H, N, D = case["batch"], case["heads"], case["tokens"], case["head_dim"]
    out = [torch.empty(B, H, N, D, dtype=torch.float64, device=DEVICE) for _ in range(4)]
    for b in range(B):
        q, k, v = (t[b].detach().double().requires_grad_(True) for t in state["qkv"])
        allowed = _unpack(state["bits"][b], N)
        logits = (q @ k.mT) / math.sqrt(D)
        weights = torch.softmax(torch.where(allowed, logits, -1e300), dim=-1)
        y = torch.where(allowed, weights, 0.0) @ v
        grads = torch.autograd.grad(y, (q, k, v), state["grad"][b].double())
        for o, t in zip(out, (y, *grads)):
            o[b] = t.detach()
    return out


def _exact_gated(case, state):
    F = torch.nn.functional
    act = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu,
           "sigmoid": torch.sigmoid}[case["activation"]]
    leaves = [t.detach().double().requires_grad_(True)
              for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    gate, up = F.linear(*leaves).chunk(2, dim=-1)
    y = act(gate) * up
    if not case["train"]:
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["grad"].double())]
