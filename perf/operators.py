"""Timing cases of the operators around the attention of a transformer block: the
residual addition with its RMS norm (training, and with 8-bit rows and their scales),
rotary positions, the 8-bit projection, and gradient clipping.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes
a case's inputs on the GPU from a seed, ``run()`` makes one pass -- in elementary torch
operations, or with the framework's kernels where ``own`` is true -- ``work()`` counts the
bytes and operations that a pass cannot do without, and ``exact()`` evaluates the same
definitions in 64 bits.
"""
import math
import random

import torch

own = False

EPS = 1e-6
FP8_MAX = 448.0         # largest finite e4m3 value
SCALE_FLOOR = 2.0 ** -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------ cases
def listed():
    return [
        # one token's residual and norm: latency only
        {"name": "norm_token", "op": "norm", "mode": "fwd", "type": "bf16", "rows": 1, "cols": 5120},
        # the whole 720p grid of the 5120-wide layer, forward and backward in training
        {"name": "norm_train_720p", "op": "norm", "mode": "train", "type": "bf16", "rows": 75600, "cols": 5120},
        # an audio-width (1536) stream with one column dropped: odd rows and columns, in fp32
        {"name": "norm_train_odd", "op": "norm", "mode": "train", "type": "fp32", "rows": 4095, "cols": 1535},
        # one of eight sequence-parallel ranks of the 720p grid, 8-bit rows for the projections
        {"name": "norm_8bit_sp8", "op": "norm", "mode": "fp8", "type": "bf16", "rows": 9450, "cols": 5120},
        # decoding: 16 sequences, one token each, far into a long context, 4 query heads a key head
        {"name": "rotary_decode", "op": "rotary", "mode": "fwd", "type": "bf16", "batch": 16, "seq": 1, "hq": 32,
         "hk": 8, "dim": 128, "rot": 128, "layout": "half", "axes": 1, "scaling": "yarn", "start": 130001},
        # the 720p grid with frame / height / width positions, 40 + 40 heads
        {"name": "rotary_3d_720p", "op": "rotary", "mode": "fwd", "type": "bf16", "batch": 1, "seq": 75600, "hq": 40,
         "hk": 40, "dim": 128, "rot": 128, "layout": "interleaved", "axes": 3, "scaling": "none", "start": 0},
        # training on ragged sequences, three quarters of each head rotated, shared key heads
        {"name": "rotary_train_partial", "op": "rotary", "mode": "train", "type": "bf16", "batch": 2, "seq": 4093,
         "hq": 24, "hk": 4, "dim": 128, "rot": 96, "layout": "half", "axes": 1, "scaling": "ntk", "start": 17},
        # the vectors of a few layers (norm weights and biases): many small tensors, latency
        {"name": "clip_vectors", "op": "clip", "kind": "ragged", "type": "fp32", "tensors": 60, "largest": 5120,
         "sizes": 1},
        # one block of the 5120-wide model with its 13824-wide feed-forward layer
        {"name": "clip_block", "op": "clip", "kind": "block", "type": "mixed", "hidden": 5120, "ffn": 13824,
         "blocks": 1},
        # one token through a 5120 x 5120 projection: the weight's bytes
        {"name": "linear8_token", "op": "linear8", "m": 1, "n": 5120, "k": 5120, "bias": True},
        # the 125 audio tokens into the video width
        {"name": "linear8_audio", "op": "linear8", "m": 125, "n": 5120, "k": 1536, "bias": True},
        # a projection of the whole 720p grid
        {"name": "linear8_720p", "op": "linear8", "m": 75600, "n": 5120, "k": 5120, "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        if 3072 not in case.values():   # a size that nothing in this repository has
            return case


def _draw(rng):
    op = rng.choice(["norm", "rotary", "clip", "linear8"])
    if op == "norm":
        mode = rng.choice(["fwd", "train", "fp8"])
        cols = _log(rng, 64, 13824)
        # hidden widths are multiples of 8 as a rule; one in four is not
        cols = cols if rng.random() < 0.25 else max(64, cols // 8 * 8)
        kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rows = _log(rng, 1, min(131072, 75600 * 5120 * 2 // (cols * SIZE[kind])))
        return {"op": op, "mode": mode, "type": kind, "rows": rows, "cols": cols}
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 4 * 2, dim // 4 * 3 // 2 * 2])
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 1, 2, 4, 5])
        batch = rng.choice([1, 1, 2, 3, 8, 64])
        mode, kind = rng.choice(["fwd", "train"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
        token = batch * (hq + hk) * dim * SIZE[kind] * (2 if mode == "train" else 1)
        seq = _log(rng, 1, min(131072, 75600 * 80 * 128 * 2 // token))
        axes = rng.choice([1, 1, 1, 3])
        return {"op": op, "mode": mode, "type": kind, "batch": batch, "seq": seq, "hq": hq, "hk": hk, "dim": dim,
                "rot": rot,
                "layout": rng.choice(["interleaved", "half"]), "axes": axes,
                "scaling": "none" if axes == 3 else rng.choice(["none", "linear", "ntk", "yarn"]),
                "start": _log(rng, 1, 1000000)}
    if op == "clip":
        if rng.random() < 0.3:
            kind = rng.choice(["bf16", "mixed", "fp32"])
            hidden = 128 * _log(rng, 4, 28 if kind == "fp32" else 40)
            return {"op": op, "kind": "block", "type": kind, "hidden": hidden, "ffn": hidden * 27 // 10 // 8 * 8,
                    "blocks": rng.randint(1, max(1, min(40, 13000000 // hidden ** 2)))}
        tensors = _log(rng, 1, 1500)
        return {"op": op, "kind": "ragged", "type": rng.choice(["bf16", "mixed", "fp32", "fp16"]), "tensors": tensors,
                "largest": _log(rng, 64, min(100000000, 200000000 // tensors)), "sizes": rng.randrange(1 << 20)}
    n, k = 8 * _log(rng, 16, 1728), 16 * _log(rng, 8, 864)
    m = _log(rng, 1, min(131072, 75600 * 5120 * 5120 // (n * k)))
    return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5}


# ----------------------------------------------------------------------- inputs
def _frequencies(rot, scaling):
    """Radians per position of each of the rot / 2 pairs, float64, and the factor on the
    rotated values: base 10000; "linear" divides positions by 4, "ntk" widens the base,
    "yarn" interpolates the slow pairs by 8 over an original length of 4096."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    base = 10000.0
    if scaling == "ntk":
        base *= 4.0 ** (rot / max(rot - 2.0, 1.0))
    f = base ** (-i / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":
        turns = 4096 * f / (2 * math.pi)       # over the original length
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * keep + f / 8.0 * (1 - keep), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _sections(rot, axes):
    """Pairs that follow each position axis: the last two thirds of the head's pairs, in
    equal parts, follow height and width, the first the frame."""
    if axes == 1:
        return (rot // 2,)
    third = rot // 2 // 3
    return (rot // 2 - 2 * third, third, third)


def _sizes(case):
    """(type, number of elements) of each gradient."""
    if case["kind"] == "block":
        h, f = case["hidden"], case["ffn"]
        vec = "bf16" if case["type"] == "bf16" else "fp32"
        mat = "fp32" if case["type"] == "fp32" else "bf16"
        one = [(mat, h * h), (vec, h)] * 4 + [(vec, h)] * 4 + [(mat, h * f), (vec, f), (mat, f * h), (vec, h)]
        return one * case["blocks"]
    rng = random.Random(case["sizes"])
    out = []
    for _ in range(case["tensors"]):
        n = max(1, int(case["largest"] ** rng.uniform(0.5, 1.0)))
        n = n if rng.random() < 0.25 else max(8, n // 8 * 8)
        t = case["type"] if case["type"] != "mixed" else rng.choice(["bf16", "bf16", "fp32"])
        out.append((t, n))
    return out


def _rows_8bit(x):
    scale = (x.float().abs().amax(1) / FP8_MAX).clamp_min(SCALE_FLOOR)
    return (x.float() / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = dict(case)
    if case["op"] == "norm":
        dt, shape = TYPES[case["type"]], (case["rows"], case["cols"])
        wide = torch.exp(rnd(case["cols"]))   # channels of a residual stream differ in size
        s["x"] = rnd(*shape, dtype=dt)
        s["r"] = rnd(*shape, dtype=dt).mul_(wide.to(dt))
        s["w"] = 1.0 + 0.2 * rnd(case["cols"])
        if case["mode"] == "train":
            s["dy"], s["dh"] = rnd(*shape, dtype=dt), rnd(*shape, dtype=dt)
            for n in ("x", "r", "w"):
                s[n].requires_grad_()
    elif case["op"] == "rotary":
        dt, b, n = TYPES[case["type"]], case["batch"], case["seq"]
        heads = case["hq"] + 2 * case["hk"]
        # q and k are slices of a fused projection's output, as a layer has them
        qkv = rnd(b, n, heads, case["dim"], dtype=dt)
        s["q"], s["k"] = qkv[:, :, :case["hq"]], qkv[:, :, case["hq"]:case["hq"] + case["hk"]]
        f, s["scale"] = _frequencies(case["rot"], case["scaling"])
        s["freqs"], s["sections"] = f.cuda(), _sections(case["rot"], case["axes"])
        first = torch.randint(0, max(1, case["start"]), (b, 1), generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        if case["axes"] == 3:   # frame, row and column of a grid 45 rows high and 80 columns wide
            s["pos"] = torch.stack([at // 3600, at // 80 % 45, at % 80], -1).expand(b, n, 3) + first[..., None] % 7
        else:
            s["pos"] = first + at
        if case["mode"] == "train":
            s["dq"], s["dk"] = rnd(b, n, case["hq"], case["dim"], dtype=dt), rnd(b, n, case["hk"], case["dim"], dtype=dt)
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    elif case["op"] == "clip":
        sizes = _sizes(case)
        size = torch.exp(2.0 * torch.randn(len(sizes), generator=torch.Generator().manual_seed(seed))) * 1e-3
        s["grads"] = [rnd(n, dtype=TYPES[t]).mul_(float(a)) for (t, n), a in zip(sizes, size)]
        # the optimizer's gradient buffers, one flat buffer a type
        s["flat"] = {t: torch.zeros(sum(n for u, n in sizes if u == t), dtype=TYPES[t], device="cuda")
                     for t in sorted({t for t, _ in sizes})}
        views = {t: iter(s["flat"][t].split([n for u, n in sizes if u == t])) for t in s["flat"]}
        s["out"] = [next(views[t]) for t, _ in sizes]
        s["max_norm"] = 1.0e-2
    else:
        x = rnd(case["m"], case["k"]).mul_(torch.exp(0.5 * rnd(case["k"])))
        s["x8"], s["xs"] = _rows_8bit(x.to(torch.bfloat16))
        s["w8"], s["ws"] = _rows_8bit(rnd(case["n"], case["k"], dtype=torch.bfloat16).mul_(case["k"] ** -0.5))
        s["b"] = rnd(case["n"]) if case["bias"] else None
    return s


# -------------------------------------------------------------------- one pass
def run(s):
    return (_OWN if own else _PLAIN)[s["op"]](s)


def _own_norm(s):
    from prism_b200.norm import add_rms_norm, add_rms_norm_fp8
    if s["mode"] == "fp8":
        y8, scale, h = add_rms_norm_fp8(s["x"], s["r"], s["w"], eps=EPS)
        return {"y8": y8, "scale": scale, "h": h}
    y, h = add_rms_norm(s["x"], s["r"], s["w"], eps=EPS)
    if s["mode"] == "fwd":
        return {"y": y, "h": h}
    dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
    return {"y": y, "h": h, "dx": dx, "dr": dr, "dw": dw}


def _plain_norm(s):
    with torch.no_grad():
        x, w = s["x"], s["w"]
        h = (x.float() + s["r"].float()).to(x.dtype)      # the residual stream as it is kept
        hf = h.float()
        rs = torch.rsqrt(hf.square().mean(1, keepdim=True) + EPS)
        if s["mode"] == "fp8":
            y = hf * rs * w
            scale = (y.abs().amax(1) / FP8_MAX).clamp_min(SCALE_FLOOR)
            y8 = (y / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
            return {"y8": y8, "scale": scale, "h": h}
        y = (hf * rs * w).to(x.dtype)
        if s["mode"] == "fwd":
            return {"y": y, "h": h}
        dy = s["dy"].float()
        gy = dy * w
        xhat = hf * rs
        dx = (rs * (gy - xhat * (gy * xhat).mean(1, keepdim=True)) + s["dh"].float()).to(x.dtype)
        return {"y": y, "h": h, "dx": dx, "dr": dx, "dw": (dy * xhat).sum(0)}


def _own_rotary(s):
    from prism_b200.rotary import apply_rotary
    sections = s["sections"] if s["axes"] > 1 else None
    q, k = apply_rotary(s["q"], s["k"], s["pos"], s["freqs"], layout=s["layout"], sections=sections, scale=s["scale"])
    if s["mode"] == "fwd":
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _angles(s):
    """Angle of each pair of each token, in radians: 64 bits, because a product of a long
    position and a frequency does not fit 32."""
    pos = s["pos"].double()
    if s["axes"] == 1:
        return pos[..., None] * s["freqs"]
    axis = torch.repeat_interleave(torch.arange(s["axes"], device=pos.device),
                                   torch.tensor(s["sections"], device=pos.device), output_size=s["rot"] // 2)
    return pos[..., axis] * s["freqs"]


def _rotate(x, cos, sin, s):
    rot = s["rot"]
    a, b = ((x[..., 0:rot:2], x[..., 1:rot:2]) if s["layout"] == "interleaved"
            else (x[..., :rot // 2], x[..., rot // 2:rot]))
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if s["layout"] == "interleaved" else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rotary(s):
    with torch.no_grad():
        angle = _angles(s)
        cos, sin = (f(angle).float().mul(s["scale"])[:, :, None] for f in (torch.cos, torch.sin))
        dt = s["q"].dtype
        out = {n: _rotate(s[n].float(), cos, sin, s).to(dt) for n in ("q", "k")}
        if s["mode"] == "train":   # the transposed rotation
            out |= {n: _rotate(s[n].float(), cos, -sin, s).to(dt) for n in ("dq", "dk")}
        return out


def _own_clip(s):
    from prism_b200.grad_clip import clip_grad_norm
    norm = clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
    return {"norm": norm, "flat": s["flat"]}


def _plain_clip(s):
    flat = {t: torch.cat([g for g in s["grads"] if g.dtype == TYPES[t]]).float() for t in s["flat"]}
    norm = torch.stack([f.square().sum() for f in flat.values()]).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "flat": {t: s["flat"][t].copy_(f * coef) for t, f in flat.items()}}


def _own_linear8(s):
    from prism_b200.linear import linear_fp8
    return linear_fp8(s["x8"], s["xs"], s["w8"], s["ws"], bias=s["b"])


def _plain_linear8(s):
    y = s["x8"].float() @ s["w8"].float().t() * s["xs"][:, None] * s["ws"]
    return (y if s["b"] is None else y + s["b"]).to(torch.bfloat16)


_OWN = {"norm": _own_norm, "rotary": _own_rotary, "clip": _own_clip, "linear8": _own_linear8}
_PLAIN = {"norm": _plain_norm, "rotary": _plain_rotary, "clip": _plain_clip, "linear8": _plain_linear8}


# ------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "norm":
        n, c, e = case["rows"] * case["cols"], case["cols"], SIZE[case["type"]]
        if case["mode"] == "fp8":
            return {"bytes": n * (3 * e + 1) + 4 * c + 4 * case["rows"], "flops": 7 * n}
        if case["mode"] == "fwd":
            return {"bytes": n * 4 * e + 4 * c, "flops": 5 * n}
        # x, r, dy, dh in; y, h, dx out (dr is dx)
        return {"bytes": n * 7 * e + 8 * c, "flops": 16 * n}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        heads = case["hq"] + case["hk"]
        n, passes = tokens * heads * case["dim"], 2 if case["mode"] == "train" else 1
        return {"bytes": passes * (2 * n * SIZE[case["type"]]) + 8 * tokens * case["axes"] + 4 * case["rot"],
                "flops": passes * 3 * tokens * heads * case["rot"]}
    if case["op"] == "clip":
        sizes = _sizes(case)
        return {"bytes": sum(2 * n * SIZE[t] for t, n in sizes), "flops": 3 * sum(n for _, n in sizes)}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * k + n * k + 2 * m * n + 4 * (m + 2 * n), "flops": 2 * m * n * k}


# -------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s)
        if case["op"] == "rotary":
            return _exact_rotary(s)
        if case["op"] == "clip":
            # one sum a type: the gradients' squares, then the factor of all of them
            per_type = {t: torch.cat([g.double() for g in s["grads"] if g.dtype == TYPES[t]]) for t in s["flat"]}
            norm = math.sqrt(sum(float(torch.dot(f, f)) for f in per_type.values()))
            factor = min(1.0, s["max_norm"] / (norm + 1e-6))
            return {"norm": torch.tensor(norm, dtype=torch.float64), "flat": {t: f * factor for t, f in per_type.items()}}
        x = s["x8"].double() * s["xs"].double()[:, None]
        y = torch.mm(x, (s["w8"].double() * s["ws"].double()[:, None]).t())
        return y if s["b"] is None else y + s["b"].double()


def _exact_norm(s):
    # the stream is kept in the inputs' type; everything after that is in 64 bits
    h = (s["x"].double() + s["r"].double()).to(s["x"].dtype).double()
    w, n = s["w"].double(), s["cols"]
    inv = 1.0 / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / n + EPS)
    y = h * inv * w
    if s["mode"] == "fp8":
        top = torch.maximum(y.amax(1), -y.amin(1))
        scale = torch.clamp(top / FP8_MAX, min=SCALE_FLOOR)
        return {"y8": y / scale[:, None], "scale": scale, "h": h}   # y8 before its rounding to 8 bits
    if s["mode"] == "fwd":
        return {"y": y, "h": h}
    # y_i = w_i h_i u, u = (mean h^2 + eps)^(-1/2): dy_i/dh_j = w_i u [i = j] - w_i h_i u^3 h_j / n
    dy = s["dy"].double()
    along = torch.einsum("rc,rc,c->r", dy, h, w)[:, None]
    dx = dy * w * inv - h * inv ** 3 * along / n + s["dh"].double()
    return {"y": y, "h": h, "dx": dx, "dr": dx, "dw": torch.einsum("rc,rc,r->c", dy, h, inv[:, 0])}


def _exact_rotary(s):
    # each pair as a complex number, multiplied by scale * exp(i angle); the gradient by its conjugate
    sizes = torch.tensor(s["sections"])
    axis = torch.repeat_interleave(torch.arange(len(sizes)), sizes).cuda()
    pos = s["pos"].double() if s["axes"] > 1 else s["pos"].double()[..., None]
    turn = torch.polar(torch.full((), float(s["scale"]), dtype=torch.float64, device="cuda").expand(
        *pos.shape[:2], s["rot"] // 2), pos.index_select(-1, axis) * s["freqs"])[:, :, None]
    out = {}
    names = ("q", "k", "dq", "dk") if s["mode"] == "train" else ("q", "k")
    for name in names:
        x = s[name].double()
        half = s["rot"] // 2
        pair = (x[..., :s["rot"]].unflatten(-1, (half, 2)) if s["layout"] == "interleaved"
                else x[..., :s["rot"]].unflatten(-1, (2, half)).transpose(-1, -2))
        z = torch.view_as_complex(pair.contiguous()) * (turn.conj() if name[0] == "d" else turn)
        y = torch.view_as_real(z)
        y = y if s["layout"] == "interleaved" else y.transpose(-1, -2)
        out[name] = torch.cat((y.flatten(-2), x[..., s["rot"]:]), -1)
    return out
