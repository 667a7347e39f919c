"""The attention operators of a decoder over an encoder's states: what a pass
through each of them is, in a plain form and as the library's calls.

* ``rotary``: positions rotated into queries and keys (sam3cu.rope_pos);
* ``qk_norm``: queries and keys normalised head by head and rotated, in one
  pass (sam3cu.qk_norm_rope);
* ``cross``: attention of queries over states of another length
  (sam3cu.cross_attention).

A case is a dict of plain values.  Tensors are [batch, tokens, heads, head_dim]
in that order of dimensions; ``order`` says how they lie in memory.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _lib():
    """The library's Python module."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sam3.c_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import sam3cu
    return sam3cu


# ------------------------------------------------------------------ cases
def _rotary(name, batch, tokens, q_heads, k_heads, head_dim, rot, dtype, layout="half", scaling="none", factor=1.0,
            far=0, order="bshd", op="rotary", norm="none"):
    c = {"op": op, "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim,
         "rot": rot, "dtype": dtype, "layout": layout, "scaling": scaling, "factor": factor, "far": far,
         "order": order, "norm": norm}
    return dict(c, name=name) if name else c


def _cross(name, batch, queries, keys, q_heads, kv_heads, head_dim, dtype, mask="none", order="bshd"):
    c = {"op": "cross", "batch": batch, "queries": queries, "keys": keys, "q_heads": q_heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "dtype": dtype, "mask": mask, "order": order}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token: the launch itself counts
        _rotary("rotary, one token", 1, 1, 16, 4, 64, 64, "bf16"),
        # the tokens of eight 1008-pixel images (72 x 72 patches each)
        _rotary("rotary, image tokens", 8, 5184, 16, 16, 64, 64, "bf16", layout="interleaved"),
        # a long prompt far behind its start, half of each head rotated
        _rotary("rotary, far positions", 5, 1237, 20, 4, 128, 64, "f16", scaling="yarn", factor=8.0, far=200000,
                order="bhsd"),
        # a batch of sequences, one new token each
        _rotary("norm and rotary, single tokens", 64, 1, 32, 8, 128, 128, "bf16", far=4000, op="qk_norm", norm="rms"),
        # image tokens, queries and keys as columns of the fused projection's rows
        _rotary("norm and rotary, fused rows", 16, 5184, 16, 4, 64, 64, "bf16", order="fused", op="qk_norm",
                norm="layer"),
        # 32-bit activations, heads of 80 with 48 of them rotated
        _rotary("norm and rotary, f32", 3, 777, 12, 12, 80, 48, "f32", layout="interleaved", scaling="bands",
                factor=8.0, far=30000, op="qk_norm", norm="rms"),
        # a mask decoder's few tokens over a 64 x 64 feature map
        _cross("cross, mask tokens", 1, 7, 4096, 8, 8, 16, "f16"),
        # single tokens over long states of several lengths, eight query heads to a key head
        _cross("cross, one query, long states", 2, 1, 65521, 32, 4, 128, "bf16", mask="lengths"),
        # a detector's queries over an image's tokens with a position bias
        _cross("cross, detector queries, bias", 4, 201, 5184, 8, 8, 32, "bf16", mask="bias"),
        # image tokens over a padded text
        _cross("cross, image to text", 8, 5184, 77, 8, 8, 32, "bf16", mask="keys", order="bhsd"),
        # shared key heads, heads of 128, a batch of padded states
        _cross("cross, shared heads, lengths", 2, 1729, 6001, 20, 4, 128, "f16", mask="lengths", order="bhsd"),
        # an image's tokens over those of four frames
        _cross("cross, image to frames", 2, 5184, 20736, 16, 16, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most_bytes = max(work(c)["bytes"] for c in listed())
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        if rng.random() < 0.5:
            op = rng.choice(["rotary", "qk_norm"])
            k_heads = rng.choice([1, 2, 4, 8, 12, 16])
            q_heads = k_heads * rng.choice([1, 1, 2, 4, 5, 8])
            head_dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 256])
            rot = head_dim if rng.random() < 0.6 else 2 * rng.randint(4, head_dim // 2)
            scaling = rng.choice(["none", "none", "linear", "ntk", "yarn", "bands"])
            c = _rotary("", _log_int(rng, 1, 64), _log_int(rng, 1, 6000), q_heads, k_heads, head_dim, rot,
                        rng.choice(["bf16", "f16", "f32"]), rng.choice(["half", "interleaved"]), scaling,
                        1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 32])), _log_int(rng, 1, 1000000),
                        rng.choice(["bshd", "bhsd", "fused"]), op,
                        "none" if op == "rotary" else rng.choice(["rms", "layer"]))
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 16])
            q_heads = kv_heads * rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
            c = _cross("", _log_int(rng, 1, 32), _log_int(rng, 1, 6000), _log_int(rng, 1, 70000), q_heads, kv_heads,
                       rng.choice([16, 32, 32, 40, 64, 64, 72, 96, 128, 128]), rng.choice(["bf16", "f16"]),
                       rng.choice(["none", "none", "lengths", "lengths", "keys", "bias"]),
                       rng.choice(["bshd", "bhsd"]))
            if 4 * c["batch"] * q_heads * c["queries"] * c["keys"] > 12e9:  # the plain form's 32-bit scores
                continue
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return c


# ----------------------------------------------------------------- inputs
def _lengths(batch, keys):
    """Valid keys of each sequence of a padded batch: whole, then shorter by even steps; a batch of more than eight
    has an empty one."""
    n = [keys - (b * keys) // (2 * batch) for b in range(batch)]
    if batch > 8:
        n[-1] = 0
    return n


def _holes(length):
    """Masked keys inside a sequence's valid part."""
    return length // 8


def _tensor(gen, batch, tokens, heads, head_dim, dtype, order):
    shape = (batch, heads, tokens, head_dim) if order == "bhsd" else (batch, tokens, heads, head_dim)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(DTYPES[dtype])
    return x.transpose(1, 2) if order == "bhsd" else x


def _inverse_frequencies(c):
    """Angles per position in turns, [rot / 2] in 64 bits, and the amplitude of the rotated part."""
    rot, factor, theta, trained = c["rot"], c["factor"], 10000.0, 4096
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    amplitude = 1.0
    if c["scaling"] == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    w = theta ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        w = w / factor
    elif c["scaling"] == "yarn":
        lo = max(0, math.floor(rot * math.log(trained / (32 * 2 * math.pi)) / (2 * math.log(theta))))
        hi = min(rot - 1, math.ceil(rot * math.log(trained / (1 * 2 * math.pi)) / (2 * math.log(theta))))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        w = w / factor * ramp + w * (1 - ramp)
        amplitude = 0.1 * math.log(factor) + 1.0
    elif c["scaling"] == "bands":
        smooth = ((trained * w / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        w = (1 - smooth) * w / factor + smooth * w
    return w / (2 * math.pi), amplitude


def _plan(c):
    m = _lib()
    return m.RopeFreqs(c["rot"], layout={"half": m.ROPE_HALF, "interleaved": m.ROPE_INTERLEAVED}[c["layout"]],
                       scaling={"none": m.ROPE_SCALE_NONE, "linear": m.ROPE_SCALE_LINEAR, "ntk": m.ROPE_SCALE_NTK,
                                "yarn": m.ROPE_SCALE_YARN, "bands": m.ROPE_SCALE_BANDS}[c["scaling"]],
                       factor=c["factor"], trained_len=4096)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    host = np.random.default_rng(int(seed))
    if c["op"] == "cross":
        q = _tensor(gen, c["batch"], c["queries"], c["q_heads"], c["head_dim"], c["dtype"], c["order"])
        k = _tensor(gen, c["batch"], c["keys"], c["kv_heads"], c["head_dim"], c["dtype"], c["order"])
        v = _tensor(gen, c["batch"], c["keys"], c["kv_heads"], c["head_dim"], c["dtype"], c["order"])
        s = {"case": c, "q": q, "k": k, "v": v, "lengths": None, "keys": None, "bias": None}
        if c["mask"] == "lengths":
            n = host.permutation(_lengths(c["batch"], c["keys"]))
            s["lengths"] = torch.from_numpy(n.astype(np.int32)).cuda()
        elif c["mask"] == "keys":
            m = np.zeros((c["batch"], c["keys"]), np.bool_)
            for row, n in zip(m, host.permutation(_lengths(c["batch"], c["keys"]))):
                row[:n] = True
                row[host.permutation(n)[:_holes(n)]] = False
            s["keys"] = torch.from_numpy(m).cuda()
        elif c["mask"] == "bias":
            s["bias"] = torch.randn((c["batch"], c["q_heads"], c["queries"], c["keys"]), generator=gen, device="cuda")
        return s
    hq, hk, hd = c["q_heads"], c["k_heads"], c["head_dim"]
    if c["order"] == "fused":  # rows of queries, keys and values
        rows = _tensor(gen, c["batch"], c["tokens"], hq + 2 * hk, hd, c["dtype"], "bshd")
        q, k = rows[:, :, :hq], rows[:, :, hq:hq + hk]
    else:
        q = _tensor(gen, c["batch"], c["tokens"], hq, hd, c["dtype"], c["order"])
        k = _tensor(gen, c["batch"], c["tokens"], hk, hd, c["dtype"], c["order"])
    turns, amplitude = _inverse_frequencies(c)
    first = torch.from_numpy(host.integers(0, c["far"] + 1, (c["batch"], 1))).cuda()
    s = {"case": c, "q": q, "k": k, "turns": turns, "amplitude": amplitude,
         "positions": first + torch.arange(c["tokens"], device="cuda")[None],
         "plan": _plan(c) if own else None}
    if c["op"] == "qk_norm":
        for n in ("q", "k"):
            s[n + "_gamma"] = 1.0 + 0.1 * torch.randn(hd, generator=gen, device="cuda")
            s[n + "_beta"] = 0.1 * torch.randn(hd, generator=gen, device="cuda") if c["norm"] == "layer" else None
    return s


# ------------------------------------------------------------- plain form
def _rotated(x, cos, sin, c):
    """x [batch, tokens, heads, head_dim] in 32 bits, cos and sin [batch, tokens, 1, rot / 2]."""
    rot = c["rot"]
    part = x[..., :rot]
    if c["layout"] == "half":
        u, w = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((u * cos - w * sin, u * sin + w * cos), -1)
    else:
        u, w = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((u * cos - w * sin, u * sin + w * cos), -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _normed(x, gamma, beta, c):
    if c["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
    return x if beta is None else x + beta


def _plain_rotary(s):
    c = s["case"]
    angle = (2 * math.pi) * torch.frac(s["positions"].double()[..., None, None] * s["turns"])
    cos, sin = (s["amplitude"] * angle.cos()).float(), (s["amplitude"] * angle.sin()).float()
    q, k = s["q"].float(), s["k"].float()
    if c["op"] == "qk_norm":
        q, k = _normed(q, s["q_gamma"], s["q_beta"], c), _normed(k, s["k_gamma"], s["k_beta"], c)
    return tuple(_rotated(x, cos, sin, c).to(s["q"].dtype) for x in (q, k))


def _plain_cross(s):
    c = s["case"]
    group = c["q_heads"] // c["kv_heads"]
    q = s["q"].float().transpose(1, 2).unflatten(1, (c["kv_heads"], group)) * c["head_dim"] ** -0.5
    k, v = s["k"].float().transpose(1, 2)[:, :, None], s["v"].float().transpose(1, 2)[:, :, None]
    scores = torch.matmul(q, k.transpose(-1, -2))  # [batch, kv_heads, group, queries, keys]
    if s["bias"] is not None:
        scores += s["bias"].unflatten(1, (c["kv_heads"], group))
    valid = s["keys"]
    if s["lengths"] is not None:
        valid = torch.arange(c["keys"], device="cuda")[None] < s["lengths"][:, None]
    if valid is not None:
        scores.masked_fill_(~valid[:, None, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    o = torch.matmul(scores, v) / total.masked_fill(total == 0, 1.0)
    return o.flatten(1, 2).transpose(1, 2).to(s["q"].dtype)


# -------------------------------------------------------------------- run
def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_cross(s) if c["op"] == "cross" else _plain_rotary(s)
    m = _lib()
    if c["op"] == "cross":
        return m.cross_attention(s["q"], s["k"], s["v"], k_lens=s["lengths"], key_mask=s["keys"], bias=s["bias"])
    if c["op"] == "rotary":
        return m.rope_pos(s["q"], s["plan"], s["positions"], k=s["k"])
    return m.qk_norm_rope(s["q"], s["k"], s["q_gamma"], s["k_gamma"], q_beta=s["q_beta"], k_beta=s["k_beta"],
                          norm=m.NORM_LAYER if c["norm"] == "layer" else m.NORM_RMS, eps=1e-6, freqs=s["plan"],
                          positions=s["positions"])


def work(case):
    c = case
    es = BYTES[c["dtype"]]
    if c["op"] != "cross":
        n = c["batch"] * c["tokens"] * (c["q_heads"] + c["k_heads"]) * c["head_dim"]
        return {"bytes": 2 * es * n + 8 * c["batch"] * c["tokens"], "flops": (3 if c["op"] == "rotary" else 7) * n}
    valid = c["batch"] * c["keys"]
    if c["mask"] in ("lengths", "keys"):
        n = _lengths(c["batch"], c["keys"])
        valid = sum(x - (_holes(x) if c["mask"] == "keys" else 0) for x in n)
    rows = c["q_heads"] * c["queries"]
    extra = {"bias": 4 * rows * c["batch"] * c["keys"], "keys": c["batch"] * c["keys"], "lengths": 4 * c["batch"],
             "none": 0}[c["mask"]]
    return {"bytes": 2 * es * c["batch"] * rows * c["head_dim"] + 2 * es * valid * c["kv_heads"] * c["head_dim"] + extra,
            "flops": 4 * valid * rows * c["head_dim"]}


# ------------------------------------------------------------------ exact
def _exact_turns(c):
    """The definition, frequency by frequency, with Python's floats."""
    rot, out = c["rot"], []
    base = 10000.0
    if c["scaling"] == "ntk" and rot > 2:
        base *= c["factor"] ** (rot / (rot - 2))
    for i in range(rot // 2):
        f = base ** (-(2 * i) / rot)
        if c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "yarn":
            def index_of(turns):  # the dimension that makes so many turns over the trained length
                return rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
            lo, hi = max(math.floor(index_of(32)), 0), min(math.ceil(index_of(1)), rot - 1)
            t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = t * (f / c["factor"]) + (1 - t) * f
        elif c["scaling"] == "bands":
            length = 2 * math.pi / f
            if length > 4096 / 1.0:
                f = f / c["factor"]
            elif length >= 4096 / 4.0:
                t = (4096 / length - 1.0) / 3.0
                f = (1 - t) * f / c["factor"] + t * f
        out.append(f / (2 * math.pi))
    return np.array(out), (0.1 * math.log(c["factor"]) + 1.0) if c["scaling"] == "yarn" else 1.0


def _exact_rotary(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    turns, amplitude = _exact_turns(c)
    at = s["positions"].double()[:, :, None] * torch.from_numpy(turns).cuda()
    angle = (at - at.round()) * 2 * math.pi
    cos, sin = (f(angle)[:, :, None] * amplitude for f in (torch.cos, torch.sin))
    first = torch.arange(half, device="cuda") * (1 if c["layout"] == "half" else 2)
    second = first + (half if c["layout"] == "half" else 1)
    out = []
    for n in ("q", "k"):
        x = s[n].double()
        if c["op"] == "qk_norm":
            if c["norm"] == "layer":
                var, mean = torch.var_mean(x, -1, keepdim=True, correction=0)
                x = (x - mean) / torch.sqrt(var + 1e-6) * s[n + "_gamma"].double() + s[n + "_beta"].double()
            else:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["head_dim"] + 1e-6) * s[n + "_gamma"].double()
        y = x.clone()
        y[..., first] = x[..., first] * cos - x[..., second] * sin
        y[..., second] = x[..., second] * cos + x[..., first] * sin
        out.append(y)
    return tuple(out)


def _exact_cross(s):
    """Head by head over the keys that count."""
    c = s["case"]
    out = torch.zeros((c["batch"], c["queries"], c["q_heads"], c["head_dim"]), dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        keep = torch.arange(c["keys"], device="cuda")
        if s["lengths"] is not None:
            keep = keep[:int(s["lengths"][b])]
        if s["keys"] is not None:
            keep = keep[s["keys"][b]]
        if not len(keep):
            continue
        for h in range(c["q_heads"]):
            at = h // (c["q_heads"] // c["kv_heads"])
            scores = s["q"][b, :, h].double() @ s["k"][b, keep, at].double().T / math.sqrt(c["head_dim"])
            if s["bias"] is not None:
                scores += s["bias"][b, h][:, keep].double()
            out[b, :, h] = torch.softmax(scores, -1) @ s["v"][b, keep, at].double()
    return out


def exact(case, seed):
    if work(case)["flops"] > 2e12:
        return None
    s = prepare(case, seed)
    return _exact_cross(s) if case["op"] == "cross" else _exact_rotary(s)
