"""GPU parity of the rotary positions and the head norms against their
formulas in 64 bits, element by element.

Tolerances, per element: half a step of the output type (eps/2 of the
value, the smallest subnormal's half below the normal range) for the one
rounding, plus the F32 work before it: the angle (2^-23 of a revolution's
2 pi, so 2^-20), cosine, sine, two products and a sum stay below 2^-19 of
|u| + |w|; a norm adds (n + 16) 2^-23 of the head's largest normalised
value (sums of n squares and of n elements, one root, one division)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = ("bf16", "f16", "f32")


def _torch_dtype(dt):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dt]


def _tensor(shape, dt, seed, order="bshd"):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, s, h, d = shape
    x = torch.randn((b, h, s, d) if order == "bhsd" else shape, generator=g, device="cuda").to(_torch_dtype(dt))
    return x.transpose(1, 2) if order == "bhsd" else x


def _norm64(x, norm, gamma, beta, eps):
    import torch
    if norm == 2:
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if gamma is not None:
        x = x * gamma.double()
    return x if beta is None else x + beta.double()


def _rotate64(x, freqs, pos, half):
    """x float64 [b, s, h, d], pos float64 [b, s]; the rotation and |u| + |w| per element."""
    import torch
    if freqs is None:
        return x, torch.zeros_like(x)
    n = len(freqs.turns)
    t = pos[:, :, None, None] * torch.from_numpy(freqs.turns).cuda()
    a = (t - t.round()) * 2 * math.pi
    cos, sin = a.cos() * freqs.amplitude, a.sin() * freqs.amplitude
    i = torch.arange(n, device="cuda")
    iu, iw = (i, i + n) if half else (2 * i, 2 * i + 1)
    u, w = x[..., iu], x[..., iw]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., iu], y[..., iw] = u * cos - w * sin, u * sin + w * cos
    size[..., iu] = size[..., iw] = (u.abs() + w.abs()) * freqs.amplitude
    return y, size


def _within(y, ref, slack):
    import torch
    fi = torch.finfo(y.dtype)
    tol = torch.maximum(ref.abs() * (fi.eps / 2), torch.full_like(ref, fi.tiny * fi.eps / 2)) + slack
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def _check(shape, kh, dt, rot, half, norm=0, far=1000, seed=0, order="bshd", affine=True, scaling=0, inplace=False,
           per_batch=True):
    import torch
    import sam3cu
    b, s, h, d = shape
    q, k = _tensor(shape, dt, seed, order), _tensor((b, s, kh, d), dt, seed + 1, order)
    freqs = sam3cu.RopeFreqs(rot, layout=1 if half else 0, scaling=scaling, factor=8.0) if rot else None
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    pos = torch.randint(-far, far + 1, (b, s) if per_batch else (s,), generator=g, device="cuda")
    par = {}
    if norm and affine:
        for n in ("q", "k"):
            par[n + "_gamma"] = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
            par[n + "_beta"] = 0.2 * torch.randn(d, generator=g, device="cuda")
    ref = []
    for n, x in (("q", q), ("k", k)):
        x, scale = x.double(), torch.zeros((), device="cuda", dtype=torch.float64)
        if norm:
            x = _norm64(x, norm, par.get(n + "_gamma"), par.get(n + "_beta"), 1e-6)
            scale = (d + 16) * 2.0 ** -23 * x.abs().amax(-1, keepdim=True) * 2
        y, size = _rotate64(x, freqs, pos.double() if per_batch else pos.double()[None], half)
        ref.append((y, size * 2.0 ** -19 + scale))
    out = dict(out=q, k_out=k) if inplace else {}
    if norm:
        got = sam3cu.qk_norm_rope(q, k, norm=norm, freqs=freqs, positions=pos, **par, **out)
    else:
        got = sam3cu.rope_pos(q, freqs, pos, k=k, **out)
    torch.cuda.synchronize()
    for y, (r, slack) in zip(got, ref):
        _within(y, r, slack)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 32), (128, 128), (128, 64), (32, 32), (16, 16), (80, 48), (96, 96),
                                    (256, 256), (240, 16), (64, 2), (64, 50), (72, 72), (40, 8), (2, 2), (7, 4),
                                    (130, 66), (255, 254), (96, 70), (128, 18), (256, 250),
                                    (48, 34), (80, 20)])
def test_rope(cuda, dt, half, hd, rot):
    _check((3, 5, 6, hd), 2, dt, rot, half, seed=hd + rot)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("norm", [1, 2])
@pytest.mark.parametrize("hd,rot,half", [(64, 64, True), (64, 64, False), (128, 64, True), (80, 48, False), (32, 0, True),
                                         (256, 128, True), (72, 40, True), (7, 2, False), (1, 0, True), (250, 0, True),
                                         (16, 16, True), (96, 70, True), (96, 70, False), (256, 250, True),
                                         (48, 2, True), (16, 6, True), (128, 36, False)])
def test_norm(cuda, dt, norm, hd, rot, half):
    _check((2, 7, 5, hd), 3, dt, rot, half, norm=norm, seed=hd + rot)


@pytest.mark.parametrize("order", ["bshd", "bhsd"])
@pytest.mark.parametrize("norm", [0, 1])
@pytest.mark.parametrize("shape,kh", [((1, 1, 1, 64), 1), ((1, 1, 128, 64), 16), ((1, 1201, 20, 128), 4), ((64, 1, 33, 64), 1),
                                      ((2, 5184, 16, 64), 16)])
def test_sizes(cuda, order, norm, shape, kh):
    _check(shape, kh, "bf16", 64, True, norm=norm, order=order, far=10 ** 6, seed=5)


@pytest.mark.parametrize("norm", [0, 1])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 32), (72, 20), (96, 70), (256, 4)])
@pytest.mark.parametrize("order", ["bshd", "bhsd"])
def test_in_place(cuda, norm, hd, rot, order):
    _check((2, 9, 4, hd), 2, "f16", rot, True, norm=norm, inplace=True, order=order)


@pytest.mark.parametrize("scaling", range(5))
def test_scalings(cuda, scaling):
    _check((2, 33, 4, 64), 2, "f32", 64, True, scaling=scaling, far=10 ** 5)


def test_shared_positions_and_no_affine(cuda):
    _check((3, 9, 4, 64), 2, "bf16", 64, True, per_batch=False)
    _check((3, 9, 4, 64), 2, "f32", 64, True, norm=2, affine=False)


def test_far_positions_f32(cuda):
    """At 2^40 positions the angle still has 2^-13 of a revolution in 64 bits
    (53 bits of a 40-bit count); the formula above makes the same product."""
    _check((2, 4, 4, 64), 2, "f32", 64, True, far=2 ** 40)


def test_start_counts_tokens(cuda):
    import torch
    import sam3cu
    q = _tensor((2, 11, 3, 64), "f32", 1)
    f = sam3cu.RopeFreqs(64)
    pos = torch.arange(11, device="cuda") + 1234567
    assert torch.equal(sam3cu.rope_pos(q, f, start=1234567), sam3cu.rope_pos(q, f, pos))


def test_negative_positions_undo(cuda):
    """Rotation by p and then by -p: two roundings, F32."""
    import torch
    import sam3cu
    q = _tensor((2, 50, 3, 64), "f32", 2)
    f = sam3cu.RopeFreqs(64, layout=sam3cu.ROPE_INTERLEAVED)
    pos = torch.arange(50, device="cuda") * 977
    back = sam3cu.rope_pos(sam3cu.rope_pos(q, f, pos), f, -pos)
    assert float((back - q).abs().max()) <= 2.0 ** -18 * 2 * float(q.abs().max())


def test_fused_rows(cuda):
    """Queries and keys as columns of a projection's rows, and their values
    and everything around left as they were."""
    import torch
    import sam3cu
    rows = _tensor((2, 13, 16 + 4 + 4, 64), "bf16", 3)
    before = rows.clone()
    f = sam3cu.RopeFreqs(64)
    q, k = rows[:, :, :16], rows[:, :, 16:20]
    want = sam3cu.qk_norm_rope(q.contiguous(), k.contiguous(), freqs=f)
    sam3cu.qk_norm_rope(q, k, freqs=f, out=q, k_out=k)
    assert torch.equal(rows[:, :, :16], want[0]) and torch.equal(rows[:, :, 16:20], want[1])
    assert torch.equal(rows[:, :, 20:], before[:, :, 20:])


def test_misaligned_rows(cuda):
    """Rows that start on 2 bytes only."""
    import torch
    import sam3cu
    buf = torch.randn(2 * 5 * 3 * 65 + 1, device="cuda").bfloat16()
    q = buf[1:].view(2, 5, 3, 65)[..., :64]
    f = sam3cu.RopeFreqs(64)
    assert torch.equal(sam3cu.rope_pos(q, f), sam3cu.rope_pos(q.contiguous(), f))


def test_expanded_input(cuda):
    import torch
    import sam3cu
    x = _tensor((1, 6, 2, 64), "bf16", 4)
    f = sam3cu.RopeFreqs(64)
    assert torch.equal(sam3cu.rope_pos(x.expand(3, 6, 2, 64), f), sam3cu.rope_pos(x, f).expand(3, 6, 2, 64))


def test_empty(cuda):
    import torch
    import sam3cu
    f = sam3cu.RopeFreqs(64)
    x = torch.zeros(0, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    assert sam3cu.rope_pos(x, f).shape == x.shape
    x = torch.zeros(2, 4, 0, 64, device="cuda", dtype=torch.bfloat16)
    assert sam3cu.qk_norm_rope(x, x)[1].shape == x.shape


def test_zero_and_infinite_heads(cuda):
    """A head of zeros stays zero (eps keeps the root off 0); infinities stay
    in their own head, and out of elements that do not rotate."""
    import torch
    import sam3cu
    x = torch.zeros(1, 1, 3, 64, device="cuda")
    x[0, 0, 1] = torch.randn(64, device="cuda")
    x[0, 0, 2, 5] = float("inf")
    f = sam3cu.RopeFreqs(32)
    y = sam3cu.qk_norm_rope(x, None, freqs=f, start=7)
    assert bool((y[0, 0, 0] == 0).all()) and bool(torch.isfinite(y[0, 0, 1]).all())
    z = sam3cu.rope_pos(x, f, start=7)
    assert torch.equal(z[0, 0, 2, 32:], x[0, 0, 2, 32:]) and bool(torch.isfinite(z[0, 0, :2]).all())


def test_wrapper_refusals(cuda):
    import torch
    import sam3cu
    f = sam3cu.RopeFreqs(64)
    x = _tensor((2, 4, 2, 64), "bf16", 6)
    for bad in (lambda: sam3cu.rope_pos(x, f, torch.zeros(2, 4, device="cuda", dtype=torch.int32)),
                lambda: sam3cu.rope_pos(x, f, torch.zeros(3, 4, device="cuda", dtype=torch.int64)),
                lambda: sam3cu.rope_pos(x, f, torch.zeros(2, 5, device="cuda", dtype=torch.int64)),
                lambda: sam3cu.rope_pos(x, f, torch.zeros(2, 4, dtype=torch.int64)),
                lambda: sam3cu.rope_pos(x, f, k=x.half()),
                lambda: sam3cu.rope_pos(x, f, k=x[:, :3]),
                lambda: sam3cu.rope_pos(x, f, out=x.float()),
                lambda: sam3cu.rope_pos(x.transpose(2, 3), f),
                lambda: sam3cu.qk_norm_rope(x, x, q_gamma=torch.ones(32, device="cuda")),
                lambda: sam3cu.rope_pos(x[0], f)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        sam3cu.qk_norm_rope(x, x, q_gamma=torch.ones(64, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(sam3cu.Sam3cuError):
        sam3cu.rope_pos(x[..., :32], f)
    with pytest.raises(sam3cu.Sam3cuError):
        sam3cu.rope_pos(x, f, out=x.new_empty(64).expand(2, 4, 2, 64))


def test_captured_and_other_stream(cuda):
    import torch
    import sam3cu
    f = sam3cu.RopeFreqs(64)
    q = _tensor((4, 3, 8, 64), "bf16", 7)
    out, pos = torch.empty_like(q), torch.zeros(4, 3, device="cuda", dtype=torch.int64)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        with torch.cuda.graph(g, stream=st):
            sam3cu.rope_pos(q, f, pos, out=out)
    for n in (0, 77):
        q.copy_(_tensor((4, 3, 8, 64), "bf16", 8 + n))
        pos.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sam3cu.rope_pos(q, f, pos))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("norm", [0, 2])
@pytest.mark.parametrize("hd", [48, 80, 96, 112, 144, 160, 176, 192, 208, 224, 240])
def test_exchange_with_lanes_left_over(cuda, dt, norm, hd):
    """Halves that are not multiples of 8 elements go through shared memory;
    where head_dim / 16 is no power of two some lanes of a group hold no part
    of the head and must leave its words to the lanes that do."""
    _check((3, 41, 9, hd), 5, dt, hd - 2, True, norm=norm, seed=hd)
    _check((3, 41, 9, hd), 5, dt, hd // 2 + 2 - hd // 2 % 2, True, norm=norm, seed=hd, inplace=True)


@pytest.mark.parametrize("norm", [0, 1, 2])
@pytest.mark.parametrize("hd,rot", [(64, 64), (80, 20), (72, 40)])
def test_heads_of_k_alone(cuda, norm, hd, rot):
    """No heads of q, with and without memory of its own; the result is that
    of the same heads taken as q's."""
    import torch
    import sam3cu
    x, f = _tensor((3, 17, 5, hd), "bf16", 9), sam3cu.RopeFreqs(rot)
    gamma = 1 + 0.1 * torch.arange(hd, device="cuda", dtype=torch.float32) / hd
    for none in (x[:, :, :0], torch.empty(3, 17, 0, hd, device="cuda", dtype=x.dtype)):
        if norm:
            want = sam3cu.qk_norm_rope(x, None, gamma, norm=norm, freqs=f, start=3)
            q, k = sam3cu.qk_norm_rope(none, x, None, gamma, norm=norm, freqs=f, start=3)
        else:
            want = sam3cu.rope_pos(x, f, start=3)
            q, k = sam3cu.rope_pos(none, f, start=3, k=x)
        assert q.shape == (3, 17, 0, hd) and torch.equal(k, want)


@pytest.mark.parametrize("norm", [0, 1])
@pytest.mark.parametrize("hd,rot", [(64, 64), (80, 20), (72, 40)])
def test_offsets_past_32_bits(cuda, norm, hd, rot):
    """Tokens that begin beyond 2^32 bytes (and 2^31 elements) into the input
    and the output, with heads of q and k side by side."""
    import torch
    import sam3cu
    tokens, pitch = 1100, 1 << 21
    f = sam3cu.RopeFreqs(rot)
    small = _tensor((1, tokens, 4, hd), "bf16", 10)
    big = torch.empty(tokens * pitch, dtype=torch.bfloat16, device="cuda").as_strided((1, tokens, 4, hd),
                                                                                      (0, pitch, hd, 1))
    out = torch.empty(tokens * pitch, dtype=torch.bfloat16, device="cuda").as_strided((1, tokens, 4, hd),
                                                                                      (0, pitch, hd, 1))
    big.copy_(small)

    def call(x, **out):
        if norm:
            return sam3cu.qk_norm_rope(x[:, :, :3], x[:, :, 3:], freqs=f, start=9, **out)
        return sam3cu.rope_pos(x[:, :, :3], f, start=9, k=x[:, :, 3:], **out)
    want = call(small)
    call(big, out=out[:, :, :3], k_out=out[:, :, 3:])
    assert torch.equal(out[:, :, :3], want[0]) and torch.equal(out[:, :, 3:], want[1])
    call(big, out=big[:, :, :3], k_out=big[:, :, 3:])
    assert torch.equal(big[:, :, :3], want[0]) and torch.equal(big[:, :, 3:], want[1])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("norm", [0, 1])
def test_rows_aligned_to_an_element(cuda, dt, norm):
    """Inputs and outputs whose rows start on one element's size only."""
    import torch
    import sam3cu
    f = sam3cu.RopeFreqs(64)
    buf, back = (torch.randn(2 * 5 * 3 * 65 + 1, device="cuda").to(_torch_dtype(dt)) for _ in range(2))
    q, out = buf[1:].view(2, 5, 3, 65)[..., :64], back[1:].view(2, 5, 3, 65)
    rest = out[..., 64].clone()
    # (products and sums in another order than in the kernel of aligned rows: against the formula)
    x, slack = q.double(), 0.0
    if norm:
        sam3cu.qk_norm_rope(q, None, freqs=f, start=2, out=out[..., :64])
        x = _norm64(x, 1, None, None, 1e-6)
        slack = (64 + 16) * 2.0 ** -23 * x.abs().amax(-1, keepdim=True) * 2
    else:
        sam3cu.rope_pos(q, f, start=2, out=out[..., :64])
    ref, size = _rotate64(x, f, (torch.arange(5, device="cuda", dtype=torch.float64) + 2)[None], True)
    _within(out[..., :64], ref, size * 2.0 ** -19 + slack)
    assert torch.equal(out[..., 64], rest)
