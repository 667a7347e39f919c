"""GPU parity of the cross attention against its formula in 64 bits, element
by element.

Tolerance of an element: with e = eps/2 of the type (half a step), A = sum_j
p_j |v_j| / sum_j p_j and d = head_dim 2^-23 max_j scale sum |q||k_j| (the
F32 accumulation of a score, twice 2^-24 for the tensor cores' truncation),
  e |o|                 the output's rounding
  + e A                 P rounded to the type before P.V
  + 2 d A               a score off by d moves p_j / sum p by a factor e^(2d)
  + 2^-18 A             exponentials, sums over keys and the division in F32
and for f16, whose P below 2^-14 has steps of 2^-24: 2^-25 sum_j |v_j| / sum p."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def _make(b, sq, sk, hq, hkv, hd, dt, seed=0, order="bshd", sharp=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(s, h, f=1.0):
        x = torch.randn((b, h, s, hd) if order == "bhsd" else (b, s, h, hd), generator=g, device="cuda") * f
        x = x.to(_dt(dt))
        return x.transpose(1, 2) if order == "bhsd" else x
    return one(sq, hq, sharp), one(sk, hkv), one(sk, hkv)


def _reference(q, k, v, k_lens=None, key_mask=None, bias=None, scale=0.0):
    """o and the tolerance, float64 [b, sq, hq, hd]."""
    import torch
    b, sq, hq, hd = q.shape
    sk, g = k.shape[1], hq // k.shape[2]
    scale = scale or 1 / math.sqrt(hd)
    half = torch.finfo(q.dtype).eps / 2
    o = torch.zeros(b, sq, hq, hd, dtype=torch.float64, device=q.device)
    tol = torch.full_like(o, torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps / 2)
    full = None if bias is None else bias.expand(b, hq, sq, sk)
    for i in range(b):
        keep = torch.ones(sk, dtype=torch.bool, device=q.device)
        if k_lens is not None:
            keep &= torch.arange(sk, device=q.device) < k_lens[i]
        if key_mask is not None:
            keep &= key_mask[i if key_mask.shape[0] > 1 else 0] != 0
        if not bool(keep.any()):
            continue
        for h in range(hq):
            kk, vv = k[i, keep, h // g].double(), v[i, keep, h // g].double()
            s = q[i, :, h].double() @ kk.T * scale
            d = hd * 2.0 ** -23 * (q[i, :, h].double().abs() @ kk.abs().T * scale).amax(-1, keepdim=True)
            if full is not None:
                s = s + full[i, h][:, keep].double()
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
            l = p.sum(-1, keepdim=True)
            dead = l == 0
            l = torch.where(dead, torch.ones_like(l), l)
            a = p @ vv.abs() / l
            o[i, :, h] = p @ vv / l
            tol[i, :, h] += half * o[i, :, h].abs() + (half + 2 * d + 2.0 ** -18) * a
            if q.dtype == torch.float16:
                tol[i, :, h] += 2.0 ** -25 * vv.abs().sum(0) / l
    return o, tol


def _check(q, k, v, **kw):
    import torch
    import sam3cu
    o = sam3cu.cross_attention(q, k, v, **kw)
    torch.cuda.synchronize()
    assert sam3cu.device_error() == 0
    ref, tol = _reference(q, k, v, **kw)
    off = (o.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    return o


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [8, 16, 32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 257), (7, 64), (16, 129), (17, 33), (64, 65), (130, 300), (300, 130),
                                   (257, 1000)])
def test_sizes(cuda, dt, hd, sq, sk):
    _check(*_make(2, sq, sk, 3, 3, hd, dt, seed=sq + sk))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv", [(8, 1), (6, 2), (5, 1), (32, 4), (16, 16), (128, 1), (100, 1), (96, 3)])
@pytest.mark.parametrize("sq,sk", [(1, 1111), (3, 70), (77, 200), (201, 700)])
def test_shared_heads(cuda, dt, hq, hkv, sq, sk):
    _check(*_make(2, sq, sk, hq, hkv, 64, dt, seed=hq, order="bhsd"))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq", [1, 40, 500])
def test_lengths(cuda, hd, sq):
    import torch
    lens = [0, 1, 63, 64, 65, 127, 128, 129, 300, 999, 1000, 2000, -5]
    q, k, v = _make(len(lens), sq, 1000, 4, 2, hd, "bf16", seed=sq)
    o = _check(q, k, v, k_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert bool((o[0] == 0).all()) and bool((o[-1] == 0).all())


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq,sk", [(1, 77), (9, 1000), (100, 513), (400, 77), (300, 2100)])
def test_key_mask(cuda, hd, sq, sk):
    import torch
    q, k, v = _make(6, sq, sk, 4, 4, hd, "f16", seed=sk)
    g = torch.Generator(device="cuda").manual_seed(3)
    mask = torch.rand(6, sk, generator=g, device="cuda") < 0.5
    mask[1] = True
    mask[2] = False                       # nothing left
    mask[3, : sk - 1] = False             # the last key alone
    mask[4, min(128, sk // 2):] = False   # a padded end
    mask[5, : sk // 2] = False            # a padded beginning
    o = _check(q, k, v, key_mask=mask)
    assert bool((o[2] == 0).all())
    _check(q, k, v, key_mask=mask[:1])    # shared by the batch
    _check(q, k, v, key_mask=mask.to(torch.uint8) * 255,
           k_lens=torch.tensor([sk, sk // 2, sk, sk, 1, sk], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq", [1, 60, 333])
def test_padding_may_hold_anything(cuda, hd, sq):
    """Infinities and NaN in the K and V rows of keys that do not count."""
    import torch
    sk = 700
    q, k, v = _make(3, sq, sk, 2, 2, hd, "bf16", seed=1)
    lens = torch.tensor([700, 333, 0], dtype=torch.int32, device="cuda")
    mask = torch.ones(3, sk, dtype=torch.bool, device="cuda")
    mask[0, 100:200] = False
    mask[0, 513] = False
    want = _check(q, k, v, k_lens=lens, key_mask=mask)
    for x in (k, v):
        x[0, 100:150] = float("nan")
        x[0, 150:200] = float("inf")
        x[0, 513] = -float("inf")
        x[1, 333:] = float("nan")
        x[2] = float("nan")
    import sam3cu
    assert torch.equal(sam3cu.cross_attention(q, k, v, k_lens=lens, key_mask=mask), want)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq,sk", [(1, 300), (5, 1027), (201, 517), (300, 129)])
def test_bias(cuda, hd, sq, sk):
    import torch
    q, k, v = _make(2, sq, sk, 4, 2, hd, "bf16", seed=9)
    g = torch.Generator(device="cuda").manual_seed(4)
    bias = torch.randn(2, 4, sq, sk, generator=g, device="cuda") * 2
    _check(q, k, v, bias=bias)
    for part in (bias[:1], bias[:, :1], bias[:, :, :1], bias[0, 0], bias[0, 0, 0]):
        _check(q, k, v, bias=part)
    wide = torch.randn(2, 4, sq, sk + 3, generator=g, device="cuda")
    _check(q, k, v, bias=wide[..., 1: sk + 1], k_lens=torch.tensor([sk, sk // 3], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("sq", [1, 200])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_rows_without_keys(cuda, sq, low):
    """-inf leaves rows empty (zeros); the type's lowest value on a whole row
    leaves its scores as they round beside it: equal, the mean of V."""
    import torch
    q, k, v = _make(1, sq, 500, 2, 2, 64, "f16", seed=5)
    value = -math.inf if low == "inf" else torch.finfo(torch.float32).min
    bias = torch.zeros(1, 2, sq, 500, device="cuda")
    bias[0, 0, 0] = value              # a whole row
    bias[0, 1, :, 100:] = value        # all but 100 keys
    o = _check(q, k, v, bias=bias)
    if low == "inf":
        assert bool((o[0, 0, 0] == 0).all())
    else:
        mean = v[0, :, 0].double().mean(0)
        assert float((o[0, 0, 0].double() - mean).abs().max()) <= 2.0 ** -11 * (
            float(mean.abs().max()) + float(v[0, :, 0].double().abs().mean(0).max()))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("sq", [1, 20, 300])
def test_sharp_and_growing_scores(cuda, dt, sq):
    """Scores of some hundreds that grow along the keys: every tile raises
    the running maximum."""
    import torch
    q, k, v = _make(1, sq, 1500, 2, 2, 64, dt, seed=6, sharp=2.0)
    k = (k.double() * torch.linspace(0.1, 8, 1500, device="cuda", dtype=torch.float64)[None, :, None, None]).to(k.dtype)
    _check(q, k, v)
    _check(q, k.flip(1), v)  # and falling ones


@pytest.mark.parametrize("sq", [1, 150])
def test_equal_large_scores(cuda, sq):
    """One value for all scores, 10^4: the softmax is uniform."""
    import torch
    q, k, v = _make(1, sq, 999, 1, 1, 64, "bf16", seed=7)
    q[:] = 40.0
    k[:] = 31.25
    _check(q, k, v)


@pytest.mark.parametrize("sq", [1, 70, 400])
def test_strides(cuda, sq):
    """States shared by a batch, heads expanded, columns of wider rows, a
    given output with gaps that stay as they are."""
    import torch
    import sam3cu
    q, k, v = _make(1, sq, 300, 4, 4, 64, "bf16", seed=8)
    q = q.expand(3, sq, 4, 64)
    _check(q, k.expand(3, 300, 4, 64), v.expand(3, 300, 4, 64))
    _check(q, k[:, :, :1].expand(3, 300, 4, 64), v[:, :, 1:2].expand(3, 300, 4, 64))
    rows = torch.randn(2, 300, 4 + 4, 72, device="cuda").half()
    q2 = torch.randn(2, sq, 6, 72, device="cuda").half()
    kk, vv = rows[:, :, :4, :64], rows[:, :, 4:, :64]
    out = torch.full((2, sq + 3, 6, 72), 7.0, device="cuda").half()
    got = _check(q2[:, :, 1:5, 8:], kk, vv)
    sam3cu.cross_attention(q2[:, :, 1:5, 8:], kk, vv, out=out[:, :sq, 1:5, :64])
    assert torch.equal(out[:, :sq, 1:5, :64], got)
    out[:, :sq, 1:5, :64] = 7.0
    assert bool((out == 7.0).all())


def test_scale(cuda):
    q, k, v = _make(2, 50, 200, 2, 2, 64, "bf16", seed=10)
    _check(q, k, v, scale=1.0)
    _check(q, k, v, scale=1e-3)


@pytest.mark.parametrize("sq", [1, 5, 300])
def test_no_keys(cuda, sq):
    import sam3cu
    q, k, v = _make(2, sq, 0, 2, 2, 64, "bf16")
    assert bool((sam3cu.cross_attention(q, k, v) == 0).all())
    assert sam3cu.cross_attention(q[:, :0], k, v).shape == (2, 0, 2, 64)


def test_nan_query_stays_in_its_row(cuda):
    import torch
    import sam3cu
    for sq in (3, 300):
        q, k, v = _make(1, sq, 600, 2, 2, 64, "bf16", seed=11)
        want = sam3cu.cross_attention(q, k, v)
        q[0, 1, 1] = float("nan")
        got = sam3cu.cross_attention(q, k, v)
        assert bool(got[0, 1, 1].isnan().all())
        got[0, 1, 1] = want[0, 1, 1]
        assert torch.equal(got, want)


@pytest.mark.parametrize("b,sq,sk,hq,hkv,hd,dt", [(1, 1, 70001, 8, 2, 128, "bf16"), (4, 7, 4096, 8, 8, 16, "f16"),
                                                  (1, 2047, 5184, 4, 4, 64, "bf16"), (2, 600, 2500, 10, 2, 128, "f16"),
                                                  (200, 1, 33, 8, 8, 64, "bf16"), (1, 5184, 32, 8, 8, 32, "f16"),
                                                  (1, 40, 20000, 1, 1, 128, "bf16")])
def test_long_and_many(cuda, b, sq, sk, hq, hkv, hd, dt):
    _check(*_make(b, sq, sk, hq, hkv, hd, dt, seed=12))


@pytest.mark.parametrize("hd,dt", [(32, "f16"), (64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("sq,hq,hkv", [(1, 8, 2), (16, 1, 1), (5, 8, 1)])
def test_few_rows_over_long_states(cuda, hd, dt, sq, hq, hkv):
    """Keys split over all SMs and joined by a second launch: lengths (an empty
    sequence among them), a mask that leaves whole splits out, a bias."""
    import torch
    sk = (24 << 20) // (4 * hd * hkv * 3) // 8 * 8 + 13
    q, k, v = _make(3, sq, sk, hq, hkv, hd, dt, seed=sq)
    _check(q, k, v)
    o = _check(q, k, v, k_lens=torch.tensor([sk, 0, 700], dtype=torch.int32, device="cuda"))
    assert bool((o[1] == 0).all())
    mask = torch.zeros(3, sk, dtype=torch.bool, device="cuda")
    mask[0, -1] = True
    mask[1, 100:sk // 2: 3] = True
    _check(q, k, v, key_mask=mask)
    _check(q, k, v, bias=torch.randn(1, hq, 1, sk, device="cuda"))


@pytest.mark.parametrize("sq", [1, 300])
def test_offsets_past_32_bits(cuda, sq):
    """Rows that begin beyond 2^32 bytes into the states (and 2^31 elements)."""
    import torch
    sk, pitch = 1100, 1 << 21
    buf = torch.empty(sk * pitch, dtype=torch.bfloat16, device="cuda")
    k = buf.as_strided((1, sk, 2, 64), (0, pitch, 64, 1))
    v = buf.as_strided((1, sk, 2, 64), (0, pitch, 64, 1), 128)
    q, k0, v0 = _make(1, sq, sk, 2, 2, 64, "bf16", seed=13)
    k.copy_(k0)
    v.copy_(v0)
    _check(q, k, v)


@pytest.mark.parametrize("sq", [1, 300])
def test_same_answer_every_time(cuda, sq):
    import torch
    import sam3cu
    q, k, v = _make(1, sq, 9000, 4, 4, 64, "bf16", seed=14)
    first = sam3cu.cross_attention(q, k, v)
    for _ in range(5):
        assert torch.equal(sam3cu.cross_attention(q, k, v), first)


@pytest.mark.parametrize("sq,sk", [(2, 3000), (300, 3000), (2, 30000)])
def test_captured_graphs_and_streams(cuda, sq, sk):
    """Two captured graphs replayed at once on two streams, with new inputs
    and new lengths, against plain calls."""
    import torch
    import sam3cu
    sets = []
    for i in range(2):
        q, k, v = _make(2, sq, sk, 4, 2, 64, "bf16", seed=20 + i)
        lens = torch.tensor([sk, 5], dtype=torch.int32, device="cuda")
        out, st, g = torch.empty_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            sam3cu.cross_attention(q, k, v, k_lens=lens, out=out)
        sets.append((q, k, v, lens, out, st, g))
    for i, (q, k, v, lens, out, st, g) in enumerate(sets):
        for x, y in zip((q, k, v), _make(2, sq, sk, 4, 2, 64, "bf16", seed=30 + i)):
            x.copy_(y)
        lens.copy_(torch.tensor([17 + i, sk - 100], dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(4):
        for q, k, v, lens, out, st, g in sets:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for q, k, v, lens, out, st, g in sets:
        assert torch.equal(out, sam3cu.cross_attention(q, k, v, k_lens=lens))
        _check(q, k, v, k_lens=lens)


def test_first_call_may_be_captured():
    """In a fresh process the first call of each kernel is one that a graph
    captures (each takes its attributes, tables and pool on first use)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys
sys.path.insert(0, %r)
import torch, sam3cu
sam3cu.init(0)
f = sam3cu.RopeFreqs(64)
for sq, sk in ((1, 200), (1, 40000), (40, 300), (300, 77), (300, 2000)):
    q = torch.randn(1, sq, 4, 64, device="cuda").bfloat16()
    k = torch.randn(1, sk, 4, 64, device="cuda").bfloat16()
    v = torch.randn(1, sk, 4, 64, device="cuda").bfloat16()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = sam3cu.cross_attention(sam3cu.rope_pos(q, f), k, v)
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, sam3cu.cross_attention(sam3cu.rope_pos(q, f), k, v)), (sq, sk)
    assert sam3cu.device_error() == 0
print("done")
""" % os.path.join(root, "sam3.c_b200")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


def test_two_threads(cuda):
    """Calls from two host threads, each on a stream of its own."""
    import threading

    import torch
    import sam3cu
    sets = [_make(1, sq, 3000, 4, 2, 64, "bf16", seed=sq) for sq in (2, 300)]
    want = [sam3cu.cross_attention(*s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        torch.cuda.set_device(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = sam3cu.cross_attention(*sets[i])
            torch.cuda.current_stream().synchronize()
            if not torch.equal(got, want[i]):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_wrapper_refusals(cuda):
    import torch
    import sam3cu
    q, k, v = _make(2, 3, 10, 4, 2, 64, "bf16")
    i32 = dict(dtype=torch.int32, device="cuda")
    for bad in (dict(k=k[:1]), dict(v=v[:, :9]), dict(v=v.half()), dict(k=k[..., :32]), dict(q=q[0]),
                dict(k=k.transpose(2, 3)), dict(k_lens=torch.ones(2, device="cuda", dtype=torch.int64)),
                dict(k_lens=torch.ones(3, **i32)), dict(k_lens=torch.ones(2, dtype=torch.int32)),
                dict(key_mask=torch.ones(2, 9, dtype=torch.bool, device="cuda")),
                dict(key_mask=torch.ones(2, 10, device="cuda")),
                dict(key_mask=torch.ones(3, 10, dtype=torch.bool, device="cuda")),
                dict(bias=torch.zeros(2, 4, 3, 9, device="cuda")),
                dict(bias=torch.zeros(2, 4, 3, 10, device="cuda").half()),
                dict(out=torch.empty(2, 3, 4, 32, device="cuda", dtype=q.dtype)), dict(out=q.float())):
        with pytest.raises(ValueError):
            sam3cu.cross_attention(**{**dict(q=q, k=k, v=v), **bad})
    for bad in (dict(q=q[:, :, :3]), dict(scale=-1.0), dict(q=q[..., :20], k=k[..., :20], v=v[..., :20]),
                dict(k=torch.empty(2 * 10 * 2 * 64 + 1, device="cuda", dtype=q.dtype)[1:].view(2, 10, 2, 64))):
        with pytest.raises(sam3cu.Sam3cuError):
            sam3cu.cross_attention(**{**dict(q=q, k=k, v=v), **bad})
    with pytest.raises(KeyError):
        sam3cu.cross_attention(q.double(), k.double(), v.double())


@pytest.mark.parametrize("hd,dt", [(32, "f16"), (64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("sq,sk", [(130, 300), (1000, 200), (300, 3000)])
def test_without_the_tcgen05_kernel(cuda, hd, dt, sq, sk):
    """Where a compiler spilled that kernel the warp-MMA ones take its calls."""
    import torch
    import sam3cu
    q, k, v = _make(2, sq, sk, 6, 3, hd, dt, seed=hd)
    lens = torch.tensor([sk, sk // 3], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    mask = torch.rand(2, sk, generator=g, device="cuda") < 0.5
    sam3cu.lib().sam3cu_selftest_cross_spilled(1)
    try:
        _check(q, k, v)
        _check(q, k, v, k_lens=lens, key_mask=mask)
    finally:
        sam3cu.lib().sam3cu_selftest_cross_spilled(0)
    _check(q, k, v, k_lens=lens, key_mask=mask)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_the_tcgen05_kernel_is_not_spilled(cuda, hd, dt, masked):
    """Each build of it is the one that runs: none was left to the warp MMAs."""
    import torch
    import sam3cu
    q, k, v = _make(1, 300, 1000, 2, 2, hd, dt, seed=hd)
    mask = torch.arange(1000, device="cuda")[None] % 3 > 0 if masked else None
    _check(q, k, v, key_mask=mask)
    assert sam3cu.lib().sam3cu_selftest_cross_spilled(0) == 0


@pytest.mark.parametrize("b,sq,sk,hq,hkv,hd,dt", [
    (2, 1729, 1001, 20, 4, 128, "f16"), (2, 500, 1001, 6, 2, 64, "bf16"), (2, 901, 1500, 5, 1, 32, "f16")])
def test_what_ran_before_has_no_say(cuda, b, sq, sk, hq, hkv, hd, dt):
    """Groups that do not divide 128 leave rows of a tile without a query.
    Whatever earlier kernels left in their shared memory, the other rows come
    out the same, to the bit."""
    import torch
    import sam3cu
    q, k, v = _make(b, sq, sk, hq, hkv, hd, dt, seed=18)
    lens = torch.tensor([sk * 2 // 3, sk * 3 // 5], dtype=torch.int32, device="cuda")
    first = [sam3cu.cross_attention(q, k, v, k_lens=n) for n in (None, lens)]
    for i in range(9):
        x = _make(1, 1000, 1000, 4, 4, hd, dt, seed=i, sharp=10.0 ** (i % 3))
        sam3cu.cross_attention(*x)
        for n, want in zip((None, lens), first):
            assert torch.equal(sam3cu.cross_attention(q, k, v, k_lens=n), want)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("value", [(40.0, 31.25), (800.0, 640.0)])
@pytest.mark.parametrize("sq,sk", [(1, 999), (20, 999), (150, 999), (150, 77), (300, 5000), (1, 70000)])
def test_equal_large_scores_give_the_mean(cuda, dt, value, sq, sk):
    """One value for all scores, 10^4 or 4 10^6: the mean of V.  The dot
    products are sums of equal powers of two and small factors, exact in F32,
    so every P is the same number: the rounding of P (half a step), of the
    sums and of the output remain, and nothing for the scores."""
    import torch
    import sam3cu
    q, k, v = _make(1, sq, sk, 1, 1, 64, dt, seed=7)
    q[:], k[:] = value
    o = sam3cu.cross_attention(q, k, v).double()
    mean, size = v[0, :, 0].double().mean(0), v[0, :, 0].double().abs().mean(0)
    half = torch.finfo(v.dtype).eps / 2
    tol = half * mean.abs() + (half + 2.0 ** -18) * size
    assert bool(((o - mean).abs() <= tol).all())


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq,sk", [(1, 300), (5, 1027), (40, 517), (201, 517), (300, 129)])
def test_bias_with_masks(cuda, hd, sq, sk):
    """A bias beside lengths and a key mask; what it holds at keys that do not
    count, NaN and infinities, stays out."""
    import torch
    import sam3cu
    q, k, v = _make(3, sq, sk, 4, 2, hd, "bf16", seed=15)
    g = torch.Generator(device="cuda").manual_seed(5)
    bias = torch.randn(3, 4, sq, sk, generator=g, device="cuda") * 2
    bias[0, 1, 0] = -math.inf
    mask = torch.rand(3, sk, generator=g, device="cuda") < 0.6
    mask[1] = False
    lens = torch.tensor([sk, sk, sk // 2], dtype=torch.int32, device="cuda")
    o = _check(q, k, v, bias=bias, key_mask=mask, k_lens=lens)
    assert bool((o[1] == 0).all()) and bool((o[0, 0, 1] == 0).all())
    off = ~mask | (torch.arange(sk, device="cuda") >= lens[:, None])
    for value in (math.nan, math.inf):
        assert torch.equal(sam3cu.cross_attention(q, k, v, bias=bias.masked_fill(off[:, None, None], value),
                                                  key_mask=mask, k_lens=lens), o)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq,sk", [(1, 400), (40, 400), (300, 400), (300, 77)])
def test_expanded_keys_and_queries(cuda, hd, sq, sk):
    """Stride 0 along the keys, the queries and the heads of the queries,
    which tensor maps cannot describe."""
    import torch
    q, k, v = _make(2, sq, sk, 4, 4, hd, "bf16", seed=16)
    one = k[:, :1].expand(2, sk, 4, hd)
    _check(q, one, v)
    _check(q, k, v[:, :1].expand(2, sk, 4, hd))
    _check(q, one, v[:, :1].expand(2, sk, 4, hd), k_lens=torch.tensor([3, sk], dtype=torch.int32, device="cuda"))
    _check(q[:, :1].expand(2, sq, 4, hd), k, v)
    _check(q[:, :, :1].expand(2, sq, 4, hd), k, v)


@pytest.mark.parametrize("b,sq,sk,hq,hkv,hd,dt", [
    (2, 5, 300, 8, 2, 64, "bf16"), (1, 7, 4096, 8, 8, 16, "f16"), (2, 1, 65521, 32, 4, 128, "bf16"),
    (2, 40, 5000, 4, 4, 32, "f16"), (4, 300, 77, 8, 8, 32, "bf16"), (2, 1729, 1001, 20, 4, 128, "f16"),
    (1, 300, 9000, 2, 2, 128, "bf16"), (2, 2000, 1500, 4, 4, 64, "bf16")])
def test_repeats_exactly(cuda, b, sq, sk, hq, hkv, hd, dt):
    """Every kernel and every split of the keys has a fixed order of sums."""
    import torch
    import sam3cu
    q, k, v = _make(b, sq, sk, hq, hkv, hd, dt, seed=17)
    lens = torch.randint(0, sk + 1, (b,), device="cuda", dtype=torch.int32)
    first, masked = sam3cu.cross_attention(q, k, v), sam3cu.cross_attention(q, k, v, k_lens=lens)
    for _ in range(4):
        assert torch.equal(sam3cu.cross_attention(q, k, v), first)
        assert torch.equal(sam3cu.cross_attention(q, k, v, k_lens=lens), masked)


def test_every_result_of_four_threads(cuda):
    """Calls from four host threads, each on a stream of its own, with a
    workspace, a cluster and the tensor cores among them: what a thread raises
    is raised here, and every result counts."""
    from concurrent.futures import ThreadPoolExecutor

    import torch
    import sam3cu
    f = sam3cu.RopeFreqs(64)
    sets = [_make(1, sq, sk, 4, 2, 64, "bf16", seed=sq + sk) for sq, sk in ((2, 40000), (20, 3000), (300, 3000), (300, 77))]
    want = [sam3cu.cross_attention(sam3cu.rope_pos(q, f, start=5), k, v) for q, k, v in sets]
    torch.cuda.synchronize()

    def work(i):
        torch.cuda.set_device(0)
        q, k, v = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            wrong = torch.zeros((), device="cuda", dtype=torch.int64)
            for _ in range(50):
                wrong += (sam3cu.cross_attention(sam3cu.rope_pos(q, f, start=5), k, v) != want[i]).sum()
            return int(wrong)
    with ThreadPoolExecutor(4) as pool:
        assert [t.result() for t in [pool.submit(work, i) for i in range(4)]] == [0] * 4
    assert sam3cu.device_error() == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("sq,sk", [(1, 999), (20, 999), (150, 77), (150, 999), (1, 70000)])
@pytest.mark.parametrize("size", [4096.0, 65024.0])
def test_huge_scores(cuda, dt, sq, sk, size):
    """Scores of 10^8 and 3 10^10, from finite 16-bit queries and keys, equal
    but for keys whose score is lower by much more than F32 resolves: the
    mean of V over the others.  (The dot products are exact: one product of
    powers of two times 64.)"""
    import torch
    import sam3cu
    q, k, v = _make(1, sq, sk, 1, 1, 64, dt, seed=19)
    q[:], k[:] = size, size
    k[:, ::3] = size / 2
    o = sam3cu.cross_attention(q, k, v).double()
    keep = torch.arange(sk, device="cuda") % 3 != 0
    vv = v[0, keep, 0].double()
    mean, mag = vv.mean(0), vv.abs().mean(0)
    half = torch.finfo(v.dtype).eps / 2
    assert bool(((o - mean).abs() <= half * mean.abs() + (half + 2.0 ** -18) * mag).all())


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sq,sk", [(3, 500), (40, 500), (150, 77), (300, 1500)])
def test_rows_of_large_scores_among_others(cuda, dt, hd, sq, sk):
    """Scores around 32768 / sqrt(head_dim), 2900 to 5800, in every third row,
    around as much below 0 in every third, small ones in the rest, with
    lengths and a key mask."""
    import torch
    q, k, v = _make(2, sq, sk, 4, 2, hd, dt, seed=21)
    k[..., 0] = 256.0
    q[..., 0] = torch.tensor([0.0, 128.0, -128.0], device="cuda").to(q.dtype)[torch.arange(sq, device="cuda") % 3, None]
    lens = torch.tensor([sk, sk // 2], dtype=torch.int32, device="cuda")
    _check(q, k, v, k_lens=lens)
    _check(q, k, v, k_lens=lens, key_mask=torch.arange(sk, device="cuda")[None] % 5 > 1)


@pytest.mark.parametrize("sq,sk", [(1, 999), (20, 999), (150, 77), (300, 1500)])
def test_scores_whose_exponents_pass_f32(cuda, sq, sk):
    """Finite dot products whose product with the scale is none: equal scores
    still give the mean of V."""
    import torch
    import sam3cu
    q, k, v = _make(1, sq, sk, 1, 1, 64, "bf16", seed=22)
    q[:], k[:] = 32.0, 32.0
    o = sam3cu.cross_attention(q, k, v, scale=2.0 ** 120).double()
    mean, mag = v[0, :, 0].double().mean(0), v[0, :, 0].double().abs().mean(0)
    assert bool(((o - mean).abs() <= 2.0 ** -8 * mean.abs() + (2.0 ** -8 + 2.0 ** -18) * mag).all())


@pytest.mark.parametrize("sq", [1, 40, 300])
def test_overlapping_rows(cuda, sq):
    """Strides shorter than a row: keys, heads and sequences that share data
    (windows over one buffer)."""
    import torch
    buf, other = (torch.randn(40000, device="cuda").bfloat16() for _ in range(2))
    q, k, v = _make(2, sq, 300, 4, 2, 64, "bf16", seed=23)
    _check(q, buf.as_strided((2, 300, 2, 64), (8, 16, 64, 1)), other.as_strided((2, 300, 2, 64), (24, 8, 8, 1)))
    _check(buf.as_strided((2, sq, 4, 64), (16, 8, 24, 1)), k, v)


@pytest.mark.parametrize("sq,sk,hd", [(300000, 5, 32), (300000, 130, 64), (1, 2000000, 16), (100, 500000, 16)])
def test_largest_sides(cuda, sq, sk, hd):
    _check(*_make(1, sq, sk, 1, 1, hd, "bf16", seed=24))
