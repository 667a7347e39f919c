"""The operators together, as a decoder layer over an encoder's states uses
them: projections (sam3cu_linear), norms of the heads with the rotation,
attention over states of another length, output projection onto the
residual - for a prompt and then for single tokens, as plain calls and as one
captured graph - against the same layer in 64 bits.

Tolerance (normwise, as for the other 16-bit paths): the layer rounds seven
times to bf16 (q, k, v, the normalised q and k, P, o), each by at most 2^-8
of a value and independently, so sqrt(7) 2^-8 = 1.04e-2 of the attention's
part, which the output projection averages; the residual is F32 and larger.
1e-2 of the largest output is above that by more than the residual's share."""
import math

import pytest

from _util import rel_err, to_np

pytestmark = pytest.mark.gpu

E, HEADS, KV, HD = 256, 4, 2, 64


def _weights(seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def w(n, k):
        return (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).bfloat16()
    return {"q": w(HEADS * HD, E), "kv": w(2 * KV * HD, E), "o": w(E, HEADS * HD),
            "gq": 1 + 0.1 * torch.randn(HD, generator=g, device="cuda"),
            "gk": 1 + 0.1 * torch.randn(HD, generator=g, device="cuda")}


def _layer(w, x, states, lens, freqs, start):
    """x [b, sq, E] bf16 -> [b, sq, E] f32."""
    import sam3cu
    b, sq, sk = x.shape[0], x.shape[1], states.shape[1]
    q = sam3cu.linear(x.reshape(-1, E), w["q"]).view(b, sq, HEADS, HD)
    kv = sam3cu.linear(states.reshape(-1, E), w["kv"]).view(b, sk, 2 * KV, HD)
    k, v = kv[:, :, :KV], kv[:, :, KV:]
    q = sam3cu.qk_norm_rope(q, None, w["gq"], freqs=freqs, start=start, out=q)
    sam3cu.qk_norm_rope(k, None, w["gk"], freqs=freqs, out=k)
    o = sam3cu.cross_attention(q, k, v, k_lens=lens)
    return sam3cu.linear(o.view(-1, HEADS * HD), w["o"], residual=x.reshape(-1, E).float(),
                         out_dtype=_f32()).view(b, sq, E)


def _f32():
    import torch
    return torch.float32


def _layer64(w, x, states, lens, freqs, start):
    import torch
    d = {n: t.double() for n, t in w.items()}
    b, sq, sk = x.shape[0], x.shape[1], states.shape[1]
    turns = torch.from_numpy(freqs.turns).cuda()

    def norm_rope(t, gamma, first):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * gamma
        a = 2 * math.pi * (torch.arange(t.shape[1], device="cuda", dtype=torch.float64) + first)[:, None, None] * turns
        u, v = t[..., :HD // 2], t[..., HD // 2:]
        return torch.cat((u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()), -1)
    q = norm_rope((x.double() @ d["q"].T).view(b, sq, HEADS, HD), d["gq"], start)
    kv = (states.double() @ d["kv"].T).view(b, sk, 2 * KV, HD)
    k = norm_rope(kv[:, :, :KV], d["gk"], 0).repeat_interleave(HEADS // KV, 2)
    v = kv[:, :, KV:].repeat_interleave(HEADS // KV, 2)
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(HD)
    s.masked_fill_(torch.arange(sk, device="cuda") >= lens[:, None, None, None], -math.inf)
    o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v).reshape(b, sq, -1)
    return o @ d["o"].T + x.double()


@pytest.mark.parametrize("sq", [1, 37, 300])
def test_layer(cuda, sq):
    import torch
    import sam3cu
    w, freqs = _weights(1), sam3cu.RopeFreqs(HD)
    g = torch.Generator(device="cuda").manual_seed(sq)
    x = torch.randn(2, sq, E, generator=g, device="cuda").bfloat16()
    states = torch.randn(2, 576, E, generator=g, device="cuda").bfloat16()
    lens = torch.tensor([576, 333], dtype=torch.int32, device="cuda")
    y = _layer(w, x, states, lens, freqs, 5)
    assert rel_err(to_np(y), _layer64(w, x, states, lens, freqs, 5).cpu().numpy()) < 1e-2
    assert sam3cu.device_error() == 0


def test_layer_captured(cuda):
    """The layer as one graph: replayed with new inputs it gives what the
    plain calls give, bit for bit."""
    import torch
    import sam3cu
    w, freqs = _weights(2), sam3cu.RopeFreqs(HD)
    x = torch.randn(3, 1, E, device="cuda").bfloat16()
    states = torch.randn(3, 576, E, device="cuda").bfloat16()
    lens = torch.tensor([576, 1, 100], dtype=torch.int32, device="cuda")
    _layer(w, x, states, lens, freqs, 9)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = _layer(w, x, states, lens, freqs, 9)
    for i in range(3):
        x.copy_(torch.randn(3, 1, E, device="cuda").bfloat16())
        states.copy_(torch.randn(3, 576, E, device="cuda").bfloat16())
        lens.copy_(torch.tensor([i, 200 * i + 1, 576], dtype=torch.int32))
        g.replay()
        assert torch.equal(y, _layer(w, x, states, lens, freqs, 9))
