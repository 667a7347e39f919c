"""Host side of the rotary positions, head norms and cross attention: the
frequency tables against their formulas, and every refusal (no GPU: a
refused call returns before it touches a device)."""
import ctypes as C
import math
import struct

import numpy as np
import pytest

import sam3cu

EINVAL, EDTYPE, ESHAPE = -1, -6, -101


def _formula(rot, scaling, theta, factor, trained=4096.0, fast=32.0, slow=1.0, low=1.0, high=4.0):
    base = theta
    if scaling == sam3cu.ROPE_SCALE_NTK and rot > 2:
        base = theta * factor ** (rot / (rot - 2))
    out = []
    for i in range(rot // 2):
        w = base ** (-2 * i / rot)
        turns = trained * w / (2 * math.pi)
        if scaling == sam3cu.ROPE_SCALE_LINEAR:
            w /= factor
        elif scaling == sam3cu.ROPE_SCALE_YARN:
            def at(n):
                return rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))
            a, b = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
            t = min(max((i - a) / max(b - a, 0.001), 0), 1)
            w = (w / factor) * t + w * (1 - t)
        elif scaling == sam3cu.ROPE_SCALE_BANDS:
            if turns < low:
                w /= factor
            elif turns <= high:
                t = (turns - low) / (high - low)
                w = (1 - t) * w / factor + t * w
        out.append(w / (2 * math.pi))
    return np.array(out)


@pytest.mark.parametrize("scaling", range(5))
@pytest.mark.parametrize("rot,theta,factor", [(2, 10000.0, 4.0), (64, 10000.0, 1.0), (64, 10000.0, 8.0),
                                              (96, 500000.0, 32.0), (256, 1e6, 2.5)])
def test_frequencies(scaling, rot, theta, factor):
    f = sam3cu.RopeFreqs(rot, scaling=scaling, theta=theta, factor=factor)
    want = _formula(rot, scaling, theta, factor)
    assert f.turns.shape == (rot // 2,)
    # a power, a logarithm or two and a handful of products in 64 bits
    np.testing.assert_allclose(f.turns, want, rtol=1e-13)
    amp = 0.1 * math.log(factor) + 1 if scaling == sam3cu.ROPE_SCALE_YARN else 1.0
    assert abs(f.amplitude - amp) <= 2.0 ** -24 * amp


def test_frequencies_given_amplitude():
    assert sam3cu.RopeFreqs(8, scaling=sam3cu.ROPE_SCALE_YARN, factor=4, amplitude=0.5).amplitude == 0.5


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("bad", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(rot_dim=-2), dict(layout=2), dict(layout=-1),
    dict(scaling=5), dict(scaling=-1), dict(theta=1.0), dict(theta=NAN), dict(theta=INF), dict(amplitude=-1.0),
    dict(amplitude=NAN), dict(scaling=1, factor=0.5), dict(scaling=2, factor=NAN), dict(scaling=3, trained_len=0),
    dict(scaling=3, beta_fast=1.0), dict(scaling=3, beta_slow=0.0), dict(scaling=4, low_freq=0.0),
    dict(scaling=4, high_freq=1.0), dict(scaling=4, trained_len=NAN)])
def test_frequencies_refused(bad):
    with pytest.raises(sam3cu.Sam3cuError):
        sam3cu.RopeFreqs(**{"rot_dim": 64, **bad})


def _view(x=4096, xs=(1024, 64, 64), y=8192, ys=(1024, 64, 64), heads=1, gamma=0, beta=0):
    return struct.pack("P3qP3qi4xPP", x, *xs, y, *ys, heads, gamma, beta)


def _rope(q=None, k=None, dtype=sam3cu.BF16, batch=2, seq=2, hd=64, pos=None, stride=0, freqs=True):
    table = sam3cu.RopeFreqs(64)
    f = table.ptr if freqs is True else freqs
    return sam3cu.lib().sam3cu_rope_pos(_view() if q is None else q, k, dtype, batch, seq, hd, pos, stride, 0, f, None)


def test_rope_refused():
    assert _rope(dtype=sam3cu.Q8_0) == EDTYPE
    assert _rope(batch=-1) == EINVAL and _rope(seq=-1) == EINVAL and _rope(hd=0) == EINVAL
    assert _rope(hd=257) == ESHAPE
    assert _rope(hd=62) == ESHAPE               # less than what rotates
    assert _rope(freqs=0) == EINVAL
    assert _rope(stride=-1) == EINVAL
    assert _rope(pos=4097) == EINVAL            # misaligned positions
    assert _rope(q=_view(x=0)) == EINVAL and _rope(q=_view(y=0)) == EINVAL
    assert _rope(q=_view(x=4097)) == EINVAL     # misaligned elements
    assert _rope(q=_view(heads=-1)) == EINVAL
    assert _rope(q=_view(xs=(-1, 64, 64))) == EINVAL and _rope(q=_view(ys=(1024, -64, 64))) == EINVAL
    assert _rope(q=_view(ys=(0, 64, 64))) == EINVAL      # sequences written over each other
    assert _rope(q=_view(y=4096, ys=(2048, 64, 64))) == EINVAL  # in place, elsewhere
    assert _rope(k=_view(x=0)) == EINVAL
    bad = sam3cu._RopeFreqs(n_pairs=129, layout=1)
    assert _rope(freqs=C.addressof(bad), hd=256) == EINVAL
    bad = sam3cu._RopeFreqs(n_pairs=0, layout=1)
    assert _rope(freqs=C.addressof(bad)) == EINVAL
    bad = sam3cu._RopeFreqs(n_pairs=2, layout=7)
    assert _rope(freqs=C.addressof(bad)) == EINVAL
    L = sam3cu.lib()
    f = sam3cu.RopeFreqs(64)
    assert L.sam3cu_rope_pos(None, None, 2, 1, 1, 64, None, 0, 0, f.ptr, None) == EINVAL


def test_rope_nothing_to_do():
    assert _rope(batch=0) == 0 and _rope(seq=0) == 0
    assert _rope(q=_view(heads=0, x=0, y=0)) == 0


def test_qk_norm_refused():
    L, f = sam3cu.lib(), sam3cu.RopeFreqs(64)

    def call(norm=1, eps=1e-6, q=None, hd=64, freqs=f.ptr, dtype=2):
        return L.sam3cu_qk_norm_rope(q or _view(), None, dtype, 2, 2, hd, norm, eps, None, 0, 0, freqs, None)
    assert call(norm=0) == EINVAL and call(norm=3) == EINVAL
    assert call(eps=-1.0) == EINVAL and call(eps=NAN) == EINVAL
    assert call(q=_view(gamma=4097)) == EINVAL and call(q=_view(beta=4098)) == EINVAL
    assert call(hd=300, freqs=None) == ESHAPE
    assert call(dtype=7) == EDTYPE


def _cross(ptr=(4096, 8192, 12288, 16384), qs=(64, 64, 64), ks=(64, 64, 64), vs=(64, 64, 64), os_=(4096, 128, 64),
           dtype=sam3cu.BF16, batch=2, sq=2, sk=2, qh=2, kh=1, hd=64, scale=0.0, lens=0, mask=0, ms=0, bias=0,
           bs=(0, 0, 0)):
    a = struct.pack("4P12q7ifPPqP3q", *ptr, *qs, *ks, *vs, *os_, dtype, batch, sq, sk, qh, kh, hd, scale, lens, mask,
                    ms, bias, *bs)
    return sam3cu.lib().sam3cu_cross_attention(a, None)


def test_cross_attention_refused():
    assert sam3cu.lib().sam3cu_cross_attention(None, None) == EINVAL
    assert _cross(dtype=sam3cu.F32) == EDTYPE and _cross(dtype=sam3cu.Q8_0) == EDTYPE
    for bad in (dict(batch=-1), dict(sq=-1), dict(sk=-1), dict(qh=-2), dict(kh=0), dict(hd=0), dict(qh=3, kh=2),
                dict(scale=-1.0), dict(scale=NAN), dict(scale=INF), dict(qs=(-64, 64, 64)), dict(ks=(64, -64, 64)),
                dict(os_=(0, 128, 64)), dict(os_=(4096, 0, 64)), dict(os_=(4096, 128, 0)), dict(lens=4098),
                dict(mask=4096, ms=-1), dict(bias=4097), dict(bias=4096, bs=(0, -1, 0)), dict(ptr=(0, 8192, 8192, 4096)),
                dict(ptr=(4096, 0, 8192, 4096)), dict(ptr=(4096, 8192, 0, 4096)), dict(ptr=(4096, 8192, 8192, 0))):
        assert _cross(**bad) == EINVAL, bad
    for bad in (dict(hd=68), dict(hd=136), dict(hd=4), dict(qs=(64, 60, 64)), dict(vs=(64, 4, 64)),
                dict(ptr=(4104, 8192, 8192, 4096)), dict(ptr=(4096, 8200, 8192, 4096)), dict(qh=258, kh=2),
                dict(sk=0x7fffffff), dict(sq=0x7fffffff, qh=1)):
        assert _cross(**bad) == ESHAPE, bad


def test_cross_attention_nothing_to_do():
    assert _cross(batch=0) == 0 and _cross(sq=0) == 0 and _cross(qh=0) == 0


def test_wrappers_want_cuda_tensors():
    import torch
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        sam3cu.cross_attention(x, x, x)
    with pytest.raises(ValueError):
        sam3cu.rope_pos(x, sam3cu.RopeFreqs(64))
    with pytest.raises(ValueError):
        sam3cu.qk_norm_rope(x, None)


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle"])
def test_copied_frequencies_point_to_their_own_table(how):
    """A copied or unpickled table (a module's deepcopy, another process) hands
    the library its own memory, not that of the object it was made from."""
    import copy
    import pickle
    f = sam3cu.RopeFreqs(64, theta=500.0)
    g = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x))}[how](f)
    want = f.turns
    assert g.rot_dim == 64 and np.array_equal(g.turns, want)
    assert g.ptr == C.addressof(g._c)
    if how != "copy":
        assert g.ptr != f.ptr
    del f
    assert sam3cu._RopeFreqs.from_address(g.ptr).n_pairs == 32
    assert np.array_equal(np.array(sam3cu._RopeFreqs.from_address(g.ptr).turns[:32]), want)


@pytest.mark.parametrize("bad", [
    dict(amplitude=1e39), dict(scaling=sam3cu.ROPE_SCALE_NTK, factor=1e200, rot_dim=4),
    dict(scaling=sam3cu.ROPE_SCALE_NTK, factor=1e10, theta=1e300)])
def test_tables_that_do_not_fit_are_refused(bad):
    """An amplitude past F32, a base past F64: the table would hold
    infinities, or zeros in place of every frequency but the first."""
    with pytest.raises(sam3cu.Sam3cuError):
        sam3cu.RopeFreqs(**{"rot_dim": 64, **bad})


def test_largest_tables():
    assert np.isfinite(sam3cu.RopeFreqs(64, amplitude=3e38).amplitude)
    assert (sam3cu.RopeFreqs(64, scaling=sam3cu.ROPE_SCALE_NTK, factor=1e6, theta=1e300).turns > 0).all()


def test_start_out_of_range():
    """start + seq - 1 has to be a 64-bit position; a Python integer that is
    none must not wrap into one."""
    L, f = sam3cu.lib(), sam3cu.RopeFreqs(64)

    def call(start, seq=2, batch=2):
        rope = L.sam3cu_rope_pos(_view(), None, sam3cu.BF16, batch, seq, 64, None, 0, start, f.ptr, None)
        norm = L.sam3cu_qk_norm_rope(_view(), None, sam3cu.BF16, batch, seq, 64, 1, 1e-6, None, 0, start, f.ptr, None)
        assert rope == norm
        return rope
    assert call(2 ** 63 - 1) == EINVAL and call(2 ** 63 - 5, seq=7) == EINVAL
    assert call(2 ** 63 - 1, batch=0) == 0
    for start in (2 ** 63, 2 ** 64 + 1, -2 ** 63 - 1):
        with pytest.raises(ValueError):
            sam3cu._positions(None, start, 1, 1, 0)
    assert sam3cu._positions(None, -2 ** 63, 1, 1, 0) == (None, 0)


def test_cross_attention_scale_out_of_range():
    """Scores are taken in base 2: scale * log2(e) has to be finite, or a score
    of 0 becomes NaN."""
    for scale in (3.4e38, 2.4e38):
        assert _cross(scale=scale) == EINVAL
