"""CPU: the rotary tables, and what the rotary entry points refuse."""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from cast_b200 import _lib, rotary
from oracle import rotary as ora


@pytest.fixture(scope="module")
def lib():
    from cast_b200 import build

    build.build()
    return _lib.load()


def test_frequencies_of_one_axis_and_three():
    f = rotary.rope_frequencies(128)
    assert f.dtype == torch.float64 and f.shape == (64,)
    for j in (0, 1, 17, 63):
        assert f[j].item() == pytest.approx(10000.0 ** (-2 * j / 128), rel=1e-14)
    g = rotary.rope_frequencies(128, axes=(22, 21, 21))
    assert g[22].item() == 1.0 and g[43].item() == 1.0
    assert g[23].item() == pytest.approx(10000.0 ** (-1 / 21), rel=1e-14)


def test_frequencies_scaled_for_long_contexts():
    f = rotary.rope_frequencies(64, base=500.0)
    assert torch.equal(rotary.rope_frequencies(64, base=500.0, scaling=("linear", 4.0)), f / 4)
    n = rotary.rope_frequencies(64, base=500.0, scaling=("ntk", 4.0))
    assert n[0] == f[0] and n[-1].item() == pytest.approx(f[-1].item() / 4, rel=1e-12)
    assert (n[1:] < f[1:]).all()
    y = rotary.rope_frequencies(64, scaling=("yarn", 8.0, 4096))
    f = rotary.rope_frequencies(64)
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(y[turns > 40], f[turns > 40])
    assert torch.allclose(y[turns < 0.7], f[turns < 0.7] / 8, rtol=1e-12)
    assert ((y <= f) & (y >= f / 8 * (1 - 1e-12))).all()


@pytest.mark.parametrize("kwargs", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0),
                                    dict(rotary_dim=8, axes=(1, 1, 1)), dict(rotary_dim=8, scaling=("other", 2.0)),
                                    dict(rotary_dim=8, scaling=("linear", 0.0))])
def test_frequencies_refused(kwargs):
    with pytest.raises(ValueError):
        rotary.rope_frequencies(**kwargs)


def test_table_holds_far_positions():
    f = rotary.rope_frequencies(16)
    t = rotary.rope_table(f, 200001, amplitude=0.5, device="cpu")
    assert t.shape == (200001, 8, 2) and t.dtype == torch.float32
    theta = ora.angles(torch.tensor([[200000]]), f)[0, 0]
    # float32 rounding of a value up to 1/2; float64 angles are off by 200000 * 2^-53
    assert torch.allclose(t[200000, :, 0].double(), 0.5 * theta.cos(), rtol=0, atol=2.0 ** -25 * 1.01)
    assert torch.allclose(t[200000, :, 1].double(), 0.5 * theta.sin(), rtol=0, atol=2.0 ** -25 * 1.01)
    with pytest.raises(ValueError):
        rotary.rope_table(f, 0, device="cpu")


def test_a_turn_by_an_inverse_turn_is_the_identity():
    x = torch.randn(1, 3, 2, 16, dtype=torch.float64)
    theta = torch.randn(1, 3, 6, dtype=torch.float64)
    for inter in (False, True):
        back = ora.turn(ora.turn(x, theta, inter), -theta, inter)
        assert torch.allclose(back, x, atol=1e-14)
        # scores depend on the distance of positions alone
        y = torch.randn(1, 3, 2, 16, dtype=torch.float64)
        a = (ora.turn(x, theta, inter) * ora.turn(y, theta + 0.3, inter)).sum(-1)
        b = (ora.turn(x, theta + 5, inter) * ora.turn(y, theta + 5.3, inter)).sum(-1)
        assert torch.allclose(a, b, atol=1e-12)


def test_python_refuses_host_tensors():
    x = torch.zeros(1, 2, 2, 16)
    with pytest.raises(ValueError, match="CUDA"):
        rotary.rope(x, torch.zeros(2, 8, 2))
    with pytest.raises(ValueError, match="CUDA"):
        rotary.qk_norm_rope(x, x, None, None)


def _rope(lib, **kw):
    a = dict(x=4096, dtype=0, table=4096, rows=4, positions=None, p64=0, batch=0, first=0, axes=None, B=1, L=2, H=2,
             D=128, R=128, flags=1, strides=[512, 256, 128] * 2, out=8192)
    a.update(kw)
    st = (ctypes.c_longlong * 6)(*a["strides"])
    ax = None if a["axes"] is None else (ctypes.c_int * 3)(*a["axes"])
    return lib.cast_rope(a["x"], a["dtype"], a["table"], a["rows"], a["positions"], a["p64"], a["batch"], a["first"], ax,
                         a["B"], a["L"], a["H"], a["D"], a["R"], a["flags"], st, a["out"], None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(x=None), 1, b"required"),
    (dict(dtype=3), 1, b"dtype"),
    (dict(L=0), 1, b"non-positive"),
    (dict(D=260), 2, b"head_dim"),
    (dict(D=20, R=16), 2, b"head_dim"),
    (dict(R=130), 1, b"rotated part"),
    (dict(R=12), 2, b"rotated part"),
    (dict(R=24, flags=0), 2, b"rotated part"),
    (dict(flags=4), 1, b"flags"),
    (dict(table=None), 1, b"table"),
    (dict(rows=0), 1, b"table"),
    (dict(table=4100), 3, b"table"),
    (dict(axes=(22, 21, 20), positions=4096), 1, b"axes"),
    (dict(axes=(22, 21, 21)), 1, b"positions"),
    (dict(x=4098), 3, b"16-byte"),
    (dict(strides=[512, 252, 128] * 2), 3, b"16-byte"),
])
def test_rope_refused(lib, kw, status, text):
    assert _rope(lib, **kw) == status
    assert text in lib.cast_last_error_message()


def _norm(lib, **kw):
    a = dict(q=4096, k=4096, v=None, dtype=0, out_dtype=0, eps=1e-6, Hq=4, Hk=2, D=128, qo=4096, ko=4096, vo=None,
             slots=None, pages=0, page=0, qw=4096, strides=[1024, 512, 128] * 5)
    a.update(kw)
    st = (ctypes.c_longlong * 15)(*a["strides"])
    return lib.cast_qk_norm_rope(a["q"], a["k"], a["v"], a["dtype"], a["out_dtype"], a["qw"], 4096, 0, 0, a["eps"], 4096,
                                 4, None, 0, 0, 0, None, 1, 2, a["Hq"], a["Hk"], a["D"], 64, 1, st, a["qo"], a["ko"],
                                 a["vo"], a["slots"], 0, a["pages"], a["page"], None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(k=None), 1, b"required"),
    (dict(out_dtype=2), 2, b"out_dtype"),
    (dict(dtype=2, out_dtype=0), 2, b"out_dtype"),
    (dict(v=4096), 1, b"together"),
    (dict(v=4096, vo=4096), 1, b"together"),
    (dict(v=4096, vo=4096, slots=4096), 1, b"cache"),
    (dict(eps=-1.0), 1, b"eps"),
    (dict(eps=float("nan")), 1, b"eps"),
    (dict(Hk=0), 1, b"heads"),
    (dict(qw=4100), 3, b"16-byte"),
    (dict(strides=[1024, 512, 128] * 4 + [1024, 512, 4]), 3, b"16-byte"),
])
def test_qk_norm_rope_refused(lib, kw, status, text):
    assert _norm(lib, **kw) == status
    assert text in lib.cast_last_error_message()


@pytest.mark.parametrize("r,base,factor,length,fast,slow", [
    (128, 10000.0, 8.0, 131072, 32.0, 1.0),   # the slowest pair turns 2.4 times over the learned length
    (64, 500.0, 4.0, 32768, 32.0, 1.0),       # 8 times or so
    (128, 10000.0, 8.0, 4096, 32.0, 1.0),
    (64, 10000.0, 16.0, 10 ** 7, 8.0, 2.0),   # every pair turns often: all are kept
    (128, 1000000.0, 4.0, 32768, 32.0, 1.0)])
def test_blended_frequencies_pair_by_pair(r, base, factor, length, fast, slow):
    """Each pair by itself: kept above `fast` turns over the learned length,
    divided below `slow`, and between them linear in the pair's index, from the
    last whole index of the first kind to the first one of the second (the
    head's last value at most)."""
    got = rotary.rope_frequencies(r, base=base, scaling=("yarn", factor, length, fast, slow))
    # base^(-2j/r) length / (2 pi) = turns
    place = [r / 2 * math.log(length / (2 * math.pi * t), base) for t in (fast, slow)]
    first, last = math.floor(place[0]), min(math.ceil(place[1]), r - 1)
    assert first >= 0
    for j in range(r // 2):
        step = base ** (-2 * j / r)
        turns = step * length / (2 * math.pi)
        if turns >= fast:
            want = step
        elif turns <= slow:
            want = step / factor
        else:
            share = min(max((j - first) / (last - first), 0.0), 1.0)
            want = step * (1 - share) + step / factor * share
        assert got[j].item() == pytest.approx(want, rel=1e-12), (j, turns)
        if turns > slow and j < last:
            assert got[j].item() > step / factor  # never divided by the whole factor


@pytest.mark.parametrize("scaling", [("yarn", 4.0), ("yarn", 4.0, 4096, 32.0), ("yarn", 4.0, 0), ("yarn", 4.0, -5.0),
                                     ("yarn", 4.0, 4096, 1.0, 32.0), ("yarn", 4.0, 4096, 32.0, 0.0),
                                     ("yarn", 4.0, float("inf")), ("ntk", float("nan"))])
def test_scalings_refused(scaling):
    with pytest.raises(ValueError, match="scaling"):
        rotary.rope_frequencies(64, scaling=scaling)


def test_blended_frequencies_of_a_length_that_no_pair_turns_over():
    f = rotary.rope_frequencies(64)
    for length in (1, 6):  # the fastest pair turns once over 6.3 positions
        assert torch.allclose(rotary.rope_frequencies(64, scaling=("yarn", 4.0, length)), f / 4, rtol=1e-14)
    assert rotary.rope_frequencies(64, scaling=("yarn", 4.0, 7))[0] == f[0]


def test_options_are_read_at_every_call(monkeypatch):
    """An option given as a tensor that changes in place between two calls."""
    seen = []

    def rope(x, table, positions, interleaved, axes, inverse, start, out):
        seen.append((interleaved, axes, inverse, start))
        return True, 0, 0, 0, ()

    def norm(q, k, qw, kw, table, positions, interleaved, axes, start, out_dtype, *rest):
        seen.append((interleaved, axes, start))
        return True, 0, q.dtype, (1,), (1,), (), (), 0, (), ()

    monkeypatch.setattr(rotary, "_rope_plan", rope)
    monkeypatch.setattr(rotary, "_norm_plan", norm)
    monkeypatch.setattr(rotary, "_rope_plans", {})
    monkeypatch.setattr(rotary, "_norm_plans", {})
    x, table = torch.zeros(1, 2, 2, 16), torch.zeros(9, 8, 2)
    start, inter, inv, axes = torch.tensor(1), torch.tensor(True), torch.tensor(False), torch.tensor([4, 2, 2])
    for change in (lambda: None, lambda: start.add_(1), lambda: inter.logical_not_(), lambda: inv.logical_not_(),
                   lambda: axes.copy_(torch.tensor([2, 2, 4]))):
        change()
        rotary.rope(x, table, interleaved=inter, inverse=inv, axes=axes, start=start)
        rotary.qk_norm_rope(x, x, None, None, table, interleaved=inter, axes=axes, start=start)
    a, b = (4, 2, 2), (2, 2, 4)
    assert [s for s in seen if len(s) == 4] == [(True, a, False, 1), (True, a, False, 2), (False, a, False, 2),
                                                (False, a, True, 2), (False, b, True, 2)]
    assert [s for s in seen if len(s) == 3] == [(True, a, 1), (True, a, 2), (False, a, 2), (False, b, 2)]


def test_gradients_of_both_modes_refused():
    x, y = torch.zeros(3), torch.zeros(3, requires_grad=True)
    rotary._refuse_gradients(x, None)
    with pytest.raises(ValueError, match="gradient"):
        rotary._refuse_gradients(x, None, y)
    with torch.no_grad():
        rotary._refuse_gradients(x, None, y)
        with forward_ad.dual_level():
            rotary._refuse_gradients(x, None)
            with pytest.raises(ValueError, match="tangent"):  # no_grad does not end forward mode
                rotary._refuse_gradients(None, forward_ad.make_dual(x, torch.ones(3)))
