"""CPU: the visibility rule of the window attention, and what it refuses."""

import ctypes

import pytest
import torch

from cast_b200 import _lib, window
from oracle import window as ora


@pytest.fixture(scope="module")
def lib():
    from cast_b200 import build

    build.build()
    return _lib.load()


def test_the_rule_token_by_token():
    s = ora.sees(7, 3, 2, 1, 1)
    assert s.tolist() == [[True, False, False, True, True, False, False],
                          [True, False, False, False, True, True, False],
                          [True, False, False, False, False, True, True]]
    # frames of 2: the chunk's frame sees itself whole, one frame back, and the first frame
    s = ora.sees(8, 2, 2, 1, 2)
    assert s.tolist() == [[True, True, False, False, True, True, True, True]] * 2
    # more queries than keys: the first ones have no position
    s = ora.sees(1, 3, 5, 4, 1)
    assert s.tolist() == [[False], [False], [True]]


def test_oracle_keeps_hidden_values_out():
    q, k, v = torch.randn(2, 4), torch.randn(3, 4), torch.randn(3, 4)
    seen = torch.tensor([[True, True, False], [False, False, False]])
    v[2] = float("nan")
    out, size, _, _ = ora.attention(q, k, v, seen)
    assert torch.isfinite(out).all() and (out[1] == 0).all() and (size[1] == 0).all()
    seen[1, 2] = True
    assert torch.isnan(ora.attention(q, k, v, seen)[0][1]).all()


def test_python_refuses_host_tensors():
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        window.window_attention(x, x, x, window=4)
    with pytest.raises(ValueError, match="CUDA"):
        window.paged_window_attention(x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                      window=4)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1),
                                dict(window=4, frame_tokens=0)])
def test_rule_refused(kw):
    with pytest.raises(ValueError, match="window"):
        window._rule(kw["window"], kw.get("sinks", 0), kw.get("frame_tokens", 1))


def test_rule_takes_any_size():
    assert window._rule(None, 0, 1)[0] >= 1 << 31
    assert window._rule(1 << 70, 1 << 70, 1 << 70) == (1 << 40, 1 << 40, 1 << 30)


def _call(lib, **kw):
    a = dict(q=4096, k=4096, v=4096, dtype=0, lens=None, B=1, Hq=4, Hk=2, Lq=8, Lk=16, D=128,
             strides=[4096, 1024, 128] * 4, window=8, sinks=0, frame=1, scale=0.1, out=4096)
    a.update(kw)
    st = (ctypes.c_longlong * 12)(*a["strides"])
    return lib.cast_window_attention(a["q"], a["k"], a["v"], a["dtype"], a["lens"], a["B"], a["Hq"], a["Hk"], a["Lq"],
                                     a["Lk"], a["D"], st, a["window"], a["sinks"], a["frame"], a["scale"], a["out"], None,
                                     0, None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(q=None), 1, b"required"),
    (dict(dtype=1), 2, b"dtype"),
    (dict(B=0), 1, b"non-positive"),
    (dict(Lk=0), 1, b"non-positive"),
    (dict(Hq=3), 1, b"evenly"),
    (dict(D=96), 2, b"head_dim"),
    (dict(window=0), 1, b"window"),
    (dict(sinks=-1), 1, b"sinks"),
    (dict(frame=0), 1, b"frame_tokens"),
    (dict(scale=0.0), 1, b"sm_scale"),
    (dict(scale=float("inf")), 1, b"sm_scale"),
    (dict(k=4104), 3, b"16-byte"),
    (dict(strides=[4096, 1024, 132] * 4), 3, b"16-byte"),
    (dict(Lk=1 << 30), 2, b"index range"),
])
def test_window_attention_refused(lib, kw, status, text):
    assert _call(lib, **kw) == status
    assert text in lib.cast_last_error_message()


def _paged(lib, **kw):
    a = dict(table=4096, max_pages=4, n_pages=8, page=16, lens=4096, D=64, scale=0.1)
    a.update(kw)
    st = (ctypes.c_longlong * 12)(*([2048, 512, 64] * 4))
    return lib.cast_paged_window_attention(4096, 4096, 4096, 0, a["table"], a["max_pages"], a["n_pages"], a["page"],
                                           a["lens"], 2, 4, 2, 1, a["D"], st, 8, 0, 1, a["scale"], 4096, None, 0, None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(table=None), 1, b"block_table"),
    (dict(lens=None), 1, b"kv_lens"),
    (dict(page=0), 1, b"cache"),
    (dict(n_pages=0), 1, b"cache"),
    (dict(max_pages=1 << 28), 2, b"keys in one session"),
    (dict(D=32), 2, b"head_dim"),
])
def test_paged_window_attention_refused(lib, kw, status, text):
    assert _paged(lib, **kw) == status
    assert text in lib.cast_last_error_message()


def test_python_refuses_what_is_no_tensor():
    with pytest.raises(ValueError, match="CUDA"):
        window.window_attention([1], None, None, window=4)
    with pytest.raises(ValueError, match="CUDA"):
        window.paged_window_attention(None, None, None, None, None, window=4)


def test_options_are_read_at_every_call(monkeypatch):
    """An option given as a tensor that changes in place between two calls."""
    seen = []

    def plan(q, k, v, win, sinks, frame, *rest):
        seen.append((win, sinks, frame))
        return True, False, 0, 0, 0.0, (), ()

    def paged(q, k, v, table, lens, win, sinks, frame, *rest):
        seen.append((win, sinks, frame))
        return True, False, 0, 0, 0.0, (), (), ()

    monkeypatch.setattr(window, "_window_plan", plan)
    monkeypatch.setattr(window, "_paged_plan", paged)
    monkeypatch.setattr(window, "_plans", {})
    monkeypatch.setattr(window, "_paged_plans", {})
    x, n = torch.zeros(1, 2, 4, 64), torch.zeros(1, dtype=torch.int32)
    for call in (lambda *a: window.window_attention(x, x, x, window=a[0], sinks=a[1], frame_tokens=a[2]),
                 lambda *a: window.paged_window_attention(x, x, x, n[None], n, window=a[0], sinks=a[1], frame_tokens=a[2])):
        opts = [torch.tensor(9), torch.tensor(2), torch.tensor(3)]
        seen.clear()
        call(*opts)
        for o in opts:
            o.add_(1)
            call(*opts)
        assert seen == [(9, 2, 3), (10, 2, 3), (10, 3, 3), (10, 3, 4)]
        assert all(type(v) is int for s in seen for v in s)
