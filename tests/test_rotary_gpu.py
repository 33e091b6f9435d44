"""Rotary positions and the norm of query / key heads on the GPU, against the
formulas in 64 bits.

Tolerances (u = half a step of the output type, eps / 2): the output is
rounded once, u |y|.  Before that, in float32 (2^-24 a rounding): a turn takes
the table's rounded cos and sin, two products and a sum, 4 * 2^-24 (|a| + |b|)
of its pair; the norm takes a sum of D squares, eight by eight in a lane and
then over at most 32 lanes (16 roundings), halved by the root, a reciprocal
root off by 2 * 2^-24 * 2, a division, and two products: 16 * 2^-24 more.
float16 results below its normal range are off by 2^-25.
"""

import pytest
import torch

from cast_b200 import _lib, rotary
from cast_b200._lib import CastError
from oracle import rotary as ora

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _close(got, want, size, units, dtype=None):
    dtype = dtype or got.dtype
    tol = torch.finfo(dtype).eps / 2 * want.abs() + units * 2.0 ** -24 * size
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = (got.double() - want).abs()
    assert (off <= tol * 1.01).all(), f"off by {(off / tol.clamp_min(1e-300)).max().item():.3f} of the tolerance"


def _x(*shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * 2).to(dtype)


def _quiet():
    """No device error is pending."""
    _lib.check_device(torch.cuda.current_stream().cuda_stream, "test")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,l,h,d,r", [(1, 1, 1, 8, 0), (1, 1, 24, 128, 128), (2, 5, 3, 64, 32), (3, 7, 1, 80, 80),
                                       (1, 33, 5, 96, 48), (2, 130, 9, 256, 256), (1, 4, 40, 256, 16)])
def test_rope(cuda, dtype, interleaved, b, l, h, d, r):
    if r == 0:
        r = 8 if interleaved else 0
        if not r:
            d, r = 16, 16
    f = rotary.rope_frequencies(r)
    table = rotary.rope_table(f, 700)
    x = _x(b, l, h, d, dtype=dtype)
    pos = torch.randint(0, 700, (b, l), device="cuda", dtype=torch.int32)
    want = ora.turn(x.double(), ora.angles(pos, f), interleaved)
    size = ora.pair_size(x.double(), r, interleaved)
    _close(rotary.rope(x, table, pos, interleaved=interleaved), want, size, 4)
    # positions of 64 bits, shared by the batch
    want = ora.turn(x.double(), ora.angles(pos[:1].expand(b, l), f), interleaved)
    _close(rotary.rope(x, table, pos[0].long(), interleaved=interleaved), want, size, 4)
    # none: one after the other
    want = ora.turn(x.double(), ora.angles(torch.arange(3, 3 + l, device="cuda").expand(b, l), f), interleaved)
    _close(rotary.rope(x, table, interleaved=interleaved, start=3), want, size, 4)
    _quiet()


@pytest.mark.parametrize("interleaved", [True, False])
def test_rope_axes_far_and_scaled(cuda, interleaved):
    axes = (22, 21, 21)
    f = rotary.rope_frequencies(128, axes=axes, scaling=("ntk", 4.0))
    table = rotary.rope_table(f, 64)
    x = _x(2, 50, 3, 128, dtype=torch.bfloat16)
    pos = torch.randint(0, 64, (2, 50, 3), device="cuda")
    want = ora.turn(x.double(), ora.angles(pos, f, axes), interleaved)
    got = rotary.rope(x, table, pos, interleaved=interleaved, axes=axes)
    _close(got, want, ora.pair_size(x.double(), 128, interleaved), 4)
    f = rotary.rope_frequencies(64, scaling=("yarn", 8.0, 4096))
    table = rotary.rope_table(f, 1_000_001)
    x = _x(1, 4, 2, 64, dtype=torch.float32)
    pos = torch.tensor([[0, 131071, 999999, 1000000]], device="cuda")
    want = ora.turn(x.double(), ora.angles(pos, f), interleaved)
    _close(rotary.rope(x, table, pos, interleaved=interleaved), want, ora.pair_size(x.double(), 64, interleaved), 4)


@pytest.mark.parametrize("interleaved", [True, False])
def test_rope_strides_in_place_and_back(cuda, interleaved):
    f = rotary.rope_frequencies(64)
    table = rotary.rope_table(f, 100)
    qkv = _x(2, 9, 12, 128, dtype=torch.bfloat16)
    before = qkv.clone()
    part = qkv[:, :, 4:8]  # a slice of a projection
    pos = torch.arange(9, device="cuda").flip(0)
    theta = ora.angles(pos.expand(2, 9), f)
    want, size = ora.turn(part.double(), theta, interleaved), ora.pair_size(part.double(), 64, interleaved)
    out = torch.empty(2, 4, 9, 128, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    assert rotary.rope(part, table, pos, interleaved=interleaved, out=out) is out
    _close(out, want, size, 4)
    rotary.rope(part, table, pos, interleaved=interleaved, out=part)  # in place
    assert torch.equal(part, out)
    assert torch.equal(qkv[:, :, :4], before[:, :, :4]) and torch.equal(qkv[:, :, 8:], before[:, :, 8:])
    back = rotary.rope(part, table, pos, interleaved=interleaved, inverse=True)
    _close(back, ora.turn(part.double(), -theta, interleaved), ora.pair_size(part.double(), 64, interleaved), 4)
    # a head that all heads share (stride 0), and head-major tensors
    one = _x(2, 9, 1, 128, dtype=torch.bfloat16).expand(2, 9, 5, 128)
    want = ora.turn(one.double(), theta, interleaved)
    _close(rotary.rope(one, table, pos, interleaved=interleaved), want, ora.pair_size(one.double(), 64, interleaved), 4)


def test_rope_special_values(cuda):
    f = rotary.rope_frequencies(16)
    table = rotary.rope_table(f, 8)
    x = _x(1, 3, 2, 32, dtype=torch.float16)
    x[0, 1, 0, 0] = float("inf")
    x[0, 1, 1, 31] = float("nan")  # not turned: stays alone
    x[0, 2, 0, 3] = 6e-8
    y = rotary.rope(x, table)
    bad = ~torch.isfinite(y)
    assert bad[0, 1, 0, :2].any() and bad[0, 1, 1, 31] and int(bad.sum()) <= 3
    assert not bad[0, 0].any() and not bad[0, 2].any()


def test_unknown_positions_are_zeros_and_reported(cuda):
    table = rotary.rope_table(rotary.rope_frequencies(64), 10)
    x = _x(1, 4, 3, 64, dtype=torch.bfloat16)
    pos = torch.tensor([3, 10, -1, 9], device="cuda")
    y = rotary.rope(x, table, pos)
    with pytest.raises(CastError):
        _quiet()
    assert (y[0, 1:3] == 0).all() and (y[0, 0] != 0).any() and (y[0, 3] != 0).any()
    _quiet()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,l,hq,hk,d,r,f32,per_head", [
    (1, 1, 1, 1, 64, 64, False, False), (3, 1, 32, 8, 128, 128, True, False), (2, 37, 6, 2, 128, 64, False, True),
    (1, 130, 5, 5, 80, 48, True, True), (2, 9, 3, 1, 256, 256, False, False), (1, 17, 24, 24, 96, 0, False, False)])
def test_qk_norm_rope(cuda, dtype, interleaved, b, l, hq, hk, d, r, f32, per_head):
    qkv = _x(b, l, hq + 2 * hk, d, dtype=dtype)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    wt = torch.float32 if f32 else dtype
    qw, kw = (1 + _x(*((h, d) if per_head else (d,)), dtype=torch.float32, seed=h) / 8 for h in (hq, hk))
    qw, kw = qw.to(wt), kw.to(wt)
    f = rotary.rope_frequencies(r) if r else None
    table = rotary.rope_table(f, 300) if r else None
    pos = torch.randint(0, 300, (b, l), device="cuda") if r else None
    got = rotary.qk_norm_rope(q, k, qw, kw, table, pos, eps=1e-5, interleaved=interleaved)
    for y, x, w in zip(got, (q, k), (qw, kw)):
        assert y.shape == (b, x.shape[2], l, d) and y.is_contiguous()
        z = ora.norm(x, w, 1e-5)
        want = ora.turn(z, ora.angles(pos, f), interleaved) if r else z
        size = ora.pair_size(z, r, interleaved) if r else z.abs()
        _close(y.transpose(1, 2), want, size, 20)
    _quiet()


def test_qk_norm_rope_one_side_types_and_out(cuda):
    f = rotary.rope_frequencies(128)
    table = rotary.rope_table(f, 64)
    q, k = _x(2, 11, 4, 128, dtype=torch.float32), _x(2, 11, 2, 128, dtype=torch.float32, seed=1)
    qw = 1 + _x(128, dtype=torch.float32, seed=2) / 8
    qo = torch.empty(2, 11, 4, 128, dtype=torch.bfloat16, device="cuda")
    got = rotary.qk_norm_rope(q, k, qw, None, table, out_dtype=torch.bfloat16, out=(qo.transpose(1, 2), None))
    assert got[0].data_ptr() == qo.data_ptr() and got[1].dtype == torch.bfloat16
    theta = ora.angles(torch.arange(11, device="cuda").expand(2, 11), f)
    for y, z in ((qo, ora.norm(q, qw, 1e-6)), (got[1].transpose(1, 2), k.double())):
        _close(y, ora.turn(z, theta, True), ora.pair_size(z, 128, True), 20)
    # a head of zeros: the norm of nothing is nothing
    q[0, 0, 0] = 0
    assert (rotary.qk_norm_rope(q, k, qw, None, table)[0][0, 0, 0] == 0).all()


@pytest.mark.parametrize("slot_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("interleaved", [True, False])
def test_qk_norm_rope_into_pages(cuda, slot_type, interleaved):
    b, l, hq, hk, d, page = 2, 21, 4, 2, 64, 16
    f = rotary.rope_frequencies(d)
    table = rotary.rope_table(f, 64)
    qkv = _x(b, l, hq + 2 * hk, d, dtype=torch.bfloat16)
    q, k, v = qkv[:, :, :hq], qkv[:, :, hq:hq + hk], qkv[:, :, hq + hk:]
    w = 1 + _x(d, dtype=torch.bfloat16, seed=3) / 8
    kp, vp = _x(6, hk, page, d, dtype=torch.bfloat16, seed=4), _x(6, hk, page, d, dtype=torch.bfloat16, seed=5)
    k0, v0 = kp.clone(), vp.clone()
    slots = torch.randperm(6 * page, device="cuda")[:b * l].view(b, l).to(slot_type)
    slots[0, 3], slots[1, 20] = -1, 6 * page  # not written; past the end
    got, pages = rotary.qk_norm_rope(q, k, w, w, table, interleaved=interleaved, v=v, cache=(kp, vp), slots=slots)
    assert pages[0] is kp and pages[1] is vp
    with pytest.raises(CastError):
        _quiet()
    theta = ora.angles(torch.arange(l, device="cuda").expand(b, l), f)
    z = ora.norm(q, w, 1e-6)
    _close(got.transpose(1, 2), ora.turn(z, theta, interleaved), ora.pair_size(z, d, interleaved), 20)
    plain_k = rotary.qk_norm_rope(q, k, w, w, table, interleaved=interleaved)[1]
    touched = torch.zeros(6, page, dtype=torch.bool, device="cuda")
    for bb in range(b):
        for t in range(l):
            s = int(slots[bb, t])
            if 0 <= s < 6 * page:
                assert torch.equal(kp[s // page, :, s % page], plain_k[bb, :, t])
                assert torch.equal(vp[s // page, :, s % page], v[bb, t])
                touched[s // page, s % page] = True
    left = ~touched[:, None, :, None].expand_as(kp)
    assert torch.equal(kp[left], k0[left]) and torch.equal(vp[left], v0[left])
    _quiet()


def test_rotary_refusals(cuda):
    table = rotary.rope_table(rotary.rope_frequencies(64), 10)
    x = _x(1, 4, 3, 64, dtype=torch.bfloat16)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(x=x.transpose(2, 3)), dict(x=x[..., :32]),
                dict(table=table.double()), dict(table=table.cpu()), dict(start=7),
                dict(positions=torch.zeros(5, device="cuda", dtype=torch.int32)),
                dict(positions=torch.zeros(4, device="cuda")), dict(positions=torch.zeros(4, dtype=torch.int32)),
                dict(axes=(16, 16)), dict(out=torch.empty_like(x[:, :2])), dict(out=x[:, :, :1].expand(1, 4, 3, 64)),
                dict(x=x.clone().requires_grad_())):
        args = dict(x=x, table=table)
        args.update(bad)
        with pytest.raises(ValueError):
            rotary.rope(args.pop("x"), args.pop("table"), args.pop("positions", None), **args)
    with pytest.raises(CastError, match="16-byte"):
        rotary.rope(torch.zeros(1, 2, 2, 65, dtype=torch.bfloat16, device="cuda")[..., 1:], table)
    y = x.clone().requires_grad_()
    with torch.no_grad():
        assert torch.equal(rotary.rope(y, table), rotary.rope(x, table))
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    kp = torch.zeros(2, 3, 8, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    for bad in (dict(k=x[:, :2]), dict(kw=w.float()), dict(kw=w[:32]), dict(qw=w.double()), dict(v=x), dict(cache=(kp, kp)),
                dict(v=x, slots=slots, cache=(kp, kp[:1])), dict(v=x, slots=slots[:, :3], cache=(kp, kp)),
                dict(v=x, slots=slots, cache=(kp.half(), kp.half())), dict(out_dtype=torch.float16)):
        args = dict(k=x, qw=w, kw=w)
        args.update(bad)
        with pytest.raises(ValueError):
            rotary.qk_norm_rope(x, args.pop("k"), args.pop("qw"), args.pop("kw"), table, **args)
    assert rotary.rope(x[:, :0], table).shape == (1, 0, 3, 64)
    assert rotary.qk_norm_rope(x[:0], x[:0], w, w, table)[0].shape == (0, 3, 4, 64)


def test_rotary_on_another_stream_and_in_a_graph(cuda):
    f = rotary.rope_frequencies(128)
    table = rotary.rope_table(f, 256)
    x = _x(2, 64, 8, 128, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    want = rotary.rope(x, table)
    wq, wk = rotary.qk_norm_rope(x, x[:, :, :2], w, w, table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary.rope(x, table)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    still = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rotary.rope(still, table)
        gq, gk = rotary.qk_norm_rope(still, still[:, :, :2], w, w, table)
    still.zero_()
    g.replay()
    assert (y == 0).all() and (gq == 0).all()
    still.copy_(x)
    g.replay()
    assert torch.equal(y, want) and torch.equal(gq, wq) and torch.equal(gk, wk)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("b,l,hq,hk,d,r", [(1, 2100, 24, 24, 128, 128), (3, 700, 8, 2, 128, 128), (1, 5000, 3, 1, 64, 32),
                                           (2, 1500, 16, 16, 64, 64), (1, 4097, 1, 1, 48, 48), (1, 1300, 5, 2, 256, 256),
                                           (1, 3001, 4, 4, 24, 16 * 1), (1, 9, 2, 1, 40, 32)])
def test_many_tokens_and_every_lane_layout(cuda, interleaved, b, l, hq, hk, d, r):
    """The layouts that the launch picks from: one or two pieces a lane, few or many heads a lane, runs of tokens."""
    f = rotary.rope_frequencies(r)
    table = rotary.rope_table(f, l + 3)
    q, k = _x(b, l, hq, d, dtype=torch.bfloat16), _x(b, l, hk, d, dtype=torch.bfloat16, seed=1)
    w = 1 + _x(d, dtype=torch.float32, seed=2) / 8
    theta = ora.angles(torch.arange(3, l + 3, device="cuda").expand(b, l), f)
    for y, x in zip(rotary.qk_norm_rope(q, k, w, w, table, start=3, interleaved=interleaved), (q, k)):
        z = ora.norm(x, w, 1e-6)
        _close(y.transpose(1, 2), ora.turn(z, theta, interleaved), ora.pair_size(z, r, interleaved), 20)
    want = ora.turn(q.double(), theta, interleaved)
    _close(rotary.rope(q, table, start=3, interleaved=interleaved), want, ora.pair_size(q.double(), r, interleaved), 4)
    _quiet()


def test_unknown_positions_under_the_norm(cuda):
    table = rotary.rope_table(rotary.rope_frequencies(128), 10)
    x = _x(1, 4, 8, 128, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    pos = torch.tensor([3, 10, -1, 9], device="cuda")
    for eps in (1e-6, 0.0):
        for y in rotary.qk_norm_rope(x, x[:, :, :2], w, w, table, pos, eps=eps):
            assert (y[0, :, 1:3] == 0).all() and (y[0, :, 0] != 0).any() and (y[0, :, 3] != 0).any()
        with pytest.raises(CastError):
            _quiet()


def test_single_precision_into_half_precision_pages(cuda):
    table = rotary.rope_table(rotary.rope_frequencies(64), 16)
    q, k, v = (_x(2, 5, h, 64, dtype=torch.float32, seed=h) for h in (4, 2, 2))
    v = v * 1.001
    w = torch.ones(64, device="cuda")
    kp = torch.zeros(3, 2, 8, 64, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    slots = torch.arange(10, device="cuda").view(2, 5) + 7
    rotary.qk_norm_rope(q, k, w, w, table, v=v, cache=(kp, vp), slots=slots, out_dtype=torch.bfloat16)
    want = rotary.qk_norm_rope(q, k, w, w, table, out_dtype=torch.bfloat16)[1]
    s = slots.view(-1)
    assert torch.equal(kp[s // 8, :, s % 8], want.transpose(1, 2).reshape(10, 2, 64))
    assert torch.equal(vp[s // 8, :, s % 8], v.bfloat16().reshape(10, 2, 64))
    _quiet()


def test_inputs_with_tangents_and_outs_with_gradients_refused(cuda):
    from torch.autograd import forward_ad

    from cast_b200 import window

    table = rotary.rope_table(rotary.rope_frequencies(64), 10)
    x = _x(1, 4, 3, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    pages = torch.zeros(1, dtype=torch.int32, device="cuda")[None]

    def calls(y, out=None):
        yield lambda: rotary.rope(y, table, out=out)
        yield lambda: rotary.qk_norm_rope(x, y, w, w, table, out=None if out is None else (None, out.transpose(1, 2)))
        yield lambda: window.window_attention(x, x, y, window=2, out=out)
        yield lambda: window.paged_window_attention(x, x, y, pages, n, window=2, out=out)

    for call in calls(x):
        call()  # as it is (and kept as checked)
    with forward_ad.dual_level(), torch.no_grad():
        for call in calls(forward_ad.make_dual(x, torch.ones_like(x))):
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in calls(x):
            call()
    for call in calls(x, out=torch.zeros_like(x, requires_grad=True)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        for call in calls(x, out=torch.zeros_like(x, requires_grad=True)):
            call()
    with pytest.raises(ValueError, match="gradient"):
        rotary.qk_norm_rope(x, x, w.clone().requires_grad_(), w, table)
    _quiet()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,r,l,h", [(128, 128, 4, 5), (128, 64, 4, 3), (64, 64, 300, 7), (256, 256, 4, 2), (80, 48, 9, 3)])
def test_unknown_positions_are_zeros_whatever_weights_and_table_hold(cuda, interleaved, d, r, l, h):
    table = rotary.rope_table(rotary.rope_frequencies(r), 10)
    table[0] = float("nan")
    x = _x(2, l, h, d, dtype=torch.bfloat16)
    pos = torch.randint(1, 10, (2, l), device="cuda")
    pos[:, 1], pos[1, 2] = 10, -1
    unknown = (pos < 0) | (pos > 9)
    y = rotary.rope(x, table, pos, interleaved=interleaved)
    assert (y[unknown] == 0).all() and torch.isfinite(y).all() and (y[~unknown] != 0).any()
    x0 = x.clone()
    assert torch.equal(rotary.rope(x0, table, pos, interleaved=interleaved, out=x0), y)
    kp = torch.full((2 * l // 4 + 1, h, 4, d), 3.0, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    slots = torch.randperm(2 * l, device="cuda").view(2, l)
    for w in (torch.full((d,), float("inf"), device="cuda"), torch.full((h, d), float("nan"), device="cuda").bfloat16()):
        for got in rotary.qk_norm_rope(x, x, w, w, table, pos, interleaved=interleaved):
            assert (got.transpose(1, 2)[unknown] == 0).all() and not torch.isfinite(got.transpose(1, 2)[~unknown]).any()
        q, _ = rotary.qk_norm_rope(x, x, w, w, table, pos, interleaved=interleaved, v=x, cache=(kp, vp), slots=slots)
        s = slots[unknown]
        assert (q.transpose(1, 2)[unknown] == 0).all() and (kp[s // 4, :, s % 4] == 0).all()
        s = slots.view(-1)
        assert torch.equal(vp[s // 4, :, s % 4], x.view(2 * l, h, d))  # values are copied whatever the position
    with pytest.raises(CastError):
        _quiet()
    _quiet()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,l,hq,hk,d", [(1, 9, 17, 24, 128), (1, 9, 16, 24, 128), (2, 130, 18, 18, 128), (1, 77, 25, 23, 128),
                                         (1, 3001, 22, 20, 128), (1, 5921, 18, 17, 128), (3, 21, 10, 12, 256),
                                         (1, 40, 33, 48, 64), (1, 40, 23, 23, 72), (5, 1200, 17, 17, 128)])
def test_head_counts_around_a_batch_of_three_a_lane(cuda, dtype, b, l, hq, hk, d):
    f = rotary.rope_frequencies(d)
    table = rotary.rope_table(f, l)
    x = _x(b, l, hq + hk, d, dtype=dtype)
    q, k = x[:, :, :hq], x[:, :, hq:]
    qw, kw = (1 + _x(d, dtype=torch.float32, seed=s) / 8 for s in (2, 3))
    theta = ora.angles(torch.arange(l, device="cuda").expand(b, l), f)
    for y, x, w in zip(rotary.qk_norm_rope(q, k, qw, kw, table), (q, k), (qw, kw)):
        z = ora.norm(x, w, 1e-6)
        _close(y.transpose(1, 2), ora.turn(z, theta, True), ora.pair_size(z, d, True), 20)
    _quiet()


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("hq,hk,l", [(2, 40, 3), (24, 24, 3), (24, 24, 2500), (3, 1, 4)])
def test_values_of_unknown_positions_are_copied(cuda, normed, hq, hk, l):
    """However many heads a lane takes one after the other; keys and queries are zeros."""
    d = 128
    table = rotary.rope_table(rotary.rope_frequencies(d), 10)
    x = _x(1, l, hq + 2 * hk, d, dtype=torch.bfloat16)
    q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
    pos = torch.randint(0, 10, (l,), device="cuda")
    pos[1], pos[2] = 10, -7
    w = torch.full((d,), float("inf"), device="cuda") if normed else None
    kp = torch.full((l // 4 + 1, hk, 4, d), 3.0, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    slots = torch.randperm(l, device="cuda")[None]
    got, _ = rotary.qk_norm_rope(q, k, w, w, table, pos, v=v, cache=(kp, vp), slots=slots)
    s = slots[0]
    assert torch.equal(vp[s // 4, :, s % 4], v[0])
    assert (got[0, :, 1:3] == 0).all() and (kp[s[1:3] // 4, :, s[1:3] % 4] == 0).all()
    if not normed:
        plain = rotary.qk_norm_rope(q, k, None, None, table, pos)
        assert torch.equal(got, plain[0]) and torch.equal(kp[s // 4, :, s % 4], plain[1][0].transpose(0, 1))
        assert torch.isfinite(got).all() and (got[0, :, 0] != 0).any()
    with pytest.raises(CastError):
        _quiet()
    _quiet()
