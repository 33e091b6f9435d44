"""Sliding-window attention with sinks on the GPU, dense and paged, against
``oracle.window`` in 64 bits; the tolerance is derived there."""

import pytest
import torch

from cast_b200 import _lib, rotary, window
from cast_b200._lib import CastError
from oracle import rotary as ora_rotary
from oracle import window as ora

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _quiet():
    _lib.check_device(torch.cuda.current_stream().cuda_stream, "test")


def _data(b, hq, hk, d, lq, lk, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda")

    return ((normal(b, hq, lq, d) * spread).to(dtype), normal(b, hk, lk, d).to(dtype),
            (normal(b, hk, lk, d) + 0.5 * normal(hk, 1, d)).to(dtype))


def _check(got, q, k, v, lens, *, window, sinks=0, frame=1, scale=None, heads=None):
    """Every (or the given) head of every session against the oracle."""
    b, hq, lq, d = q.shape
    group = hq // k.shape[1]
    for bb in range(b):
        n = k.shape[2] if lens is None else int(lens[bb])
        seen = ora.sees(n, lq, window, sinks, frame, device=q.device)
        for h in range(hq) if heads is None else heads:
            want, size, top, spread = ora.attention(q[bb, h], k[bb, h // group, :n], v[bb, h // group, :n], seen, scale)
            tol = ora.tolerance(want, size, top, spread, d, n, q.dtype)
            x = got[bb, h].double()
            fine = torch.isfinite(want)
            assert torch.equal(torch.isfinite(x), fine), (bb, h)
            assert torch.equal(torch.isnan(x), torch.isnan(want)), (bb, h)
            off = torch.where(fine, (x - want).abs(), torch.zeros_like(x))
            assert (off <= tol).all(), (bb, h, (off / tol.clamp_min(1e-300)).max().item())
            assert (x[~seen.any(-1)] == 0).all()


CASES = [
    # b, hq, hk, d, lq, lk, window, sinks, frame, lens, dtype
    (1, 1, 1, 128, 1, 1, 1, 0, 1, None, BF16),
    (1, 2, 1, 64, 1, 17, None, 0, 1, None, FP16),
    (2, 24, 24, 128, 1, 300, 100, 3, 1, [300, 1], BF16),
    (1, 8, 2, 128, 1, 5000, 4096, 4, 1, None, BF16),
    (1, 3, 1, 64, 4, 90, 17, 2, 1, None, BF16),          # 12 rows
    (2, 16, 1, 128, 2, 700, 600, 130, 1, [700, 611], BF16),  # 32 rows
    (1, 4, 4, 128, 16, 40, 5, 0, 1, None, FP16),
    (2, 6, 2, 64, 11, 64, 1, 1, 1, [3, 64], FP16),       # queries without a position, a window of one
    (1, 4, 2, 128, 40, 333, 50, 7, 1, None, BF16),
    (1, 2, 2, 128, 128, 128, None, 0, 1, None, BF16),
    (1, 4, 1, 128, 100, 1000, 128, 128, 1, None, BF16),
    (2, 3, 1, 64, 129, 700, 77, 0, 1, [500, 640], FP16),
    (1, 2, 1, 128, 260, 1030, 3, 1, 110, None, BF16),    # frames
    (1, 6, 2, 128, 300, 900, 2, 1, 64, None, FP16),
    (1, 2, 2, 64, 513, 1025, 1, 0, 880, None, BF16),     # a frame larger than a tile
    (3, 4, 2, 128, 257, 1111, 200, 20, 1, [1111, 257, 100], BF16),
    (1, 8, 8, 128, 384, 384, 100000, 100000, 1, None, BF16),
    (1, 12, 4, 64, 200, 4000, None, 5, 1, None, BF16),
    (1, 2, 1, 128, 88, 20000, None, 0, 1, None, BF16),
    (2, 2, 1, 128, 70, 900, 300, 0, 1, [0, 900], BF16),  # an empty session
]


@pytest.mark.parametrize("b,hq,hk,d,lq,lk,win,sinks,frame,lens,dtype", CASES)
def test_window_attention(cuda, b, hq, hk, d, lq, lk, win, sinks, frame, lens, dtype):
    q, k, v = _data(b, hq, hk, d, lq, lk, dtype, seed=lq + lk)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = window.window_attention(q, k, v, window=win, sinks=sinks, frame_tokens=frame, kv_lens=n)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    _check(got, q, k, v, lens, window=win, sinks=sinks, frame=frame)
    _quiet()
    again = window.window_attention(q, k, v, window=win, sinks=sinks, frame_tokens=frame, kv_lens=n)
    assert torch.equal(got, again)  # every sum has one order


@pytest.mark.parametrize("lq", [1, 9, 150, 300])
def test_what_a_query_does_not_see_never_reaches_it(cuda, lq):
    """NaN and infinities behind the lengths, before the window and at keys
    that only some rows of a tile see."""
    lk, win, sinks = 700, 60, 5
    lens = [700, 512]
    q, k, v = _data(2, 4, 2, 128, lq, lk, BF16, seed=lq)
    for bb, n in enumerate(lens):
        k[bb, :, n:], v[bb, :, n:] = float("nan"), float("inf")
        first = max(0, n - lq - win)
        k[bb, :, sinks:first], v[bb, :, sinks:first] = float("inf"), float("nan")
    if lq > 1:
        v[0, 0, 698, 7], v[0, 1, 700 - lq + 2, 100] = float("inf"), float("nan")
        k[1, 0, 511 - lq // 2] = float("nan")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = window.window_attention(q, k, v, window=win, sinks=sinks, kv_lens=n)
    for bb in range(2):  # a NaN score makes its row NaN: the oracle's softmax does the same
        seen = ora.sees(lens[bb], lq, win, sinks, 1, device="cuda")
        for h in range(4):
            kk, vv = k[bb, h // 2, :lens[bb]], v[bb, h // 2, :lens[bb]]
            sick = (seen & torch.isnan(kk).any(-1)).any(-1)
            assert torch.isnan(got[bb, h][sick]).all()
            kk = torch.where(torch.isnan(kk).any(-1, keepdim=True), torch.zeros_like(kk), kk)
            want, size, top, spread = ora.attention(q[bb, h], kk, vv, seen)
            tol = ora.tolerance(want, size, top, spread, 128, lens[bb], BF16)
            x = got[bb, h].double()
            well = torch.isfinite(want) & ~sick[:, None]
            assert torch.equal(torch.isfinite(x)[~sick], torch.isfinite(want)[~sick])
            assert ((x - want).abs() <= tol)[well].all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lq", [1, 200])
def test_large_scores_and_a_scale(cuda, dtype, lq):
    q, k, v = _data(1, 4, 2, 64, lq, 600, dtype, seed=3, spread=6.0)
    k[:, :, 300:] *= 3  # the maximum moves late
    got = window.window_attention(q, k, v, window=500, sinks=2, sm_scale=0.31)
    _check(got, q, k, v, None, window=500, sinks=2, scale=0.31)


@pytest.mark.parametrize("lq", [1, 3, 90, 333])
def test_strides_and_out(cuda, lq):
    b, hq, hk, d, lk = 2, 8, 2, 128, 500
    q0, k0, v0 = _data(b, hq, hk, d, lq, lk, BF16, seed=5)
    want = window.window_attention(q0, k0, v0, window=200, sinks=3)
    q = q0.transpose(1, 2).contiguous().transpose(1, 2)      # token-major, as a projection leaves it
    kv = torch.empty(b, lk, 2 * hk, d, dtype=BF16, device="cuda")
    kv[:, :, :hk], kv[:, :, hk:] = k0.transpose(1, 2), v0.transpose(1, 2)
    k, v = kv[:, :, :hk].transpose(1, 2), kv[:, :, hk:].transpose(1, 2)
    room = torch.full((b, lq, hq + 1, d), 7.0, dtype=BF16, device="cuda")
    out = room[:, :, :hq].transpose(1, 2)
    assert window.window_attention(q, k, v, window=200, sinks=3, out=out) is out
    assert torch.equal(out, want) and (room[:, :, hq] == 7).all()
    # one cache for the whole batch
    one = window.window_attention(q0, k0[:1].expand(b, hk, lk, d), v0[:1].expand(b, hk, lk, d), window=200, sinks=3)
    assert torch.equal(one[0], want[0])


def _pages(k, v, page, extra=3, seed=0):
    """The dense keys of every session in shuffled pages; unused rows are NaN."""
    b, hk, lk, d = k.shape
    each = -(-lk // page)
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.randperm(b * each + extra, generator=g, device="cuda")[:b * each].view(b, each)
    kp = torch.full((b * each + extra, hk, page, d), float("nan"), dtype=k.dtype, device="cuda")
    vp = kp.clone()
    j = torch.arange(lk, device="cuda")
    for bb in range(b):
        kp[order[bb, j // page], :, j % page] = k[bb].transpose(0, 1)
        vp[order[bb, j // page], :, j % page] = v[bb].transpose(0, 1)
    return kp, vp, order.to(torch.int32)


PAGED = [
    # b, hq, hk, d, lq, lens, window, sinks, page, dtype
    (1, 1, 1, 64, 1, [1], 1, 0, 16, BF16),
    (3, 8, 2, 128, 1, [100, 1, 37], 20, 3, 16, BF16),
    (4, 32, 8, 128, 1, [3000, 2999, 17, 512], 1024, 4, 64, BF16),
    (2, 8, 8, 64, 3, [531, 438], 200, 5, 16, FP16),
    (2, 12, 2, 128, 7, [90, 4], None, 0, 13, FP16),    # a page of 13, more queries than keys
    (1, 4, 1, 64, 40, [777], 50, 70, 128, BF16),       # many rows
    (16, 4, 4, 128, 1, [64 * i + 1 for i in range(16)], 300, 16, 256, BF16),
    (1, 2, 1, 128, 1, [30000], None, 0, 64, BF16),     # more parts than a cluster has
]


@pytest.mark.parametrize("b,hq,hk,d,lq,lens,win,sinks,page,dtype", PAGED)
def test_paged_window_attention(cuda, b, hq, hk, d, lq, lens, win, sinks, page, dtype):
    lk = max(lens)
    q, k, v = _data(b, hq, hk, d, lq, lk, dtype, seed=lk)
    for bb, n in enumerate(lens):
        k[bb, :, n:], v[bb, :, n:] = float("nan"), float("inf")
    kp, vp, table = _pages(k, v, page)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = window.paged_window_attention(q, kp, vp, table, n, window=win, sinks=sinks)
    _check(got, q, k, v, lens, window=win, sinks=sinks)
    assert torch.equal(got, window.paged_window_attention(q, kp, vp, table, n, window=win, sinks=sinks))
    # pages that left the window are not looked up
    if win is not None:
        gone = table.clone()
        for bb, m in enumerate(lens):
            first = max(0, m - lq - win + 1)
            for pg in range(table.shape[1]):
                if pg * page >= sinks and (pg + 1) * page <= first:
                    gone[bb, pg] = -1
        assert torch.equal(got, window.paged_window_attention(q, kp, vp, gone, n, window=win, sinks=sinks))
    _quiet()


def test_frames_in_pages_and_one_tensor_for_keys_and_values(cuda):
    q, k, v = _data(2, 4, 2, 64, 6, 300, BF16, seed=9)
    kp, vp, table = _pages(k, v, 32)
    both = torch.stack([kp, vp], 1)  # [pages, 2, Hk, page, D]
    n = torch.tensor([300, 250], dtype=torch.int32, device="cuda")
    got = window.paged_window_attention(q, both[:, 0], both[:, 1], table, n, window=3, sinks=1, frame_tokens=25)
    _check(got, q, k, v, [300, 250], window=3, sinks=1, frame=25)


def test_bad_pages_and_lengths_are_reported(cuda):
    q, k, v = _data(1, 2, 1, 64, 1, 96, BF16, seed=2)
    kp, vp, table = _pages(k, v, 32)
    n = torch.tensor([96], dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[0, 1] = kp.shape[0]
    got = window.paged_window_attention(q, kp, vp, bad, n, window=None)
    with pytest.raises(CastError):
        _quiet()
    keep = torch.cat([torch.arange(32), torch.arange(64, 96)]).cuda()  # the keys that are left
    want = window.window_attention(q, k[:, :, keep], v[:, :, keep], window=None)
    assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -6, atol=1e-3)
    for lens, clipped in ((97, 96), (-5, 0)):
        n.fill_(lens)
        got = window.window_attention(q, k, v, window=None, kv_lens=n)
        with pytest.raises(CastError):
            _quiet()
        n.fill_(clipped)
        assert torch.equal(got, window.window_attention(q, k, v, window=None, kv_lens=n))
        _quiet()


def test_window_refusals(cuda):
    q, k, v = _data(1, 4, 2, 64, 3, 20, BF16)
    n = torch.tensor([20], dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(v=v[:, :, :9]), dict(k=k[:, :1], v=v), dict(q=q[:, :3]),
                dict(q=q[..., :32], k=k[..., :32], v=v[..., :32]), dict(k=k.transpose(2, 3)), dict(kv_lens=n.long()),
                dict(kv_lens=n.expand(2)), dict(kv_lens=n.cpu()), dict(window=0), dict(sinks=-1), dict(frame_tokens=0),
                dict(out=q[:, :2]), dict(out=q[:, :1].expand_as(q)), dict(q=q.clone().requires_grad_())):
        args = dict(q=q, k=k, v=v, window=8)
        args.update(bad)
        with pytest.raises(ValueError):
            window.window_attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)
    with pytest.raises(CastError, match="16-byte"):
        window.window_attention(q, k[:, :, :, 0:].as_strided(k.shape, (k.stride(0), k.stride(1), 60, 1)), v, window=8)
    with pytest.raises(CastError, match="sm_scale"):
        window.window_attention(q, k, v, window=8, sm_scale=-1.0)
    kp, vp, table = _pages(k, v, 16)
    for bad in (dict(table=table.long()), dict(table=table[:0]), dict(vp=vp[:1]), dict(n=n.long()), dict(kp=kp.half())):
        args = dict(kp=kp, vp=vp, table=table, n=n)
        args.update(bad)
        with pytest.raises(ValueError):
            window.paged_window_attention(q, args["kp"], args["vp"], args["table"], args["n"], window=8)
    assert window.window_attention(q[:, :, :0], k, v, window=8).shape == (1, 4, 0, 64)
    assert (window.window_attention(q, k[:, :, :0], v[:, :, :0], window=8) == 0).all()
    assert (window.paged_window_attention(q, kp, vp, table[:, :0], n, window=8) == 0).all()


@pytest.mark.parametrize("lq,lk", [(1, 20000), (64, 3000), (88, 20000)])
def test_two_graphs_and_an_eager_call_at_once(cuda, lq, lk):
    """No call shares scratch memory with another that may run beside it."""
    data = [_data(1, 2, 1, 128, lq, lk, BF16, seed=s) for s in range(3)]
    want = [window.window_attention(*d, window=None) for d in data]
    graphs, outs = [], []
    for d in data[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(window.window_attention(*d, window=None))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = window.window_attention(*data[2], window=None)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


def test_a_session_token_by_token(cuda):
    """The operators together, as a rollout uses them: a prompt through the
    norm, the rotation and the chunk's attention into the cache, then single
    tokens over the pages, every output against the formulas over the whole
    session."""
    hq, hk, d, page, win, sinks, prompt, steps = 8, 2, 64, 16, 50, 4, 70, 6
    total = prompt + steps
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(1, total, hq + 2 * hk, d, generator=g, device="cuda").to(BF16)
    w = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(BF16)
    f = rotary.rope_frequencies(d)
    table = rotary.rope_table(f, 128)
    kp = torch.zeros(8, hk, page, d, dtype=BF16, device="cuda")
    vp = torch.zeros_like(kp)
    blocks = torch.randperm(8, device="cuda")[None, :-(-total // page)].to(torch.int32)
    place = torch.arange(total, device="cuda")
    slots = (blocks[0, place // page].long() * page + place % page)[None]

    def step(a, b):
        part = qkv[:, a:b]
        pos = torch.arange(a, b, device="cuda")
        q, _ = rotary.qk_norm_rope(part[:, :, :hq], part[:, :, hq:hq + hk], w, w, table, pos, v=part[:, :, hq + hk:],
                                   cache=(kp, vp), slots=slots[:, a:b].contiguous())
        n = torch.tensor([b], dtype=torch.int32, device="cuda")
        return q, window.paged_window_attention(q, kp, vp, blocks, n, window=win, sinks=sinks)

    done = [step(0, prompt)] + [step(t, t + 1) for t in range(prompt, total)]
    _quiet()
    q, got = (torch.cat([x[i] for x in done], 2) for i in range(2))
    k = kp[blocks[0].long()].transpose(1, 2).flatten(0, 1)[:total].transpose(0, 1)[None]
    v = vp[blocks[0].long()].transpose(1, 2).flatten(0, 1)[:total].transpose(0, 1)[None]
    assert torch.equal(v, qkv[:, :, hq + hk:].transpose(1, 2))
    theta = ora_rotary.angles(place[None], f)
    for x, y in ((qkv[:, :, :hq], q), (qkv[:, :, hq:hq + hk], k)):
        z = ora_rotary.norm(x, w, 1e-6)
        want = ora_rotary.turn(z, theta, True).transpose(1, 2)
        size = ora_rotary.pair_size(z, d, True).transpose(1, 2)
        assert ((y.double() - want).abs() <= (2.0 ** -8 * want.abs() + 20 * 2.0 ** -24 * size) * 1.01).all()
    _check(got, q, k, v, None, window=win, sinks=sinks)
    # the chunk's attention over dense keys gives what the pages gave
    dense = window.window_attention(q, k, v, window=win, sinks=sinks)
    _check(dense, q, k, v, None, window=win, sinks=sinks)


@pytest.mark.parametrize("d,dtype,lq,hq,hk", [(64, FP16, 1, 2, 1), (64, BF16, 3, 4, 1), (64, BF16, 5, 6, 1),
                                              (128, FP16, 16, 2, 1)])
def test_many_parts_of_few_rows(cuda, d, dtype, lq, hq, hk):
    """More parts than a cluster has, joined by a second launch; 8, 16 and 32 rows a tile."""
    q, k, v = _data(1, hq, hk, d, lq, 30011, dtype, seed=d + lq)
    v[0, 0, 30010, 3] = float("inf")  # seen by the last query alone
    v[0, 0, 5, 2] = float("nan")      # seen by none: behind the window
    got = window.window_attention(q, k, v, window=30000, sinks=2)
    _check(got, q, k, v, None, window=30000, sinks=2)
    kp, vp, table = _pages(k, v, 64)
    n = torch.tensor([30011], dtype=torch.int32, device="cuda")
    _check(window.paged_window_attention(q, kp, vp, table, n, window=30000, sinks=2), q, k, v, None, window=30000, sinks=2)
    _quiet()


@pytest.mark.parametrize("d,dtype,hq,hk,lq,lk,lens", [
    (64, BF16, 4, 2, 90, 9000, None),          # few items: many parts
    (128, FP16, 2, 1, 100, 9000, [9000, 40]),  # a session with fewer tiles than parts
    (128, BF16, 24, 24, 1700, 2600, None),     # a last wave in few parts
    (64, FP16, 24, 24, 3300, 3300, None)])
def test_parts_of_tiles(cuda, d, dtype, hq, hk, lq, lk, lens):
    b = 1 if lens is None else len(lens)
    q, k, v = _data(b, hq, hk, d, lq, lk, dtype, seed=lk)
    last = lk if lens is None else lens[0]
    v[0, 0, last - 1, 3] = float("inf")     # seen by the last query alone
    v[0, 0, last - lq + 1, 5] = float("nan")  # not by the first one
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = window.window_attention(q, k, v, window=None, kv_lens=n)
    _check(got, q, k, v, lens, window=None, heads=sorted({0, hq // hk - 1, hq - 1}))
    _quiet()


def test_a_maximum_that_rises_all_the_way(cuda):
    """Every step's scores are far above the last one's: sums, O and weights
    already stored are scaled again and again."""
    for dtype in (BF16, FP16):
        for d in (64, 128):
            q, k, v = _data(1, 2, 1, d, 130, 700, dtype, seed=d)
            q.fill_(1.0)
            ramp = torch.arange(700, device="cuda").float()[:, None] * (200.0 / 700 / d ** 0.5)
            k[0, 0] = ramp.to(dtype).expand(700, d)
            for lq in (1, 20, 130):
                got = window.window_attention(q[:, :, :lq], k, v, window=650, sinks=3)
                _check(got, q[:, :, :lq], k, v, None, window=650, sinks=3)


@pytest.mark.parametrize("lq", [1, 4, 96])
def test_offsets_past_32_bits(cuda, lq):
    """Keys of the last head lie more than 2^31 elements (4 GB) in."""
    hk, lk, d, win = 3, 6 << 20, 128, 300
    k = torch.empty(1, hk, lk, d, dtype=BF16, device="cuda")
    v = torch.empty(1, hk, lk, d, dtype=BF16, device="cuda")
    assert k.numel() > 1 << 31
    q, kt, vt = _data(1, hk, hk, d, lq, win + lq, BF16, seed=lq)
    k[:, :, -(win + lq):], v[:, :, -(win + lq):] = kt, vt
    got = window.window_attention(q, k, v, window=win)
    _check(got, q, kt, vt, None, window=win)
    if lq < 96:  # the same memory as a paged cache
        kp, vp = k.view(-1, hk, 64, d), v.view(-1, hk, 64, d)
        pages = -(-(win + lq) // 64)
        for j in range(pages):
            kp[-1 - j, :, :min(64, win + lq - 64 * j)] = kt[0, :, 64 * j:64 * j + 64]
            vp[-1 - j, :, :min(64, win + lq - 64 * j)] = vt[0, :, 64 * j:64 * j + 64]
        table = (kp.shape[0] - 1 - torch.arange(pages, device="cuda")).to(torch.int32)[None]
        n = torch.tensor([win + lq], dtype=torch.int32, device="cuda")
        _check(window.paged_window_attention(q, kp, vp, table, n, window=win), q, kt, vt, None, window=win)
    _quiet()


def test_strides_that_tensor_maps_cannot_hold(cuda):
    """One key for all positions (a stride of 0 along the tokens)."""
    q, k, v = _data(1, 2, 1, 64, 70, 1, BF16)
    got = window.window_attention(q, k.expand(1, 1, 200, 64), v.expand(1, 1, 200, 64), window=50)
    _check(got, q, k.expand(1, 1, 200, 64), v.expand(1, 1, 200, 64), None, window=50)
    # and of 0 along batch and heads of q: queries that all heads share
    one = q[:, :1].expand(1, 4, 70, 64)
    k, v = (t.contiguous() for t in _data(1, 4, 4, 64, 70, 200, BF16)[1:])
    _check(window.window_attention(one, k, v, window=50), one, k, v, None, window=50)


@pytest.mark.parametrize("lq", [8, 30, 140, 300])
@pytest.mark.parametrize("d", [64, 128])
def test_a_first_token_that_the_first_queries_do_not_see(cuda, lq, d):
    """Sinks ahead of the first queries of a prompt: hidden from these alone."""
    q, k, v = _data(1, 2, 1, d, lq, lq, BF16, seed=lq)
    v[0, 0, 5, 1], v[0, 0, 6, 2] = float("inf"), float("nan")
    for win in (2, 4, None):
        got = window.window_attention(q, k, v, window=win, sinks=20)
        _check(got, q, k, v, None, window=win, sinks=20)
        kp, vp, table = _pages(k, v, 16)
        n = torch.tensor([lq], dtype=torch.int32, device="cuda")
        _check(window.paged_window_attention(q, kp, vp, table, n, window=win, sinks=20), q, k, v, None, window=win, sinks=20)
    _quiet()


@pytest.mark.parametrize("lq", [1, 50])
def test_sizes_that_mean_everything(cuda, lq):
    q, k, v = _data(1, 2, 1, 64, lq, 90, BF16)
    seen = window.window_attention(q, k, v, window=1, frame_tokens=1 << 45)  # one frame: all see all
    assert torch.equal(seen, window.window_attention(q, k, v, window=1, frame_tokens=90))
    _check(seen, q, k, v, None, window=1, frame=90)
    assert torch.equal(window.window_attention(q, k, v, window=1 << 60, sinks=1 << 60),
                       window.window_attention(q, k, v, window=None))


@pytest.mark.parametrize("dtype,rise,fall", [(BF16, 18, 10), (FP16, 10, 3)])
@pytest.mark.parametrize("lq", [40, 128, 200])
def test_a_maximum_that_rises_twice_within_a_step(cuda, dtype, rise, fall, lq):
    """Scores `rise` powers of two above the last ones every 32 keys: a step of
    64 keys scales O in both its halves.  Values fall by `fall` powers of two at
    the same places: an O that missed one of the two scales in the last step
    holds 2^(2 fall - rise) of the result too much, 2^2 and 2^-4 of it, where
    the type's rounding is 2^-8 and 2^-11."""
    d, lk = 64, 256
    q, k, v = _data(1, 2, 1, d, lq, lk, dtype, seed=rise + lq)
    chunk = torch.arange(lk, device="cuda") // 32
    q.fill_(1.0)
    k.copy_(chunk.to(dtype)[:, None].expand(lk, d))
    v.mul_((2.0 ** (fall * (3.0 - chunk))).to(dtype)[:, None])
    scale = rise * 0.6931471805599453 / d  # q.k scale: rise ln 2 a chunk
    for win, sinks in ((None, 0), (150, 40)):
        got = window.window_attention(q, k, v, window=win, sinks=sinks, sm_scale=scale)
        _check(got, q, k, v, None, window=win, sinks=sinks, scale=scale)
    _quiet()


@pytest.mark.parametrize("d,dtype,hq,hk,lq,lk,lens", [
    (64, BF16, 4, 2, 90, 9000, None), (64, FP16, 3, 1, 150, 6000, [6000, 900]),
    (128, BF16, 2, 1, 100, 9000, [9000, 40]), (128, BF16, 24, 24, 1700, 2600, None)])
def test_scores_that_are_nan_in_items_cut_into_parts(cuda, d, dtype, hq, hk, lq, lk, lens):
    """A NaN in a query, and keys that make all scores of a part NaN, reach every
    row that sees them and no other, however its keys are cut."""
    b = 1 if lens is None else len(lens)
    q, k, v = _data(b, hq, hk, d, lq, lk, dtype, seed=lk + d)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    some = sorted({0, hq // hk - 1, hq - 1})
    with torch.cuda.device(q.device):
        assert _lib.load().cast_window_attention_workspace_bytes(b, hq, hk, lq, lk, d, lk, 0, 1) > 0  # (cut)
    q[0, :, 3, 5], q[0, hq - 1, lq - 1] = float("nan"), float("nan")
    for win in (None, lk - lq // 2):
        got = window.window_attention(q, k, v, window=win, kv_lens=n)
        assert torch.isnan(got[0, :, 3]).all() and torch.isfinite(got[0, 0, 4:10]).all()
        _check(got, q, k, v, lens, window=win, heads=some)
    # the last keys: seen by the last rows alone; and with a window, a long run that the last rows do not see
    q = _data(b, hq, hk, d, lq, lk, dtype, seed=lk + d)[0]
    end = lk if lens is None else lens[0]
    k[0, :, end - 7:end] = float("nan")
    k[0, 0, 2:end - lq // 2 - 100] = float("nan")
    for win in (None, 100 + lq // 4):
        got = window.window_attention(q, k, v, window=win, kv_lens=n, sinks=1)
        _check(got, q, k, v, lens, window=win, sinks=1, heads=some)
    _quiet()


@pytest.mark.parametrize("lq", [2, 88])
def test_plans_of_windows_of_any_size(cuda, lq):
    """From C, window and sinks may be the largest numbers there are (their sum is not one)."""
    lib, most = _lib.load(), (1 << 63) - 1

    def need(win, sinks):
        return lib.cast_window_attention_workspace_bytes(1, 2, 1, lq, 20000, 128, win, sinks, 1)

    assert need(20000, 0) > 0
    for win, sinks in ((most, most), (most, 1), (1, most), (most, 0)):
        assert need(win, sinks) == need(20000, 0), (win, sinks)


FORMS = [(1, 8, 2, 128, 1, 200), (1, 2, 1, 64, 3, 3000), (1, 2, 1, 128, 4, 30000), (1, 4, 1, 64, 7, 4000),
         (2, 4, 2, 128, 150, 700), (1, 2, 1, 64, 90, 20000), (1, 4, 2, 128, 600, 600)]


@pytest.mark.parametrize("b,hq,hk,d,lq,lk", FORMS)
def test_scores_that_are_not_finite(cuda, b, hq, hk, d, lq, lk):
    """NaN and +infinity in queries and keys make the rows that see them NaN, in
    every way a call is cut; -infinity hides a key."""
    q, k, v = _data(b, hq, hk, d, lq, lk, BF16, seed=lk)
    q[0, 0, 0, 1] = float("nan")
    k[0, 0, lk - 1] = float("nan")                       # the last row's
    k[b - 1, hk - 1, lk // 2] = float("-inf")
    q[b - 1, hq - 1, lq - 1].abs_()                      # q.k = -infinity
    for win in (None, lk // 3 + lq):
        got = window.window_attention(q, k, v, window=win)
        _check(got, q, k, v, None, window=win)
    q[0, 0, 0, 1] = float("inf")
    k[0, 0, lk - 1] = 1.0
    k[b - 1, hk - 1, lk // 2] = 1.0
    got = window.window_attention(q, k, v, window=None)
    _check(got, q, k, v, None, window=None)
    kp, vp, table = _pages(k, v, 64)
    n = torch.full((b,), lk, dtype=torch.int32, device="cuda")
    _check(window.paged_window_attention(q, kp, vp, table, n, window=None), q, k, v, None, window=None)
    _quiet()


@pytest.mark.parametrize("b,hq,hk,d,lq,lk", FORMS)
def test_out_may_be_q(cuda, b, hq, hk, d, lq, lk):
    q, k, v = _data(b, hq, hk, d, lq, lk, BF16, seed=lk)
    want = window.window_attention(q, k, v, window=None)
    kp, vp, table = _pages(k, v, 64)
    n = torch.full((b,), lk, dtype=torch.int32, device="cuda")
    paged = window.paged_window_attention(q, kp, vp, table, n, window=None)
    for _ in range(3):
        x, y = q.clone(), q.transpose(1, 2).clone().transpose(1, 2)
        assert torch.equal(window.window_attention(x, k, v, window=None, out=x), want)
        assert torch.equal(window.window_attention(y, k, v, window=None, out=y), want)
        y.copy_(q)
        assert torch.equal(window.paged_window_attention(y, kp, vp, table, n, window=None, out=y), paged)


def test_an_option_that_changes_in_place(cuda):
    q, k, v = _data(1, 2, 1, 64, 5, 90, BF16)
    win, sinks = torch.tensor(9), torch.tensor(0)
    for w, s in ((9, 0), (30, 0), (30, 4)):
        win.fill_(w), sinks.fill_(s)
        _check(window.window_attention(q, k, v, window=win, sinks=sinks), q, k, v, None, window=w, sinks=s)
