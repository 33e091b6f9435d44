"""The measured cases of the rotary, norm and sliding-window attention operators.

Four operators that a streaming rollout runs around its sparse layers:

* ``rope``: rotary positions, interleaved or half layout, a part of the head or all of it, one
  position a token or three (frame, row, column), frequencies scaled for long contexts.
* ``norm``: RMS norm of queries and keys for each head with the rotation in the same pass; with a
  paged cache, keys and values go straight to their slots.
* ``window``: attention of a chunk of queries over its last frames (or tokens) and the first ones.
* ``paged``: the same for a few new tokens of many sessions over a paged key-value cache.

``run`` computes them in elementary torch operations, or calls the framework's where ``own`` is
true; ``exact`` computes them in 64 bits.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6
_AXES = (22, 21, 21)  # pairs of a 128-wide head that turn with the frame, the row and the column
_GRID = (22, 40)      # rows and columns of one latent frame


def _rope(name, dtype, B, L, H, D, R, half, axes=False, far=0, scale=1.0):
    return {"name": name, "op": "rope", "dtype": dtype, "B": B, "L": L, "H": H, "D": D, "R": R, "half": half,
            "axes": axes, "far": far, "scale": scale}


def _norm(name, dtype, B, L, Hq, Hk, D, R, half, axes=False, far=0, scale=1.0, page=0):
    return {"name": name, "op": "norm", "dtype": dtype, "B": B, "L": L, "Hq": Hq, "Hk": Hk, "D": D, "R": R,
            "half": half, "axes": axes, "far": far, "scale": scale, "page": page}


def _window(name, dtype, B, Hq, Hk, D, Lq, Lk, window, sinks, frame=1, short=0):
    return {"name": name, "op": "window", "dtype": dtype, "B": B, "Hq": Hq, "Hk": Hk, "D": D, "Lq": Lq, "Lk": Lk,
            "window": window, "sinks": sinks, "frame": frame, "short": short}


def _paged(name, dtype, B, Hq, Hk, D, Lq, Lk, window, sinks, page, short=0):
    return {"name": name, "op": "paged", "dtype": dtype, "B": B, "Hq": Hq, "Hk": Hk, "D": D, "Lq": Lq, "Lk": Lk,
            "window": window, "sinks": sinks, "frame": 1, "page": page, "short": short}


def listed():
    return [
        # the heads of one new token: nothing but latency
        _rope("rope one token", "fp32", 1, 1, 24, 128, 128, False),
        # two odd-length prompts far into a context stretched four times, half layout on half of the head
        _rope("rope long partial half", "fp16", 2, 4093, 16, 128, 64, True, far=100000, scale=4.0),
        # the whole 36-frame history of a layer turned in (frame, row, column)
        _rope("rope history axes", "bf16", 1, 31680, 24, 128, 128, False, axes=True),
        # one new token of eight sessions, keys and values into the paged cache
        _norm("norm tokens to pages", "bf16", 8, 1, 32, 8, 128, 128, True, far=30000, page=64),
        # the 4-frame chunk of a layer call
        _norm("norm chunk axes", "bf16", 1, 3520, 24, 24, 128, 128, False, axes=True),
        # one query over the newest thousand keys and the first ones
        _window("window one query", "bf16", 1, 24, 24, 128, 1, 1760, 1024, 64),
        # the layer call: 4 current frames over the last 8 frames and the first one
        _window("window chunk of frames", "bf16", 1, 24, 24, 128, 3520, 31680, 8, 1, frame=880),
        # a prompt with grouped heads, a window of tokens and a few sinks
        _window("window prompt grouped", "bf16", 1, 32, 8, 128, 8192, 8192, 1024, 4),
        # a padded batch of odd lengths, small heads, half precision
        _window("window padded batch", "fp16", 3, 16, 4, 64, 1001, 4099, 777, 13, short=611),
        # a few rows over the whole long history: work has to come from the keys
        _window("window few rows long", "bf16", 1, 4, 2, 128, 88, 112640, 112640, 0),
        # one new token of sixteen sessions with long, ragged histories
        _paged("paged tokens", "bf16", 16, 32, 8, 128, 1, 32768, 8192, 16, 64, short=1777),
        # three drafted tokens of two sessions, small pages
        _paged("paged drafted tokens", "fp16", 2, 8, 8, 64, 3, 1531, 600, 5, 16, short=93),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    g = rng.choice([1, 1, 2, 3, 4, 8])
    hk = rng.choice([1, 2, 3, 4, 6, 8, 16, 24])
    return (g * hk, hk) if g * hk <= most else (hk, hk)


def _cost(c):
    w = work(c)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["rope", "norm", "window", "window", "paged"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"] if op in ("rope", "norm") else ["bf16", "bf16", "fp16"])
        if op in ("rope", "norm"):
            half = rng.random() < 0.5
            D = rng.choice([64, 80, 96, 128, 256])
            R = D if rng.random() < 0.5 else 16 * rng.randint(1, D // 16)
            axes = D == 128 and R == 128 and rng.random() < 0.5
            L = 1 if rng.random() < 0.2 else _log(rng, 2, 40000)
            B = 1 if L > 8000 else rng.randint(1, 8)
            far = 0 if axes else rng.choice([0, 0, _log(rng, 1000, 500000)])
            scale = rng.choice([1.0, 1.0, 2.0, 4.0, 8.0])
            Hq, Hk = _heads(rng, 32)
            if op == "rope":
                c = _rope("", dtype, B, L, Hq, D, R, half, axes, far, scale)
            else:
                page = rng.choice([16, 64, 128]) if L < 4000 and rng.random() < 0.4 else 0
                c = _norm("", dtype, B, L, Hq, Hk, D, R, half, axes, far, scale, page)
        elif op == "window":
            D = rng.choice([64, 128, 128])
            Hq, Hk = _heads(rng, 32)
            frame = rng.choice([1, 1, 1, 64, 110, 880])
            Lq = rng.choice([1, rng.randint(2, 40), _log(rng, 32, 8192)])
            Lk = Lq + _log(rng, 1, 32000)
            window = _log(rng, 1, max(2, Lk // frame))
            sinks = rng.choice([0, 1, 4, _log(rng, 4, 600)]) if frame == 1 else rng.choice([0, 1])
            B = rng.randint(1, 4)
            short = rng.randint(1, max(1, Lk // 5)) if B > 1 and rng.random() < 0.5 else 0
            c = _window("", dtype, B, Hq, Hk, D, Lq, Lk, window, sinks, frame, short)
            if B * Hq * Lq * Lk > 2.6e9:
                continue
        else:
            D = rng.choice([64, 128, 128])
            Hq, Hk = _heads(rng, 32)
            Lq = rng.choice([1, 1, 1, rng.randint(2, 9)])
            Lk = Lq + _log(rng, 1, 40000)
            window = _log(rng, 1, Lk)
            B = rng.randint(1, 16)
            short = rng.randint(0, max(1, Lk // B))
            c = _paged("", dtype, B, Hq, Hk, D, Lq, Lk, window, rng.choice([0, 4, 16, 130]), rng.choice([16, 32, 64, 256]),
                       short)
            if B * Lk * Hk * D > 6e8:
                continue
        if _cost(c) <= most:
            del c["name"]
            return c


def _lens(case):
    """Keys of each session of the batch: each `short` fewer than the one before, one at least."""
    return [max(1, case["Lk"] - b * case["short"]) for b in range(case["B"])]


def _frequencies(R, axes, scale):
    """Angle of one position step for each pair, in 64 bits; a stretched context divides the steps."""
    if axes:
        parts = [10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in _AXES]
        return torch.cat(parts) / scale
    return 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R) / scale


def _positions(case, gen):
    """int32 positions of the tokens: [B, L], or [B, L, 3] of frame, row and column; and their bound."""
    B, L = case["B"], case["L"]
    if case["axes"]:
        h, w = _GRID
        t = torch.arange(L, device="cuda")
        p = torch.stack([t // (h * w), t // w % h, t % w], -1).expand(B, L, 3)
        first = torch.randint(0, 8, (B, 1, 1), generator=gen, device="cuda")
        p = p + first * torch.tensor([1, 0, 0], device="cuda")
        return p.to(torch.int32).contiguous(), max(L // (h * w) + 9, w)
    first = torch.randint(0, case["far"] + 1, (B, 1), generator=gen, device="cuda")
    return (first + torch.arange(L, device="cuda")).to(torch.int32), case["far"] + L


def _table(freq, count):
    """float32 (cos, sin) of every position and pair, from angles in 64 bits."""
    a = torch.arange(count, dtype=torch.float64, device="cuda")[:, None] * freq.to("cuda")
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 7919 + 17)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    def heads(n):  # the spread that heads of one layer have
        return 0.5 + 1.5 * torch.rand(n, generator=gen, device="cuda")

    B, D = case["B"], case["D"]
    s = {"case": dict(case)}
    if case["op"] in ("rope", "norm"):
        L = case["L"]
        s["freq"] = _frequencies(case["R"], case["axes"], case["scale"])
        s["positions"], count = _positions(case, gen)
        s["table"] = _table(s["freq"], count)
    if case["op"] == "rope":
        s["x"] = (normal(B, L, case["H"], D) * heads(case["H"])[:, None]).to(dtype)
    elif case["op"] == "norm":
        Hq, Hk, page = case["Hq"], case["Hk"], case["page"]
        # the projection of a layer leaves q, k and v beside one another in one tensor
        qkv = normal(B, L, Hq + 2 * Hk, D) * heads(Hq + 2 * Hk)[:, None]
        qkv = qkv.to(dtype)
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
        s["q_weight"] = (1.0 + 0.2 * normal(D)).to(dtype)
        s["k_weight"] = (1.0 + 0.2 * normal(D)).to(dtype)
        if page:
            pages = -(-L // page) * B + 5
            s["k_pages"] = normal(pages, Hk, page, D).to(dtype)
            s["v_pages"] = normal(pages, Hk, page, D).to(dtype)
            each = -(-L // page)
            order = torch.randperm(pages, generator=gen, device="cuda")[:each * B].view(B, each)
            t = torch.arange(L, device="cuda")
            s["slots"] = (order[:, t // page] * page + t % page).to(torch.int32)
    else:
        Hq, Hk, Lq, Lk = case["Hq"], case["Hk"], case["Lq"], case["Lk"]
        s["q"] = (normal(B, Hq, Lq, D) * heads(Hq)[:, None, None]).to(dtype)
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        if case["op"] == "window":
            s["k"] = normal(B, Hk, Lk, D).to(dtype)
            s["v"] = (0.8 * normal(B, Hk, Lk, D) + 0.6 * normal(Hk, 1, D)).to(dtype)
        else:
            page = case["page"]
            each = -(-Lk // page)
            s["k_pages"] = normal(B * each + 3, Hk, page, D).to(dtype)
            s["v_pages"] = (0.8 * normal(B * each + 3, Hk, page, D) + 0.6 * normal(Hk, 1, D)).to(dtype)
            order = torch.randperm(B * each + 3, generator=gen, device="cuda")[:B * each]
            s["block_table"] = order.view(B, each).to(torch.int32)
    return s


def _angles(s):
    """Angles [B, L, pairs] in 64 bits: far positions turn through many circles."""
    p, f = s["positions"].double(), s["freq"].to("cuda")
    if s["case"]["axes"]:
        axis = torch.tensor([a for a, n in enumerate(_AXES) for _ in range(n)], device="cuda")
        return p[..., axis] * f
    return p[..., None] * f


def _turn(x, cos, sin, R, half):
    """x float32 [B, L, H, D] with the pairs of its first R values turned."""
    if half:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., R:]], -1)
    a, b = x[..., 0:R:2], x[..., 1:R:2]
    y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([y, x[..., R:]], -1)


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * w


def _visible(case, lens, Lk):
    """Which of the keys 0..Lk-1 each query sees: [B, Lq, Lk]."""
    F = case["frame"]
    p = lens[:, None].long() - case["Lq"] + torch.arange(case["Lq"], device="cuda")
    j = torch.arange(Lk, device="cuda")
    fp, fj = torch.div(p, F, rounding_mode="floor")[..., None], j // F
    return (j < lens[:, None, None]) & (fj <= fp) & ((fj > fp - case["window"]) | (fj < case["sinks"])) & (p >= 0)[..., None]


def _attend(q, k, v, seen):
    """Softmax attention in float32; a query that sees nothing gives zeros."""
    B, Hq, Lq, D = q.shape
    Hk = k.shape[1]
    s = q.float().reshape(B, Hk, Hq // Hk * Lq, D) @ k.float().mT * D ** -0.5
    s = s.view(B, Hk, Hq // Hk, Lq, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-1e30)
    s = s.sub_(m).exp_()
    total = s.sum(-1, keepdim=True)
    o = s.view(B, Hk, Hq // Hk * Lq, -1) @ v.float()
    return (o.view(B, Hq, Lq, D) / total.view(B, Hq, Lq, 1).clamp_min(1e-30)).to(q.dtype)


def _plain(s):
    c = s["case"]
    if c["op"] in ("rope", "norm"):
        a = _angles(s)
        cos, sin = a.cos().float()[:, :, None], a.sin().float()[:, :, None]
    if c["op"] == "rope":
        return _turn(s["x"].float(), cos, sin, c["R"], c["half"]).to(s["x"].dtype)
    if c["op"] == "norm":
        q = _turn(_rms(s["q"].float(), s["q_weight"].float()), cos, sin, c["R"], c["half"]).to(s["q"].dtype)
        k = _turn(_rms(s["k"].float(), s["k_weight"].float()), cos, sin, c["R"], c["half"]).to(s["k"].dtype)
        q = q.transpose(1, 2).contiguous()
        if not c["page"]:
            return q, k.transpose(1, 2).contiguous()
        at = s["slots"].long()
        s["k_pages"][at // c["page"], :, at % c["page"]] = k
        s["v_pages"][at // c["page"], :, at % c["page"]] = s["v"]
        return q, s["k_pages"], s["v_pages"]
    if c["op"] == "window":
        return _attend(s["q"], s["k"], s["v"], _visible(c, s["lens"], c["Lk"]))
    table = s["block_table"].long()
    k, v = (s[n][table].transpose(2, 3).flatten(1, 2).transpose(1, 2) for n in ("k_pages", "v_pages"))
    return _attend(s["q"], k, v, _visible(c, s["lens"], k.shape[2]))


def run(s):
    if not own:
        return _plain(s)
    from cast_b200 import rotary, window

    c = s["case"]
    axes = _AXES if c.get("axes") else None
    if c["op"] == "rope":
        return rotary.rope(s["x"], s["table"], s["positions"], interleaved=not c["half"], axes=axes)
    if c["op"] == "norm":
        cache = (s["k_pages"], s["v_pages"]) if c["page"] else None
        q, k = rotary.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], s["positions"], eps=_EPS,
                                   interleaved=not c["half"], axes=axes, v=s["v"] if cache else None, cache=cache,
                                   slots=s["slots"] if cache else None)
        return (q, *cache) if cache else (q, k)
    if c["op"] == "window":
        return window.window_attention(s["q"], s["k"], s["v"], window=c["window"], sinks=c["sinks"],
                                       frame_tokens=c["frame"], kv_lens=s["lens"])
    return window.paged_window_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lens"],
                                         window=c["window"], sinks=c["sinks"], frame_tokens=c["frame"])


def _spans(case, n):
    """(first, end) of the window and of the sinks for each query of a session of n keys."""
    F, got = case["frame"], []
    for i in range(case["Lq"]):
        p = n - case["Lq"] + i
        if p >= 0:
            end = min(n, (p // F + 1) * F)
            first = max(0, (p // F - case["window"] + 1) * F)
            got.append((first, end, min(case["sinks"] * F, first)))
    return got


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] in ("rope", "norm"):
        tokens, R, D = case["B"] * case["L"], case["R"], case["D"]
        rows = tokens if not case["axes"] else min(tokens, 64)
        plan = rows * R * 4 + tokens * (12 if case["axes"] else 4)
        if case["op"] == "rope":
            return {"bytes": 2 * tokens * case["H"] * D * e + plan, "flops": 3 * R * tokens * case["H"]}
        h = case["Hq"] + case["Hk"]
        copied = 2 * case["Hk"] * D * e * tokens + 4 * tokens if case["page"] else 0
        return {"bytes": 2 * tokens * h * D * e + plan + copied, "flops": (4 * D + 3 * R) * tokens * h}
    pairs = keys = 0
    for n in _lens(case):
        spans = _spans(case, n)
        pairs += sum(end - first + sinks for first, end, sinks in spans)
        if spans:
            first, end = spans[0][0], spans[-1][1]
            keys += end - first + min(case["sinks"] * case["frame"], first)
    B, D = case["B"], case["D"]
    return {"bytes": 2 * B * case["Hq"] * case["Lq"] * D * e + 2 * keys * case["Hk"] * D * e + 4 * B,
            "flops": 4 * D * pairs * case["Hq"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rope", "norm"):
        pos, freq = s["positions"].double(), s["freq"].to("cuda")
        if case["axes"]:
            ends = [sum(_AXES[:n + 1]) for n in range(3)]
            theta = torch.cat([pos[..., n:n + 1] * freq[e - w:e] for n, (e, w) in enumerate(zip(ends, _AXES))], -1)
        else:
            theta = pos.unsqueeze(-1) * freq
        unit = torch.polar(torch.ones_like(theta), theta).unsqueeze(2)

        def turned(x):
            R = case["R"]
            y = x.clone()
            one, two = (slice(0, R // 2), slice(R // 2, R)) if case["half"] else (slice(0, R, 2), slice(1, R, 2))
            z = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * unit
            y[..., one], y[..., two] = z.real, z.imag
            return y

        def normed(x, w):
            x = x.double()
            return x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + _EPS) * w.double()

        if case["op"] == "rope":
            return turned(s["x"].double())
        q = turned(normed(s["q"], s["q_weight"])).permute(0, 2, 1, 3).contiguous()
        k = turned(normed(s["k"], s["k_weight"]))
        if not case["page"]:
            return q, k.permute(0, 2, 1, 3).contiguous()
        pages = []
        for kept, new in ((s["k_pages"], k), (s["v_pages"], s["v"].double())):
            flat = kept.double().permute(0, 2, 1, 3).flatten(0, 1)
            flat[s["slots"].long().flatten()] = new.flatten(0, 1)
            pages.append(flat.unflatten(0, (-1, case["page"])).permute(0, 2, 1, 3).contiguous())
        return q, pages[0], pages[1]
    B, Hq, Lq, D = s["q"].shape
    out = torch.zeros(B, Hq, Lq, D, dtype=torch.float64, device="cuda")
    F, group = case["frame"], Hq // case["Hk"]
    for b, n in enumerate(_lens(case)):
        if case["op"] == "paged":
            j = torch.arange(n, device="cuda")
            page = s["block_table"][b, j // case["page"]].long()
            kb, vb = (s[m][page, :, j % case["page"]].transpose(0, 1).double() for m in ("k_pages", "v_pages"))
        else:
            kb, vb = s["k"][b, :, :n].double(), s["v"][b, :, :n].double()
        frame_of = torch.arange(n, device="cuda") // F
        skip = max(0, Lq - n)  # queries before the first key see nothing
        mine = frame_of[n - (Lq - skip):, None]
        hidden = (frame_of > mine) | ((frame_of <= mine - case["window"]) & (frame_of >= case["sinks"]))
        for h in range(Hq):
            z = s["q"][b, h, skip:].double() @ kb[h // group].mT / math.sqrt(D)
            z[hidden] = -math.inf
            out[b, h, skip:] = torch.softmax(z, -1) @ vb[h // group]
    return out
