"""The attention-block operators for long contexts, as they are measured: rotary positions, the rotary append to a K/V
cache, attention with a sliding window and sinks (forward and backward), and the same attention over a cache.

With `own` false, run() computes an operator in its plain form: elementary torch operations in fp32 (angles in fp64),
rounded once at the end.  With `own` true it makes the calls a user makes of metalllm_b200.attention.

Shapes: q [B, T, NH*D], k and v [B, T, NKV*D], caches [B, cap, NKV*D]; query head h reads K/V head h // (NH // NKV).
Query i (position start + i) sees key j when j <= start + i and (start + i - j < window or j < sinks) and i < lens.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------ cases
def listed():
    return [
        # rotary: a long document's q and k (grouped heads), half layout, positions far into a stretched context
        dict(name="rotary_long", op="rotary", B=2, T=8192, NH=32, NKV=8, D=128, rot=128, inter=False, far=1000000,
             amp=1.2079441541679836, back=False),
        # rotary backward at the smallest training shape (B=16, T=256, 6 heads of 64): fp32 dQ and bf16 dK as the attention's
        # backward gives them, interleaved layout on half of the head
        dict(name="rotary_back_small", op="rotary", B=16, T=256, NH=6, NKV=6, D=64, rot=32, inter=True, far=0, amp=1.0,
             back=True),
        # one decoding step of 64 requests: rotate q and k, store k and v; latency counts
        dict(name="append_step", op="append", B=64, M=1, NH=32, NKV=8, D=128, cap=2048, rot=128, inter=False, ragged=False),
        # prompts of odd lengths, padded to the longest, entering the cache
        dict(name="append_prompts", op="append", B=8, M=1999, NH=12, NKV=4, D=64, cap=4096, rot=64, inter=False,
             ragged=True),
        # training forward at the smallest training shape
        dict(name="forward_small", op="forward", B=16, T=256, NH=6, NKV=6, D=64, window=128, sinks=4, ragged=False),
        # a long sequence, grouped heads: the work is the window's, not the sequence's square
        dict(name="forward_long", op="forward", B=1, T=8192, NH=32, NKV=8, D=128, window=1024, sinks=16, ragged=False),
        # training backward at the smallest training shape
        dict(name="backward_small", op="backward", B=16, T=256, NH=6, NKV=6, D=64, window=128, sinks=4, ragged=False),
        # the benchmark's B=64, T=1024, 12 heads of 64, padded to the longest sequence
        dict(name="backward_padded", op="backward", B=64, T=1024, NH=12, NKV=12, D=64, window=250, sinks=4, ragged=True),
        # T=4096 with 16 heads of 128, grouped: gradients of shared heads, sinks that every query reaches
        dict(name="backward_long", op="backward", B=2, T=4096, NH=16, NKV=4, D=128, window=1000, sinks=64, ragged=False),
        # one decoding step of 64 requests of different lengths
        dict(name="cached_step", op="cached", B=64, M=1, NH=32, NKV=8, D=128, cap=8192, window=4096, sinks=4, ragged=True),
        # one request, one token, everything visible: few rows, a very long axis
        dict(name="cached_long", op="cached", B=1, M=1, NH=32, NKV=8, D=128, cap=131072, window=131072, sinks=0,
             ragged=False),
        # a piece of a prompt against what the cache holds already
        dict(name="cached_chunk", op="cached", B=2, M=500, NH=16, NKV=4, D=64, cap=8192, window=2048, sinks=4, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "forward", "backward", "cached"])
    D = rng.choice([64, 128])
    NKV = rng.choice([1, 2, 4, 6])
    NH = NKV * rng.choice([1, 2, 4])
    window, sinks = _log(rng, 1, 3000), rng.choice([0, 1, 4, 16, rng.randint(0, 300)])
    ragged = rng.random() < 0.5
    if op == "rotary":
        rot = rng.choice([D, D // 2, 2 * rng.randint(1, D // 2)])
        return dict(op=op, B=rng.randint(1, 8), T=_log(rng, 1, 4000), NH=NH, NKV=NKV, D=D, rot=rot, inter=rng.random() < 0.5,
                    far=rng.choice([0, rng.randint(0, 4000000)]), amp=rng.choice([1.0, 1.0 + rng.random()]),
                    back=rng.random() < 0.5)
    if op == "append":
        M = rng.choice([1, _log(rng, 1, 2000)])
        rot = rng.choice([D, D // 2, 2 * rng.randint(1, D // 2)])
        return dict(op=op, B=rng.randint(1, 32), M=M, NH=NH, NKV=NKV, D=D, cap=M + rng.randint(1, 2000), rot=rot,
                    inter=rng.random() < 0.5, ragged=ragged)
    if op == "cached":
        M = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 400)])
        return dict(op=op, B=rng.randint(1, 16), M=M, NH=NH, NKV=NKV, D=D, cap=M + _log(rng, 1, 16000), window=window,
                    sinks=sinks, ragged=ragged)
    # where every query sees one key, dQ and dK are 0 but for rounding: a backward starts at two keys and some rows
    low = (16, 2) if op == "backward" else (1, 1)
    c = dict(op=op, B=rng.randint(1, 4), T=_log(rng, low[0], 8000), NH=NH, NKV=NKV, D=D, window=max(low[1], window),
             sinks=sinks, ragged=ragged)
    # no dearer than the dearest listed case, and the plain form's score matrices within 16 GB each
    while work(c)["flops"] > 1.5e11 or c["B"] * NH * c["T"] ** 2 > 4e9:
        c["T"] = c["T"] * 2 // 3
    return c


# ------------------------------------------------- what the sizes give, without data
def _lens(c):
    """Valid new tokens of each sequence: all of them, or from about half up to all."""
    n = c.get("M", c.get("T"))
    return [n - (b * 37 % 64) * (n // 2) // 64 if c.get("ragged") else n for b in range(c["B"])]


def _starts(c):
    """Tokens a cache holds before the new ones: almost all it has room for, or down to about half of that."""
    room = c["cap"] - c["M"]
    return [room - (b * 41 % 64) * (room // 2) // 64 if c.get("ragged") else room for b in range(c["B"])]


def _pairs(c):
    """Visible (query, key) pairs of one head over the batch, and the distinct keys they reach."""
    pairs = keys = 0
    W, S = c["window"], c["sinks"]
    starts = _starts(c) if c["op"] == "cached" else [0] * c["B"]
    for s, n in zip(starts, _lens(c)):
        pos = s + np.arange(n, dtype=np.int64)
        low = np.maximum(pos + 1 - W, 0)
        pairs += int((pos + 1 - low + np.minimum(S, low)).sum())
        if n:
            first = max(s + 1 - W, 0)
            keys += s + n - first + min(S, first)
    return pairs, keys


def work(case):
    c = case
    n = c["B"] * c.get("M", c.get("T"))
    q, kv = n * c["NH"] * c["D"], n * c["NKV"] * c["D"]
    if c["op"] == "rotary":
        return {"bytes": 2 * ((4 if c["back"] else 2) * q + 2 * kv), "flops": 3 * (q + kv)}
    if c["op"] == "append":
        return {"bytes": 2 * 2 * (q + 2 * kv), "flops": 3 * (q + kv)}
    pairs, keys = _pairs(c)
    if c["op"] == "forward":
        return {"bytes": 2 * (2 * q + 2 * kv) + 4 * n * c["NH"], "flops": 4 * c["D"] * c["NH"] * pairs}
    if c["op"] == "backward":
        return {"bytes": 2 * (4 * q + 4 * kv) + 4 * n * c["NH"], "flops": 10 * c["D"] * c["NH"] * pairs}
    return {"bytes": 2 * (2 * q + 2 * keys * c["NKV"] * c["D"]) + 4 * n * c["NH"], "flops": 4 * c["D"] * c["NH"] * pairs}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    B, n, NH, NKV, D = c["B"], c.get("M", c.get("T")), c["NH"], c["NKV"], c["D"]
    s = {"case": c}
    whole = torch.int32
    lens = torch.tensor(_lens(c), dtype=whole, device=dev)
    if c["op"] == "rotary":
        # a backward's dQ stays in fp32, as the attention's backward accumulates it
        s["q"] = normal(B, n, NH * D, dtype=torch.float32 if c["back"] else torch.bfloat16)
        s["k"] = normal(B, n, NKV * D)
        s["positions"] = None
        if c["far"]:
            s["positions"] = (torch.arange(n, device=dev) + c["far"]).to(whole).expand(B, n).contiguous()
    elif c["op"] == "append":
        s["q"], s["k"], s["v"] = normal(B, n, NH * D), normal(B, n, NKV * D), normal(B, n, NKV * D)
        s["k_cache"], s["v_cache"] = normal(B, c["cap"], NKV * D), normal(B, c["cap"], NKV * D)
    elif c["op"] == "cached":
        s["q"] = normal(B, n, NH * D)
        s["k_cache"] = torch.empty(B, c["cap"], NKV * D, dtype=torch.bfloat16, device=dev)
        s["v_cache"] = torch.empty_like(s["k_cache"])
        s["k_cache"].normal_(generator=gen)
        s["v_cache"].normal_(generator=gen)
    else:
        s["q"], s["k"], s["v"] = normal(B, n, NH * D), normal(B, n, NKV * D), normal(B, n, NKV * D)
    if c["op"] in ("append", "cached"):
        s["start"] = torch.tensor(_starts(c), dtype=whole, device=dev)
    if c["op"] in ("rotary", "append"):
        i = torch.arange(c["rot"] // 2, dtype=torch.float64, device=dev)
        s["inv_freq"] = 10000.0 ** (-2.0 * i / c["rot"])
    s["lens"] = lens if c.get("ragged") else None
    if c["op"] == "backward":
        s["dO"] = normal(B, n, NH * D)
        s["out"], s["l"] = _plain_attention(s["q"], s["k"], s["v"], c, None, s["lens"])
    return s


# ------------------------------------------------------------- plain forms
def _visible(c, n, keys, start, lens, dev):
    """[B, n, keys] truth values (B = 1 where all sequences are alike)."""
    i = torch.arange(n, device=dev)
    pos = (start[:, None] if start is not None else 0) + i[None]
    j = torch.arange(keys, device=dev)
    see = (j <= pos[..., None]) & ((pos[..., None] - j < c["window"]) | (j < c["sinks"]))
    return see if lens is None else see & (i[None, :, None] < lens[:, None, None])


def _heads(x, heads, D):
    """[B, n, heads*D] -> fp32 [B, heads, n, D]."""
    return x.float().view(x.shape[0], x.shape[1], heads, D).transpose(1, 2)


def _rows(x):
    return x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1)


def _grouped(x, c):
    """[B, NH, n, D] -> [B, NKV, G*n, D]: the query heads of a K/V head one below the other."""
    return x.reshape(x.shape[0], c["NKV"], -1, c["D"])


def _scores(q, k, c, see):
    """Scaled scores [B, NKV, G, n, keys], -inf where a key is not visible."""
    s = _grouped(q, c) @ k.transpose(2, 3)
    s = s.view(s.shape[0], c["NKV"], c["NH"] // c["NKV"], q.shape[2], k.shape[2]).mul_(c["D"] ** -0.5)
    return s.masked_fill_(~see[:, None, None], -math.inf)


def _plain_attention(q, k, v, c, start, lens):
    n = q.shape[1]
    see = _visible(c, n, k.shape[1], start, lens, q.device)
    s = _scores(_heads(q, c["NH"], c["D"]), _heads(k, c["NKV"], c["D"]), c, see)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = e.view(e.shape[0], c["NKV"], -1, e.shape[4]) @ _heads(v, c["NKV"], c["D"])
    o = o.view(o.shape[0], c["NKV"], -1, n, c["D"]) / total
    o = torch.where(total > 0, o, torch.zeros_like(o))
    l = (top + total.log()).view(q.shape[0], c["NH"], n)
    return _rows(o.view(q.shape[0], c["NH"], n, c["D"])).to(torch.bfloat16), l.transpose(1, 2).contiguous()


def _plain_backward(st, c):
    q, k, v, d = (_heads(st[x], h, c["D"]) for x, h in (("q", c["NH"]), ("k", c["NKV"]), ("v", c["NKV"]), ("dO", c["NH"])))
    n = q.shape[2]
    see = _visible(c, n, n, None, st["lens"], q.device)
    delta = (d * _heads(st["out"], c["NH"], c["D"])).sum(-1)
    lse = st["l"].transpose(1, 2)
    lse = torch.where(lse == -math.inf, torch.zeros_like(lse), lse)
    shape = (q.shape[0], c["NKV"], c["NH"] // c["NKV"], n, 1)
    p = _scores(q, k, c, see).sub_(lse.reshape(shape)).exp_()
    flat = (q.shape[0], c["NKV"], -1, n)
    dv = p.view(flat).transpose(2, 3) @ _grouped(d, c)
    ds = (_grouped(d, c) @ v.transpose(2, 3)).view(p.shape).sub_(delta.reshape(shape)).mul_(p).mul_(c["D"] ** -0.5)
    dq = (ds.view(flat) @ k).reshape(q.shape)
    dk = ds.view(flat).transpose(2, 3) @ _grouped(q, c)
    return tuple(_rows(x).to(torch.bfloat16) for x in (dq, dk, dv))


def _plain_rotate(x, heads, c, inv_freq, pos, back):
    """x [B, n, heads*D] turned by pos [B, n] (in the backward by its negative); angles in fp64."""
    amp = c.get("amp", 1.0)
    angle = pos[..., None].double() * inv_freq
    cos, sin = ((f(angle) * amp).float()[:, :, None] for f in (torch.cos, torch.sin))
    sin = -sin if back else sin
    y = x.float().view(x.shape[0], x.shape[1], heads, c["D"])
    turned, rest = y[..., : c["rot"]], y[..., c["rot"]:]
    if c["inter"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1).view(x.shape).to(x.dtype)


def _plain_append(st, c):
    B, n = st["k"].shape[:2]
    i = torch.arange(n, device=st["k"].device)
    pos = st["start"][:, None].long() + i[None]
    q = _plain_rotate(st["q"], c["NH"], c, st["inv_freq"], pos, False)
    k = _plain_rotate(st["k"], c["NKV"], c, st["inv_freq"], pos, False)
    row = torch.arange(B, device=pos.device)[:, None].expand_as(pos)
    if st["lens"] is None:
        st["k_cache"][row, pos] = k
        st["v_cache"][row, pos] = st["v"]
    else:  # rows past a sequence's length keep what the cache holds there
        keep = (i[None] < st["lens"][:, None])[..., None]
        st["k_cache"][row, pos] = torch.where(keep, k, st["k_cache"][row, pos])
        st["v_cache"][row, pos] = torch.where(keep, st["v"], st["v_cache"][row, pos])
        q = torch.where(keep, q, torch.zeros_like(q))
    return q, st["k_cache"], st["v_cache"]


# -------------------------------------------------------------------- run
def _own_run(st, c):
    from metalllm_b200 import attention as A
    B, NKV = c["B"], c["NKV"]
    p = A.make_params(c.get("M", c.get("T")), c["NH"], c["D"])
    if c["op"] == "rotary":
        f = A.rotaryBackward if c["back"] else A.rotaryForward
        return f(st["q"], st["k"], st["inv_freq"], p, B, NKV=NKV, positions=st["positions"], interleaved=c["inter"],
                 amplitude=c["amp"])
    if c["op"] == "append":
        q = A.rotaryCacheAppend(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["start"], st["inv_freq"], p, B,
                                NKV=NKV, lens=st["lens"], interleaved=c["inter"])
        return q, st["k_cache"], st["v_cache"]
    mask = dict(window=c["window"], sinks=c["sinks"], NKV=NKV, lens=st["lens"])
    if c["op"] == "forward":
        return A.windowAttentionForward(st["q"], st["k"], st["v"], p, B, **mask)
    if c["op"] == "backward":
        return A.windowAttentionBackward(st["dO"], st["out"], st["l"], st["q"], st["k"], st["v"], p, B,
                                         dQ_dtype=torch.bfloat16, **mask)
    return A.windowAttentionCached(st["q"], st["k_cache"], st["v_cache"], st["start"], p, B, **mask)


def run(state):
    c = state["case"]
    if own:
        return _own_run(state, c)
    if c["op"] == "rotary":
        pos = state["positions"]
        if pos is None:
            pos = torch.arange(c["T"], device=state["q"].device).expand(c["B"], c["T"])
        return tuple(_plain_rotate(state[x], h, c, state["inv_freq"], pos, c["back"]) for x, h in (("q", c["NH"]), ("k", c["NKV"])))
    if c["op"] == "append":
        return _plain_append(state, c)
    if c["op"] == "forward":
        return _plain_attention(state["q"], state["k"], state["v"], c, None, state["lens"])
    if c["op"] == "backward":
        return _plain_backward(state, c)
    return _plain_attention(state["q"], state["k_cache"], state["v_cache"], c, state["start"], state["lens"])


# ------------------------------------------------------------------ exact
def _exact_turn(x, c, pos, inv_freq, back):
    """Rotation by complex numbers, fp64: x [rows, heads, D], pos [rows]."""
    w = torch.polar(torch.full((1,), c.get("amp", 1.0), dtype=torch.float64, device=x.device), pos.double()[:, None] * inv_freq)
    w = (w.conj() if back else w)[:, None]
    y, r = x.double().clone(), c["rot"]
    re, im = (y[..., 0:r:2], y[..., 1:r:2]) if c["inter"] else (y[..., : r // 2], y[..., r // 2: r])
    z = torch.complex(re.contiguous(), im.contiguous()) * w
    re.copy_(z.real)
    im.copy_(z.imag)
    return y


def _exact_keys(c, first, last, held):
    """Positions of the keys that queries at positions first..last can see, and the truth of each pair."""
    dev = held
    low = max(0, first - c["window"] + 1)
    ks = torch.cat((torch.arange(min(c["sinks"], low), device=dev), torch.arange(low, last + 1, device=dev)))
    qs = torch.arange(first, last + 1, device=dev)
    gap = qs[:, None] - ks[None]
    return ks, (gap >= 0) & ((gap < c["window"]) | (ks < c["sinks"])[None])


def exact(case, seed):
    c, st = case, prepare(case, seed)
    B, n, NH, NKV, D = c["B"], c.get("M", c.get("T")), c["NH"], c["NKV"], c["D"]
    f64, dev = torch.float64, st["q"].device
    lens = _lens(c)
    if c["op"] == "rotary":
        got = []
        for x, h in (("q", NH), ("k", NKV)):
            y = torch.empty(B, n, h * D, dtype=f64, device=dev)
            for b in range(B):
                pos = st["positions"][b] if st["positions"] is not None else torch.arange(n, device=dev)
                y[b] = _exact_turn(st[x][b].view(n, h, D), c, pos, st["inv_freq"], c["back"]).view(n, h * D)
            got.append(y)
        return tuple(got)
    starts = _starts(c) if "start" in st else [0] * B
    if c["op"] == "append":
        q = torch.zeros(B, n, NH * D, dtype=f64, device=dev)
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        for b, (s, m) in enumerate(zip(starts, lens)):
            pos = torch.arange(s, s + m, device=dev)
            q[b, :m] = _exact_turn(st["q"][b, :m].view(m, NH, D), c, pos, st["inv_freq"], False).view(m, -1)
            kc[b, s: s + m] = _exact_turn(st["k"][b, :m].view(m, NKV, D), c, pos, st["inv_freq"], False).view(m, -1)
            vc[b, s: s + m] = st["v"][b, :m].double()
        return q, kc, vc
    G, rows = NH // NKV, 512
    back = c["op"] == "backward"
    K, V = (st["k_cache"], st["v_cache"]) if c["op"] == "cached" else (st["k"], st["v"])
    o = torch.zeros(B, n, NH, D, dtype=f64, device=dev)
    l = torch.full((B, n, NH), -math.inf, dtype=f64, device=dev)
    dk, dv = (torch.zeros(B, n, NKV, D, dtype=f64, device=dev) for _ in range(2)) if back else (None, None)
    for b, (s, m) in enumerate(zip(starts, lens)):
        for r in range(0, m, rows):
            e = min(r + rows, m)
            ks, see = _exact_keys(c, s + r, s + e - 1, dev)
            k, v = (x[b, ks].view(-1, NKV, 1, D).double().permute(1, 2, 0, 3) for x in (K, V))  # [NKV, 1, keys, D]
            q = st["q"][b, r:e].view(-1, NKV, G, D).double().permute(1, 2, 0, 3)  # [NKV, G, rows, D]
            x = (q @ k.transpose(2, 3)) / math.sqrt(D)
            x[:, :, ~see] = -math.inf
            if not back:
                lse = torch.logsumexp(x, -1)
                l[b, r:e] = lse.permute(2, 0, 1).reshape(-1, NH)
                o[b, r:e] = (torch.exp(x - lse[..., None]) @ v).permute(2, 0, 1, 3).reshape(-1, NH, D)
                continue
            d, w = (st[y][b, r:e].view(-1, NKV, G, D).double().permute(1, 2, 0, 3) for y in ("dO", "out"))
            lse = st["l"][b, r:e].double().view(-1, NKV, G).permute(1, 2, 0)
            p = torch.exp(x - lse[..., None])
            t = p * (d @ v.transpose(2, 3) - (d * w).sum(-1, keepdim=True)) / math.sqrt(D)
            o[b, r:e] = (t @ k).permute(2, 0, 1, 3).reshape(-1, NH, D)  # dQ
            dk[b].index_add_(0, ks, (t.transpose(2, 3) @ q).sum(1).transpose(0, 1))
            dv[b].index_add_(0, ks, (p.transpose(2, 3) @ d).sum(1).transpose(0, 1))
    if back:
        return o.view(B, n, -1), dk.view(B, n, -1), dv.view(B, n, -1)
    return o.view(B, n, -1), l
