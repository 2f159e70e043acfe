"""GPU tests of the long-context operators (rotary positions, windowed
attention forward and backward, the cache append and the attention over a
cache) against plain fp64 forms, element by element, within the error that
their roundings allow (long_context_ref)."""
import math

import pytest

torch = pytest.importorskip("torch")

import long_context_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.fixture(scope="module")
def A():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from metalllm_b200.build import build_cuda
    build_cuda()
    from metalllm_b200 import attention
    yield attention
    torch.cuda.synchronize()
    assert attention.device_status() == 0


def randn(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def near(name, got, want, tol):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), name
    assert torch.isfinite(got[~inf]).all(), f"{name}: not finite"
    off = ((got - want).abs() / tol)[~inf]
    assert off.numel() == 0 or off.max().item() <= 1.0, f"{name}: {off.max().item():.3f} of the error allowed"


def check_forward(A, q, k, v, NH, NKV, D, window, sinks, lens=None, **kw):
    B, T = q.shape[:2]
    p = A.make_params(T, NH, D)
    out, l = A.windowAttentionForward(q, k, v, p, B, window, sinks, NKV, lens=None if lens is None else i32(lens), **kw)
    for b in range(B):
        n = T if lens is None else max(0, min(T, lens[b]))
        o64, l64, to, tl = ref.forward(q[b], k[b], v[b], NH, NKV, D, window, sinks, 0, n)
        near(f"out[{b}]", out[b], o64, to)
        near(f"l[{b}]", l[b], l64, tl)
    return out, l


def check_backward(A, dO, out, l, q, k, v, NH, NKV, D, window, sinks, lens=None, dtype=torch.bfloat16, **kw):
    B, T = q.shape[:2]
    p = A.make_params(T, NH, D)
    got = A.windowAttentionBackward(dO, out, l, q, k, v, p, B, window, sinks, NKV,
                                    lens=None if lens is None else i32(lens), dQ_dtype=dtype, **kw)
    for b in range(B):
        n = T if lens is None else max(0, min(T, lens[b]))
        want, tol = ref.backward(dO[b], out[b], l[b], q[b], k[b], v[b], NH, NKV, D, window, sinks, n,
                                 dtype == torch.float32)
        for name, g, w, t in zip(("dQ", "dK", "dV"), got, want, tol):
            near(f"{name}[{b}]", g[b], w, t)
            if n < T:
                assert not g[b][n:].any(), f"{name}[{b}]: padding rows"
    return got


# B, T, NH, NKV, D, window, sinks, lens
MASKS = [
    (1, 1, 1, 1, 64, 1, 0, None), (2, 2, 2, 1, 128, 1, 0, None), (1, 5, 2, 2, 64, 2, 1, None),
    (1, 64, 2, 2, 64, 1 << 31, 0, None),              # plain causal: a window past any sequence
    (2, 127, 2, 1, 64, 31, 3, None), (1, 128, 4, 1, 128, 128, 0, None), (1, 129, 2, 2, 128, 127, 129, None),
    (1, 300, 3, 1, 64, 128, 4, None), (1, 300, 2, 1, 128, 129, 1, None), (1, 513, 2, 2, 64, 1, 1, None),
    (1, 640, 4, 2, 64, 65, 200, None), (1, 640, 2, 2, 128, 200, 300, None),
    (1, 700, 2, 1, 64, 257, 5000, None),              # every key is a sink
    (1, 2300, 2, 1, 64, 300, 4, None),                # more than 16 tiles
    (1, 2300, 2, 2, 128, 1000, 130, None),
    (1, 4200, 3, 1, 64, 70, 2, None),
    (2, 2900, 4, 1, 128, 40, 20, [2900, 1500]),       # sinks reached by many queries of a group
    # padded batches: empty sequences, one row, whole tiles, a cut inside a tile
    (5, 260, 2, 2, 64, 100, 4, [0, 1, 128, 200, 260]), (5, 260, 4, 2, 128, 100, 4, [260, 0, 129, 256, 7]),
    (3, 2200, 2, 1, 64, 500, 10, [2200, 3, 1025]), (2, 300, 2, 2, 128, 1 << 31, 0, [-5, 1000]),
]


@pytest.mark.parametrize("B,T,NH,NKV,D,window,sinks,lens", MASKS)
def test_window_forward_and_backward(A, B, T, NH, NKV, D, window, sinks, lens):
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    out, l = check_forward(A, q, k, v, NH, NKV, D, window, sinks, lens)
    check_backward(A, dO, out, l, q, k, v, NH, NKV, D, window, sinks, lens)
    check_backward(A, dO, out, l, q, k, v, NH, NKV, D, window, sinks, lens, torch.float32)


@pytest.mark.parametrize("D", [64, 128])
def test_window_many_heads_and_sequences(A, D):
    """More units than the GPU holds at once."""
    B, T, NH, NKV, W, S = 6, 520, 24, 12, 150, 6
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    lens = [520, 300, 519, 0, 129, 384]
    out, l = check_forward(A, q, k, v, NH, NKV, D, W, S, lens)
    check_backward(A, dO, out, l, q, k, v, NH, NKV, D, W, S, lens)


@pytest.mark.parametrize("D", [64, 128])
def test_window_peaked_scores(A, D):
    """Scores of some hundreds: one key takes all, running maxima jump."""
    B, T, NH, NKV, W, S = 1, 700, 2, 1, 200, 4
    q, k = randn(B, T, NH * D, seed=1, scale=6.0), randn(B, T, NKV * D, seed=2, scale=6.0)
    v, dO = randn(B, T, NKV * D, seed=3), randn(B, T, NH * D, seed=4)
    out, l = check_forward(A, q, k, v, NH, NKV, D, W, S)
    check_backward(A, dO, out, l, q, k, v, NH, NKV, D, W, S)


@pytest.mark.parametrize("D", [64, 128])
def test_window_equals_causal_attention(A, D):
    """A window over everything, equal heads and no padding: flashAttentionForward's case, whose kernel
    rounds in the same places; l to fp32 rounding and out to one bf16 step."""
    B, T, H = 2, 400, 3
    q, k, v = (randn(B, T, H * D, seed=s) for s in (1, 2, 3))
    p = A.make_params(T, H, D)
    o1, l1 = A.flashAttentionForward(q, k, v, p, B)
    o2, l2 = A.windowAttentionForward(q, k, v, p, B, T)
    assert (l1 - l2).abs().max().item() <= 2.0 ** -18 * l1.abs().max().item()
    assert (o1.float() - o2.float()).abs().max().item() <= 4 * ref.BF * v.float().abs().max().item()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fill", [NAN, math.inf, 3e38])
def test_window_padding_holds_anything(A, D, fill):
    """Padding rows of every input, and their l, may hold NaN or infinity: nothing reaches a valid row."""
    B, T, NH, NKV, W, S = 4, 400, 4, 2, 90, 5
    lens = [250, 128, 0, 399]
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    out, l = check_forward(A, q, k, v, NH, NKV, D, W, S, lens)
    want = check_backward(A, dO, out, l, q, k, v, NH, NKV, D, W, S, lens, torch.float32)
    bad = [x.clone() for x in (q, k, v, dO, out, l)]
    for b, n in enumerate(lens):
        for x in bad:
            x[b, n:] = fill
    q2, k2, v2, dO2, out2, l2 = bad
    o, ll = A.windowAttentionForward(q2, k2, v2, A.make_params(T, NH, D), B, W, S, NKV, lens=i32(lens))
    assert torch.equal(o, out) and torch.equal(ll, l)
    got = check_backward(A, dO2, out2, l2, q2, k2, v2, NH, NKV, D, W, S, lens, torch.float32)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("D", [64, 128])
def test_window_units_of_padding_come_first(A, D):
    """Sequences cut in their first or second tile, more units than the GPU holds at once: a SM's first units
    store zeros only, and the units with keys that follow leave the padding rows zero, run after run."""
    B, T, NH, NKV, W, S = 24, 2048, 16, 4, 300, 4
    q = randn(B, T, NH * D, seed=1)
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    lens = [1 + (37 * b) % 250 for b in range(B)]
    p, ln = A.make_params(T, NH, D), i32(lens)
    pad = torch.arange(T, device="cuda")[None, :] >= ln[:, None]
    first = None
    for _ in range(10):
        out = torch.full_like(q, NAN)
        out, l = A.windowAttentionForward(q, k, v, p, B, W, S, NKV, lens=ln, out=out)
        assert not out[pad].any() and torch.isneginf(l[pad]).all()
        first = first or (out, l)
        assert torch.equal(out, first[0]) and torch.equal(l, first[1])
    for b in (0, 11, 23):
        o64, l64, to, tl = ref.forward(q[b], k[b], v[b], NH, NKV, D, W, S, 0, lens[b])
        near(f"out[{b}]", first[0][b], o64, to)
        near(f"l[{b}]", first[1][b], l64, tl)


@pytest.mark.parametrize("D", [64, 128])
def test_window_thousands_of_padding_units(A, D):
    """Units that take a microsecond each, 27 and more a SM: every one is taken once and its rows are written, in
    the forward, the backward and over a cache, run after run."""
    B, T, NH, NKV, W, S = 32, 4096, 8, 4, 300, 4
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    lens = [(37 * b) % 250 for b in range(B)]
    p, ln, st = A.make_params(T, NH, D), i32(lens), i32([0] * B)
    pad = torch.arange(T, device="cuda")[None, :] >= ln[:, None]

    def run():
        out, dQ = torch.full_like(q, NAN), torch.full_like(q, NAN)
        l = torch.full((B, T, NH), NAN, device="cuda")
        dK, dV = torch.full_like(k, NAN), torch.full_like(v, NAN)
        o2, l2 = torch.full_like(q, NAN), torch.full_like(l, NAN)
        A.windowAttentionForward(q, k, v, p, B, W, S, NKV, lens=ln, out=out, l=l)
        A.windowAttentionBackward(dO, out, l, q, k, v, p, B, W, S, NKV, lens=ln, dQ=dQ, dK=dK, dV=dV)
        A.windowAttentionCached(q, k, v, st, p, B, W, S, NKV, lens=ln, out=o2, l=l2)
        return out, l, dQ, dK, dV, o2, l2

    first = run()
    for _ in range(15):
        got = run()
        for name, x, y in zip(("out", "l", "dQ", "dK", "dV", "out over a cache", "l over a cache"), got, first):
            assert torch.isneginf(x[pad]).all() if name[0] == "l" else not x[pad].any(), name
            assert torch.equal(x, y), name
    for b in (1, 20):
        o64, l64, to, tl = ref.forward(q[b], k[b], v[b], NH, NKV, D, W, S, 0, lens[b])
        near(f"out[{b}]", first[0][b], o64, to)
        near(f"l[{b}]", first[1][b], l64, tl)


def test_window_outputs_written_whole(A):
    """Outputs given, full of NaN, come back written, and the bytes around them stay."""
    B, T, NH, NKV, D, W, S = 2, 200, 2, 1, 64, 50, 2
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))

    def inside(heads, dt):
        whole = torch.full((B * T * heads + 128,), NAN, dtype=dt, device="cuda")
        return whole, whole[64:64 + B * T * heads].view(B, T, heads)

    wo, o = inside(NH * D, torch.bfloat16)
    wl, l = inside(NH, torch.float32)
    check_forward(A, q, k, v, NH, NKV, D, W, S, [130, 200], out=o, l=l)
    wq, dQ = inside(NH * D, torch.bfloat16)
    wk, dK = inside(NKV * D, torch.bfloat16)
    wv, dV = inside(NKV * D, torch.bfloat16)
    check_backward(A, dO, o, l, q, k, v, NH, NKV, D, W, S, [130, 200], dQ=dQ, dK=dK, dV=dV)
    for w in (wo, wl, wq, wk, wv):
        assert torch.isnan(w[:64]).all() and torch.isnan(w[-64:]).all()


@pytest.mark.parametrize("D", [64, 128])
def test_window_gradient_against_differences(A, D):
    """The gradient of sum(dO * out) along a direction, against fp64 differences of the formula."""
    B, T, NH, NKV, W, S = 1, 150, 2, 1, 40, 3
    q, dO, uq = (randn(B, T, NH * D, seed=s) for s in (1, 4, 5))
    k, v, uk, uv = (randn(B, T, NKV * D, seed=s) for s in (2, 3, 6, 7))
    out, l = A.windowAttentionForward(q, k, v, A.make_params(T, NH, D), B, W, S, NKV)
    dQ, dK, dV = A.windowAttentionBackward(dO, out, l, q, k, v, A.make_params(T, NH, D), B, W, S, NKV)

    def f(e):
        o = ref.forward(q[0].double() + e * uq[0].double(), k[0].double() + e * uk[0].double(),
                        v[0].double() + e * uv[0].double(), NH, NKV, D, W, S, 0, T)[0]
        return (o * dO[0].double()).sum().item()

    h = 1e-4
    want = (f(h) - f(-h)) / (2 * h)
    got = sum((g.double() * u.double()).sum().item() for g, u in ((dQ, uq), (dK, uk), (dV, uv)))
    _, tol = ref.backward(dO[0], out[0], l[0], q[0], k[0], v[0], NH, NKV, D, W, S, T, True)
    # out enters delta rounded to bf16: D's error, through dS, moves dQ and dK by at most
    # P |delta error| scale, summed here over keys and directions; differences are exact to h^2
    eo = (out[0].double().abs() * ref.BF * dO[0].double().abs()).view(T, NH, D).sum(-1).transpose(0, 1)
    slack = sum((t * u[0].double().abs()).sum().item() for t, u in zip(tol, (uq, uk, uv)))
    span = max(uk.abs().max().item() * q.abs().max().item(), uq.abs().max().item() * k.abs().max().item())
    assert abs(got - want) <= slack + 2 * math.sqrt(D) * span * eo.sum().item() + 1e-6 * abs(want)


@pytest.mark.parametrize("D", [64, 128])
def test_window_other_stream_and_graph(A, D):
    """On a stream of the caller's, and captured: two graphs that replay in turn give what eager calls gave."""
    B, T, NH, NKV, W, S = 2, 500, 4, 2, 130, 4
    data = []
    for s in (0, 100):
        q, dO = (randn(B, T, NH * D, seed=s + i) for i in (1, 4))
        k, v = (randn(B, T, NKV * D, seed=s + i) for i in (2, 3))
        data.append((q, k, v, dO))
    p = A.make_params(T, NH, D)

    def step(x, stream=None):
        q, k, v, dO = x
        out, l = A.windowAttentionForward(q, k, v, p, B, W, S, NKV, stream=stream)
        return (out, l) + A.windowAttentionBackward(dO, out, l, q, k, v, p, B, W, S, NKV, dQ_dtype=torch.bfloat16,
                                                    stream=stream)

    want = [step(x) for x in data]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(data[0], side)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for x in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(x)
        graphs.append((g, y))
    for _ in range(3):
        for g, _y in graphs:
            g.replay()
    torch.cuda.synchronize()
    for y, w in ((got, want[0]), (graphs[0][1], want[0]), (graphs[1][1], want[1])):
        for name, a, b in zip(("out", "l", "dQ", "dK", "dV"), y, w):
            assert torch.equal(a, b), name


def test_outputs_on_another_stream_take_no_block_of_this_one(A):
    """A block freed on the current stream, whose work may still be queued, is not the output of a call on another
    stream; a dropped output is not handed out on its own stream while the current one may read it."""
    B, T, NH, D = 2, 300, 4, 64
    p = A.make_params(T, NH, D)
    q, k, v = (randn(B, T, NH * D, seed=s) for s in (1, 2, 3))
    want = A.windowAttentionForward(q, k, v, p, B, 50)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    x = torch.empty_like(q)
    ptr = x.data_ptr()
    del x
    out, l = A.windowAttentionForward(q, k, v, p, B, 50, stream=side)
    assert out.data_ptr() != ptr
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want[0]) and torch.equal(l, want[1])
    torch.cuda._sleep(200_000_000)  # the current stream is busy for about 0.1 s
    got = out + 0.0
    ptr = out.data_ptr()
    del out
    with torch.cuda.stream(side):
        y = torch.empty_like(q)
    assert y.data_ptr() != ptr
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])


def test_window_calls_at_once(A):
    """Two streams, each with its own backward and its own split attention over a cache, workspaces and all."""
    B, T, NH, NKV, D, W, S = 1, 2300, 4, 1, 64, 90, 3  # split sink tiles: partial sums in the workspace
    p, p1 = A.make_params(T, NH, D), A.make_params(1, NH, D)
    data = []
    for s in (0, 50):
        q, dO, k, v = (randn(B, T, h * D, seed=s + i) for i, h in ((1, NH), (2, NH), (3, NKV), (4, NKV)))
        out, l = A.windowAttentionForward(q, k, v, p, B, W, S, NKV)
        data.append((dO, out, l, q, k, v))

    def both(x):
        g = A.windowAttentionBackward(*x, p, B, W, S, NKV)
        return g + A.windowAttentionCached(x[3][:, -1:].contiguous(), x[4], x[5], i32([T - 1]), p1, B, T, 0, NKV)

    want = [both(x) for x in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for _ in range(5):
        for n, (st, x) in enumerate(zip(streams, data)):
            with torch.cuda.stream(st):
                got[n].append(both(x))
    torch.cuda.synchronize()
    for n in range(2):
        for g in got[n]:
            for a, b in zip(g, want[n]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_window_far_offsets(A, D):
    """q, out and the gradients of more than 2^31 elements: the last sequence and head."""
    T, NH, W, S = 8192, 32, 20, 3
    B = 2 ** 31 // (T * NH * D) + 1
    p = A.make_params(T, NH, D)
    q, dO = torch.zeros(B, T, NH * D, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, T, NH * D, dtype=torch.bfloat16, device="cuda")
    k, v = randn(B, T, D, seed=2), randn(B, T, D, seed=3)
    q[-1], dO[-1] = randn(T, NH * D, seed=1), randn(T, NH * D, seed=4)
    out, l = A.windowAttentionForward(q, k, v, p, B, W, S, 1)
    dQ, dK, dV = A.windowAttentionBackward(dO, out, l, q, k, v, p, B, W, S, 1, dQ_dtype=torch.bfloat16)
    f = A.rotaryFrequencies(D)
    qr, _ = A.rotaryForward(q, k, f, p, B, 1)
    r0, cols = T - 300, slice((NH - 1) * D, NH * D)  # the last rows see keys from r0 - W + 1 on, and the sinks
    rows = list(range(S)) + list(range(r0 - W + 1, T))
    x = [t[-1][rows] for t in (k, v)]
    # the same keys one after the other: positions move by the gap, the mask with them
    gap = r0 - W + 1 - S
    n = len(rows)
    qs = torch.zeros(n, D, dtype=torch.bfloat16, device="cuda")
    qs[S + W - 1:] = q[-1][r0:, cols]
    o64, l64, to, tl = ref.forward(qs, x[0], x[1], 1, 1, D, W, S, 0, n)
    assert gap > 0
    near("out", out[-1][r0:, cols], o64[S + W - 1:], to[S + W - 1:])
    near("l", l[-1][r0:, NH - 1:], l64[S + W - 1:], tl[S + W - 1:])
    full = [torch.zeros(n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    full[0][S + W - 1:], full[1][S + W - 1:] = dO[-1][r0:, cols], out[-1][r0:, cols]
    ls = l64.float().clone()
    ls[S + W - 1:] = l[-1][r0:, NH - 1:]
    want, tol = ref.backward(full[0], full[1], ls, qs, x[0], x[1], 1, 1, D, W, S, n, False)
    near("dQ", dQ[-1][r0:, cols], want[0][S + W - 1:], tol[0][S + W - 1:])
    wq, mq = ref.rotate(q[-1][r0:, cols], 1, D, D, False, 1.0, f, torch.arange(r0, T, device="cuda"))
    near("rotary", qr[-1][r0:, cols], wq, rotary_tol(wq, mq, torch.bfloat16))
    assert not dQ[0].any() and torch.isfinite(dK.float()).all() and torch.isfinite(dV.float()).all()
    del q, dO, out, dQ, qr
    torch.cuda.empty_cache()


def test_many_short_sequences(A):
    """70000 sequences of two rows: each as it would be alone, in every operator."""
    B, T, NH, NKV, D, W = 70000, 2, 2, 1, 64, 2
    p, f = A.make_params(T, NH, D), A.rotaryFrequencies(D)
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    ln = (torch.arange(B, device="cuda") % 3).to(torch.int32)

    def calls(i):
        n, x = len(i), [t[i].contiguous() for t in (q, k, v, dO, ln)]
        out, l = A.windowAttentionForward(*x[:3], p, n, W, 0, NKV, lens=x[4])
        g = A.windowAttentionBackward(x[3], out, l, *x[:3], p, n, W, 0, NKV, lens=x[4])
        kc, vc = torch.zeros_like(x[1]), torch.zeros_like(x[2])
        st = torch.zeros(n, dtype=torch.int32, device="cuda")
        qr = A.rotaryCacheAppend(*x[:3], kc, vc, st, f, p, n, NKV, lens=x[4])
        return (out, l) + g + (qr, kc, vc) + A.windowAttentionCached(qr, kc, vc, st, p, n, W, 0, NKV, lens=x[4])

    some = torch.tensor([0, 1, 2, 65535, 65536, B - 2, B - 1], device="cuda")
    for a, b in zip(calls(torch.arange(B, device="cuda")), calls(some)):
        assert torch.equal(a[some], b)


def test_refuses_layouts(A):
    """Strided, misaligned, mistyped and misplaced tensors are refused before anything runs."""
    B, T, NH, NKV, D = 2, 8, 2, 1, 64
    p, f = A.make_params(T, NH, D), A.rotaryFrequencies(D)
    q, k, v = randn(B, T, NH * D), randn(B, T, NKV * D), randn(B, T, NKV * D)
    qkv = randn(B, T, (NH + 2 * NKV) * D)
    st = i32([0, 0])
    shifted = randn(B * T * NH * D + 1).view(-1)[1:].view(B, T, NH * D)  # 2 bytes off a 16-byte boundary
    fwd = lambda x, **kw: A.windowAttentionForward(x, k, v, p, B, 4, 0, NKV, **kw)
    step = lambda x, **kw: A.windowAttentionCached(x, k, v, kw.pop("start", st), p, B, 4, 0, NKV, **kw)
    rot = lambda x, **kw: A.rotaryForward(x, k, kw.pop("f", f), p, B, NKV, **kw)
    for call in (fwd, step, rot):
        with pytest.raises(ValueError, match="contiguous"):
            call(qkv[..., :NH * D])
        with pytest.raises(A.MetalAttnError, match="aligned"):
            call(shifted)
        with pytest.raises(TypeError, match="bfloat16"):
            call(q.float())
        with pytest.raises(ValueError, match="CUDA"):
            call(q.cpu())
        with pytest.raises(ValueError, match="shape"):
            call(q[:1].contiguous())
    with pytest.raises(TypeError, match="int32"):
        fwd(q, lens=torch.tensor([3, 8], device="cuda"))
    with pytest.raises(ValueError, match="CUDA"):
        step(q, start=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="float64"):
        rot(q, f=f.float())
    with pytest.raises(A.MetalAttnError, match="overlaps"):
        fwd(q, out=q)
    with pytest.raises(A.MetalAttnError, match="window"):
        A.windowAttentionForward(q, k, v, p, B, 0, 0, NKV)
    with pytest.raises(A.MetalAttnError, match="cap=0"):
        A.windowAttentionCached(q, k[:, :0], v[:, :0], st, p, B, 4, 0, NKV)
    assert A.device_status() == 0


def test_window_results_repeat(A):
    """The same call gives the same bits: no sum's order is left to chance."""
    B, T, NH, NKV, D, W, S = 2, 2500, 8, 2, 128, 300, 70
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    p, ln = A.make_params(T, NH, D), i32([2500, 1800])
    runs = []
    for _ in range(4):
        out, l = A.windowAttentionForward(q, k, v, p, B, W, S, NKV, lens=ln)
        runs.append((out, l) + A.windowAttentionBackward(dO, out, l, q, k, v, p, B, W, S, NKV, lens=ln))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


# ------------------------------------------------------------------- cached
def cache_case(B, M, NH, NKV, D, cap, seed=0, fill=NAN):
    """q, and caches whose every row is `fill` until a test writes the visible ones."""
    q = randn(B, M, NH * D, seed=seed)
    kc = torch.full((B, cap, NKV * D), fill, dtype=torch.bfloat16, device="cuda")
    return q, kc, kc.clone()


def check_cached(A, q, kc, vc, start, NH, NKV, D, window, sinks, lens=None, **kw):
    B, M = q.shape[:2]
    out, l = A.windowAttentionCached(q, kc, vc, i32(start), A.make_params(M, NH, D), B, window, sinks, NKV,
                                     lens=None if lens is None else i32(lens), **kw)
    for b in range(B):
        n = M if lens is None else max(0, min(M, lens[b]))
        o64, l64, to, tl = ref.forward(q[b], kc[b], vc[b], NH, NKV, D, window, sinks, start[b], n)
        near(f"out[{b}]", out[b], o64, to)
        near(f"l[{b}]", l[b], l64, tl)
    return out, l


# B, M, NH, NKV, D, cap, window, sinks, start, lens
CACHED = [
    (1, 1, 1, 1, 64, 1, 1, 0, [0], None), (2, 1, 8, 2, 128, 70, 1000, 0, [69, 0], None),
    (3, 1, 4, 4, 64, 700, 64, 4, [699, 3, 200], None), (2, 1, 32, 2, 128, 900, 300, 1, [899, 511], None),
    (4, 1, 6, 1, 64, 5000, 4096, 16, [4999, 4100, 0, 17], [1, 1, 0, 1]),
    (1, 1, 8, 8, 128, 20000, 1 << 31, 0, [19999], None), (1, 1, 40, 1, 64, 9000, 9000, 0, [8999], None),
    (2, 2, 4, 2, 64, 300, 33, 2, [298, 100], None), (2, 5, 8, 2, 128, 1300, 1, 0, [1295, 600], [5, 3]),
    (2, 8, 8, 4, 64, 3000, 700, 130, [2992, 1000], [8, 0]), (1, 16, 2, 1, 128, 600, 100, 60, [500], None),
    (1, 17, 16, 1, 64, 2000, 513, 3, [1900], None),
    (2, 40, 4, 2, 64, 1000, 90, 3, [960, 130], [40, 11]), (2, 200, 4, 1, 128, 3000, 500, 140, [2800, 77], [200, 130]),
    (1, 300, 2, 2, 64, 4096, 4096, 0, [3796], None), (2, 260, 2, 1, 64, 700, 100, 4, [0, 440], None),
    # 128 query heads of one K/V head; padding rows of a split call
    (2, 1, 128, 1, 128, 900, 200, 5, [899, 3], None), (3, 3, 4, 2, 64, 9000, 9000, 0, [8000, 20, 8990], [3, 1, 0]),
    # a window without end, from a position inside a tile
    (1, 200, 2, 1, 64, 700, 2 ** 32 - 1, 0, [77], None), (2, 3, 4, 1, 128, 700, 2 ** 32 - 1, 2 ** 32 - 1, [77, 690], None),
    # more query tiles than SMs: units are pairs of tiles, which start inside the cache
    (3, 700, 12, 2, 64, 3000, 400, 70, [2300, 129, 0], [700, 500, 257]),
    (2, 1100, 10, 5, 128, 2000, 300, 3, [900, 13], None),
]


@pytest.mark.parametrize("B,M,NH,NKV,D,cap,window,sinks,start,lens", CACHED)
def test_cached(A, B, M, NH, NKV, D, cap, window, sinks, start, lens):
    """Rows no query sees hold NaN: the cache's end, what has left the window, padding."""
    q, kc, vc = cache_case(B, M, NH, NKV, D, cap)
    full_k, full_v = randn(B, cap, NKV * D, seed=2), randn(B, cap, NKV * D, seed=3)
    for b in range(B):
        n = M if lens is None else lens[b]
        used = ref.visible(M, cap, window, sinks, start[b], n, "cuda").any(0)
        kc[b, used], vc[b, used] = full_k[b, used], full_v[b, used]
    check_cached(A, q, kc, vc, start, NH, NKV, D, window, sinks, lens)


@pytest.mark.parametrize("B,M,NH,NKV,D,cap,window,sinks", [(64, 1, 32, 8, 128, 4300, 4096, 4), (64, 4, 16, 4, 64, 4300, 4096, 0),
                                                            (2, 1, 32, 8, 128, 60000, 60000, 0), (4, 100, 16, 4, 128, 5000, 2000, 4)])
def test_cached_results_repeat(A, B, M, NH, NKV, D, cap, window, sinks):
    """Many blocks through the ring of every SM: each of ten calls gives the same bits, and the right ones."""
    q = randn(B, M, NH * D, seed=1)
    kc, vc = randn(B, cap, NKV * D, seed=2), randn(B, cap, NKV * D, seed=3)
    start = [cap - M - 17 * (b % 8) for b in range(B)]
    p, st = A.make_params(M, NH, D), i32(start)
    runs = [A.windowAttentionCached(q, kc, vc, st, p, B, window, sinks, NKV) for _ in range(10)]
    for o, l in runs[1:]:
        assert torch.equal(o, runs[0][0]) and torch.equal(l, runs[0][1])
    o, l = runs[0]
    for b in range(0, B, 9):
        o64, l64, to, tl = ref.forward(q[b], kc[b], vc[b], NH, NKV, D, window, sinks, start[b], M)
        near("out", o[b], o64, to)
        near("l", l[b], l64, tl)


def test_cached_far_rows(A):
    """A cache of more than 2^32 bytes and more than 2^31 elements: the last sequence's rows."""
    B, M, NH, NKV, D, cap, W, S = 3, 1, 8, 8, 128, 1 << 20, 200, 4
    q = randn(B, M, NH * D, seed=1)
    kc = torch.empty((B, cap, NKV * D), dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    start = [cap - 1, 5, cap - 2]
    rows = [list(range(S)) + list(range(max(S, s - W + 1), s + 1)) for s in start]
    out = A.windowAttentionCached
    for b, r in enumerate(rows):
        kc[b, r], vc[b, r] = randn(len(r), NKV * D, seed=20 + b), randn(len(r), NKV * D, seed=30 + b)
    o, l = out(q, kc, vc, i32(start), A.make_params(M, NH, D), B, W, S, NKV)
    for b, r in enumerate(rows):  # the same keys without the gap between sinks and window
        o64, l64, to, tl = ref.forward(q[b], kc[b, r], vc[b, r], NH, NKV, D, len(r), 0, len(r) - 1, 1)
        near("out", o[b], o64, to)
        near("l", l[b], l64, tl)
    del kc, vc
    torch.cuda.empty_cache()


def test_cached_past_the_end_stays_inside(A):
    """start + M past the cache, negative or huge: no fault, rows that fit are right."""
    B, M, NH, NKV, D, cap = 3, 4, 2, 1, 64, 300
    q = randn(B, M, NH * D, seed=1)
    kc, vc = randn(B, cap, NKV * D, seed=2), randn(B, cap, NKV * D, seed=3)
    start = [cap - 2, -7, 2 ** 31 - 2]
    out, l = A.windowAttentionCached(q, kc, vc, i32(start), A.make_params(M, NH, D), B, 50, 2, NKV)
    assert torch.isfinite(out.float()).all() and torch.isfinite(l).all()
    o64, l64, to, tl = ref.forward(q[0, :2], kc[0], vc[0], NH, NKV, D, 50, 2, cap - 2, 2)
    near("out", out[0, :2], o64, to)


# ------------------------------------------------------------------- rotary
def rotary_tol(want, mag, dtype):
    """bf16: half a step of the value; fp32: the angle's 2^-24 turns (2^-21 rad), sincos and four roundings."""
    return (ref.BF if dtype == torch.bfloat16 else 0.0) * want.abs() + 2.0 ** -20 * mag + 1e-30


# B, T, NH, NKV, D, rot, interleaved, positions
ROTARY = [
    (1, 1, 1, 1, 64, 64, False, None), (2, 3, 4, 2, 64, 64, True, None), (2, 100, 3, 1, 128, 128, False, 999999),
    (1, 257, 6, 6, 64, 32, True, None), (1, 50, 2, 1, 128, 64, False, 4000000), (1, 33, 2, 2, 64, 2, False, None),
    (1, 33, 2, 2, 64, 6, True, 12), (2, 65, 3, 3, 128, 126, False, -30), (1, 40, 5, 1, 64, 48, False, None),
    (1, 40, 5, 1, 128, 72, True, 2 ** 31 - 100), (3, 1, 32, 8, 128, 128, True, 7),
    (2, 37, 3, 1, 64, 24, False, None), (2, 37, 3, 1, 64, 20, False, None), (1, 37, 4, 2, 128, 100, True, 5),
    (1, 37, 4, 2, 128, 118, True, None), (1, 300, 4, 2, 64, 18, False, None),
]


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("B,T,NH,NKV,D,rot,inter,far", ROTARY)
def test_rotary(A, B, T, NH, NKV, D, rot, inter, far, back):
    f = A.rotaryFrequencies(rot)
    amp = 1.0 if rot == D else 1.25
    pos = torch.arange(T).expand(B, T) + torch.arange(B)[:, None] * 3 if far is None else (torch.arange(B * T) % T).view(B, T) + far
    given = None if far is None else pos.to(torch.int32).cuda().contiguous()
    if far is None:
        pos = torch.arange(T).expand(B, T)
    p = A.make_params(T, NH, D)
    k = randn(B, T, NKV * D, seed=2)
    for dt in ((torch.bfloat16, torch.float32) if back else (torch.bfloat16,)):
        q = randn(B, T, NH * D, seed=1, dtype=dt)
        call = A.rotaryBackward if back else A.rotaryForward
        got = call(q, k, f, p, B, NKV, positions=given, interleaved=inter, amplitude=amp)
        for name, x, y, h in (("q", q, got[0], NH), ("k", k, got[1], NKV)):
            assert y.dtype == x.dtype
            for b in range(B):
                want, mag = ref.rotate(x[b], h, D, rot, inter, amp, f, pos[b].cuda(), back)
                near(name, y[b], want, rotary_tol(want, mag, x.dtype))
                assert torch.equal(y[b].view(T, h, D)[..., rot:], x[b].view(T, h, D)[..., rot:])
        q2, k2 = q.clone(), k.clone()  # in place
        out = {"dQ_out": q2, "dK_out": k2} if back else {"q_out": q2, "k_out": k2}
        call(q2, k2, f, p, B, NKV, positions=given, interleaved=inter, amplitude=amp, **out)
        assert torch.equal(q2, got[0]) and torch.equal(k2, got[1])


def test_rotary_frequencies(A):
    f = A.rotaryFrequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(A.rotaryFrequencies(8, base=100.0, factor=4.0, device="cpu"), f / 4)
    g = A.rotaryFrequencies(64, factor=8.0, original_length=4096, device="cpu")
    full = A.rotaryFrequencies(64, device="cpu")
    assert torch.equal(g[:2], full[:2])           # many turns within 4096: kept
    assert torch.allclose(g[-1], full[-1] / 8)    # less than one: stretched
    assert (g <= full).all() and (g >= full / 8).all()


# B, M, NH, NKV, D, cap, rot, interleaved, start, lens
APPEND = [
    (1, 1, 1, 1, 64, 1, 64, False, [0], None), (4, 1, 8, 2, 128, 50, 128, False, [49, 0, 7, 33], [1, 1, 0, 1]),
    (2, 70, 4, 1, 64, 200, 32, True, [0, 130], [70, 33]), (1, 9, 2, 2, 128, 40, 6, False, [31], None),
    (3, 33, 4, 2, 64, 90, 18, False, [3, 0, 57], [33, 1, 30]), (2, 12, 4, 2, 128, 90, 100, True, [3, 0], [0, 12]),
    (2, 12, 3, 1, 64, 90, 24, False, [3, 70], [5, 12]), (1, 12, 3, 1, 64, 90, 28, False, [3], [5]),
    (2, 5, 3, 3, 64, 8, 64, True, [6, -2], None),     # rows past the end and before the start are not stored
]


@pytest.mark.parametrize("B,M,NH,NKV,D,cap,rot,inter,start,lens", APPEND)
def test_cache_append(A, B, M, NH, NKV, D, cap, rot, inter, start, lens):
    f = A.rotaryFrequencies(rot)
    q, k, v = randn(B, M, NH * D, seed=1), randn(B, M, NKV * D, seed=2), randn(B, M, NKV * D, seed=3)
    k0, v0 = randn(B, cap, NKV * D, seed=4), randn(B, cap, NKV * D, seed=5)
    for place in (False, True):
        kc, vc, q1 = k0.clone(), v0.clone(), q.clone()
        got = A.rotaryCacheAppend(q1, k, v, kc, vc, i32(start), f, A.make_params(M, NH, D), B, NKV,
                                  lens=None if lens is None else i32(lens), interleaved=inter,
                                  q_out=q1 if place else None)
        for b in range(B):
            n = M if lens is None else lens[b]
            pos = torch.arange(start[b], start[b] + M, device="cuda")
            wq, mq = ref.rotate(q[b], NH, D, rot, inter, 1.0, f, pos)
            wk, mk = ref.rotate(k[b], NKV, D, rot, inter, 1.0, f, pos)
            near("q", got[b, :n], wq[:n], rotary_tol(wq, mq, q.dtype)[:n])
            assert not got[b, n:].any()
            left = torch.ones(cap, dtype=torch.bool, device="cuda")
            for i in range(n):
                t = start[b] + i
                if 0 <= t < cap:
                    left[t] = False
                    near("k", kc[b, t], wk[i], rotary_tol(wk, mk, k.dtype)[i])
                    assert torch.equal(vc[b, t], v[b, i])
            assert torch.equal(kc[b, left], k0[b, left]) and torch.equal(vc[b, left], v0[b, left])


# --------------------------------------------------------- together, as used
@pytest.mark.parametrize("D,inter,lens", [(64, False, None), (128, True, [333, 128])])
def test_training_chain(A, D, inter, lens):
    """Rotary, attention, its backward and the rotary backward, against the whole chain's gradient by autograd
    in fp64.  bf16 intermediates: a handful of roundings of q, k, P, dS, dK, out, each 2^-8 of a term; the
    norm of their sum stays within 4 of them."""
    B, T, NH, NKV, W, S, rot = 2, 333, 4, 2, 100, 4, D // 2
    f = A.rotaryFrequencies(rot)
    q, dO = (randn(B, T, NH * D, seed=s) for s in (1, 4))
    k, v = (randn(B, T, NKV * D, seed=s) for s in (2, 3))
    p = A.make_params(T, NH, D)
    ln = None if lens is None else i32(lens)
    qr, kr = A.rotaryForward(q, k, f, p, B, NKV, interleaved=inter)
    out, l = A.windowAttentionForward(qr, kr, v, p, B, W, S, NKV, lens=ln)
    dQ, dK, dV = A.windowAttentionBackward(dO, out, l, qr, kr, v, p, B, W, S, NKV, lens=ln)
    dQ, dK = A.rotaryBackward(dQ, dK, f, p, B, NKV, interleaved=inter, dQ_out=dQ, dK_out=dK)
    pos = torch.arange(T, device="cuda")
    for b in range(B):
        n = T if lens is None else lens[b]
        x = [t[b].double().requires_grad_() for t in (q, k, v)]

        def turn(y, h):
            ang = pos.double()[:, None] * f
            c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
            y = y.view(T, h, D)
            a, e = (y[..., 0:rot:2], y[..., 1:rot:2]) if inter else (y[..., :rot // 2], y[..., rot // 2:rot])
            u, w = a * c - e * s, a * s + e * c
            z = torch.stack((u, w), -1).flatten(-2) if inter else torch.cat((u, w), -1)
            return torch.cat((z, y[..., rot:]), -1).transpose(0, 1)

        Q, K = turn(x[0], NH), turn(x[1], NKV).repeat_interleave(NH // NKV, 0)
        V = x[2].view(T, NKV, D).transpose(0, 1).repeat_interleave(NH // NKV, 0)
        see = ref.visible(T, T, W, S, 0, T, "cuda")
        o = torch.softmax((Q @ K.transpose(1, 2) / math.sqrt(D)).masked_fill(~see, -math.inf), -1) @ V
        o = o.transpose(0, 1).reshape(T, -1)
        (o[:n] * dO[b, :n].double()).sum().backward()
        for name, g, w in (("out", out[b, :n], o[:n].detach()), ("dQ", dQ[b], x[0].grad), ("dK", dK[b], x[1].grad),
                           ("dV", dV[b], x[2].grad)):
            off = (g.double() - w).norm() / w.norm()
            assert off.item() <= 4 * ref.BF, f"{name}: {off.item():.2e}"


@pytest.mark.parametrize("D,NH,NKV,M", [(64, 4, 2, 50), (128, 8, 1, 200)])
def test_serving_chain(A, D, NH, NKV, M):
    """Prompts of different lengths enter the cache in one padded piece, a second piece follows, then single
    tokens: every row equals the row of one windowed forward over the whole rotated sequence."""
    B, cap, W, S, steps = 3, 512, 60, 3, 3
    f = A.rotaryFrequencies(D)
    first = [M, M // 2, 1]
    total = [n + 30 + steps for n in first]
    q, k, v = (randn(B, cap, h * D, seed=s) for h, s in ((NH, 1), (NKV, 2), (NKV, 3)))
    p = A.make_params(cap, NH, D)
    qr, kr = A.rotaryForward(q, k, f, p, B, NKV)
    want, wl = A.windowAttentionForward(qr, kr, v, p, B, W, S, NKV, lens=i32(total))
    kc, vc = torch.full((2, B, cap, NKV * D), NAN, dtype=torch.bfloat16, device="cuda")
    start = [0] * B
    pieces = [(M, first), (30, [30] * B)] + [(1, [1] * B)] * steps
    for m, lens in pieces:
        new = [torch.zeros(B, m, x.shape[2], dtype=x.dtype, device="cuda") for x in (q, k, v)]
        for b in range(B):
            for y, x in zip(new, (q, k, v)):
                y[b, :lens[b]] = x[b, start[b]:start[b] + lens[b]]
        pm = A.make_params(m, NH, D)
        qn = A.rotaryCacheAppend(*new, kc, vc, i32(start), f, pm, B, NKV, lens=i32(lens))
        out, l = A.windowAttentionCached(qn, kc, vc, i32(start), pm, B, W, S, NKV, lens=i32(lens))
        for b in range(B):
            s, n = start[b], lens[b]
            assert (l[b, :n] - wl[b, s:s + n]).abs().max().item() <= 2.0 ** -18 * wl[b, s:s + n].abs().max().item()
            # both round P and the output to bf16, each 2^-8 of sums within |v|'s largest
            assert (out[b, :n].float() - want[b, s:s + n].float()).abs().max().item() <= 4 * ref.BF * v.float().abs().max().item()
            assert not out[b, n:].any() and torch.isneginf(l[b, n:]).all()
            start[b] += n


def test_append_and_step_in_a_graph(A):
    """A decoding step captured once and replayed while start grows on the device."""
    B, NH, NKV, D, cap, W, S = 2, 4, 2, 64, 300, 80, 2
    f = A.rotaryFrequencies(D)
    kc, vc = randn(B, cap, NKV * D, seed=2), randn(B, cap, NKV * D, seed=3)
    kc2, vc2 = kc.clone(), vc.clone()
    q, k, v = randn(B, 1, NH * D, seed=4), randn(B, 1, NKV * D, seed=5), randn(B, 1, NKV * D, seed=6)
    p = A.make_params(1, NH, D)
    start = i32([100, 250])

    def step(kc, vc, start):
        qn = A.rotaryCacheAppend(q, k, v, kc, vc, start, f, p, B, NKV)
        return A.windowAttentionCached(qn, kc, vc, start, p, B, W, S, NKV)

    step(kc.clone(), vc.clone(), start)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, l = step(kc, vc, start)
    for i in range(4):
        g.replay()
        o2, l2 = step(kc2, vc2, i32([100 + i, 250 + i]))
        torch.cuda.synchronize()
        assert torch.equal(out, o2) and torch.equal(l, l2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
        start += 1
