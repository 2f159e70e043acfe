"""What the long-context entry points refuse, checked on the host before any
device work (no GPU needed): shapes, grouped heads, windows, pointers,
overlapping tensors, workspaces."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from metalllm_b200 import _lib  # noqa: E402
from metalllm_b200._lib import AttentionParams, Rotary, Window  # noqa: E402

GAP = 1 << 30  # fake, 16-byte aligned, never dereferenced addresses, far apart


def at(n):
    return (n + 1) * GAP


def name(rc):
    return _lib.ERROR_NAMES.get(rc, rc)


def params(M=256, D=64, NH=6, N=None):
    return AttentionParams(M, NH * D if N is None else N, D, NH)


def rotary(NKV=2, rot=64, inter=0, freq=at(20)):
    return Rotary(freq, rot, inter, NKV, 1.0)


def forward(lib, p=None, r=None, ptrs=None, pos=None, B=1):
    x = ptrs or [at(i) for i in range(4)]
    return lib.ma_rotaryForward(*x, ctypes.byref(r) if r is not None else None, pos, ctypes.byref(p or params()), B, None)


@pytest.mark.parametrize("kw,code", [
    (dict(rot=0), "MA_ERR_SHAPE"), (dict(rot=63), "MA_ERR_SHAPE"), (dict(rot=66), "MA_ERR_SHAPE"),
    (dict(NKV=0), "MA_ERR_SHAPE"), (dict(NKV=4), "MA_ERR_SHAPE"), (dict(NKV=12), "MA_ERR_SHAPE"),
    (dict(inter=2), "MA_ERR_SHAPE"), (dict(freq=None), "MA_ERR_NULL"), (dict(freq=at(20) + 4), "MA_ERR_ALIGN"),
])
def test_rotary_refuses(cuda_lib, kw, code):
    assert name(forward(cuda_lib, r=rotary(**kw))) == code
    assert _lib.load().ma_last_error_string()


def test_rotary_refuses_pointers_and_overlaps(cuda_lib):
    lib, r = cuda_lib, rotary()
    assert name(forward(lib, r=None)) == "MA_ERR_NULL"
    for i in range(4):
        x = [at(j) for j in range(4)]
        x[i] = None
        assert name(forward(lib, r=r, ptrs=x)) == "MA_ERR_NULL"
        x[i] = at(i) + 8
        assert name(forward(lib, r=r, ptrs=x)) == "MA_ERR_ALIGN"
    assert name(forward(lib, r=r, pos=at(9) + 2)) == "MA_ERR_ALIGN"
    for x in ([at(0), at(1), at(0) + 16, at(3)], [at(0), at(1), at(1), at(3)], [at(0), at(1), at(2), at(0)],
              [at(0), at(1), at(2), at(2)], [at(0), at(1), at(2), at(1) + 32]):
        assert name(forward(lib, r=r, ptrs=x)) == "MA_ERR_RANGE", x
    assert name(forward(lib, p=params(D=96), r=r)) == "MA_ERR_SHAPE"
    assert name(forward(lib, p=params(N=100), r=r)) == "MA_ERR_SHAPE"
    assert name(forward(lib, r=r, B=0)) == "MA_ERR_SHAPE"
    rc = lib.ma_rotaryBackward(at(0), at(1), at(0) + 16, at(3), 1, ctypes.byref(r), None, ctypes.byref(params()), 1, None)
    assert name(rc) == "MA_ERR_RANGE"


def test_append_refuses(cuda_lib):
    lib, r, p = cuda_lib, rotary(), params(M=4)

    def call(x, start=at(7), lens=None, cap=64, B=1):
        return name(lib.ma_rotaryCacheAppend(*x, start, lens, ctypes.byref(r), ctypes.byref(p), B, cap, None))

    x = [at(i) for i in range(6)]
    assert call(x, cap=0) == "MA_ERR_SHAPE"
    assert call(x, cap=(1 << 30) + 1) == "MA_ERR_LIMIT"
    assert call(x, cap=1 << 30, B=1 << 10) == "MA_ERR_LIMIT"
    assert call(x, start=None) == "MA_ERR_NULL"
    assert call(x, start=at(7) + 2) == "MA_ERR_ALIGN"
    assert call(x, lens=at(8) + 1) == "MA_ERR_ALIGN"
    for i in range(6):
        y = list(x)
        y[i] = None
        assert call(y) == "MA_ERR_NULL"
    for i, j in ((4, 1), (5, 2), (5, 4), (3, 1), (4, 0)):  # outputs on inputs and on each other
        y = list(x)
        y[i] = y[j]
        assert call(y) == "MA_ERR_RANGE", (i, j)


def window(NKV=2, window=10, sinks=0):
    return Window(NKV, window, sinks)


@pytest.mark.parametrize("kw,code", [(dict(NKV=0), "MA_ERR_SHAPE"), (dict(NKV=4), "MA_ERR_SHAPE"),
                                     (dict(window=0), "MA_ERR_SHAPE")])
def test_window_refuses(cuda_lib, kw, code):
    lib, p, w = cuda_lib, params(), window(**kw)
    x = [at(i) for i in range(5)]
    n = ctypes.c_uint64()
    assert name(lib.ma_windowAttentionForward(*x, None, ctypes.byref(w), ctypes.byref(p), 1, None)) == code
    assert name(lib.ma_windowAttentionBackward_workspace(ctypes.byref(w), ctypes.byref(p), 1, ctypes.byref(n))) == code
    assert name(lib.ma_windowAttentionCached_workspace(ctypes.byref(w), ctypes.byref(p), 1, 64, ctypes.byref(n))) == code


def test_window_forward_refuses_pointers(cuda_lib):
    lib, p, w = cuda_lib, params(), window()

    def call(x, lens=None):
        return name(lib.ma_windowAttentionForward(*x, lens, ctypes.byref(w), ctypes.byref(p), 1, None))

    x = [at(i) for i in range(5)]
    for i in range(5):
        y = list(x)
        y[i] = None
        assert call(y) == "MA_ERR_NULL"
        y[i] = at(i) + 4
        assert call(y) == "MA_ERR_ALIGN"
    assert call(x, lens=at(8) + 2) == "MA_ERR_ALIGN"
    for i, j in ((3, 0), (3, 1), (4, 2), (4, 3)):
        y = list(x)
        y[i] = y[j]
        assert call(y) == "MA_ERR_RANGE", (i, j)
    assert name(lib.ma_windowAttentionForward(*x, None, None, ctypes.byref(p), 1, None)) == "MA_ERR_NULL"


def test_window_backward_refuses(cuda_lib):
    lib, p, w = cuda_lib, params(), window()
    n = ctypes.c_uint64()
    assert lib.ma_windowAttentionBackward_workspace(ctypes.byref(w), ctypes.byref(p), 1, ctypes.byref(n)) == 0
    assert name(lib.ma_windowAttentionBackward_workspace(ctypes.byref(w), ctypes.byref(p), 1, None)) == "MA_ERR_NULL"
    need = n.value

    def call(x, ws=at(12), have=need):
        return name(lib.ma_windowAttentionBackward(*x, 0, None, ctypes.byref(w), ctypes.byref(p), 1, ws, have, None))

    x = [at(i) for i in range(9)]
    assert call(x, have=need - 1) == "MA_ERR_LIMIT"
    assert call(x, ws=None) == "MA_ERR_NULL"
    assert call(x, ws=at(12) + 8) == "MA_ERR_ALIGN"
    assert call(x, ws=at(3)) == "MA_ERR_RANGE"
    for i in range(9):
        y = list(x)
        y[i] = None
        assert call(y) == "MA_ERR_NULL"
    for i, j in ((6, 3), (7, 4), (8, 7), (6, 0)):
        y = list(x)
        y[i] = y[j]
        assert call(y) == "MA_ERR_RANGE", (i, j)


def test_cached_refuses(cuda_lib):
    lib, p, w = cuda_lib, params(M=1), window()
    n = ctypes.c_uint64()
    assert name(lib.ma_windowAttentionCached_workspace(ctypes.byref(w), ctypes.byref(p), 1, 0, ctypes.byref(n))) == "MA_ERR_SHAPE"
    assert lib.ma_windowAttentionCached_workspace(ctypes.byref(w), ctypes.byref(p), 1, 64, ctypes.byref(n)) == 0

    def call(x, start=at(8), lens=None, cap=64, ws=at(12)):
        return name(lib.ma_windowAttentionCached(*x, start, lens, ctypes.byref(w), ctypes.byref(p), 1, cap, ws, n.value, None))

    x = [at(i) for i in range(5)]
    assert call(x, start=None) == "MA_ERR_NULL"
    assert call(x, start=at(8) + 1) == "MA_ERR_ALIGN"
    assert call(x, cap=0) == "MA_ERR_SHAPE"
    assert call(x, cap=(1 << 30) + 1) == "MA_ERR_LIMIT"
    for i, j in ((3, 0), (3, 1), (4, 2)):
        y = list(x)
        y[i] = y[j]
        assert call(y) == "MA_ERR_RANGE", (i, j)


def test_outputs_over_index_arrays_are_refused(cuda_lib):
    """positions, inv_freq, lens and start are inputs too: an output, a cache or a workspace over one of them is
    refused."""
    lib, p, w = cuda_lib, params(M=4), window()
    r, B, i = rotary(), 3, at(20)
    n = ctypes.c_uint64()

    def fwd(x, pos):
        return name(lib.ma_rotaryForward(*x, ctypes.byref(rotary(freq=at(21))), pos, ctypes.byref(p), B, None))

    def append(x, start=at(22), lens=None, freq=at(21)):
        return name(lib.ma_rotaryCacheAppend(*x, start, lens, ctypes.byref(rotary(freq=freq)), ctypes.byref(p), B, 8, None))

    def cached(x, start, lens=None, ws=at(12)):
        return name(lib.ma_windowAttentionCached(*x, start, lens, ctypes.byref(w), ctypes.byref(p), B, 512, ws, n.value, None))

    assert lib.ma_windowAttentionCached_workspace(ctypes.byref(w), ctypes.byref(p), B, 512, ctypes.byref(n)) == 0
    ends = 2 * B * 4 * 6 * 64  # bytes of q
    x = [at(j) for j in range(9)]
    assert fwd([x[0], x[1], i, x[3]], i + 64) == "MA_ERR_RANGE"
    assert "positions" in lib.ma_last_error_string().decode()
    assert fwd([x[0], x[1], i - ends + 16, x[3]], i) == "MA_ERR_RANGE"
    assert name(forward(lib, p=p, r=rotary(freq=i), ptrs=[x[0], x[1], x[2], i + 240])) == "MA_ERR_RANGE"
    assert "inv_freq" in lib.ma_last_error_string().decode()
    rc = lib.ma_rotaryBackward(x[0], x[1], i, x[3], 1, ctypes.byref(r), i + 2 * ends - 4, ctypes.byref(p), B, None)
    assert name(rc) == "MA_ERR_RANGE"  # fp32: twice the bytes
    for kw, word in ((dict(start=i + 4), "start"), (dict(lens=i + 8), "lens"), (dict(freq=i + 8), "inv_freq")):
        for j in (3, 4, 5):
            y = x[:6]
            y[j] = i
            assert append(y, **kw) == "MA_ERR_RANGE"
            assert word in lib.ma_last_error_string().decode()
    for j in (3, 4):
        y = x[:5]
        y[j] = i
        assert name(lib.ma_windowAttentionForward(*y, i + 4, ctypes.byref(w), ctypes.byref(p), B, None)) == "MA_ERR_RANGE"
        assert cached(y, i + 4) == "MA_ERR_RANGE"
        assert cached(y, at(22), i + 4) == "MA_ERR_RANGE"
    assert n.value == 0 or cached(x[:5], i + 4, ws=i) == "MA_ERR_RANGE"
    assert lib.ma_windowAttentionBackward_workspace(ctypes.byref(w), ctypes.byref(p), B, ctypes.byref(n)) == 0
    for j in (6, 7, 8, None):
        y, ws = list(x), at(12)
        if j is None:
            ws = i
        else:
            y[j] = i
        rc = lib.ma_windowAttentionBackward(*y, 0, i + 4, ctypes.byref(w), ctypes.byref(p), B, ws, n.value, None)
        assert name(rc) == "MA_ERR_RANGE"
        assert "lens" in lib.ma_last_error_string().decode()


def test_python_layer_refuses():
    """The Python layer's own checks: types, devices, groups, signs."""
    from metalllm_b200 import attention as A
    p = A.make_params(8, 4, 64)
    q = torch.zeros(1, 8, 256, dtype=torch.bfloat16)
    k = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    f = A.rotaryFrequencies(64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        A.rotaryForward(q, k, f, p, 1, NKV=2)
    with pytest.raises(ValueError, match="divide"):
        A.windowAttentionForward(q, k, k, p, 1, 4, NKV=3)
    with pytest.raises(ValueError, match="negative"):
        A.windowAttentionForward(q, k, k, p, 1, -1, NKV=2)
    with pytest.raises(ValueError, match="negative"):
        A.windowAttentionForward(q, k, k, p, 1, 4, sinks=-2, NKV=2)
    with pytest.raises(ValueError, match="CUDA"):
        A.windowAttentionForward(q, k, k, p, 1, 4, NKV=2)
    with pytest.raises(TypeError, match="inv_freq"):
        A.rotaryForward(q, k, [1.0], p, 1, NKV=2)
    with pytest.raises(TypeError, match="'?q'? must"):
        A.windowAttentionForward(None, k, k, p, 1, 4, NKV=2)
    with pytest.raises(TypeError, match="cap"):
        A.windowAttentionCached(q, k[0], k[0], None, p, 1, 4, NKV=2)
    with pytest.raises(ValueError, match="even"):
        A.rotaryFrequencies(7)


def test_outputs_of_a_call_on_another_stream(monkeypatch):
    """They are allocated in that stream's order and recorded for the current one; on the current stream itself,
    and without stream=, neither is done."""
    from contextlib import contextmanager

    from metalllm_b200 import attention as A
    inside, made, recorded = [], [], []

    @contextmanager
    def on(stream):
        inside.append(stream)
        yield
        inside.pop()

    class Stream:
        def __init__(self, handle):
            self.cuda_stream = handle

    here, side = Stream(5), Stream(9)
    empty, empty_like = torch.empty, torch.empty_like
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: here)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(A, "_raw_stream", lambda device: here.cuda_stream)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (made.append(tuple(inside)), empty(*a, **k))[1])
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: (made.append(tuple(inside)), empty_like(*a, **k))[1])
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: recorded.append(s))
    monkeypatch.setattr(A, "_check_all", lambda *a: None)
    monkeypatch.setattr(A, "_check", lambda *a: None)
    monkeypatch.setattr(A._lib, "call", lambda *a: None)
    monkeypatch.setattr(A, "_workspace", lambda *a, **k: torch.zeros(1))
    p, f = A.make_params(8, 4, 64), torch.ones(32, dtype=torch.float64)
    q, k = torch.zeros(2, 8, 256, dtype=torch.bfloat16), torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    st = torch.zeros(2, dtype=torch.int32)
    l = torch.zeros(2, 8, 4)
    calls = {
        2: [lambda s: A.rotaryForward(q, k, f, p, 2, 2, stream=s), lambda s: A.rotaryBackward(q, k, f, p, 2, 2, stream=s),
            lambda s: A.windowAttentionForward(q, k, k, p, 2, 4, 0, 2, stream=s),
            lambda s: A.windowAttentionCached(q, k, k, st, p, 2, 4, 0, 2, stream=s),
            lambda s: A.flashAttentionForward(q, q, q, p, 2, stream=s)],
        1: [lambda s: A.rotaryCacheAppend(q, k, k, k, k, st, f, p, 2, 2, stream=s)],
        3: [lambda s: A.windowAttentionBackward(q, q, l, q, k, k, p, 2, 4, 0, 2, stream=s)],
    }
    for n, group in calls.items():
        for call in group:
            for stream, want in ((side, [(side,)] * n), (here, [()] * n), (None, [()] * n)):
                made.clear(), recorded.clear()
                call(stream)
                assert made == want
                assert recorded == ([here] * n if stream is side else [])
