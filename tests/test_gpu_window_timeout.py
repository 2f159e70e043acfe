"""The time-out path of the windowed kernels' bounded waits, on the GPU, without a
fault: ma_debug_expire_next_wait lets one wait of the next launch run out after
1 ms on a barrier that nothing arrives at, with copies and products in flight.
Each test checks that the status names that kernel, and that the calls after it
give the bits of the calls before it.  Every wait, those of the wind-down
included, is bounded."""
import pytest

torch = pytest.importorskip("torch")

from metalllm_b200 import _lib  # noqa: E402

pytestmark = pytest.mark.gpu

LIMIT_NS = 1_000_000


@pytest.fixture(scope="module")
def A():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from metalllm_b200.build import build_cuda
    build_cuda()
    from metalllm_b200 import attention
    yield attention
    attention.debug_expire_next_wait(0)


def randn(*shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").bfloat16()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def expire(A, bit, call):
    """call() three times: as it is, with a wait that runs out, and as it is again."""
    want = call()
    torch.cuda.synchronize()
    assert A.device_status() == 0
    A.debug_expire_next_wait(bit, LIMIT_NS)
    call()
    torch.cuda.synchronize()
    assert A.device_status() == bit
    for _ in range(2):  # the request was consumed: ordinary calls again
        for a, b in zip(call(), want):
            assert torch.equal(a, b)
    assert A.device_status() == 0


# B, T, NH, NKV, lens: units of one tile (one key tile, several), units of two, and more of them than SMs, so that
# a launch-control request is in flight; padded batches, whose units of padding have no product to wait for
FORWARD = [(1, 100, 2, 1, None), (1, 500, 3, 1, None), (2, 700, 24, 4, None), (2, 2304, 24, 4, None),
           (8, 1500, 16, 16, [1500, 3, 0, 129, 700, 1500, 1, 256])]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,NH,NKV,lens", FORWARD)
def test_forward(A, D, B, T, NH, NKV, lens):
    q, k, v = (randn(B, T, h * D, seed=s) for h, s in ((NH, 1), (NKV, 2), (NKV, 3)))
    p, ln = A.make_params(T, NH, D), None if lens is None else i32(lens)
    expire(A, _lib.STATUS_FWD_TIMEOUT, lambda: A.windowAttentionForward(q, k, v, p, B, 300, 4, NKV, lens=ln))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,NH", [(200, 4), (700, 48)])
def test_cached_many_rows(A, D, M, NH):
    B, NKV, cap = 2, 2, 3000
    q, kc, vc = randn(B, M, NH * D, seed=1), randn(B, cap, NKV * D, seed=2), randn(B, cap, NKV * D, seed=3)
    p, start = A.make_params(M, NH, D), i32([2000, 77])
    expire(A, _lib.STATUS_FWD_TIMEOUT, lambda: A.windowAttentionCached(q, kc, vc, start, p, B, 900, 4, NKV))


# B, T, NH, NKV, window, lens: few units; more of them than SMs in each pass; sink tiles cut into units of their own,
# whose partial sums a last kernel adds up; padded batches
BACKWARD = [(1, 100, 2, 1, 300, None), (2, 1024, 24, 24, 300, None), (1, 4200, 3, 1, 70, None),
            (8, 1500, 16, 16, 300, [1500, 3, 0, 129, 700, 1500, 1, 256])]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,NH,NKV,window,lens", BACKWARD)
def test_backward(A, D, B, T, NH, NKV, window, lens):
    q, k, v, dO = (randn(B, T, h * D, seed=s) for h, s in ((NH, 1), (NKV, 2), (NKV, 3), (NH, 4)))
    p, ln = A.make_params(T, NH, D), None if lens is None else i32(lens)
    out, l = A.windowAttentionForward(q, k, v, p, B, window, 4, NKV, lens=ln)
    expire(A, _lib.STATUS_BWD_TIMEOUT,
           lambda: A.windowAttentionBackward(dO, out, l, q, k, v, p, B, window, 4, NKV, lens=ln))


# B, M, NH, NKV, cap: one split, the key axis split and joined, some requests of padding
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,M,NH,NKV,cap,lens", [(64, 1, 32, 8, 1500, None), (1, 1, 8, 2, 20000, None),
                                                 (3, 5, 8, 2, 3000, [5, 0, 2])])
def test_cached_few_rows(A, D, B, M, NH, NKV, cap, lens):
    q, kc, vc = randn(B, M, NH * D, seed=1), randn(B, cap, NKV * D, seed=2), randn(B, cap, NKV * D, seed=3)
    p, start, ln = A.make_params(M, NH, D), i32([cap - M] * B), None if lens is None else i32(lens)
    expire(A, _lib.STATUS_FWD_TIMEOUT, lambda: A.windowAttentionCached(q, kc, vc, start, p, B, cap, 0, NKV, lens=ln))
