"""The k largest of each row against a stable 64-bit sort: ties, masked rows, NaN, rows that end inside a piece or a split, and the
calls that are refused."""
import ctypes

import pytest
import torch

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _check(x, k, got=None):
    from gmk import ops
    v, i = ops.topk_rows(x.cuda(), k) if got is None else got
    # a stable sort keeps equal values by rising index, has -0 equal 0 and puts NaN above all
    _, ri = torch.sort(x.double(), dim=1, descending=True, stable=True)
    ri = ri[:, :k]
    assert v.dtype == x.dtype and i.dtype == torch.int32 and v.shape == i.shape == ri.shape
    assert torch.equal(i.cpu().long(), ri), (x.shape, k)
    # the values are the row's own, bit for bit
    bits = torch.int32 if x.dtype == torch.float32 else torch.int16
    assert torch.equal(v.cpu().view(bits), x.view(bits).gather(1, ri))   # of whole numbers: a gather on the CPU changes a bf16 NaN's bits


SHAPES = [(1, 1, 1), (3, 10, 3), (5, 10, 10), (256, 10, 3), (4, 63, 7), (2, 64, 64), (3, 65, 2), (7, 257, 256), (256, 1000, 10), (3, 1023, 100), (2, 2048, 128), (9, 4099, 33),
          (2, 10007, 20), (300, 5003, 5), (1, 30000, 256), (3, 32768, 64), (2, 65537, 1), (1, 150001, 50), (4, 200003, 128), (1, 1000003, 256)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_topk_rows(shape, dtype):
    n, C, k = shape
    _check((3 * _randn(C + k, n, C)).to(dtype), k)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [8191, 8192, 8193, 12287, 12289, 24577, 2093057, 2097153])
def test_topk_rows_where_parts_end(C, dtype):
    """Rows around whole numbers of parts, the last one short; the largest elements in the last part, or in the first."""
    for k in (1, 8, 50, 256):
        x = _randn(C + k, 2, C)
        x[0, C - min(k, 100):] += 20
        x[1, : min(k, 100)] += 20
        _check(x.to(dtype), k)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,k", [(9001, 100), (17001, 20), (33003, 40), (70001, 128)])
def test_topk_rows_ties_and_masks_in_whole_rows(C, k, dtype):
    """Enough rows that none is split: equal values, few different ones, masked rows, NaN, the largest all in one thread's elements."""
    from gmk import ops
    n, some = 520, 14
    g = torch.Generator().manual_seed(C)
    x = torch.randn(n, C, generator=torch.Generator("cuda").manual_seed(C), device="cuda")
    y = _randn(C, some, C)
    y[0] = 0.0
    y[1] = -float("inf")
    y[2] = torch.finfo(torch.float32).min
    y[3] = torch.randint(0, 3, (C,), generator=g).float()
    y[4, : C - k // 2] = -float("inf")
    y[5, ::3] = float("inf")
    y[6, 5:] = float("nan")
    y[7, -3:] = float("nan")
    y[8] = torch.arange(C).float()
    y[9] = -torch.arange(C).float()
    y[10, 2048:2052] += 50
    y[11, ::1024] += 50
    y[12, C - k:] += 50
    y[13, 1:] = -float("inf")
    x[:some] = y.cuda()
    x = x.to(dtype)
    v, i = ops.topk_rows(x, k)
    rows = list(range(some)) + [100, n - 1]
    _check(x[rows].cpu(), k, (v[rows], i[rows]))


@gpu
@pytest.mark.parametrize("C,k", [(10, 4), (300, 40), (5000, 256), (70001, 64), (200000, 17)])
def test_topk_rows_ties_and_masks(C, k):
    """Rows of equal values, of few different ones, masked to fewer than k, wholly masked, with NaN and both zeros, rising and
    falling rows."""
    g = torch.Generator().manual_seed(C)
    x = _randn(C, 12, C)
    x[0] = 0.0
    x[1] = -float("inf")
    x[2] = torch.finfo(torch.float32).min
    x[3] = torch.randint(0, 3, (C,), generator=g).float()
    x[4, : C - k // 2] = -float("inf")
    x[5, ::7] = float("inf")
    x[6, 5:] = float("nan")
    x[7] = torch.where(torch.rand(C, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(-0.0))
    x[8] = torch.arange(C).float()
    x[9] = -torch.arange(C).float()
    x[10] = -x[10].abs() - 1
    x[10, C // 2] = -x[10, C // 2]
    x[11] = 1.0
    x[11, -1] = 2.0
    for dtype in TYPES:
        _check(x.to(dtype), k)


@gpu
def test_topk_rows_at_any_element():
    """Rows of a contiguous view that starts at no 16-byte border, between values that must not be seen."""
    from gmk import ops
    for dtype in TYPES:
        for n, C, k in ((3, 1001, 9), (2, 70003, 30)):
            for off in (1, 3, 7):
                buf = torch.full((n * C + 64,), float("inf"), dtype=dtype, device="cuda")
                x = buf[off: off + n * C].view(n, C)
                x.copy_(_randn(off, n, C).to(dtype))
                _check(x.cpu(), k, ops.topk_rows(x, k))


@gpu
def test_topk_rows_streams_graphs_and_empty():
    from gmk import ops
    xs = [_randn(i, 3, 90001).cuda() for i in range(2)]
    ref = [ops.topk_rows(x, 40) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.topk_rows(x, 40))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eager = ops.topk_rows(xs[0], 40)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, r in zip(outs, ref) for a, b in zip(o, r))
        assert torch.equal(eager[1], ref[0][1])
    v, i = ops.topk_rows(torch.empty(0, 50, device="cuda"), 5)
    assert v.shape == i.shape == (0, 5)


@gpu
def test_scratch_under_another_stream_handle(monkeypatch):
    """Calls in SideQueue.run, where the launch goes to a side stream and torch's current stream stays: the scratch that dies with the call
    is not handed out again while the side stream, held up by a wait of some milliseconds, has yet to use it."""
    from gmk import ops
    x = _randn(1, 3, 90001).cuda()
    ref = ops.topk_rows(x, 40)
    seen = []
    real = ops._scratch
    monkeypatch.setattr(ops, "_scratch", lambda *a: [seen.append((t.data_ptr(), b)) or (t, b) for t, b in [real(*a)]][0])
    kept = ops.topk_rows(x, 40)
    again = torch.empty(seen[-1][1], dtype=torch.uint8, device="cuda")
    assert again.data_ptr() == seen[-1][0]   # a call on the current stream: its scratch is free behind it, in the stream's order
    del again, kept
    torch.cuda.synchronize()
    side = ops.SideQueue(x.device)
    for st in side.streams:
        with torch.cuda.stream(st):
            torch.cuda._sleep(20_000_000)
    out = side.run(lambda: ops.topk_rows(x, 40), x)
    others = [torch.full((seen[-1][1],), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
    at, size = seen[-1]
    assert all(o.data_ptr() >= at + size or o.data_ptr() + size <= at for o in others)
    side.join()
    torch.cuda.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


def test_topk_rows_refusals():
    from gmk import lib, ops
    h = lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    f = lambda **k: h.gmk_topk_rows(*{**dict(x=p, t=0, v=p, i=p, n=2, C=100, k=5, w=p, wb=1 << 40, st=None), **k}.values())  # noqa: E731
    assert f(t=3) == f(t=-1) == -3
    assert f(n=-1) == f(C=0) == f(k=0) == f(k=101) == -1
    assert f(k=257, C=1000) == f(C=1 << 31) == -6
    assert f(x=None) == f(v=None) == f(i=None) == -5
    assert f(x=odd) == f(v=odd) == f(i=ctypes.c_void_p(4098)) == -2
    assert f(n=0, x=None) == 0
    need = int(h.gmk_topk_rows_workspace_bytes(2, 1 << 20, 5))
    assert need == 0 or f(C=1 << 20, wb=need - 1) == -4
    with pytest.raises(ValueError):
        ops.topk_rows(torch.zeros(2, 5), 2)


def test_widest_rows():
    """2^31 - 2 classes are the most that the header allows, of a top-k and of a distillation (then the missing tensors are what is refused)."""
    from gmk import lib
    h = lib()
    for C, code in (((1 << 31) - 2, -5), ((1 << 31) - 1, -6)):
        assert h.gmk_topk_rows(None, 0, None, None, 2, C, 5, None, 0, None) == code
        assert h.gmk_distill_fwd_bwd(None, 0, None, 0, None, None, None, None, None, 2, C, 5, 1.0, 1.0, 0.0, 1.0, None, 0, None) == code


@gpu
def test_topk_rows_refuses_wrong_tensors():
    from gmk import ops
    x = torch.zeros(4, 20, device="cuda")
    for call in (lambda: ops.topk_rows(x, 0), lambda: ops.topk_rows(x, 21), lambda: ops.topk_rows(x.t(), 2), lambda: ops.topk_rows(x[0], 2),
                 lambda: ops.topk_rows(x.double(), 2), lambda: ops.topk_rows(x.long(), 2), lambda: ops.topk_rows(torch.zeros(2, 1000, device="cuda"), 257)):
        with pytest.raises(ValueError):
            call()
