"""8-bit rows and the 8-bit linear layer against 64-bit arithmetic, at the sizes where tiles, pieces and splits end, and the
calls that are refused.  The quantised values and the whole-number sums are exact; what is rounded after that is counted."""
import ctypes

import pytest
import torch

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _rows(x):
    """(q, scale) of the definition: the quotient in 64 bits, the scale a 127th of the largest magnitude in 32 bits."""
    x = x.double()
    scale = (x.abs().amax(1) / 127).float().clamp_min(2.0 ** -126)
    return (x / scale.double()[:, None]).round(), scale


def _act(name, z):
    if name == "relu":
        return z.clamp_min(0)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / 2 ** 0.5)
    if name == "elu":
        return torch.where(z > 0, z, torch.expm1(z))
    return z


def _linear_oracle(x, wq, ws, b, act):
    q, s = _rows(x)
    z = (q @ wq[:, : q.shape[1]].double().T) * s.double()[:, None] * ws.double()
    return _act(act, z if b is None else z + b.double()), z


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 15), (2, 16), (5, 17), (1, 4096), (7, 1357), (33, 2048), (2, 8192), (3, 9001), (1, 40007), (130, 256)])
def test_quantize_rows_is_exact(shape, dtype):
    from gmk import ops
    x = (_randn(1, *shape) * torch.logspace(-3, 3, shape[0])[:, None]).to(dtype)
    q, scale = ops.quantize_rows(x.cuda())
    rq, rs = _rows(x)
    assert q.shape == (shape[0], -(-shape[1] // 16) * 16)
    assert torch.equal(scale.cpu(), rs)
    assert torch.equal(q.cpu()[:, : shape[1]].double(), rq)
    assert not q[:, shape[1]:].any()


@gpu
def test_quantize_rows_halves_extremes_and_rows_without_a_scale():
    from gmk import ops
    # scale 1: halves go to the even neighbour; a hair beside them to the nearest
    halves = torch.arange(-126.5, 127, 1.0)
    up, down = halves * (1 + 2.0 ** -23), halves * (1 - 2.0 ** -23)
    rows = torch.stack([torch.cat([h, torch.tensor([127.0, 0.0])]) for h in (halves, up, down)])
    rows[:, -2] = 127.0
    # zeros, denormals, the largest numbers
    other = torch.zeros(4, rows.shape[1])
    other[1, 3] = 1e-42
    other[2] = 3.4e38
    other[2, ::2] = -1.7e38
    other[3, :5] = torch.tensor([2.0 ** -126, -(2.0 ** -120), 3 * 2.0 ** -127, 0.0, 2.0 ** -149])
    x = torch.cat([rows, other])
    q, scale = ops.quantize_rows(x.cuda())
    rq, rs = _rows(x)
    assert torch.equal(scale.cpu(), rs)
    assert torch.equal(q.cpu()[:, : x.shape[1]].double(), rq)
    # an infinity or a NaN: zeros and a NaN scale, neighbours untouched
    y = x.clone()
    y[1, 7], y[4, -1], y[5, 0] = float("inf"), float("nan"), float("-inf")
    q2, scale2 = ops.quantize_rows(y.cuda())
    bad = torch.tensor([False, True, False, False, True, True, False])
    assert torch.equal(torch.isnan(scale2.cpu()), bad)
    assert not q2.cpu()[bad].any()
    assert torch.equal(q2.cpu()[~bad], q.cpu()[~bad]) and torch.equal(scale2.cpu()[~bad], rs[~bad])


# M, K, N: single rows, few rows, tiles that end inside, K chunks that end inside, odd everything, several tiles each way
SHAPES = [(1, 30000, 40), (4, 8192, 9000), (3, 10, 9001), (1, 16, 1), (1, 256, 10), (1, 4096, 1000), (2, 100, 37), (4, 8200, 33), (5, 1, 5), (8, 4097, 129), (16, 640, 64), (17, 64, 17), (24, 8192, 200),
          (33, 2050, 1030), (64, 16384, 48), (65, 128, 257), (100, 333, 300), (128, 256, 128), (129, 1357, 131), (256, 4096, 256), (257, 144, 513), (300, 80, 1100),
          (512, 512, 512), (777, 1357, 503), (1030, 272, 770)]


@gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_i8(shape):
    from gmk import ops
    M, K, N = shape
    for i, (xt, yt, act, bias) in enumerate([(torch.float32, torch.float32, "gelu", True), (torch.bfloat16, torch.float32, None, False),
                                             (torch.bfloat16, torch.bfloat16, "relu", True), (torch.float16, torch.float16, None, True)]):
        x = _randn(10 + i, M, K).to(xt)
        wq, ws = ops.quantize_rows((_randn(20 + i, N, K) / K ** 0.5).cuda())
        b = 0.1 * _randn(30 + i, N) if bias else None
        y = ops.linear_i8(x.cuda(), wq, ws, None if b is None else b.cuda(), act=act, out_dtype=yt)
        ref, z = _linear_oracle(x, wq.cpu(), ws.cpu(), b, act)
        assert y.shape == (M, N) and y.dtype == yt
        # (float) of the sum, two products, the bias' sum: 4 roundings of half a step of 2^-23 of magnitudes up to |z - b| + |b|; the
        # gelu is the framework's own (1.5e-7 of |z|, slope up to 1.13, a few roundings of its factors); one rounding to the output
        size = z.abs() + (0 if b is None else b.abs())
        tol = 4 * 2.0 ** -24 * size * (1.13 if act == "gelu" else 1) + ((1.5e-7 + 8 * 2.0 ** -24) * size if act == "gelu" else 0)
        tol = tol + torch.finfo(yt).eps / 2 * (ref.abs() + tol) + (2.0 ** -25 if yt == torch.float16 else 0) + 1e-38
        err = (y.cpu().double() - ref).abs()
        assert (err <= tol).all(), (shape, xt, yt, act, float((err - tol).max()))


@gpu
@pytest.mark.parametrize("shape", [(1, 131056, 3), (3, 131056, 2), (70, 131056, 65)])
def test_gemm_i8_sums_at_their_largest(shape):
    """-128 times -128 over the longest K: the sum is 131056 * 16384 = 2147221504 < 2^31."""
    from gmk import ops
    M, K, N = shape
    xq = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    wq[-1] = 127
    one = torch.ones(max(M, N), device="cuda")
    y = ops.matmul_i8(xq, one[:M], wq, one[:N])
    ref = torch.full((M, N), 131056.0 * 16384)
    ref[:, -1] = -131056.0 * 16256
    assert torch.equal(y.cpu(), ref.float())


@gpu
@pytest.mark.parametrize("M", [1, 3, 16, 40, 200])
def test_gemm_i8_whole_numbers(M):
    """Scales of 1 and sums below 2^24: every output is exact, whatever kernel and split the shape takes."""
    from gmk import ops
    g = torch.Generator().manual_seed(M)
    for K, N in ((16, 7), (512, 130), (1008, 1), (1024, 515)):
        xq = torch.randint(-128, 128, (M, K), generator=g).to(torch.int8)
        wq = torch.randint(-128, 128, (N, K), generator=g).to(torch.int8)
        y = ops.matmul_i8(xq.cuda(), torch.ones(M, device="cuda"), wq.cuda(), torch.ones(N, device="cuda"))
        assert torch.equal(y.cpu().double(), xq.double() @ wq.double().T)


# shapes for each of the larger kernels (64x32, 64x64, 128x128 twice, 256x256 with one and with several tiles a workgroup), ended by all
# three sizes inside a tile; the smaller ones are in SHAPES
@gpu
@pytest.mark.parametrize("shape", [(7, 208, 20000), (30, 1040, 17000), (65, 1040, 17010), (1100, 1296, 3101), (777, 1360, 5003), (1500, 1360, 5003), (4090, 2064, 4085),
                                   (8190, 144, 8190), (8190, 1040, 4099)])
def test_gemm_i8_larger_kernels(shape):
    """Whole numbers below 2^24 in fp32 are exact; bias, activation and a 16-bit output against the same in 64 bits."""
    from gmk import ops
    M, K, N = shape
    g = torch.Generator(device="cuda").manual_seed(M + N)
    xq, wq = (torch.randint(-60, 61, (n, K), generator=g, device="cuda").to(torch.int8) for n in (M, N))
    one = torch.ones(max(M, N), device="cuda")
    ref = xq.double() @ wq.double().t().contiguous()
    assert torch.equal(ops.matmul_i8(xq, one[:M].contiguous(), wq, one[:N].contiguous()).double(), ref)
    xs, ws, b = (torch.rand(n, generator=g, device="cuda") + 0.5 for n in (M, N, N))
    xs = xs / K
    for act, dtype in (("relu", torch.bfloat16), ("gelu", torch.float16), ("elu", torch.float32)):
        y = ops.matmul_i8(xq, xs, wq, ws, b, act=act, out_dtype=dtype).double()
        z = ref * xs.double()[:, None] * ws.double() + b.double()
        r = _act(act, z)
        tol = (z.abs() + 2 * b.double()) * (4 * 2.0 ** -24 * 1.13 + 1.5e-7 + 8 * 2.0 ** -24)   # as in test_linear_i8
        tol += torch.finfo(dtype).eps / 2 * (r.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert ((y - r).abs() <= tol).all(), act


def _kernels(call):
    """The template arguments behind the type, of every 8-bit product that `call` launches: "64, 32, 2, 2, 6" (columns and rows of a tile, waves
    both ways, stages)."""
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    return [e.name.split("<")[1].split(">")[0].split(", ", 1)[1] for e in prof.events() if "gemm_i8_tile_kernel<" in e.name]


# Whole lines of y (N a multiple of 64: stores past the caches in every type), whole chunks of K (a multiple of 128) and M that ends inside a
# tile, for every tile shape above 32x32: with one tile a workgroup, and with several, whose loads run over from one tile into the next.
# The kernel that each size is here for is checked by name, so that another choice of kernels cannot leave one out.
WHOLE_LINES = [("64, 32, 2, 2, 6", (30, 1024, 17024)), ("64, 32, 2, 2, 6", (24, 256, 40000)), ("64, 64, 2, 2, 4", (36, 1920, 32960)),
               ("128, 128, 4, 2, 4", (65, 1024, 17024)), ("128, 128, 4, 2, 4", (1100, 1280, 3136)), ("128, 192, 4, 2, 3", (777, 1408, 5056)),
               ("128, 192, 4, 2, 3", (528, 896, 26304)), ("128, 128, 2, 2, 2", (1500, 1408, 5056)), ("128, 128, 2, 2, 2", (263, 128, 34688)),
               ("256, 256, 4, 2, 2", (4090, 2048, 4096)), ("256, 256, 4, 2, 2", (8100, 1024, 8256)), ("256, 256, 4, 2, 2", (649, 128, 33536))]


@gpu
@pytest.mark.parametrize("kernel,shape", WHOLE_LINES)
def test_gemm_i8_whole_lines_and_chunks(kernel, shape):
    """As test_gemm_i8_larger_kernels: exact whole numbers in fp32, then scales, bias and activation in each type."""
    from gmk import ops
    M, K, N = shape
    assert N % 64 == 0 and K % 128 == 0
    g = torch.Generator(device="cuda").manual_seed(M + N)
    xq, wq = (torch.randint(-60, 61, (n, K), generator=g, device="cuda").to(torch.int8) for n in (M, N))
    one = torch.ones(max(M, N), device="cuda")
    ref = xq.double() @ wq.double().t().contiguous()
    got = []
    ran = _kernels(lambda: got.append(ops.matmul_i8(xq, one[:M].contiguous(), wq, one[:N].contiguous())))
    assert got[0].data_ptr() % 128 == 0
    assert torch.equal(got[0].double(), ref)
    xs, ws, b = (torch.rand(n, generator=g, device="cuda") + 0.5 for n in (M, N, N))
    xs = xs / K
    for act, dtype in ((None, torch.bfloat16), ("relu", torch.bfloat16), ("gelu", torch.float16), ("elu", torch.float32)):
        y = ops.matmul_i8(xq, xs, wq, ws, b, act=act, out_dtype=dtype).double()
        z = ref * xs.double()[:, None] * ws.double() + b.double()
        r = _act(act, z)
        tol = (z.abs() + 2 * b.double()) * (4 * 2.0 ** -24 * 1.13 + 1.5e-7 + 8 * 2.0 ** -24)   # as in test_linear_i8
        tol += torch.finfo(dtype).eps / 2 * (r.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert ((y - r).abs() <= tol).all(), act
    if not ran:
        pytest.skip("the results are right, but the profiler names no kernel here")
    assert ran == [kernel]


# M ends so early inside the last tile that some of its waves have no row, and a workgroup takes another tile behind one of those (more tiles
# than run at once on 256 compute units): 64x32, 64x64, 128x192, 128x128 and 256x256
@gpu
@pytest.mark.parametrize("shape", [(10, 256, 40000), (36, 1920, 32960), (528, 896, 26304), (263, 128, 34688), (649, 128, 33536), (649, 144, 33533)])
def test_gemm_i8_next_tile_has_its_own_scales(shape):
    """Sums below 2^24 and scales that are powers of two: every output is exact, and one with another tile's scales is not."""
    from gmk import ops
    M, K, N = shape
    g = torch.Generator(device="cuda").manual_seed(M + N)
    xq, wq = (torch.randint(-60, 61, (n, K), generator=g, device="cuda").to(torch.int8) for n in (M, N))
    xs, ws = (2.0 ** torch.randint(-8, 9, (n,), generator=g, device="cuda") for n in (M, N))
    ref = (xq.double() @ wq.double().t().contiguous()) * xs.double()[:, None] * ws.double()
    for _ in range(3):
        assert torch.equal(ops.matmul_i8(xq, xs, wq, ws).double(), ref)


@gpu
@pytest.mark.parametrize("dtype,M,K,N", [(torch.bfloat16, 9001, 4100, 130), (torch.float32, 4500, 4097, 300), (torch.float16, 700, 8200, 12000)])
def test_linear_i8_large_is_its_two_steps(dtype, M, K, N):
    """Sizes at which the activations pass the caches by: the same bits as quantize_rows and matmul_i8."""
    from gmk import ops
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    wq, ws = ops.quantize_rows(torch.randn(N, K, generator=g, device="cuda"))
    assert torch.equal(ops.linear_i8(x, wq, ws, act="relu"), ops.matmul_i8(*ops.quantize_rows(x), wq, ws, act="relu", out_dtype=dtype))


@gpu
@pytest.mark.parametrize("M", [1, 4, 20, 150])
def test_linear_i8_rows_are_independent_and_nan_stays_in_its_row(M):
    from gmk import ops
    K, N = 513, 77
    x = _randn(5, M, K)
    wq, ws = ops.quantize_rows(_randn(6, N, K).cuda())
    clean = ops.linear_i8(x.cuda(), wq, ws)
    x[M - 1, 100] = float("nan")
    x[M // 2, 3] = float("inf")
    y = ops.linear_i8(x.cuda(), wq, ws)
    bad = torch.zeros(M, dtype=torch.bool)
    bad[M - 1] = bad[M // 2] = True
    assert torch.isnan(y.cpu()[bad]).all()
    assert torch.equal(y.cpu()[~bad], clean.cpu()[~bad])
    # zero rows of activations and of weights give the bias
    b = _randn(7, N)
    z = ops.linear_i8(torch.zeros(M, K, device="cuda"), wq, ws, b.cuda())
    assert torch.equal(z.cpu(), b.expand(M, N))


@gpu
@pytest.mark.parametrize("act", [None, "relu", "leaky-relu", "elu", "selu", "gelu", "swish", "mish", "sigmoid"])
@pytest.mark.parametrize("M,N", [(1, 33), (3, 9000), (9, 40), (33, 2050), (300, 1100), (1100, 3101)])
def test_linear_i8_keeps_nan_behind_every_activation(M, N, act):
    from gmk import ops
    x = _randn(5, M, 100)
    x[M // 2, 7] = float("nan")
    wq, ws = ops.quantize_rows(_randn(6, N, 100).cuda())
    nan = torch.isnan(ops.linear_i8(x.cuda(), wq, ws, act=act))
    assert nan[M // 2].all() and nan.sum() == N


@gpu
@pytest.mark.parametrize("act", ["leaky-relu", "elu", "selu", "swish", "mish", "sigmoid"])
def test_linear_i8_activations(act):
    """Every activation of the fp32 layer, on the same values: linear_fwd with the identity as its weight applies it in fp32."""
    from gmk import ops
    x = _randn(8, 20, 64).cuda()
    wq, ws = ops.quantize_rows(_randn(9, 64, 64).cuda())
    z = ops.linear_i8(x, wq, ws)
    y = ops.linear_i8(x, wq, ws, act=act)
    ref = ops.linear_fwd(z, torch.eye(64, device="cuda"), torch.zeros(64, device="cuda"), act=act)
    assert torch.allclose(y, ref, rtol=1e-6, atol=1e-6)


@gpu
def test_linear_i8_writes_its_rows_only_and_reads_only_its_own():
    """Views into larger buffers: what lies before and behind x and y is neither read into a result nor written."""
    from gmk import lib, check, ops
    for M, K, N in ((1, 250, 70), (5, 250, 70), (70, 250, 135)):
        wq, ws = ops.quantize_rows(_randn(3, N, K).cuda())
        xb = torch.full((M * K + 64,), float("nan"), device="cuda")
        xb[32: 32 + M * K] = _randn(4, M * K).cuda()
        yb = torch.full((M * N + 64,), 7.0, device="cuda")
        x, y = xb[32: 32 + M * K].view(M, K), yb[32: 32 + M * N].view(M, N)
        scratch = torch.empty(int(lib().gmk_linear_i8_workspace_bytes(M, K, N)) + 16, dtype=torch.uint8, device="cuda")
        check(lib().gmk_linear_i8_fwd(x.data_ptr(), 0, wq.data_ptr(), ws.data_ptr(), None, y.data_ptr(), 0, M, K, N, 0, scratch.data_ptr(),
                                      scratch.numel(), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(y, ops.linear_i8(x.clone(), wq, ws))
        assert (yb[:32] == 7).all() and (yb[32 + M * N:] == 7).all()


@gpu
def test_linear_i8_without_rows():
    from gmk import ops
    wq, ws = ops.quantize_rows(_randn(1, 5, 40).cuda())
    assert ops.linear_i8(torch.empty(0, 40, device="cuda"), wq, ws).shape == (0, 5)
    assert ops.quantize_rows(torch.empty(0, 40, device="cuda"))[0].shape == (0, 48)


@gpu
def test_linear_i8_on_two_streams_and_in_two_graphs():
    """Calls on two streams at once, and two graphs of the same shapes replayed side by side: no scratch is shared."""
    from gmk import ops
    M, K, N = 24, 4096, 512
    xs = [_randn(40 + i, M, K).cuda() for i in range(2)]
    w = [ops.quantize_rows(_randn(50 + i, N, K).cuda()) for i in range(2)]
    ref = [ops.linear_i8(xs[i], *w[i], act="gelu") for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        out = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                out.append(ops.linear_i8(xs[i], *w[i], act="gelu"))
        torch.cuda.synchronize()
        assert all(torch.equal(out[i], ref[i]) for i in range(2))
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.linear_i8(xs[i], *w[i], act="gelu"))
        graphs.append(g)
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], ref[i]) for i in range(2))
        assert torch.equal(ops.linear_i8(xs[0], *w[0], act="gelu"), ref[0])


# ---------------------------------------------------------------- refusals (no GPU)

def test_wrappers_refuse_cpu_tensors():
    from gmk import ops
    x, q = torch.zeros(2, 16), torch.zeros(3, 16, dtype=torch.int8)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.linear_i8(x, q, torch.ones(3)), lambda: ops.matmul_i8(q, torch.ones(3), q, torch.ones(3))):
        with pytest.raises(ValueError):
            call()


def test_wrappers_refuse_sizes_beyond_32_bits(monkeypatch):
    """Rows and columns that a C int would cut (2^32 + 5 rows to 5, with the others never written), on tensors without memory."""
    from gmk import ops
    monkeypatch.setattr(ops, "_chk_first", lambda *a: 0)
    monkeypatch.setattr(ops, "_chk_rows", lambda *a: None)

    def calls(M, K, N):
        x, q, w = (torch.empty(n, c, dtype=d, device="meta") for n, c, d in ((M, K, torch.bfloat16), (M, K, torch.int8), (N, K, torch.int8)))
        return (lambda: ops.linear_i8(x, w, None)), (lambda: ops.matmul_i8(q, None, w, None))

    for M, N in (((1 << 32) + 5, 7), (7, (1 << 32) + 5), ((1 << 30) + 1, 7), (7, (1 << 30) + 1)):
        for call in calls(M, 16, N):
            with pytest.raises(ValueError, match="rows"):
                call()
    for K in ((1 << 32) + 16, (1 << 30) + 16):
        with pytest.raises(ValueError, match="columns"):
            ops.quantize_rows(torch.empty(1, K, device="meta"))


def test_c_entries_refuse_bad_arguments():
    """Every check comes before the first launch, so that it can be made without a GPU."""
    from gmk import lib
    h = lib()
    p = ctypes.c_void_p(4096)        # never read
    odd = ctypes.c_void_p(4097)
    E = dict(shape=-1, align=-2, unsupported=-3, workspace=-4, null=-5, large=-6)
    q = lambda **k: h.gmk_quantize_rows(*{**dict(x=p, t=0, q=p, s=p, M=2, K=20, ld=32, st=None), **k}.values())  # noqa: E731
    assert q(t=3) == E["unsupported"] and q(t=-1) == E["unsupported"]
    assert q(M=-1) == q(K=0) == q(ld=16) == q(ld=24) == E["shape"]
    assert q(x=None) == q(q=None) == q(s=None) == E["null"]
    assert q(x=odd) == q(q=ctypes.c_void_p(4100)) == q(s=odd) == E["align"]
    assert q(K=1 << 30, ld=(1 << 30) + 16) == q(M=1 << 40) == E["large"]
    assert q(M=0, x=None) == 0
    g = lambda **k: h.gmk_gemm_i8(*{**dict(xq=p, xs=p, wq=p, ws=p, b=None, y=p, yt=0, M=2, K=32, N=3, act=0, st=None), **k}.values())  # noqa: E731
    assert g(yt=9) == g(act=9) == g(act=-1) == E["unsupported"]
    assert g(M=-1) == g(K=0) == g(K=20) == g(N=0) == E["shape"]
    assert g(K=131072) == g(M=(1 << 31) - 1) == g(N=(1 << 30) + 1) == g(M=1, K=16, N=1 << 28) == E["large"]
    assert g(xq=None) == g(xs=None) == g(wq=None) == g(ws=None) == g(y=None) == E["null"]
    assert g(xq=ctypes.c_void_p(4104)) == g(wq=ctypes.c_void_p(4104)) == g(b=odd) == g(y=odd) == E["align"]
    assert g(M=0) == 0
    f = lambda **k: h.gmk_linear_i8_fwd(*{**dict(x=p, xt=0, wq=p, ws=p, b=None, y=p, yt=0, M=20, K=20, N=3, act=0, w=p, wb=1 << 40, st=None), **k}.values())  # noqa: E731
    assert f(xt=5) == f(yt=5) == f(act=12) == E["unsupported"]
    assert f(M=-2) == f(K=-1) == f(N=0) == E["shape"]
    assert f(K=131057) == f(M=(1 << 31) - 1) == f(N=(1 << 31) - 1) == f(M=1, N=1 << 28) == E["large"]
    assert f(x=None) == f(w=None) == f(y=None) == E["null"]
    assert f(x=odd) == f(w=ctypes.c_void_p(4104)) == E["align"]
    assert f(wb=int(h.gmk_linear_i8_workspace_bytes(20, 20, 3)) - 1) == E["workspace"]
    assert h.gmk_linear_i8_workspace_bytes(20, 20, 3) >= 20 * 32 + 80


@gpu
def test_wrappers_refuse_wrong_tensors():
    from gmk import ops
    x = torch.zeros(4, 40, device="cuda")
    wq, ws = ops.quantize_rows(torch.ones(6, 40, device="cuda"))
    b = torch.zeros(6, device="cuda")
    ops.linear_i8(x, wq, ws, b)
    for call in (lambda: ops.linear_i8(x.double(), wq, ws, b), lambda: ops.linear_i8(x[:, ::2], wq, ws, b), lambda: ops.linear_i8(x[0], wq, ws, b),
                 lambda: ops.linear_i8(x[:, :20].contiguous(), wq, ws, b), lambda: ops.linear_i8(x, wq[:, :40], ws, b), lambda: ops.linear_i8(x, wq, ws[:5], b),
                 lambda: ops.linear_i8(x, wq, ws, b[:3]), lambda: ops.linear_i8(x, wq, ws.double(), b), lambda: ops.linear_i8(x, wq.float(), ws, b),
                 lambda: ops.linear_i8(x, wq, ws, b, out_dtype=torch.float64), lambda: ops.linear_i8(x, wq, ws.cpu(), b), lambda: ops.quantize_rows(x.int()),
                 lambda: ops.quantize_rows(torch.empty(3, 0, device="cuda")), lambda: ops.matmul_i8(wq[:, :40].contiguous(), ws, wq, ws),
                 lambda: ops.matmul_i8(wq, ws[:2], wq, ws)):
        with pytest.raises(ValueError):
            call()
