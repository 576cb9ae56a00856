"""The distillation loss and its gradient against the definition in 64 bits, with tolerances that count roundings; masked and empty
rows, repeated and missing entries, the path from a teacher's 8-bit layers to the student's gradient, and the calls that are
refused."""
import ctypes
import math

import pytest
import torch

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24   # half a step of fp32


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _oracle(z, t, idx, labels, T, soft, hard):
    """(loss, gradient of the row's loss, and for both how far fp32 arithmetic may be off), all in 64 bits.

    The bounds, in units of 2^-24: an exponential exp(d / T) carries the roundings of z - max, of 1 / T and of the product(s), each
    relative to d / T, and its own: 4 |d / T| + 4.  A sum of C of them in partial sums of C / 64 terms at most: C / 64 + 24 more.
    """
    z, t = z.double(), t.double()
    n, C = z.shape
    k = t.shape[1]
    m = z.amax(1, keepdim=True)
    live = (m > -math.inf)[:, 0]
    d = torch.where(live[:, None], z - m, torch.zeros_like(z))
    there = (idx >= 0) & (idx < C)
    at = torch.where(there, idx, torch.zeros_like(idx)).long()
    tt = torch.where(there, t, torch.full_like(t, -math.inf))
    tm = tt.amax(1, keepdim=True)
    has = (tm > -math.inf)[:, 0] & live
    a = torch.where(has[:, None], (tt - tm) / T, torch.full_like(t, -math.inf))
    p = a.exp()
    p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    rel_p = torch.where(p > 0, 8 * a.abs() + k + 16, torch.zeros_like(p))

    def soft_max(T):
        e = (d / T).exp()
        S = e.sum(1, keepdim=True)
        q = e / S
        off = 4 * torch.where(q > 0, q * d.abs() / T, torch.zeros_like(q)).sum(1, keepdim=True) + 4 + C / 64 + 24
        rel_q = 4 * torch.where(q > 0, d.abs() / T, torch.zeros_like(q)) + 8 + off
        return q, S.log(), off, rel_q

    q, lnS, off, rel_q = soft_max(T)
    dj = (d / T).gather(1, at)
    part = torch.where(p > 0, p * (p.log() - dj), torch.zeros_like(p))
    kl = part.sum(1) + lnS[:, 0] * has
    e_kl = torch.where(p > 0, p * (4 * (dj.abs() + p.log().abs()) + rel_p * (p.log().abs() + dj.abs() + lnS + 1) + 8), torch.zeros_like(p)).sum(1)
    e_kl = e_kl + off[:, 0] + 4 * lnS[:, 0] + (k / 64 + 8) * part.abs().sum(1)
    w = torch.zeros(n, C, dtype=torch.float64).scatter_add(1, at, p * there)
    w_rel = torch.zeros(n, C, dtype=torch.float64).scatter_add(1, at, p * there * (rel_p + k))
    loss = soft * T * T * kl * has
    e_loss = abs(soft) * T * T * (e_kl + 4 * kl.abs()) * has
    grad = soft * T * (q - w) * has[:, None]
    e_grad = abs(soft) * T * (q * (rel_q + 4) + w_rel + 4 * w) * has[:, None]
    if labels is not None and hard:
        ok = (labels >= 0) & (labels < C) & live
        l = torch.where(ok, labels, torch.zeros_like(labels))[:, None]
        q1, lnS1, off1, rel_q1 = soft_max(1.0)
        dl = d.gather(1, l)
        loss = loss + hard * (lnS1 - dl)[:, 0] * ok
        e_loss = e_loss + abs(hard) * (off1 + 4 * lnS1 + 4 * dl.abs())[:, 0] * ok
        one = torch.zeros(n, C, dtype=torch.float64).scatter_(1, l, 1.0)
        grad = grad + hard * (q1 - one) * ok[:, None]
        e_grad = e_grad + abs(hard) * (q1 * (rel_q1 + 4) + 4 * one) * ok[:, None]
    e_loss = U * (e_loss + 4 * loss.abs()) + 1e-37
    e_grad = U * (e_grad + 2 * grad.abs()) + 1e-37
    return loss, grad, e_loss, e_grad


def _case(seed, n, C, k, dtype, tdtype=torch.float32, pads=True):
    g = torch.Generator().manual_seed(seed)
    z = (2.5 * torch.randn(n, C, generator=g)).to(dtype)
    idx = torch.stack([torch.randperm(C, generator=g)[:k] for _ in range(n)]).int()
    t = (z.float().gather(1, idx.long()) + 3 + 2 * torch.randn(n, k, generator=g)).to(tdtype)
    labels = torch.randint(0, C, (n,), generator=g)
    if pads:
        kept = torch.randint(0, k + 1, (n, 1), generator=g)
        idx = torch.where(torch.arange(k) < kept, idx, torch.tensor(-1, dtype=torch.int32))
        labels[torch.rand(n, generator=g) < 0.2] = -100
    return z, t, idx, labels


def _within(got, ref, tol, what):
    got = got.cpu()
    t = torch.finfo(got.dtype)
    tol = tol + (ref.abs() + tol) * (t.eps / 2) + (t.smallest_normal * t.eps / 2 if got.dtype == torch.float16 else 0)
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (what, float((err / tol).max()), float(err.max()))


def _all_forms(z, t, idx, labels, T, soft, hard, weight=None, scale=0.37):
    """The two calls and the one call against the oracle."""
    from gmk import ops
    n = z.shape[0]
    loss, grad, e_loss, e_grad = _oracle(z, t, idx, labels, T, soft, hard)
    dev = [None if v is None else v.cuda() for v in (z, t, idx, labels)]
    got, stats = ops.distill_fwd(*dev, T, soft, hard)
    _within(got, loss, e_loss, "loss")
    w = torch.ones(n) if weight is None else weight
    gz = ops.distill_bwd(w.cuda(), *dev, stats, T, soft, hard)
    assert gz.dtype == z.dtype
    _within(gz, grad * w.double()[:, None], e_grad * w.abs().double()[:, None] + 4 * U * (grad * w.double()[:, None]).abs(), "bwd")
    l2, g2 = ops.distill_fwd_bwd(*dev, T, soft, hard, None if weight is None else weight.cuda(), scale)
    ws = (w * scale).double()
    _within(l2, loss * w.double(), e_loss * w.abs().double() + U * loss.abs(), "fused loss")
    _within(g2, grad * ws[:, None], e_grad * ws.abs()[:, None] + 4 * U * (grad * ws[:, None]).abs(), "fused gradient")
    return got, gz, l2, g2


SHAPES = [(1, 1, 1), (2, 2, 2), (256, 10, 3), (7, 10, 10), (300, 37, 5), (5, 64, 8), (3, 127, 64), (64, 1000, 10), (9, 2049, 100), (5, 4096, 256), (33, 8191, 20), (6, 10007, 20),
          (3, 16384, 64), (2, 32768, 64), (3, 40001, 30), (2, 65536, 128), (1, 70001, 256), (2, 131073, 64), (3, 200003, 50), (520, 34000, 3), (1, 1200001, 200)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_distill(shape, dtype):
    n, C, k = shape
    z, t, idx, labels = _case(C + k, n, C, k, dtype, tdtype=TYPES[(n + k) % 3])
    _all_forms(z, t, idx, labels, 3.0, 0.7, 0.3)
    weight = _randn(n, n).abs()
    weight[n // 2] = 0
    _all_forms(z, t, idx, None, 1.0, 1.0, 0.0, weight)
    _all_forms(z, t, idx, labels, 0.5, 0.0, 1.0, weight)


@gpu
@pytest.mark.parametrize("C", [10, 1000, 20000, 150000])
def test_distill_rows_with_masks(C):
    """-inf and the lowest value at masked classes, rows that are masked altogether, teachers with nothing to say, repeated classes,
    classes that do not exist: every row against the definition, none spoils its neighbour."""
    k, low = 6, torch.finfo(torch.float32).min
    z, t, idx, labels = _case(C, 12, C, k, torch.float32, pads=False)
    live = idx[:, 0].clone()
    z[0, :] = -math.inf                      # nothing is left of the student's row
    z[1, :] = low                            # all at the lowest: an even distribution
    keep = z[2].clone()
    z[2, :] = -math.inf
    z[2, idx[2].long()] = keep[idx[2].long()]
    labels[2] = idx[2, 1]
    keep = z[3].clone()
    z[3, :] = low
    z[3, idx[3].long()] = keep[idx[3].long()]
    labels[3] = idx[3, 0]
    idx[4] = -1                              # no entry
    t[5] = -math.inf                         # entries without weight
    t[6, 1:] = -math.inf                     # one entry with all of it
    idx[7] = live[7]                         # one class, listed k times
    idx[8, ::2] = live[8]
    idx[9] = torch.tensor([C, C + 5, -7, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32)
    t[10] = low
    labels[11] = C
    for T, soft, hard in ((2.0, 1.0, 0.5), (0.25, 1.0, 0.0), (1.0, 0.5, 0.5)):
        got, gz, l2, g2 = _all_forms(z, t, idx, labels, T, soft, hard)
        assert got[0] == 0 and l2[0] == 0 and not gz[0].any() and not g2[0].any()


@gpu
@pytest.mark.parametrize("C", [10, 3001, 100000])
def test_distill_padding_rows_and_nan(C):
    """Rows of weight 0 hold NaN and give zeros; a NaN or an infinity in a live row stays in it."""
    from gmk import ops
    z, t, idx, labels = (v.cuda() for v in _case(3, 8, C, 4, torch.float32, pads=False))
    weight = torch.ones(8, device="cuda")
    clean_l, clean_g = ops.distill_fwd_bwd(z, t, idx, labels, 2.0, 1.0, 0.5, weight)
    z[2], t[2], weight[2] = math.nan, math.nan, 0
    z[7, C // 2:], weight[7] = math.inf, 0
    z[4, C // 3] = math.nan
    z[5, C // 3] = math.inf
    l, g = ops.distill_fwd_bwd(z, t, idx, labels, 2.0, 1.0, 0.5, weight)
    assert not l[[2, 7]].any() and not g[[2, 7]].any()
    assert torch.isnan(l[[4, 5]]).all() and torch.isnan(g[[4, 5]]).all()
    others = [0, 1, 3, 6]
    assert torch.equal(l[others], clean_l[others]) and torch.equal(g[others], clean_g[others])
    loss, stats = ops.distill_fwd(z, t, idx, labels, 2.0, 1.0, 0.5)
    gb = ops.distill_bwd(weight, z, t, idx, labels, stats, 2.0, 1.0, 0.5)
    assert not gb[[2, 7]].any() and torch.isnan(gb[[4, 5]]).all()
    assert torch.isfinite(gb[others]).all() and torch.isfinite(loss[others]).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [10, 3001, 40000, 100000])
def test_distill_rows_with_nothing_to_learn(C, dtype):
    """No entry and no label: loss 0 and gradient 0 at a weight of 1, whatever the logits hold (an ignored sample of a batch); a row with one
    of the two parts still shows them."""
    from gmk import ops
    from models.classifiers import distillation_loss
    z, t, idx, labels = (v.cuda() for v in _case(C + 1, 9, C, 4, dtype, pads=False))
    clean = ops.distill_fwd_bwd(z, t, idx, labels, 2.0, 1.0, 0.5)
    idx[[1, 3, 5, 7]], labels[[1, 3, 5, 7]] = -1, -100
    z[1] = math.nan
    z[3, C // 2] = math.nan
    z[5, C - 1] = math.inf
    z[7] = math.inf
    idx[4], z[4, C // 3] = -1, math.nan         # a label is left
    labels[6], z[6, C // 3] = -100, math.nan    # entries are left
    none, bad, others = [1, 3, 5, 7], [4, 6], [0, 2, 8]
    one = torch.ones(9, device="cuda")
    for weight in (None, one):
        l, g = ops.distill_fwd_bwd(z, t, idx, labels, 2.0, 1.0, 0.5, weight)
        assert not l[none].any() and not g[none].any()
        assert torch.isnan(l[bad]).all() and torch.isnan(g[bad]).all()
        assert torch.equal(l[others], clean[0][others]) and torch.equal(g[others], clean[1][others])
    l, stats = ops.distill_fwd(z, t, idx, labels, 2.0, 1.0, 0.5)
    g = ops.distill_bwd(one, z, t, idx, labels, stats, 2.0, 1.0, 0.5)
    assert not l[none].any() and not g[none].any() and torch.isnan(g[bad]).all() and torch.isfinite(g[others]).all()
    # parts that are switched off by their weight; through autograd, whose mean the ignored samples leave as it is
    for soft, hard, row in ((0.0, 0.5, 6), (1.0, 0.0, 4)):
        l, g = ops.distill_fwd_bwd(z, t, idx, labels, 2.0, soft, hard)
        assert not l[none + [row]].any() and not g[none + [row]].any()
    live = others + none
    a = z[live].clone().requires_grad_(True)
    distillation_loss(a, t[live], idx[live], labels[live], 2.0, 1.0, 0.5).mean().backward()
    assert torch.isfinite(a.grad).all() and a.grad[:3].any() and not a.grad[3:].any()


@gpu
def test_distill_gradient_against_differences():
    """Central differences of the loss itself.  Step h = 2^-6: the loss' third derivative is at most soft / T + hard <= 1.25 and its
    error about 1e-6, so that the quotient is off by h^2 / 6 * 1.25 + 1e-6 / h < 2e-4."""
    from gmk import ops
    C, k, h = 12, 4, 2.0 ** -6
    z, t, idx, labels = _case(1, 1, C, k, torch.float32, pads=False)
    idx[0, 3] = idx[0, 0]
    for T, soft, hard in ((2.0, 1.0, 0.5), (1.0, 0.5, 0.0), (4.0, 0.0, 1.0)):
        step = h * torch.eye(C)
        zz = torch.cat([z + step, z - step])
        many = [v.expand(2 * C, *v.shape[1:]).contiguous().cuda() for v in (t, idx, labels)]
        loss, _ = ops.distill_fwd(zz.cuda(), *many, T, soft, hard)
        slope = (loss[:C] - loss[C:]) / (2 * h)
        _, g = ops.distill_fwd_bwd(z.cuda(), t.cuda(), idx.cuda(), labels.cuda(), T, soft, hard)
        assert (slope - g[0]).abs().max() < 2e-4


@gpu
def test_distill_writes_its_rows_only():
    """Contiguous views at odd elements: neighbours in the buffers keep their values."""
    from gmk import lib, check, ops
    for dtype, ztype in zip(TYPES, (0, 1, 2)):
        for n, C in ((5, 13), (3, 4097), (2, 90001)):
            z, t, idx, _ = _case(n, n, C, 3, dtype)
            t, idx = t.cuda(), idx.cuda()
            zb = torch.full((n * C + 50,), math.nan, dtype=dtype, device="cuda")
            gb = torch.full((n * C + 50,), 7.0, dtype=dtype, device="cuda")
            zv, gv = zb[3: 3 + n * C].view(n, C), gb[5: 5 + n * C].view(n, C)
            zv.copy_(z)
            loss = torch.empty(n, device="cuda")
            ws = torch.empty(int(lib().gmk_distill_workspace_bytes(n, C)) + 16, dtype=torch.uint8, device="cuda")
            check(lib().gmk_distill_fwd_bwd(zv.data_ptr(), ztype, t.data_ptr(), 0, idx.data_ptr(), None, None, loss.data_ptr(), gv.data_ptr(),
                                            n, C, 3, 2.0, 1.0, 0.0, 1.0, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
            rl, rg = ops.distill_fwd_bwd(z.cuda(), t, idx, None, 2.0)
            assert torch.equal(loss, rl) and torch.equal(gv, rg)
            assert (gb[:5] == 7).all() and (gb[5 + n * C:] == 7).all()


@gpu
def test_distill_streams_graphs_and_empty():
    from gmk import ops
    for n, C in ((64, 10), (3, 90001)):
        cases = [[v.cuda() for v in _case(i, n, C, 5, torch.float32)] for i in range(2)]
        ref = [ops.distill_fwd_bwd(*c, 2.0, 1.0, 0.5) for c in cases]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        graphs, outs = [], []
        for c in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(ops.distill_fwd_bwd(*c, 2.0, 1.0, 0.5))
            graphs.append(g)
        for _ in range(3):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            eager = ops.distill_fwd_bwd(*cases[1], 2.0, 1.0, 0.5)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for o, r in zip(outs, ref) for a, b in zip(o, r))
            assert torch.equal(eager[1], ref[1][1])
    z = torch.empty(0, 7, device="cuda")
    t, idx = torch.empty(0, 2, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda")
    loss, stats = ops.distill_fwd(z, t, idx)
    assert loss.shape == (0,) and ops.distill_bwd(loss, z, t, idx, None, stats).shape == (0, 7)
    assert ops.distill_fwd_bwd(z, t, idx)[1].shape == (0, 7)


# ---------------------------------------------------------------- the operators together

@gpu
def test_teacher_to_student_run():
    """The teacher's two fully connected layers in 8 bits, its kept logits, the student's loss and gradient: each step against the
    64-bit definition of all the steps before it, from the step's own input."""
    from gmk import ops
    B, F, L, C, k = 96, 4096, 256, 1000, 10
    x = _randn(1, B, F)
    w1, w2 = _randn(2, L, F) / 64, _randn(3, C, L) / 4
    b1, b2 = 0.1 * _randn(4, L), 0.1 * _randn(5, C)
    q1, q2 = ops.quantize_rows(w1.cuda()), ops.quantize_rows(w2.cuda())
    hid = ops.linear_i8(x.cuda(), *q1, b1.cuda(), act="gelu")
    logits = ops.linear_i8(hid, *q2, b2.cuda())
    value, index = ops.topk_rows(logits, k)

    def exact(v, w, b):
        s = (v.double().abs().amax(1) / 127).float().double()[:, None]
        sw = (w.double().abs().amax(1) / 127).float().double()[:, None]
        return ((v.double() / s).round() * s) @ ((w.double() / sw).round() * sw).T + b.double()

    h64 = exact(x, w1, b1)
    h64 = h64 * 0.5 * torch.erfc(-h64 / 2 ** 0.5)
    assert (hid.cpu().double() - h64).abs().max() < 2e-6 * h64.abs().max()
    l64 = exact(hid.cpu(), w2, b2)
    assert (logits.cpu().double() - l64).abs().max() < 2e-6 * l64.abs().max()
    # 8 bits keep the layer: rounding errors of a step / sqrt(12) on both sides, over the whole sum
    full = x.double() @ w1.double().T + b1.double()
    full = full * 0.5 * torch.erfc(-full / 2 ** 0.5) @ w2.double().T + b2.double()
    assert (l64 - full).norm() < 0.05 * full.norm()
    ri = torch.sort(logits.cpu().double(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(index.cpu().long(), ri)
    student = _randn(6, B, C)
    labels = torch.randint(0, C, (B,), generator=torch.Generator().manual_seed(7))
    _all_forms(student, value.cpu(), index.cpu(), labels, 2.0, 0.9, 0.1)


@gpu
def test_operators_in_a_launch_plan():
    """Recorded once and replayed from C on other inputs by pointer substitution: the same bits as direct calls."""
    import ctypes as C
    from gmk import lib, check, ops
    h = lib()
    B, F, classes, k = 40, 300, 50, 6
    w = ops.quantize_rows(_randn(1, classes, F).cuda())
    labels = torch.randint(0, classes, (B,), generator=torch.Generator().manual_seed(2)).cuda()
    student = [_randn(10 + i, B, classes).cuda() for i in range(3)]
    x = [_randn(20 + i, B, F).cuda() for i in range(3)]

    def step(x, student):
        value, index = ops.topk_rows(ops.linear_i8(x, *w), k)
        loss, stats = ops.distill_fwd(student, value, index, labels, 2.0, 0.5, 0.5)
        q, s = ops.quantize_rows(x)
        return [value, index, loss, stats, ops.distill_bwd(loss, student, value, index, labels, stats, 2.0, 0.5, 0.5), q, s, ops.matmul_i8(q, s, *w),
                *ops.distill_fwd_bwd(student, value, index, labels, 2.0, 0.5, 0.5)]

    want = [[t.clone() for t in step(x[i], student[i])] for i in range(3)]
    plan = C.c_void_p()
    keep = ops._rec_keep = []
    check(h.gmk_plan_begin(C.byref(plan)))
    try:
        out = step(x[0], student[0])
    finally:
        check(h.gmk_plan_end())
        ops._rec_keep = None
    assert h.gmk_plan_calls(plan) == 7
    src = (C.c_void_p * 2)(x[0].data_ptr(), student[0].data_ptr())
    nb = (C.c_size_t * 2)(x[0].numel() * 4, student[0].numel() * 4)
    for i in (1, 2, 0):
        dst = (C.c_void_p * 2)(x[i].data_ptr(), student[i].data_ptr())
        check(h.gmk_train_step_enqueue(plan, 0, h.gmk_plan_segments(plan), 2, src, dst, nb))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    h.gmk_plan_destroy(plan)
    assert len(keep) > 7


# ---------------------------------------------------------------- refusals (no GPU)

def test_distill_c_entries_refuse_bad_arguments():
    from gmk import lib
    h = lib()
    p, odd, nan = ctypes.c_void_p(4096), ctypes.c_void_p(4097), float("nan")
    base = dict(z=p, zt=0, t=p, tt=0, idx=p, lab=None, n=2, C=50, k=4, T=1.0, s=1.0, h=0.5)

    def fwd(**c):
        c = {**base, "loss": p, "st": p, "w": p, "wb": 1 << 40, **c}
        return h.gmk_distill_fwd(c["z"], c["zt"], c["t"], c["tt"], c["idx"], c["lab"], c["loss"], c["st"], c["n"], c["C"], c["k"], c["T"], c["s"], c["h"], c["w"], c["wb"], None)

    def bwd(**c):
        c = {**base, "g": p, "st": p, "dz": ctypes.c_void_p(1 << 20), **c}
        return h.gmk_distill_bwd(c["g"], c["z"], c["zt"], c["t"], c["tt"], c["idx"], c["lab"], c["st"], c["dz"], c["n"], c["C"], c["k"], c["T"], c["s"], c["h"], None)

    def both(**c):
        c = {**base, "wt": None, "loss": p, "dz": ctypes.c_void_p(1 << 20), "sc": 1.0, "w": p, "wb": 1 << 40, **c}
        return h.gmk_distill_fwd_bwd(c["z"], c["zt"], c["t"], c["tt"], c["idx"], c["lab"], c["wt"], c["loss"], c["dz"], c["n"], c["C"], c["k"], c["T"], c["s"], c["h"], c["sc"], c["w"], c["wb"], None)

    for f in (fwd, bwd, both):
        assert f(zt=3) == f(tt=-1) == f(T=0.0) == f(T=1e-20) == f(T=1e20) == f(T=-1.0) == f(T=nan) == f(T=float("inf")) == f(s=nan) == f(h=float("inf")) == -3
        assert f(n=-1) == f(C=0) == f(k=0) == -1
        assert f(k=257) == f(C=1 << 31) == -6
        assert f(z=None) == f(t=None) == f(idx=None) == -5
        assert f(z=odd) == f(t=odd) == f(idx=odd) == f(lab=ctypes.c_void_p(4100)) == -2
        assert f(n=0, z=None) == 0
    assert fwd(loss=None) == fwd(st=None) == bwd(g=None) == bwd(st=None) == bwd(dz=None) == both(loss=None) == both(dz=None) == -5
    other = ctypes.c_void_p(8192)
    assert bwd(z=other, dz=other) == both(z=other, dz=other) == -3
    assert both(wt=odd) == both(dz=odd) == both(loss=odd) == bwd(g=odd) == fwd(st=odd) == -2
    need = int(h.gmk_distill_workspace_bytes(2, 1 << 20))
    assert need == 0 or fwd(C=1 << 20, wb=need - 1) == both(C=1 << 20, wb=need - 1) == -4


def test_distill_wrappers_refuse_cpu_tensors():
    from gmk import ops
    z, t, i = torch.zeros(2, 5), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: ops.distill_fwd(z, t, i), lambda: ops.distill_fwd_bwd(z, t, i), lambda: ops.distill_bwd(torch.ones(2), z, t, i, None, torch.ones(2, 3))):
        with pytest.raises(ValueError):
            call()


@gpu
def test_operators_refuse_another_device(monkeypatch):
    """Tensors that are not on the current device, whose stream the launch would go to."""
    from gmk import ops
    x = torch.randn(4, 32, device="cuda")
    q, s = ops.quantize_rows(x)
    v, i = ops.topk_rows(x, 3)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.linear_i8(x, q, s), lambda: ops.matmul_i8(q, s, q, s), lambda: ops.topk_rows(x, 3), lambda: ops.distill_fwd(x, v, i),
                 lambda: ops.distill_fwd_bwd(x, v, i)):
        with pytest.raises(ValueError):
            call()


@gpu
def test_distill_refuses_wrong_tensors():
    from gmk import ops
    z, t, i = torch.zeros(2, 5, device="cuda"), torch.zeros(2, 3, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    l, w = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.ones(2, device="cuda")
    _, st = ops.distill_fwd(z, t, i, l, 1.0, 1.0, 1.0)
    for call in (lambda: ops.distill_fwd(z.double(), t, i), lambda: ops.distill_fwd(z.t(), t, i), lambda: ops.distill_fwd(z, t[:1], i), lambda: ops.distill_fwd(z, t, i.long()),
                 lambda: ops.distill_fwd(z, t, i[:, :2].contiguous()), lambda: ops.distill_fwd(z, t, i, l.int(), hard=1.0), lambda: ops.distill_fwd(z, t, i, l[:1], hard=1.0),
                 lambda: ops.distill_fwd(z, t, i, None, hard=0.5), lambda: ops.distill_fwd(z, t, i, T=0.0), lambda: ops.distill_fwd(z, t, i, T=math.nan),
                 lambda: ops.distill_fwd(z, t, i.cpu()), lambda: ops.distill_bwd(w[:1], z, t, i, l, st), lambda: ops.distill_bwd(w, z, t, i, l, st[:, :2]),
                 lambda: ops.distill_fwd_bwd(z, t, i, weight=w.double()), lambda: ops.distill_fwd_bwd(z, t, i, soft=math.inf)):
        with pytest.raises(ValueError):
            call()
