"""A classifier from another one: the 8-bit fully connected layers of Classifier, distillation_loss under autograd, train_classifier with
a teacher, and its command-line flags."""
import math
import os
import types

import pytest
import torch

from test_linear_i8 import _linear_oracle

gpu = pytest.mark.gpu


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _classifier(seed=0, latent=64, act="gelu", **more):
    from models.classifiers import Classifier
    from utils import get_activation_function
    torch.manual_seed(seed)
    args = types.SimpleNamespace(debug=False, latent_size=latent, dropout=0.0, act_fn=get_activation_function(act), lr=1e-3, wd=0.0, epochs=1, **more)
    return Classifier(args=args), args


@gpu
@pytest.mark.parametrize("batch", [1, 50, 256])
def test_int8_classifier_layers(monkeypatch, batch):
    """Both layers of the 8-bit forward against 64 bits, from their own inputs; the folded weights are quantised once and again after an
    update; switching back gives the fp32 answers bit for bit."""
    from gmk import ops
    m, _ = _classifier()
    m = m.cuda().eval()
    x = torch.rand(batch, 3, 32, 32, generator=torch.Generator().manual_seed(batch)).cuda()
    plain = m(x)
    seen, quantised = [], []
    real, realq = ops.linear_i8, ops.quantize_rows
    monkeypatch.setattr(ops, "linear_i8", lambda x, wq, ws, b, act=None: seen.append((x, wq, ws, b, act, real(x, wq, ws, b, act=act))) or seen[-1][-1])
    monkeypatch.setattr(ops, "quantize_rows", lambda w: quantised.append(w) or realq(w))
    m.int8_fc = True
    y = m(x)
    assert len(seen) == 2 and len(quantised) == 2 and y is seen[1][-1] and m.latent_vector is seen[0][-1]
    for xi, wq, ws, b, act, out in seen:
        ref, z = _linear_oracle(xi.cpu(), wq.cpu(), ws.cpu(), b.cpu(), "gelu" if act else None)
        tol = (4 * 1.13 + 8) * 2.0 ** -24 * (z.abs() + b.abs().cpu()) + 1.5e-7 * z.abs() + 1e-37   # as in test_linear_i8
        assert ((out.cpu().double() - ref).abs() <= tol).all()
    # rows of x and of w lose at most half a step each: |error of the sum| <= sum |x| sw / 2 + |w| sx / 2 + sx sw / 4
    xi, wq, ws, b, _, out = seen[1]
    w = m.fc_out.weight.detach().double().cpu()
    sx = xi.cpu().double().abs().amax(1, keepdim=True) / 127
    sw = ws.cpu().double()
    full = xi.cpu().double() @ w.T + b.cpu().double()
    bound = xi.cpu().double().abs().sum(1, keepdim=True) * sw / 2 + sx / 2 * w.abs().sum(1) + sx * sw / 4 * w.shape[1]
    assert ((out.cpu().double() - full).abs() <= bound * 1.001 + 1e-5).all()
    m(x)
    assert len(quantised) == 2
    with torch.no_grad():
        m.fc_out.weight.mul_(2.0)
    m(x)
    assert len(quantised) == 4
    with torch.no_grad():
        m.fc_out.weight.mul_(0.5)
    m.int8_fc = False
    assert torch.equal(m(x), plain)


@gpu
def test_int8_layers_follow_replaced_weights():
    """A weight whose storage is exchanged twice between two calls, the second time for memory that the first one left: the answers are
    those of a classifier that never saw the others."""
    m, _ = _classifier()
    m = m.cuda().eval()
    m.int8_fc = True
    x = torch.rand(8, 3, 32, 32, generator=torch.Generator().manual_seed(5)).cuda()
    m.fc.weight.data = _randn(1, *m.fc.weight.shape).cuda() / 64
    m(x)
    for seed in (2, 3):
        m.fc.weight.data = _randn(seed, *m.fc.weight.shape).cuda() / 64
    fresh, _ = _classifier()
    fresh = fresh.cuda().eval()
    fresh.load_state_dict(m.state_dict())
    fresh.int8_fc = True
    assert torch.equal(m(x), fresh(x))


@gpu
@pytest.mark.parametrize("int8", [False, True])
def test_classifier_in_a_graph(int8):
    """The eval forward captured before it ever ran: an eager call ahead of the first replay has weights of its own, and replays follow the
    weights as they are updated, with eager work between them."""
    def fresh(of):
        other, _ = _classifier()
        other = other.cuda().eval()
        other.load_state_dict(of.state_dict())
        other.int8_fc = int8
        return other

    m, _ = _classifier(3)
    m = m.cuda().eval()
    m.int8_fc = int8
    static, x = (torch.rand(16, 3, 32, 32, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2))
    fresh(m)(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        y = m(static)
    assert torch.equal(m(x), fresh(m)(x))
    for i in range(3):
        with torch.no_grad():
            m.fc.weight.mul_(1.25)
            m.fc_out.weight.add_(0.125)
            m.bn1.running_mean.add_(0.25)
            static.copy_(torch.rand(16, 3, 32, 32, generator=torch.Generator().manual_seed(10 + i)))
        junk = [torch.full((1 << 20,), 1e30, device="cuda") for _ in range(8)]   # into whatever the eager calls have let go of
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fresh(m)(static)) and torch.equal(m(x), fresh(m)(x))
        del junk


def test_folded_weights_go_with_training_and_moving():
    """Updates that no version counter shows (here through numpy's view of the memory) between two eval phases, and a move: the eval forward
    folds again, and nothing holds the old tensors."""
    m, _ = _classifier()
    m.eval()
    before = m._folded()[m.fc][0].clone()
    assert m._folded()[m.fc][0] is m._folded()[m.fc][0]
    m.train()
    m.fc.weight.detach().numpy()[:] *= 2
    m.eval()
    assert torch.equal(m._folded()[m.fc][0], 2 * before)
    m.eval()
    assert "_gmk_fold" in m.__dict__   # a call of eval() alone costs no fold
    m.to(torch.float64)
    assert "_gmk_fold" not in m.__dict__


@gpu
@pytest.mark.parametrize("int8", [False, True])
def test_classifier_after_training_with_the_fused_optimizer(int8):
    """FusedAdamW writes the parameters on raw pointers; the backward pass is made up, so that no forward touches the version counters either."""
    from gmk.optim import FusedAdamW
    m, _ = _classifier()
    m = m.cuda()
    m.int8_fc = int8
    x = torch.rand(8, 3, 32, 32, generator=torch.Generator().manual_seed(5)).cuda()
    optim = FusedAdamW(m.parameters(), lr=0.05, weight_decay=0.0)
    first = m.eval()(x).clone()
    for turn in range(2):
        m.train()
        optim.zero_grad()
        optim.flat_grad.copy_(torch.randn(optim.flat_grad.shape, generator=torch.Generator().manual_seed(turn)))
        optim.step()
        y = m.eval()(x)
        fresh, _ = _classifier()
        fresh.load_state_dict(m.state_dict())
        fresh = fresh.cuda().eval()
        fresh.int8_fc = int8
        assert torch.equal(y, fresh(x)) and not torch.equal(y, first)


@gpu
@pytest.mark.parametrize("int8", [False, True])
def test_classifier_on_two_streams(monkeypatch, int8):
    """The first forward on a stream that is held up for some milliseconds, the next on another one: it does not use what the first has only
    queued.  Each stream folds once for all its calls, and again after an update."""
    from models.classifiers import Classifier
    m, _ = _classifier(3)
    m = m.cuda().eval()
    m.int8_fc = int8
    xs = [torch.rand(16, 3, 32, 32, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    other, _ = _classifier()
    other = other.cuda().eval()
    other.load_state_dict(m.state_dict())
    other.int8_fc = int8
    want = [other(x).clone() for x in xs]
    folds = []
    real = Classifier._fold
    monkeypatch.setattr(Classifier, "_fold", lambda self: folds.append(1) or real(self))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            torch.cuda._sleep(20_000_000)
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(m(x))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert len(folds) == 2
    with torch.no_grad():
        m.fc.bias.add_(0.0)
    torch.cuda.synchronize()
    for s, x, w in zip(streams, xs, want):
        with torch.cuda.stream(s):
            assert torch.equal(m(x), w)
    assert len(folds) == 4


@gpu
@pytest.mark.parametrize("warm", [False, True])
@pytest.mark.parametrize("int8", [False, True])
def test_classifier_in_a_launch_plan(int8, warm):
    """A recorded eval forward owns the folded weights that it names: replays answer with those of the recording, whatever became of the
    classifier's own since."""
    from gmk.plan import StepPlan
    m, _ = _classifier(3)
    m = m.cuda().eval()
    m.int8_fc = int8
    xs = [torch.rand(16, 3, 32, 32, generator=torch.Generator().manual_seed(i)).cuda() for i in range(3)]
    other, _ = _classifier()
    other = other.cuda().eval()
    other.load_state_dict(m.state_dict())
    other.int8_fc = int8
    want = [other(x).clone() for x in xs]
    if warm:
        m(xs[0])
    with torch.no_grad(), StepPlan() as plan:
        y = m(xs[0])
    plan.set_inputs(xs[0])
    assert torch.equal(y, want[0])
    with torch.no_grad():
        for name, p in m.named_parameters():
            if not name.startswith("fc_out"):   # whose weight is the parameter itself, and part of no fold
                p.mul_(3.0)
    m.bn1.running_mean.add_(1.0)
    m(xs[0])
    torch.cuda.synchronize()
    junk = [torch.full((n,), 1e30, device="cuda") for n in (10, 64, 128, 256, 640, 4800, 204800, 262144, 294912) for _ in range(4)]
    for i in (1, 2, 0):
        plan.enqueue(0, plan.nseg, xs[i])
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
    del junk
    plan.close()


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_output_layer_of_another_type_is_not_cast(dtype):
    """fc_out has no BatchNorm to be folded with: its tensors reach the ops as they are, which refuse another type than fp32."""
    m, _ = _classifier()
    m.fc_out.to(dtype)
    w, b = m.eval()._folded()[m.fc_out]
    assert w.dtype == b.dtype == dtype and w.data_ptr() == m.fc_out.weight.data_ptr()


@gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_output_layer_of_another_type_is_refused(dtype, int8):
    m, _ = _classifier()
    m = m.cuda().eval()
    m.fc_out.to(dtype)
    m.int8_fc = int8
    with pytest.raises(ValueError):
        m(torch.rand(4, 3, 32, 32).cuda())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_loss_gradient(dtype):
    """The gradient through autograd, with different weights of the samples, against automatic differentiation in 64 bits."""
    from models.classifiers import distillation_loss
    n, C, k, T, soft, hard = 40, 30, 5, 3.0, 0.7, 0.3
    z, w = _randn(1, n, C).to(dtype), _randn(2, n)
    t, idx = (3 * _randn(3, n, C)).topk(k, dim=1)
    idx = idx.int()
    idx[::4, 2:] = -1
    labels = torch.randint(0, C, (n,), generator=torch.Generator().manual_seed(4))
    labels[::5] = -100
    a = z.cuda().requires_grad_(True)
    loss = distillation_loss(a, t.cuda(), idx.cuda(), labels.cuda(), T, soft, hard)
    (loss * w.cuda()).sum().backward()
    x = z.double().requires_grad_(True)
    keep = idx >= 0
    at = idx.long().clamp(min=0)
    p = torch.log_softmax((t.double() / T).masked_fill(~keep, -math.inf), 1)
    q = torch.log_softmax(x / T, 1).gather(1, at)
    ref = soft * T * T * (p.exp() * (p - q).masked_fill(~keep, 0)).nan_to_num(0).sum(1)
    ref = ref + hard * torch.nn.functional.cross_entropy(x, labels, reduction="none", ignore_index=-100)
    (ref * w.double()).sum().backward()
    eps = torch.finfo(dtype).eps / 2
    assert loss.dtype == torch.float32 and a.grad.dtype == dtype
    # loss: sums of C terms of |d / T| up to 4: about 60 roundings of 2^-24 of values up to 10; gradient the same, and its output rounding
    assert (loss.detach().cpu().double() - ref.detach()).abs().max() < 600 * 2.0 ** -24
    assert ((a.grad.cpu().double() - x.grad).abs() <= eps * x.grad.abs() + 100 * 2.0 ** -24 * w.double().abs()[:, None] * (1 + eps)).all()
    # without labels; a strided view of the logits; no gradient asked
    b = z.cuda()
    plain = distillation_loss(b, t.cuda(), idx.cuda(), None, T, soft, hard)
    wide = torch.empty(n, 2 * C, dtype=dtype, device="cuda")
    wide[:, ::2] = b
    assert torch.equal(distillation_loss(wide[:, ::2], t.cuda(), idx.cuda(), None, T, soft), plain) and not plain.requires_grad


@gpu
def test_distillation_step_in_a_graph():
    """Loss and gradient captured and replayed on new logits, with eager work of other leaves between the replays."""
    from models.classifiers import distillation_loss
    n, C, k = 64, 10, 3
    t, idx = (v.cuda() for v in _randn(1, n, C).topk(k, dim=1))
    idx = idx.int()
    labels = torch.randint(0, C, (n,), generator=torch.Generator().manual_seed(2)).cuda()
    ones = torch.full((n,), 1.0 / n, device="cuda")

    def eager(z):
        z = z.clone().requires_grad_(True)
        loss = distillation_loss(z, t, idx, labels)
        return loss.detach(), torch.autograd.grad(loss, z, ones)[0]

    static = torch.zeros(n, C, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(distillation_loss(static, t, idx, labels), static, ones)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = distillation_loss(static, t, idx, labels)
        grad = torch.autograd.grad(loss, static, ones)[0]
    for i in range(3):
        z = _randn(10 + i, n, C).cuda()
        with torch.no_grad():
            static.copy_(z)
        g.replay()
        torch.cuda.synchronize()
        want = eager(z)
        assert torch.equal(loss.detach(), want[0]) and torch.equal(grad, want[1])


@gpu
@pytest.mark.parametrize("int8", [False, True])
def test_train_classifier_with_a_teacher(tmp_path, monkeypatch, int8):
    """One epoch of two batches from a teacher: it runs, the student moves, the teacher does not, and the first step's loss is the
    definition's."""
    from models import classifiers
    monkeypatch.chdir(tmp_path)
    os.makedirs("checkpoints")
    teacher, _ = _classifier(1)
    teacher.int8_fc = int8
    student, args = _classifier(2, distill_topk=4, distill_t=2.0, distill_soft=0.8, distill_hard=0.2)
    student, teacher = student.cuda(), teacher.cuda()
    before = {k: v.clone() for k, v in teacher.state_dict().items()}
    first = {k: v.clone() for k, v in student.state_dict().items()}
    g = torch.Generator().manual_seed(3)
    data = [(torch.rand(16, 3, 32, 32, generator=g), torch.randint(0, 10, (16,), generator=g)) for _ in range(2)]
    losses = []
    real = classifiers.distillation_loss
    monkeypatch.setattr(classifiers, "distillation_loss", lambda z, v, i, l, **k: losses.append((z.detach().clone(), v, i, l, k, real(z, v, i, l, **k))) or losses[-1][-1])
    out = classifiers.train_classifier(args, student, data, data, torch.device("cuda"), teacher=teacher)
    assert out is student and len(losses) == 2
    z, v, i, l, kw, loss = losses[0]
    assert v.shape == (16, 4) and i.dtype == torch.int32 and kw == dict(T=2.0, soft=0.8, hard=0.2)
    with torch.no_grad():
        logits = teacher.eval()(data[0][0].cuda())
    assert torch.equal(i.long(), torch.sort(logits.double(), dim=1, descending=True, stable=True)[1][:, :4])
    z, v = z.double().cpu(), v.double().cpu()
    p = torch.log_softmax(v / 2, 1)
    kl = (p.exp() * (p - torch.log_softmax(z / 2, 1).gather(1, i.long().cpu()))).sum(1)
    ref = 0.8 * 4 * kl + 0.2 * torch.nn.functional.cross_entropy(z, l.cpu(), reduction="none")
    assert (loss.detach().cpu().double() - ref).abs().max() < 200 * 2.0 ** -24 * (1 + z.abs().max())
    assert all(torch.equal(v, before[k]) for k, v in teacher.state_dict().items())
    assert any(not torch.equal(v, first[k]) for k, v in student.state_dict().items())
    assert os.path.isfile("checkpoints/cifar_classifier_64.pth")
    again = torch.load("checkpoints/cifar_classifier_64.pth", weights_only=False)
    assert not again.int8_fc and "_gmk_fold" not in again.__dict__


@pytest.mark.parametrize("shared", ["itself", "inside", "a layer"])
def test_train_classifier_refuses_a_teacher_that_it_would_train(shared):
    from models.classifiers import train_classifier
    student, args = _classifier(2)
    teacher, _ = _classifier(1)
    if shared == "a layer":
        teacher.conv1 = student.conv1
    teacher = {"itself": student, "inside": torch.nn.Sequential(student), "a layer": teacher}[shared]
    with pytest.raises(ValueError, match="shares"):
        train_classifier(args, student, [], [], torch.device("cpu"), teacher=teacher)


def test_train_classifier_takes_a_teacher_of_the_same_activation_object(monkeypatch, tmp_path):
    """Two classifiers of the same arguments share the activation's module, which has no parameters."""
    from models import classifiers
    monkeypatch.chdir(tmp_path)
    os.makedirs("checkpoints")
    student, args = _classifier(2)
    args.epochs = 0
    teacher = classifiers.Classifier(args=args)
    assert teacher.act is student.act
    monkeypatch.setattr(torch.optim.lr_scheduler, "CosineAnnealingLR", lambda **k: None)
    assert classifiers.train_classifier(args, student, [], [], torch.device("cpu"), teacher=teacher) is student


def test_flags():
    from arguments import get_args_parser
    a = get_args_parser().parse_args([])
    assert a.teacher_checkpoint is None and not a.teacher_int8 and (a.distill_topk, a.distill_t, a.distill_soft, a.distill_hard) == (3, 4.0, 0.9, 0.1)
    a = get_args_parser().parse_args("--teacher_checkpoint t.pth --teacher_int8 --distill_topk 5 --distill_t 2".split())
    assert a.teacher_checkpoint == "t.pth" and a.teacher_int8 and a.distill_topk == 5 and a.distill_t == 2.0


@pytest.mark.parametrize("case", ["plain", "loaded", "trained", "int8 alone", "no flags"])
def test_main_says_which_teacher_flags_do_nothing(monkeypatch, tmp_path, capsys, case):
    """main up to the optimizer, with made-up data and models: a teacher is used where a classifier is trained, and named as ignored else."""
    import main as drv
    from arguments import get_args_parser
    from models import classifiers

    class Stop(Exception):
        pass

    def stop(*a, **k):
        raise Stop

    monkeypatch.chdir(tmp_path)
    loader = [(torch.zeros(300, 3, 32, 32), torch.zeros(300))]
    teacher, _ = _classifier(1)
    torch.save(teacher, "t.pth")
    torch.save(torch.nn.Identity(), "ae.pth")
    torch.save(torch.nn.Identity(), "c.pth")
    seen = []
    monkeypatch.setattr(drv, "init_from_env", lambda: (0, 0, 1))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(drv, "get_cifar", lambda **k: (loader, loader))
    monkeypatch.setattr(drv, "Autoencoder", lambda **k: types.SimpleNamespace(to=lambda d: torch.nn.Identity()))
    monkeypatch.setattr(drv, "FusedAdamW", stop)
    monkeypatch.setattr(classifiers, "evaluate_classifier", lambda *a, **k: 0.0)
    monkeypatch.setattr(classifiers, "train_classifier", lambda *a, **k: seen.append(k["teacher"]) or torch.nn.Identity())
    real = torch.load
    monkeypatch.setattr(torch, "load", lambda f, map_location=None, **k: real(f, map_location="cpu", **k))
    flags = {"plain": "--teacher_checkpoint t.pth --teacher_int8", "loaded": "--variational --classifier_checkpoint c.pth --teacher_checkpoint t.pth",
             "trained": "--variational --teacher_checkpoint t.pth --teacher_int8", "int8 alone": "--variational --teacher_int8", "no flags": "--variational"}[case]
    args = get_args_parser().parse_args(flags.split() + ["--ae_checkpoint", "ae.pth", "--latent_size", "64"])
    with pytest.raises(Stop):
        drv.main(args)
    said = [line for line in capsys.readouterr().out.splitlines() if "ignored" in line]
    want = {"plain": ["--teacher_checkpoint --teacher_int8 ignored: only a --variational run trains a classifier"],
            "loaded": ["--teacher_checkpoint ignored: the classifier is loaded from c.pth"], "int8 alone": ["--teacher_int8 ignored: there is no --teacher_checkpoint"]}
    assert said == want.get(case, [])
    assert len(seen) == (case in ("trained", "int8 alone", "no flags"))
    if case == "trained":
        assert isinstance(seen[0], classifiers.Classifier) and seen[0].int8_fc
    elif seen:
        assert seen == [None]


def test_teacher_int8_needs_a_classifier(tmp_path):
    """--teacher_int8 on a model without 8-bit layers would change nothing."""
    import main as drv
    torch.save(torch.nn.Linear(3, 2), tmp_path / "t.pth")
    args = types.SimpleNamespace(teacher_checkpoint=str(tmp_path / "t.pth"), teacher_int8=True)
    with pytest.raises(NotImplementedError, match="Linear"):
        drv.load_teacher(args, "cpu")
    args.teacher_int8 = False
    assert not hasattr(drv.load_teacher(args, "cpu"), "int8_fc")
    torch.save(torch.nn.Linear(3, 2).state_dict(), tmp_path / "t.pth")
    with pytest.raises(NotImplementedError, match="state_dict"):
        drv.load_teacher(args, "cpu")
