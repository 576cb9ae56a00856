"""What is measured of three operators: the 8-bit linear layer (`linear_i8`), a row's k largest logits (`topk_rows`) and
the distillation loss from a teacher's kept logits with its gradient (`distill_*`).

Together they are the way from a large classifier to a small one: the teacher's fully connected layers answer in 8-bit
integers, its k largest logits of every sample are kept, and the student learns from them.

`run` computes an operator in its plain form, from elementary torch operations, or, where `own` is set, with the calls that a
user makes of `gmk.ops`.  `exact` computes the same from the definition in 64 bits.
"""
import importlib
import math
import sys

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _gmk_ops():
    """The framework's operators; its package lies in a folder that is no Python name."""
    if "generative-models_amd" not in sys.path:
        sys.path.append("generative-models_amd")
    return importlib.import_module("gmk.ops")


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # the first fully connected layer of the CIFAR-10 classifier, 4096 features to a 256-wide latent, one training batch
        {"name": "linear fc 256", "op": "linear", "M": 256, "K": 4096, "N": 256, "x": "fp32", "y": "fp32", "act": "gelu", "bias": True},
        # one sample through a wide output layer: the weights are read once, nothing else matters
        {"name": "linear one row", "op": "linear", "M": 1, "K": 4096, "N": 32768, "x": "bf16", "y": "bf16", "act": "none", "bias": False},
        # a handful of samples answered together
        {"name": "linear few rows", "op": "linear", "M": 24, "K": 8192, "N": 8192, "x": "bf16", "y": "bf16", "act": "gelu", "bias": True},
        # odd sizes: rows that start at no 16-byte border, a last tile that is mostly empty on both sides
        {"name": "linear odd", "op": "linear", "M": 777, "K": 1357, "N": 5003, "x": "fp16", "y": "fp16", "act": "relu", "bias": True},
        # a teacher's pass over a large set: the matrix cores' own work
        {"name": "linear large", "op": "linear", "M": 8192, "K": 4096, "N": 16384, "x": "bf16", "y": "bf16", "act": "none", "bias": True},
        # a batch of the usual 1000 classes
        {"name": "topk 1000 classes", "op": "topk", "n": 256, "C": 1000, "k": 10, "x": "fp32", "masked": 0},
        # few long rows of an odd length, the last classes masked
        {"name": "topk long rows", "op": "topk", "n": 5, "C": 150001, "k": 50, "x": "fp32", "masked": 2001},
        # a teacher's pass over a large set; bf16 logits hold many equal values
        {"name": "topk large", "op": "topk", "n": 2048, "C": 65536, "k": 32, "x": "bf16", "masked": 0},
        # the CIFAR-10 classifier's own training batch, with labels: a call that is all latency
        {"name": "distill 10 classes", "op": "distill", "form": "fused", "n": 256, "C": 10, "k": 3, "x": "fp32", "t": "fp32", "T": 4.0, "soft": 0.9, "hard": 0.1},
        # the two calls of an autograd training step, odd sizes
        {"name": "distill two calls", "op": "distill", "form": "split", "n": 1001, "C": 10007, "k": 20, "x": "fp32", "t": "fp32", "T": 2.0, "soft": 0.5, "hard": 0.5},
        # few rows over very many classes
        {"name": "distill few rows", "op": "distill", "form": "fused", "n": 9, "C": 200003, "k": 64, "x": "fp16", "t": "fp32", "T": 1.0, "soft": 1.0, "hard": 0.0},
        # a training step over many classes, loss and gradient in one call
        {"name": "distill large", "op": "distill", "form": "fused", "n": 4096, "C": 32768, "k": 64, "x": "bf16", "t": "bf16", "T": 1.5, "soft": 1.0, "hard": 0.25},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "topk", "distill"])
    x = rng.choice(["fp32", "bf16", "fp16"])
    if op == "linear":
        K, N = _between(rng, 64, 8192), _between(rng, 10, 32768)
        M = _between(rng, 1, max(1, min(8192, (1 << 38) // (K * N))))
        return {"op": op, "M": M, "K": K, "N": N, "x": x, "y": rng.choice(["fp32", x]), "act": rng.choice(["none", "relu", "gelu"]), "bias": rng.random() < 0.5}
    C = _between(rng, 10, 200000)
    n = _between(rng, 1, max(1, min(8192, (1 << 26) // C)))
    k = _between(rng, 1, min(C, 128))
    if op == "topk":
        return {"op": op, "n": n, "C": C, "k": k, "x": x, "masked": rng.choice([0, 0, C // 10])}
    return {"op": op, "form": rng.choice(["fused", "split"]), "n": n, "C": C, "k": k, "x": x, "t": rng.choice(["fp32", x]),
            "T": round(rng.uniform(1.0, 8.0), 2), "soft": 1.0, "hard": rng.choice([0.0, 0.5])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "linear":
        # activations behind a gelu, a few features of them large; weights as a layer's initialisation draws them, laid out
        # once: 8-bit rows with their scales, each padded with zeros to whole 16-byte pieces
        x = normal(case["M"], case["K"])
        x = 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5)) * (1 + 7 * (torch.rand(case["K"], generator=g, device="cuda") > 0.99))
        w = normal(case["N"], case["K"]) / case["K"] ** 0.5
        wq, ws = _quantize(w)
        s["x"] = x.to(TYPES[case["x"]])
        s["wq"] = torch.nn.functional.pad(wq, (0, -case["K"] % 16)).to(torch.int8).contiguous()
        s["ws"] = ws
        s["b"] = 0.1 * normal(case["N"]) if case["bias"] else None
        return s
    n, C, k = case["n"], case["C"], case["k"]
    z = 2.5 * normal(n, C)
    if case["op"] == "topk":
        if case["masked"]:
            z[:, C - case["masked"]:] = -math.inf
        s["x"] = z.to(TYPES[case["x"]])
        return s
    # the teacher's kept logits, largest first, agree with the student's in part; some rows keep fewer than k, some samples
    # have no label, and the last rows of the batch are padding (a weight of zero)
    first = torch.randint(0, C, (n, 1), generator=g, device="cuda")
    at = (first + torch.arange(k, device="cuda") * (C // k)) % C
    t = z.gather(1, at) + 4 + 2 * normal(n, k)
    t, order = t.sort(dim=1, descending=True)
    at = at.gather(1, order)
    kept = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
    kept = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.2, kept, torch.full_like(kept, k))
    at = torch.where(torch.arange(k, device="cuda") < kept, at, torch.full_like(at, -1))
    label = torch.randint(0, C, (n,), generator=g, device="cuda")
    label[torch.rand(n, generator=g, device="cuda") < 0.1] = -100
    weight = torch.ones(n, device="cuda")
    weight[n - n // 20:] = 0
    s.update(x=z.to(TYPES[case["x"]]), t=t.to(TYPES[case["t"]]), at=at.to(torch.int32), label=label if case["hard"] else None,
             weight=weight, scale=1.0 / max(1, n - n // 20))
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    if s["op"] == "linear":
        if own:
            return _gmk_ops().linear_i8(s["x"], s["wq"], s["ws"], s["b"], act=s["act"], out_dtype=TYPES[s["y"]])
        return _linear(s)
    if s["op"] == "topk":
        if own:
            return _gmk_ops().topk_rows(s["x"], s["k"])
        return _topk(s["x"], s["k"])
    if own:
        ops = _gmk_ops()
        if s["form"] == "fused":
            return ops.distill_fwd_bwd(s["x"], s["t"], s["at"], s["label"], s["T"], s["soft"], s["hard"], s["weight"], s["scale"])
        loss, stats = ops.distill_fwd(s["x"], s["t"], s["at"], s["label"], s["T"], s["soft"], s["hard"])
        return loss, ops.distill_bwd(s["weight"], s["x"], s["t"], s["at"], s["label"], stats, s["T"], s["soft"], s["hard"])
    loss, grad = _distill(s)
    if s["form"] == "fused":
        return loss * s["weight"], (grad * (s["weight"] * s["scale"])[:, None]).to(s["x"].dtype)
    return loss, (grad * s["weight"][:, None]).to(s["x"].dtype)


def _quantize(x):
    """Rows in 8 bits: the scale is a 127th of the row's largest magnitude, rounded to 32 bits, and at least the smallest normal
    number; values go to the nearest whole number.  The quotient is taken in 64 bits, where none of them falls on a wrong side."""
    x = x.double()
    scale = (x.abs().amax(1) / torch.full((), 127.0, dtype=torch.float64, device=x.device)).float().clamp_min(2.0 ** -126)
    return (x / scale.double()[:, None]).round(), scale


def _linear(s):
    q, scale = _quantize(s["x"])
    w = s["wq"][:, : q.shape[1]]
    # the sum of whole products is exact: in 32 bits while no sum of them can pass 2^24, in 64 bits beyond
    t = torch.float32 if q.shape[1] * 127 * 127 < 1 << 24 else torch.float64
    y = (q.to(t) @ w.to(t).t()).float() * scale[:, None] * s["ws"]
    if s["b"] is not None:
        y = y + s["b"]
    if s["act"] == "relu":
        y = y.clamp_min(0)
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    return y.to(TYPES[s["y"]])


def _topk(x, k):
    """The k largest of each row in falling order, ties to the lowest index: both in one whole number, which has no ties."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    rank = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    key = (rank << 24) + ((1 << 24) - 1 - torch.arange(x.shape[1], device=x.device))
    at = (1 << 24) - 1 - (key.topk(k, dim=1).values & ((1 << 24) - 1))
    return x.gather(1, at), at.to(torch.int32)


def _distill(s):
    """The loss of each row and its gradient, in 32 bits."""
    T, soft, hard = s["T"], s["soft"], s["hard"]
    z = s["x"].float()
    C = z.shape[1]
    z = z - z.amax(1, keepdim=True)
    d = z / T
    e = d.exp()
    total = e.sum(1, keepdim=True)
    there = (s["at"] >= 0) & (s["at"] < C)
    at = torch.where(there, s["at"], torch.zeros_like(s["at"])).long()
    t = torch.where(there, s["t"].float() / T, torch.full((), -math.inf, device=z.device))
    t = t - t.amax(1, keepdim=True)
    p = t.exp()
    all_p = p.sum(1, keepdim=True)
    p = p / all_p
    logp = t - all_p.log()
    loss = soft * T * T * (torch.where(p > 0, p * (logp - d.gather(1, at)), torch.zeros_like(p)).sum(1) + total.log()[:, 0])
    grad = (soft * T) * (e / total).scatter_add(1, at, -p)
    if hard:
        has = (s["label"] >= 0) & (s["label"] < C)
        label = torch.where(has, s["label"], torch.zeros_like(s["label"]))[:, None]
        e = z.exp()
        total = e.sum(1, keepdim=True)
        loss = loss + hard * torch.where(has, (total.log() - z.gather(1, label))[:, 0], torch.zeros_like(loss))
        grad = grad + (hard * has.float())[:, None] * (e / total).scatter_add(1, label, torch.full_like(total, -1.0))
    return loss, grad


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * size[case["x"]] + N * K + 4 * N * (2 if case["bias"] else 1) + M * N * size[case["y"]], "flops": 2.0 * M * N * K}
    n, C, k = case["n"], case["C"], case["k"]
    if case["op"] == "topk":
        return {"bytes": n * C * size[case["x"]] + n * k * (size[case["x"]] + 4), "flops": n * C}
    # a row's maximum, its one or two exponentials and their sums, and the gradient
    return {"bytes": 2 * n * C * size[case["x"]] + n * k * (size[case["t"]] + 4) + n * (16 if case["hard"] else 8), "flops": n * C * (10.0 if case["hard"] else 6.0)}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "linear":
        # y = act(b + sum_k x^ w^), x^ and w^ the values that the 8-bit rows stand for
        step = torch.maximum((x.abs().max(dim=1, keepdim=True).values * (1 / 127.0)).to(torch.float32), torch.tensor(2.0 ** -126, device=x.device)).double()
        xh = torch.round(x / step) * step
        wh = s["wq"][:, : case["K"]].double() * s["ws"].double().unsqueeze(1)
        y = torch.matmul(xh, wh.transpose(0, 1).contiguous())
        y += 0.0 if s["b"] is None else s["b"].double()
        return {"none": lambda v: v, "relu": lambda v: v * (v > 0), "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2))}[case["act"]](y)
    if case["op"] == "topk":
        v, i = torch.sort(x, dim=1, descending=True, stable=True)
        return v[:, : case["k"]].clone(), i[:, : case["k"]].to(torch.int32)
    # the gradient by automatic differentiation of the loss
    n, C = x.shape
    x.requires_grad_(True)
    T = case["T"]
    keep = s["at"].ge(0)
    at = s["at"].long().clamp(min=0)
    teacher = torch.log_softmax(s["t"].double().div(T).masked_fill(~keep, -math.inf), dim=1)
    student = (x / T).gather(1, at) - torch.logsumexp(x / T, dim=1, keepdim=True)
    loss = case["soft"] * T ** 2 * (teacher.exp() * (teacher - student).masked_fill(~keep, 0.0)).masked_fill(~keep, 0.0).nan_to_num(0.0).sum(1)
    if case["hard"]:
        ce = torch.logsumexp(x, dim=1) - x.gather(1, s["label"].clamp(min=0)[:, None])[:, 0]
        loss = loss + case["hard"] * ce * s["label"].ge(0)
    weight = s["weight"].double()
    if case["form"] == "fused":
        ((loss * weight).sum() * s["scale"]).backward()
        return (loss * weight).detach(), x.grad
    (loss * weight).sum().backward()
    return loss.detach(), x.grad
