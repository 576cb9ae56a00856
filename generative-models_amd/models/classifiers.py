"""CIFAR-10 Classifier with the reference's Python surface (feature / logit provider for the metrics).

Mirrors /root/reference/models/classifiers.py: same class name and module path (the reference stores the
classifier as a full-model pickle, `models.classifiers.Classifier`, classifiers.py:111), same constructor
(`Classifier(args)`), same child modules / parameter / buffer names, `.latent_vector` after forward.

Two forward paths, chosen by the module's mode:

* eval mode (what metrics.compute_fid / compute_inception_score / compute_confidence_diversity and
  evaluate_classifier run): hand-written gfx950 kernels through libgmk -- BatchNorm is folded
  into the preceding conv / linear weights, the activation into the conv / GEMM epilogue, so the whole forward is
  3 implicit-GEMM convs, 3 max-pools and 2 GEMMs.  CUDA tensors only (no CPU path).
* train mode (train_classifier, an auxiliary model's training loop: out of the hot-path scope):
  ordinary PyTorch modules under autograd.

Beyond the reference, a classifier can learn from another one (train_classifier(teacher=...), distillation_loss) and answer with its two
fully connected layers in 8-bit integers (int8_fc): both run on libgmk.
"""
import numpy as np
import torch
import torch.nn as nn

from gmk import ops, act_id
from utils import print_debug


class Classifier(nn.Module):
    # eval mode: fc and fc_out in 8-bit integers, one scale for each sample and each output (gmk.ops.linear_i8); set it on an instance
    int8_fc = False

    def __init__(self, args=None) -> None:
        super().__init__()
        self.debug = args.debug
        self.latent_size = args.latent_size
        self.conv1 = nn.Conv2d(in_channels=3, out_channels=64, kernel_size=5, stride=1, padding=2)
        self.conv2 = nn.Conv2d(in_channels=64, out_channels=128, kernel_size=5, stride=1, padding=2)
        self.conv3 = nn.Conv2d(in_channels=128, out_channels=256, kernel_size=3, stride=1, padding=1)
        self.max_pool = nn.MaxPool2d(2, 2)
        self.fc = nn.Linear(in_features=256 * 4 * 4, out_features=self.latent_size)
        self.fc_out = nn.Linear(in_features=self.latent_size, out_features=10)
        self.bn1 = nn.BatchNorm2d(num_features=64)
        self.bn2 = nn.BatchNorm2d(num_features=128)
        self.bn3 = nn.BatchNorm2d(num_features=256)
        self.bn4 = nn.BatchNorm1d(num_features=self.latent_size)
        self.dropout = nn.Dropout(p=args.dropout, inplace=False)
        self.act = args.act_fn

    # ------------------------------------------------------------------ eval: libgmk
    def _folded(self):
        """BatchNorm (eval: running statistics) folded into the producing layer:
        bn(conv(x)) = conv(x; w * s) + (b - mean) * s + beta,  s = gamma / sqrt(var + eps).
        Cached until a parameter or buffer is modified in place (tensor version counters) or replaced, the classifier is moved or goes into
        train mode.  A graph that is being captured folds for
        itself: its replays follow the weights, and neither uses what the other frees or has yet to compute."""
        if self.fc_out.weight.is_cuda and torch.cuda.is_current_stream_capturing():
            return self._fold()
        tensors = list(self.parameters()) + list(self.buffers())
        key = (self.int8_fc,) + tuple((t.data_ptr(), t._version) for t in tensors)
        # a fold for each stream that asks: what one of them has only queued is no weight for the others
        stream = torch._C._cuda_getCurrentRawStream(tensors[0].get_device()) if tensors[0].is_cuda else None
        cache = self.__dict__.get("_gmk_fold")
        if cache is None or cache[0] != key:
            # the tensors themselves are kept too: memory that a later weight could be given is no key
            cache = self.__dict__["_gmk_fold"] = (key, {}, [t.detach() for t in tensors])
        if stream in cache[1]:
            ops.keep_recorded(*(t for layer in cache[1][stream].values() for t in layer))
        else:
            cache[1][stream] = self._fold()
        return cache[1][stream]

    def train(self, mode=True):
        # training may write parameters where no version counter sees it: optimizers on raw pointers (gmk.optim), replayed graphs
        if mode:
            self.__dict__.pop("_gmk_fold", None)
        return super().train(mode)

    def _apply(self, *args, **kwargs):
        self.__dict__.pop("_gmk_fold", None)   # or a model that moves would leave its memory behind
        return super()._apply(*args, **kwargs)

    def _fold(self):
        out = {}
        with torch.no_grad():
            for layer, bn in ((self.conv1, self.bn1), (self.conv2, self.bn2), (self.conv3, self.bn3), (self.fc, self.bn4)):
                s = bn.weight / torch.sqrt(bn.running_var + bn.eps)
                w = layer.weight * s.view(-1, *([1] * (layer.weight.dim() - 1)))
                b = (layer.bias - bn.running_mean) * s + bn.bias
                out[layer] = (w.float().contiguous(), b.float().contiguous())
            out[self.fc_out] = (self.fc_out.weight.detach(), self.fc_out.bias.detach())   # as they are: other types are refused by the ops
            ops.keep_recorded(*(t for layer in out.values() for t in layer))
            if self.int8_fc:
                for layer in (self.fc, self.fc_out):
                    w, b = out[layer]
                    out[layer] = (*ops.quantize_rows(w), b)
        return out

    def _forward_gmk(self, x):
        if not x.is_cuda:
            raise RuntimeError("Classifier eval forward runs gfx950 kernels (libgmk): move the model and the images to "
                               "an MI355X (there is no CPU path)")
        a = act_id(self.act)
        f = self._folded()
        x = x.detach().float().contiguous()
        for conv in (self.conv1, self.conv2, self.conv3):
            w, b = f[conv]
            x = ops.conv2d_fwd(x, w, b, stride=1, act=a)       # conv + folded BN + activation, classifiers.py:33,37,42
            x = ops.maxpool2_fwd(x, want_idx=False)            # :35,39,44
        x = x.view(-1, 4 * 4 * 256)                            # :46
        linear = ops.linear_i8 if self.int8_fc else ops.linear_fwd
        x = linear(x, *f[self.fc], act=a)                      # fc + folded BN1d + activation, :48 (dropout: identity in eval)
        self.latent_vector = x                                 # :51
        return linear(x, *f[self.fc_out])                      # :52

    # ------------------------------------------------------------------ train: PyTorch autograd (out of scope for libgmk)
    def _forward_torch(self, x):
        x = self.max_pool(self.act(self.bn1(self.conv1(x))))
        x = self.max_pool(self.act(self.bn2(self.conv2(x))))
        x = self.max_pool(self.act(self.bn3(self.conv3(x))))
        x = x.view(-1, 4 * 4 * 256)
        x = self.act(self.bn4(self.fc(x)))
        x = self.dropout(x)
        self.latent_vector = x
        return self.fc_out(x)

    def forward(self, x):
        print_debug(x, self.debug, name='\nClassifier: input')
        x = self._forward_torch(x) if self.training else self._forward_gmk(x)
        print_debug(x, self.debug, name='Classifier: after fc_out')
        return x

    def __getstate__(self):
        state = self.__dict__.copy()
        state.pop("_gmk_fold", None)  # the folded-weight cache is not part of a saved model
        return state


class _DistillFn(torch.autograd.Function):
    """Row losses of gmk.ops.distill_fwd with distill_bwd as their gradient; the teacher's side and the labels have none."""

    @staticmethod
    def forward(ctx, logits, value, index, labels, T, soft, hard):
        loss, stats = ops.distill_fwd(logits, value, index, labels, T, soft, hard)
        ctx.save_for_backward(logits, value, index, labels, stats)
        ctx.weights = (T, soft, hard)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        logits, value, index, labels, stats = ctx.saved_tensors
        dz = ops.distill_bwd(grad.float().contiguous(), logits, value, index, labels, stats, *ctx.weights)
        return dz, None, None, None, None, None, None


def distillation_loss(outputs, value, index, labels=None, T=4.0, soft=0.9, hard=0.1):
    """Loss of each sample (n,) of a student's logits (n, C): soft T^2 KL(teacher || student) at temperature T over the teacher's kept logits
    `value` (n, k) of the classes `index` (n, k) int32 (gmk.ops.topk_rows; -1: no entry), plus hard * cross entropy where labels (n,) are
    given (outside [0, C): none).  CUDA tensors; outputs fp32, bf16 or fp16, under autograd.  In 32 bits the soft part is known to about
    soft T^2 2^-20, so that it loses its digits at temperatures far above the logits' differences; the gradient keeps them.  As with any loss, a
    backward pass is captured into a graph only while no eager graph of the same leaves is alive (torch.autograd's own rule)."""
    if labels is None:
        hard = 0.0
    return _DistillFn.apply(outputs.contiguous(), value.detach(), index, labels, float(T), float(soft), float(hard))


def compute_accuracy(outputs, labels):
    """Top-1 accuracy of a batch in percent (same value as reference classifiers.py:69-74)."""
    with torch.no_grad():
        hits = (outputs.argmax(dim=1) == labels).sum().item()
    return 100.0 * hits / labels.size(0)


def _epoch_accuracy(classifier, dataloader, device, step=None):
    """Mean of the per-batch accuracies over one pass; `step(outputs, labels, images)` runs the optimisation when given."""
    accs = []
    for images, labels in dataloader:
        images, labels = images.to(device), labels.to(device)
        outputs = classifier(images)
        if step is not None:
            step(outputs, labels, images)
        accs.append(compute_accuracy(outputs, labels))
    return np.mean(accs)


def train_classifier(args, classifier=None, train_dataloader=None, test_dataloader=None, device=None, teacher=None):
    """Auxiliary model training (reference classifiers.py:77-113): cross entropy, AdamW, cosine LR stepped every
    iteration over epochs * len(loader) steps; the full model object is saved, as the metrics' loader expects.
    With a `teacher` (any module of logits, put on `device` and into eval mode; not in the reference) the student learns from its args.distill_topk largest logits of each
    sample and the labels (distillation_loss, temperature args.distill_t, weights args.distill_soft and args.distill_hard)."""
    print('\n\nTraining CIFAR-10 Classifier\n\n')
    classifier = Classifier(args=args).to(device) if classifier is None else classifier
    optim = torch.optim.AdamW(classifier.parameters(), lr=args.lr, weight_decay=args.wd)
    sched = torch.optim.lr_scheduler.CosineAnnealingLR(optimizer=optim, T_max=args.epochs * len(train_dataloader))
    criterion = nn.CrossEntropyLoss()
    if teacher is not None:
        learning = {id(t) for t in (*classifier.parameters(), *classifier.buffers())}
        if any(id(t) in learning for t in (*teacher.parameters(), *teacher.buffers())):
            raise ValueError("the teacher shares parameters with the classifier that learns from it, which would train the teacher too")
        teacher = teacher.to(device).eval()

    def loss_of(outputs, labels, images):
        if teacher is None:
            return criterion(outputs, labels)
        with torch.no_grad():
            logits = teacher(images).contiguous()
            value, index = ops.topk_rows(logits, min(getattr(args, "distill_topk", 3), logits.shape[1]))
        return distillation_loss(outputs, value, index, labels, T=getattr(args, "distill_t", 4.0), soft=getattr(args, "distill_soft", 0.9),
                                 hard=getattr(args, "distill_hard", 0.1)).mean()

    def step(outputs, labels, images):
        optim.zero_grad()
        loss_of(outputs, labels, images).backward()
        optim.step()
        sched.step()

    for epoch in range(args.epochs):
        classifier.train()
        train_acc = _epoch_accuracy(classifier, train_dataloader, device, step=step)
        test_acc = evaluate_classifier(classifier, test_dataloader=test_dataloader, device=device)
        print(f'Epoch {epoch}  train {train_acc:.2f}  test {test_acc:.2f}  LR {sched.get_last_lr()[0]:.4f}')
    checkpoint_path = f'checkpoints/cifar_classifier_{args.latent_size}.pth'
    print(f'\n\nSaving classifier model checkpoint to {checkpoint_path}')
    torch.save(classifier, checkpoint_path)
    return classifier


def evaluate_classifier(classifier, test_dataloader=None, device=None):
    """Eval-mode pass (libgmk forward), reference classifiers.py:115-124."""
    classifier.eval()
    with torch.no_grad():
        return _epoch_accuracy(classifier, test_dataloader, device)
