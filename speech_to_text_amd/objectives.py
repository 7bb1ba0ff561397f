"""Scoring and distillation of label tokens on the GPU: the other end of the labels that the collator makes.

The reference trains on ``labels`` padded with -100 (``src/data.py:500``) through the cross entropy inside the Hugging Face
models (``train.py:300-309``) and evaluates by decoding (``evaluation.py:261-301``).  Two operators work on the same labels and
a model's logits, in hand-written HIP kernels (``libsttfe.so``):

* ``token_logprobs``: the log probability of every label, the entropy of its distribution, the most likely alternatives --
  how sure a model is of a transcript, one decoding step's candidates, or what ``FeatureCacheWriter`` keeps of a teacher;
* ``distillation_loss``: training on those kept alternatives (``FeatureCacheDataset`` -> ``AudioCollator`` hand them out as
  ``teacher_ids`` / ``teacher_logits``) and on the labels, with its gradient.

::

    batch = collator(samples)                                    # labels padded with -100, teacher_ids with -1
    logits = model(input_features=..., labels=...).logits        # (B, T, V)
    loss = distillation_loss(logits, batch["labels"].cuda(), batch["teacher_ids"].cuda(), batch["teacher_logits"].cuda(),
                             temperature=2.0, alpha=0.8)
    loss.backward()

Results are float32 and on the logits' GPU; gradients have the logits' type.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib

MAX_TOP = 64                       # STTFE_MAX_TOP
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_REDUCE = {"none": 0, "sum": 1, "mean": 2}


class TokenScores(NamedTuple):
    """Results of ``token_logprobs``; what was not asked for is None."""
    logprobs: Optional[torch.Tensor]          # float32, shape of the labels
    entropy: Optional[torch.Tensor]           # float32, nats
    top_ids: Optional[torch.Tensor]           # int64 (..., top_k)
    top_logprobs: Optional[torch.Tensor]      # float32 (..., top_k)


def _rows(logits: torch.Tensor, what: str):
    """The C ABI's description of (..., vocab) logits: pointer, type, outer x inner rows, their strides, vocab."""
    if not torch.is_tensor(logits) or logits.dim() < 1:
        raise ValueError(f"{what}: logits are a tensor (..., vocab)")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"{what}: logits are float32, float16 or bfloat16, not {logits.dtype}")
    shape, stride = logits.shape, logits.stride()
    V = shape[-1]
    if V < 1:
        raise ValueError(f"{what}: logits have an empty vocabulary")
    if V > 1 and stride[-1] != 1:
        raise ValueError(f"{what}: the vocabulary (last) dimension of the logits has to be contiguous, its stride is "
                         f"{stride[-1]}")
    if 0 in shape:
        return logits.data_ptr(), _DTYPES[logits.dtype], 0, 0, 0, 0, V
    # leading dimensions -> (outer, inner): merge from the right what one stride describes
    outer, inner, so, si = 1, 1, 0, 0
    for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if n == 1:
            continue
        if inner == 1:
            inner, si = n, s
        elif outer == 1 and s == si * inner:
            inner *= n
        elif outer == 1:
            outer, so = n, s
        elif s == so * outer:
            outer *= n
        else:
            raise ValueError(f"{what}: logits of shape {tuple(shape)} and strides {stride} have more than two row strides; "
                             "make them contiguous")
    return logits.data_ptr(), _DTYPES[logits.dtype], outer, inner, so, si, V


def _whole(t: torch.Tensor, shape, device, what: str, name: str) -> torch.Tensor:
    if not torch.is_tensor(t) or t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: {name} is an int64 or int32 tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, the logits ask for {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, the logits are on {device}")
    return t.to(torch.int64).contiguous()


def _on_gpu(logits: torch.Tensor, what: str):
    if logits.device.type != "cuda":
        raise _lib.SttfeError(f"{what}: logits are on {logits.device}: there is no CPU path")


def _no_tangent(what: str, *tensors: torch.Tensor):
    """Forward-mode derivatives: the kernels would drop the tangent of a dual tensor without a word."""
    if getattr(forward_ad, "_current_level", 0) < 0:             # no dual level is open (looking at a tensor takes 0.7 us)
        return
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what}: a tensor carries a forward-mode tangent; there are reverse-mode derivatives only")


def _temperature(temperature: float, what: str) -> float:
    temperature = float(temperature)
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"{what}: temperature {temperature} is not in [0.001, 1000]")
    return temperature


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _call(name: str, device: torch.device, *args):
    """One entry point of the library on the device's current stream.

    The host side of a small training step costs more than its kernels: the stream comes as a number (building a Stream object
    takes 4 us, and 15 when the autograd thread builds them too), the device is only changed if it is another."""
    fn = getattr(_lib.lib(), name)
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != 0:
        _lib.check(rc, name)


def _workspace(name: str, device: torch.device, *args) -> Tuple[Optional[torch.Tensor], int]:
    n = ctypes.c_size_t()
    rc = getattr(_lib.lib(), name)(*args, ctypes.byref(n))
    if rc != 0:
        _lib.check(rc, name)
    return (torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None), n.value


# ------------------------------------------------------------------------------------------------- token_logprobs
def _logprobs_forward(logits, rows, labels, top_k, want_entropy, temperature, ignore_index, want_stats):
    device, lead = logits.device, logits.shape[:-1]
    logprobs = torch.empty(lead, dtype=torch.float32, device=device) if labels is not None else None
    entropy = torch.empty(lead, dtype=torch.float32, device=device) if want_entropy else None
    stats = torch.empty(lead + (4,), dtype=torch.float32, device=device) if want_stats else None
    ids = torch.empty(lead + (top_k,), dtype=torch.int64, device=device) if top_k else None
    top = torch.empty(lead + (top_k,), dtype=torch.float32, device=device) if top_k else None
    ws, n = _workspace("sttfe_token_logprobs_workspace_bytes", device, rows[2] * rows[3], rows[6], rows[1], top_k)
    _call("sttfe_token_logprobs", device, *rows, _ptr(labels), ignore_index, temperature, top_k, _ptr(logprobs), _ptr(entropy),
          _ptr(stats), _ptr(ids), _ptr(top), _ptr(ws), n)
    return logprobs, entropy, ids, top, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rows, labels, top_k, want_entropy, temperature, ignore_index):
        logprobs, entropy, ids, top, stats = _logprobs_forward(logits, rows, labels, top_k, want_entropy, temperature,
                                                               ignore_index, True)
        ctx.args = (top_k, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, labels, ids, stats)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return logprobs, entropy, ids, top

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprobs, g_entropy, _, g_top):
        logits, labels, ids, stats = ctx.saved_tensors
        if g_logprobs is None and g_entropy is None and g_top is None:
            return (None,) * 7
        _no_tangent("token_logprobs backward", *(t for t in (g_logprobs, g_entropy, g_top) if t is not None))
        top_k, temperature, ignore_index = ctx.args
        rows = _rows(logits, "token_logprobs")
        g = [None if t is None else t.to(torch.float32).contiguous() for t in (g_logprobs, g_entropy, g_top)]
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _call("sttfe_token_logprobs_grad", logits.device, *rows, _ptr(labels), ignore_index, temperature, _ptr(stats), _ptr(g[0]),
              _ptr(g[1]), top_k, _ptr(ids), _ptr(g[2]), _ptr(grad))
        return grad, None, None, None, None, None, None


def token_logprobs(logits: torch.Tensor, labels: Optional[torch.Tensor] = None, *, top_k: int = 0, entropy: bool = False,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenScores:
    """Log probabilities of ``labels`` under ``softmax(logits / temperature)``, with entropy and top alternatives.

    ``logits``: (..., V) float32 / float16 / bfloat16 on the GPU, V contiguous, at most two row strides (a slice of the
    positions or an expanded batch is fine).  ``labels``: (...) int64 / int32 on the same GPU, or None (one decoding step:
    entropy and alternatives only).  Positions with ``ignore_index`` are left out: 0 for their results, -1 / -inf for their
    alternatives, no gradient.  ``top_k`` <= 64: the largest logits in falling order, equal ones by index.

    ``logprobs``, ``entropy`` and ``top_logprobs`` are differentiable in the logits (once).  A label outside the vocabulary
    makes its log probability NaN, and the gradient that comes with it: it cannot be reported without a synchronisation.
    Entropy and alternatives do not depend on the label.
    """
    what = "token_logprobs"
    rows = _rows(logits, what)
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP, rows[6]):
        raise ValueError(f"{what}: top_k {top_k} is not in [0, min({MAX_TOP}, vocabulary {rows[6]})]")
    if labels is None and not top_k and not entropy:
        raise ValueError(f"{what}: nothing is asked for (labels, top_k or entropy)")
    temperature = _temperature(temperature, what)
    if labels is not None:
        labels = _whole(labels, logits.shape[:-1], logits.device, what, "labels")
    _no_tangent(what, logits)
    _on_gpu(logits, what)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenScores(*_TokenLogprobs.apply(logits, rows, labels, top_k, bool(entropy), temperature, int(ignore_index)))
    return TokenScores(*_logprobs_forward(logits, rows, labels, top_k, bool(entropy), temperature, int(ignore_index), False)[:4])


# ------------------------------------------------------------------------------------------------- distillation_loss
def _distill_args(what, logits, labels, teacher_ids, teacher_logits, temperature, alpha, ignore_index, weight, reduction):
    rows = _rows(logits, what)
    if reduction not in _REDUCE:
        raise ValueError(f"{what}: reduction {reduction!r} is not one of {tuple(_REDUCE)}")
    temperature = _temperature(temperature, what)
    alpha, weight = float(alpha), float(weight)
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"{what}: alpha {alpha} is not in [0, 1]")
    lead = tuple(logits.shape[:-1])
    labels = _whole(labels, lead, logits.device, what, "labels")
    if not torch.is_tensor(teacher_ids) or teacher_ids.dim() != len(lead) + 1 or not 1 <= teacher_ids.shape[-1] <= MAX_TOP:
        raise ValueError(f"{what}: teacher_ids is a tensor {lead + ('K',)}, K in [1, {MAX_TOP}]")
    K = int(teacher_ids.shape[-1])
    ids = _whole(teacher_ids, lead + (K,), logits.device, what, "teacher_ids")
    t = teacher_logits
    if not torch.is_tensor(t) or t.dtype not in _DTYPES or tuple(t.shape) != lead + (K,) or t.device != logits.device:
        raise ValueError(f"{what}: teacher_logits is a floating tensor of the shape and on the device of teacher_ids")
    if torch.is_grad_enabled() and t.requires_grad:
        raise ValueError(f"{what}: the teacher has no gradient here; detach() its logits")
    _no_tangent(what, logits, t)
    if reduction == "none" and weight != 1.0:
        raise ValueError(f"{what}: weight belongs to a reduced loss; weight the positions' losses themselves")
    _on_gpu(logits, what)
    return rows, labels, ids, t.detach().to(torch.float32).contiguous(), K, temperature, alpha, int(ignore_index), weight, reduction


def _distill_forward(logits, args, want_stats, want_grad):
    """-> loss, factor, stats, gradient (each None if not wanted; the factor with the stats only)."""
    rows, labels, ids, teacher, K, temperature, alpha, ignore_index, weight, reduction = args
    device, lead = logits.device, logits.shape[:-1]
    f32 = torch.float32
    losses = torch.empty(lead, dtype=f32, device=device)
    total = factor = None
    if reduction != "none":
        total, factor = torch.empty((), dtype=f32, device=device), torch.empty((), dtype=f32, device=device)
    stats = torch.empty(lead + (4,), dtype=f32, device=device) if want_stats else None
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=device) if want_grad else None
    ws, n = _workspace("sttfe_distill_workspace_bytes", device, rows[2] * rows[3], rows[6], rows[1])
    _call("sttfe_distill_loss", device, *rows, _ptr(labels), ignore_index, _ptr(ids), _ptr(teacher), K, temperature, alpha, weight,
          _REDUCE[reduction], _ptr(losses), _ptr(total), _ptr(factor), _ptr(stats), _ptr(grad), _ptr(ws), n)
    return losses if total is None else total, factor, stats, grad


def _distill_backward(logits, args, stats, factor, g, g_rows):
    rows, labels, ids, teacher, K, temperature, alpha, ignore_index, weight, reduction = args
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _call("sttfe_distill_grad", logits.device, *rows, _ptr(labels), ignore_index, _ptr(ids), _ptr(teacher), K, temperature, alpha,
          _ptr(stats), _ptr(factor), _ptr(g), _ptr(g_rows), _ptr(grad))
    return grad


class _Distillation(torch.autograd.Function):
    """Reduced losses of bfloat16 / float32 logits make their gradient in the forward pass, for an upstream gradient of 1, while
    the row is at hand; backward hands it out, multiplied in place if the upstream gradient is another.  float16 cannot hold
    a small gradient that only a loss scale lifts into its range, and unreduced losses have an upstream gradient per
    position: both compute theirs in backward, from the logits."""

    @staticmethod
    def forward(ctx, logits, args):
        fused = args[-1] != "none" and logits.dtype != torch.float16
        loss, factor, stats, ctx.grad = _distill_forward(logits, args, not fused, fused)
        ctx.scalars = args[4:]
        ctx.save_for_backward(logits, *args[1:4], stats, None if fused else factor)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, labels, ids, teacher, stats, factor = ctx.saved_tensors
        _no_tangent("distillation_loss backward", g)
        g = g.to(torch.float32).contiguous()
        grad, ctx.grad = ctx.grad, None                 # handed out once: a second pass over a kept graph computes its own
        if grad is not None:
            _call("sttfe_distill_rescale", grad.device, _ptr(grad), _DTYPES[grad.dtype], grad.numel(), _ptr(g))
            return grad, None
        args = (_rows(logits, "distillation_loss"), labels, ids, teacher) + ctx.scalars
        if stats is None:
            _, factor, stats, _ = _distill_forward(logits, args, True, False)
        if args[-1] == "none":
            return _distill_backward(logits, args, stats, None, None, g), None
        return _distill_backward(logits, args, stats, factor, g, None), None


def distillation_loss(logits: torch.Tensor, labels: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                      temperature: float = 1.0, alpha: float = 0.5, ignore_index: int = -100, weight: float = 1.0,
                      reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's K kept entries per position, mixed with the cross entropy of the labels.

    Per position, with q = softmax(teacher_logits / temperature) over the kept entries::

        alpha * temperature**2 * sum_k q_k (log q_k - log softmax(logits / temperature)[teacher_ids_k])
            + (1 - alpha) * -log softmax(logits)[label]

    ``logits`` / ``labels`` as in ``token_logprobs``; ``teacher_ids`` / ``teacher_logits``: (..., K), K <= 64, logits or log
    probabilities alike.  Entries with a negative id are padding; a position without entries has no teacher term.
    ``reduction``: "mean" over the positions whose label is not ``ignore_index`` (0 if there is none), "sum", or "none"
    (float32, shape of the labels).  ``weight`` multiplies the reduced loss (gradient accumulation: 1 / steps).

    The gradient with respect to the logits has their type.  A reduced bfloat16 loss rounds it once for an upstream gradient of
    1 and again for another one: ``weight`` rather than a factor on the loss keeps it at one.  A label or id outside the vocabulary makes its position's loss
    and gradient NaN.
    """
    args = _distill_args("distillation_loss", logits, labels, teacher_ids, teacher_logits, temperature, alpha, ignore_index, weight,
                         reduction)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Distillation.apply(logits, args)
    return _distill_forward(logits, args, False, False)[0]


def distillation_loss_and_grad(logits: torch.Tensor, labels: torch.Tensor, teacher_ids: torch.Tensor,
                               teacher_logits: torch.Tensor, *, temperature: float = 1.0, alpha: float = 0.5,
                               ignore_index: int = -100, weight: float = 1.0, reduction: str = "mean",
                               grad_scale: Union[None, float, torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``distillation_loss`` ("mean" or "sum") and the gradient of the logits in one call without autograd, for training steps
    that are captured into a graph or drive the model's backward themselves (``logits.backward(grad)``).

    ``grad_scale`` multiplies the gradient, not the loss, before the gradient is rounded to the logits' type: a number, or a
    float32 tensor of one element on the logits' GPU that the kernels read when they run.  float16 logits need a loss scale
    here: the gradient's elements are p / positions, and what is below 3e-8 becomes 0, which no later scale brings back.
    With it the logits are read a second time for the gradient."""
    what = "distillation_loss_and_grad"
    if reduction == "none":
        raise ValueError(f"{what}: reduction is 'mean' or 'sum'")
    if torch.is_tensor(grad_scale) and (grad_scale.dtype != torch.float32 or grad_scale.numel() != 1
                                        or not torch.is_tensor(logits) or grad_scale.device != logits.device):
        raise ValueError(f"{what}: grad_scale is a number or a float32 tensor of one element on the device of the logits")
    if torch.is_tensor(logits):
        _no_tangent(what, logits, *((grad_scale,) if torch.is_tensor(grad_scale) else ()))       # detach() would drop it
        logits = logits.detach()
    args = _distill_args(what, logits, labels, teacher_ids, teacher_logits, temperature, alpha, ignore_index,
                         weight, reduction)
    if grad_scale is None:
        loss, _, _, grad = _distill_forward(logits, args, False, True)
        return loss, grad
    if not torch.is_tensor(grad_scale):
        grad_scale = torch.full((), float(grad_scale), dtype=torch.float32, device=logits.device)
    loss, factor, stats, _ = _distill_forward(logits, args, True, False)
    return loss, _distill_backward(logits, args, stats, factor, grad_scale, None)
