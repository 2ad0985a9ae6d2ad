"""Operators that fine-tune a language model on rewards and preferences: log-probabilities of given tokens, the clipped policy loss
with KL and entropy terms, the preference loss over pairs, and the global gradient norm over many tensors with clipping.

On CUDA logits (BF16, FP16, FP32) every operator runs hand-written sm_100a kernels (``csrc/cuda/token_objectives.cu``); elsewhere, and for
tensors that carry a forward-mode derivative, the same mathematics runs as plain PyTorch.  All of them are reached as
``fused.ops.<name>``, beside the cross-entropy.

With x = logits / temperature over the vocabulary: logp_t = x_t - logsumexp(x), H = -sum p log p.  A target equal to `ignore_index`
takes its token out of everything (prompts, padding): its results and gradients are zeros and its logits are never read, whatever they
hold.  A target outside the vocabulary gives NaN and a gradient of zeros.  Statistics are FP32; sums over tokens FP64."""
from __future__ import annotations

import contextlib
import math
from operator import attrgetter
from typing import List, NamedTuple, Optional, Sequence

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

_KERNEL_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_KERNEL_SET = frozenset(_KERNEL_TYPES)
_BYTES = (2, 4, 2)     # of the kernels' type codes
_shape, _dtype = attrgetter("shape"), attrgetter("dtype")
_TARGET_TYPES = (torch.int32, torch.int64)
O = None     # nexus_b200.ops._objectives, once a tensor on a GPU has been met


class PolicyLoss(NamedTuple):
    """What `policy_loss` returns: the loss (differentiable with respect to the logits) and, per token and detached, the new
    log-probability, the KL estimate against the reference and the entropy (zeros where a token does not count)."""
    loss: torch.Tensor
    logp: torch.Tensor
    kl: torch.Tensor
    entropy: torch.Tensor


class PreferenceLoss(NamedTuple):
    """What `preference_loss` returns: the loss (differentiable with respect to the logits) and, detached, the log-probability of each
    sequence [2 * pairs] and the margin of each pair (log-ratio of the chosen sequence minus that of the rejected one)."""
    loss: torch.Tensor
    logp: torch.Tensor
    margin: torch.Tensor


def _check_logits(name: str, logits, targets, vocab: Optional[int], temperature: float, ignore_index: int) -> int:
    if not logits.is_floating_point() or logits.dim() < 1:
        raise ValueError(f"{name}: logits must be a floating-point tensor [..., vocabulary]")
    shape = logits.shape
    if targets.dtype not in _TARGET_TYPES:
        raise ValueError(f"{name}: targets must be int32 or int64, got {targets.dtype}")
    if targets.shape != shape[:-1]:
        raise ValueError(f"{name}: targets {tuple(targets.shape)} do not match logits {tuple(shape)}")
    if targets.device != logits.device:
        raise ValueError(f"{name}: targets on {targets.device}, logits on {logits.device}")
    _check_temperature(name, temperature)
    _check_ignored(name, ignore_index)
    V = shape[-1] if vocab is None else int(vocab)
    if not 1 <= V <= shape[-1]:
        raise ValueError(f"{name}: vocab must be between 1 and {shape[-1]}, got {V}")
    if shape[-1] >= 2 ** 31 or targets.numel() >= 2 ** 31:
        raise ValueError(f"{name}: at most 2^31 - 1 rows and columns")
    return V


def _check_temperature(name: str, temperature: float) -> None:
    if not 1e-8 <= temperature <= 1e8:     # its inverse times a logit is an FP32 number, and -inf stays far below every logit
        raise ValueError(f"{name}: temperature must be between 1e-8 and 1e8, got {temperature}")


def _check_ignored(name: str, ignore_index: int) -> None:
    if not -2 ** 63 <= ignore_index < 2 ** 63:     # the kernels would take it modulo 2^64
        raise ValueError(f"{name}: ignore_index must be a 64-bit integer, got {ignore_index}")


def _check_values(name: str, what: str, t, shapes, device) -> torch.Tensor:
    """A tensor of constants of the loss in FP32: log-probabilities, advantages."""
    if not isinstance(t, torch.Tensor) or not t.is_floating_point():
        raise ValueError(f"{name}: {what} must be a floating-point tensor")
    if t.shape not in shapes:
        raise ValueError(f"{name}: {what} must have the shape {' or '.join(map(str, shapes))}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: {what} on {t.device}, logits on {device}")
    if t.requires_grad:
        t = t.detach()
    if _dual(t):
        t = forward_ad.unpack_dual(t).primal
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


_HERE = contextlib.nullcontext()


def _on(t: torch.Tensor):
    """Makes a tensor's device the current one, where it is not: the launches go to the current device's stream."""
    return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _dual(*ts: torch.Tensor) -> bool:
    """Whether a tensor carries a forward-mode derivative, which the kernels would drop."""
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts)


def _backward_only(name: str, t: torch.Tensor) -> None:
    if _dual(t):
        raise NotImplementedError(f"{name}: its gradient has no forward-mode derivative")


def _kernels(t: torch.Tensor) -> bool:
    if not t.is_cuda or t.dtype not in _KERNEL_TYPES:
        return False
    global O
    if O is None:
        from ..ops import _cuda, _objectives
        _cuda.lib()  # raises loudly when the library is missing on a GPU machine
        O = _objectives
    return True


def _wants(*ts: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def _token_parts(logits, targets, ignore_index, temperature, V):
    """Plain form: (counted, log-probabilities of all tokens [N, V], log-probability of the target [N]); FP32, or FP64 for FP64."""
    x = logits.reshape(-1, logits.shape[-1])[:, :V]
    x = (x if x.dtype == torch.float64 else x.float()) / temperature
    t = targets.reshape(-1).long()
    keep = t != ignore_index
    x = torch.where(keep[:, None], x, torch.zeros((), dtype=x.dtype, device=x.device))
    lp = torch.log_softmax(x, -1)
    inside = (t >= 0) & (t < V)
    logp = lp.gather(1, torch.where(inside, t, 0)[:, None])[:, 0]
    logp = torch.where(inside, logp, torch.full((), math.nan, dtype=lp.dtype, device=lp.device))
    return keep, lp, torch.where(keep, logp, torch.zeros((), dtype=lp.dtype, device=lp.device))


# ------------------------------------------------------------------------------------- log-probabilities of given tokens
def _token_forward(logits, targets, vocab, ignore_index, temperature):
    with _on(logits):
        logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
        return (logits, targets, *O.token_logprobs(rows, targets))


class _TokenLogprobs(torch.autograd.Function):
    """One read of the logits forward (one logit and a sum per row are kept), one read and one write backward."""

    @staticmethod
    def forward(ctx, logits, targets, vocab, ignore_index, temperature):
        logits, targets, logp, stats = _token_forward(logits, targets, vocab, ignore_index, temperature)
        ctx.save_for_backward(logits, targets, stats)
        ctx.cfg = (vocab, ignore_index, temperature)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        _backward_only("token_logprobs", dlogp)
        logits, targets, stats = ctx.saved_tensors
        vocab, ignore_index, temperature = ctx.cfg
        with _on(logits):
            logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
            coef = dlogp.float().contiguous()
            grad = O.empty_grad(logits)
            O.token_logprobs_grad(rows, stats, coef.data_ptr(), 1, None, grad)
        return grad, None, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100, temperature: float = 1.0,
                   vocab: Optional[int] = None) -> torch.Tensor:
    """FP32 log-probability of ``targets`` [...] under ``softmax(logits / temperature)``, logits [..., V(+pad)]; zero where the target is
    `ignore_index`.  Differentiable (once) with respect to the logits; any row strides, the innermost one 1 (others are copied)."""
    V = _check_logits("token_logprobs", logits, targets, vocab, temperature, ignore_index)
    if targets.numel() and _kernels(logits) and not _dual(logits):
        if _wants(logits):
            return _TokenLogprobs.apply(logits, targets, V, ignore_index, float(temperature))
        return _token_forward(logits, targets, V, ignore_index, temperature)[2]
    return _token_parts(logits, targets, ignore_index, temperature, V)[2].view(targets.shape)


def _linear_forward(hidden, weight, targets, vocab, ignore_index, temperature, want_grad, recompute):
    with _on(hidden):
        h = O.head_rows(hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1]))
        w, t = O.head_rows(weight), targets if targets.is_contiguous() else targets.contiguous()
        return t, *O.head_logprobs(h, w, t, vocab, ignore_index, 1.0 / temperature, want_grad, recompute)


class _LinearLogprobs(torch.autograd.Function):
    """The logits exist a tile at a time, in tensor memory; what the backward pass needs of them are their exponentials in 16 bits, or it makes
    them again."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, vocab, ignore_index, temperature, recompute):
        t, logp, block, weights = _linear_forward(hidden, weight, targets, vocab, ignore_index, temperature, True, recompute)
        ctx.save_for_backward(hidden, weight, t, block, weights)
        ctx.cfg = (vocab, ignore_index, temperature)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        _backward_only("linear_logprobs", dlogp)
        hidden, weight, t, block, weights = ctx.saved_tensors
        vocab, ignore_index, temperature = ctx.cfg
        again = torch._C._autograd._get_current_graph_task_keep_graph()
        with _on(hidden):
            h, w = O.head_rows(hidden.reshape(-1, hidden.shape[-1])), O.head_rows(weight)
            dh, dw = O.head_logprobs_grad(h, w, t, vocab, ignore_index, 1.0 / temperature, block, weights, dlogp.float().contiguous(),
                                          ctx.needs_input_grad[0], ctx.needs_input_grad[1], again)
        return (None if dh is None else dh.view(hidden.shape)), dw, None, None, None, None, None


def linear_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100, temperature: float = 1.0,
                    vocab: Optional[int] = None, recompute: bool = False) -> torch.Tensor:
    """`token_logprobs` of the logits ``hidden @ weight.T`` without the logits in memory: hidden [..., d], weight [V(+pad), d] of one type,
    targets [...].  Differentiable (once) with respect to both.

    Where a gradient is wanted, d is 512 or more and there are at most 2^29 logits (of at most 65536 tokens), their exponentials are held in
    16 bits (1 GiB at most) until the backward pass turns them into the logits' gradient in place.  Else, or with ``recompute``, nothing is held
    and the backward pass makes the logits again (a third more products), their gradient of at most 2^29 logits (or of 256 rows) at a time.

    The kernels take BF16 and FP16 with d a multiple of 8.  Log-probabilities come from logits in FP32 that are rounded nowhere.  The logits'
    gradient is rounded to the operands' type for its products, once with ``recompute``; from held exponentials twice, the exponential itself and
    its product with the row's coefficient.  FP32 and other widths go through the logits of a linear layer.  Under autocast the operands are cast
    as a linear layer's are."""
    name = "linear_logprobs"
    if hidden.is_cuda and torch.is_autocast_enabled("cuda") and hidden.is_floating_point() and weight.is_floating_point():
        dtype = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dtype), weight.to(dtype)
    if not torch.is_floating_point(hidden) or hidden.dim() < 1 or weight.dim() != 2 or weight.dtype != hidden.dtype:
        raise ValueError(f"{name}: hidden [..., d] and weight [V, d] must be floating-point tensors of one type")
    if weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"{name}: hidden has {hidden.shape[-1]} columns, weight {weight.shape[1]}")
    if weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError(f"{name}: hidden on {hidden.device}, weight on {weight.device}, targets on {targets.device}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: targets must be int32 or int64, got {targets.dtype}")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"{name}: targets {tuple(targets.shape)} do not match hidden {tuple(hidden.shape)}")
    _check_temperature(name, temperature)
    _check_ignored(name, ignore_index)
    V = weight.shape[0] if vocab is None else int(vocab)
    if not 1 <= V <= weight.shape[0]:
        raise ValueError(f"{name}: vocab must be between 1 and {weight.shape[0]}, got {V}")
    d, n = hidden.shape[-1], targets.numel()
    if n and d and d % 8 == 0 and hidden.dtype != torch.float32 and max(n, V) <= 1 << 30 and _kernels(hidden) and not _dual(hidden, weight):
        if _wants(hidden, weight):
            return _LinearLogprobs.apply(hidden, weight, targets, V, ignore_index, float(temperature), bool(recompute))
        return _linear_forward(hidden, weight, targets, V, ignore_index, temperature, False, False)[1]
    return token_logprobs(torch.nn.functional.linear(hidden, weight), targets, ignore_index, temperature, V)


# ---------------------------------------------------------------------------------------------------------- policy loss
def _policy_forward(logits, targets, vocab, ignore_index, temperature, old, args, want_grad):
    with _on(logits):
        logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
        grad = O.empty_grad(logits) if want_grad else None
        return O.policy_loss(rows, args, old, grad), grad


class _PolicyLossHalf(torch.autograd.Function):
    """FP16: a loss scale has to be in the gradient before it is rounded, so the gradient is made in the backward pass, from the logits and five
    values per row."""

    @staticmethod
    def forward(ctx, logits, targets, vocab, ignore_index, temperature, old, args):
        with _on(logits):
            logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
            slopes = old.new_empty(O.POLICY_SLOPE * rows.rows)
            loss, logp, kl, entropy = O.policy_loss(rows, args, old, None, slopes)
        ctx.save_for_backward(logits, targets, slopes)
        ctx.cfg = (vocab, ignore_index, temperature)
        ctx.mark_non_differentiable(logp, kl, entropy)
        ctx.set_materialize_grads(False)
        return loss, logp, kl, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 7
        _backward_only("policy_loss", dloss)
        logits, targets, slopes = ctx.saved_tensors
        vocab, ignore_index, temperature = ctx.cfg
        with _on(logits):
            logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
            grad = O.empty_grad(logits)
            O.policy_loss_grad(rows, slopes, dloss.float(), grad)
        return (grad, *(None,) * 6)


class _PolicyLoss(torch.autograd.Function):
    """Loss and gradient from one pass; the backward pass multiplies the gradient where the loss's own is not 1."""

    @staticmethod
    def forward(ctx, logits, targets, vocab, ignore_index, temperature, old, args):
        (loss, logp, kl, entropy), grad = _policy_forward(logits, targets, vocab, ignore_index, temperature, old, args, True)
        ctx.save_for_backward(grad)
        ctx.mark_non_differentiable(logp, kl, entropy)
        ctx.set_materialize_grads(False)
        return loss, logp, kl, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 7
        _backward_only("policy_loss", dloss)
        (grad,) = ctx.saved_tensors
        with _on(grad):
            # a graph that is kept may be walked again, and then needs the gradient as it was
            if torch._C._autograd._get_current_graph_task_keep_graph():
                grad = grad.clone()
            O.scale_unless_one_(grad, dloss.float())
        return (grad, *(None,) * 6)


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                ref_logp: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: Optional[float] = None, kl_coef: float = 0.0,
                kl: str = "k3", entropy_coef: float = 0.0, temperature: float = 1.0, reduction: str = "token", scale: float = 1.0,
                ignore_index: int = -100, vocab: Optional[int] = None) -> PolicyLoss:
    """Clipped policy loss of sampled tokens, from logits [B, T, V(+pad)] and their targets [B, T].

    Per token, with r = exp(logp - old_logp) and A its advantage: ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef KL -
    entropy_coef H``; KL is the estimate of the divergence from the reference (``ref_logp``) with d = ref_logp - logp: ``"k1"`` -d, ``"k2"``
    d^2 / 2, ``"k3"`` exp(d) - d - 1.  ``advantages`` [B, T], or [B] for one per sequence.  ``reduction``: ``"token"`` the mean over all tokens
    that count, ``"sequence"`` the mean over sequences (with such tokens) of the means over their tokens, ``"sum"``; times ``scale``.
    ``old_logp``, ``ref_logp`` and the advantages are constants.

    The gradient is made together with the loss, in one read of the logits; where the gradient of the loss itself is not 1 it is
    multiplied afterwards, so the factor of an accumulated micro-batch is better given as ``scale``.  With FP16 logits it is made in the
    backward pass, with a second read of them: a loss scale must be in it before it is rounded."""
    name = "policy_loss"
    V = _check_logits(name, logits, targets, vocab, temperature, ignore_index)
    if targets.dim() != 2:
        raise ValueError(f"{name}: logits must be [B, T, V] and targets [B, T]")
    B, T = targets.shape
    clip_high = clip_low if clip_high is None else clip_high
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0 and math.isfinite(clip_high)):
        raise ValueError(f"{name}: needs 0 <= clip_low <= 1 and clip_high >= 0")
    if kl not in ("k1", "k2", "k3"):
        raise ValueError(f"{name}: kl must be 'k1', 'k2' or 'k3'")
    if reduction not in ("token", "sequence", "sum"):
        raise ValueError(f"{name}: reduction must be 'token', 'sequence' or 'sum'")
    if not all(math.isfinite(v) for v in (kl_coef, entropy_coef, scale)):
        raise ValueError(f"{name}: kl_coef, entropy_coef and scale must be finite")
    if kl_coef != 0.0 and ref_logp is None:
        raise ValueError(f"{name}: a KL term needs ref_logp")
    old = _check_values(name, "old_logp", old_logp, [(B, T)], logits.device)
    adv = _check_values(name, "advantages", advantages, [(B, T), (B,)], logits.device)
    ref = None if ref_logp is None else _check_values(name, "ref_logp", ref_logp, [(B, T)], logits.device)
    if targets.numel() and _kernels(logits) and not _dual(logits):
        a = O.PolicyArgs(old.data_ptr(), None if ref is None else ref.data_ptr(), adv.data_ptr(), T if adv.dim() == 1 else 1, T, clip_low, clip_high,
                         kl_coef, entropy_coef, scale, O.KL[kl], O.MEAN[reduction], 0)
        if _wants(logits):
            form = _PolicyLossHalf if logits.dtype == torch.float16 else _PolicyLoss
            return PolicyLoss(*form.apply(logits, targets, V, ignore_index, float(temperature), old, a))
        return PolicyLoss(*_policy_forward(logits, targets, V, ignore_index, temperature, old, a, False)[0])
    keep, lp, logp = _token_parts(logits, targets, ignore_index, temperature, V)
    zero = torch.zeros((), dtype=lp.dtype, device=lp.device)
    p = lp.exp()
    ent = torch.where(keep, -(p * torch.where(p > 0, lp, zero)).sum(-1), zero)     # the product outside: the gradient of 0 * -inf is no number
    old, adv = old.to(lp.dtype).reshape(-1), (adv if adv.dim() == 2 else adv[:, None].expand(B, T)).to(lp.dtype).reshape(-1)
    moved = logp - old
    ratio = torch.exp(torch.where((adv == 0) & torch.isinf(torch.exp(moved.detach())), zero, moved))     # beyond the type, and counted zero times
    gain = torch.minimum(ratio * adv, ratio.clamp(1.0 - clip_low, 1.0 + clip_high) * adv)
    div = torch.zeros_like(logp)
    if ref is not None:
        d = ref.to(lp.dtype).reshape(-1) - logp
        div = {"k1": -d, "k2": 0.5 * d * d, "k3": torch.expm1(d) - d}[kl]
    per = -gain
    if kl_coef:               # an estimate that is only looked at may be infinite
        per = per + kl_coef * div
    per = torch.where(keep, per - entropy_coef * ent, zero)
    counts = keep.view(B, T).sum(-1)
    if reduction == "token":
        per = per / counts.sum().clamp(min=1)
    elif reduction == "sequence":
        per = per.view(B, T) / (counts.clamp(min=1)[:, None] * (counts > 0).sum().clamp(min=1))
    loss = (per.double().sum() * scale).to(lp.dtype)
    return PolicyLoss(loss, logp.detach().view(B, T), torch.where(keep, div, zero).detach().view(B, T), ent.detach().view(B, T))


# ------------------------------------------------------------------------------------------------------ preference loss
def _preference_forward(logits, targets, vocab, ignore_index, temperature, ref, options):
    with _on(logits):
        logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
        return (logits, targets, *O.preference_loss(rows, targets, ref, targets.shape[0] // 2, ignore_index, **options))


class _PreferenceLoss(torch.autograd.Function):
    """Forward: one read of the logits, then the pairs' losses and slopes; backward: one read and one write."""

    @staticmethod
    def forward(ctx, logits, targets, vocab, ignore_index, temperature, ref, options):
        logits, targets, loss, seq, margin, kept = _preference_forward(logits, targets, vocab, ignore_index, temperature, ref, options)
        ctx.save_for_backward(logits, targets, kept)
        ctx.cfg = (vocab, ignore_index, temperature)
        ctx.mark_non_differentiable(seq, margin)
        ctx.set_materialize_grads(False)
        return loss, seq, margin

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 7
        _backward_only("preference_loss", dloss)
        logits, targets, kept = ctx.saved_tensors
        vocab, ignore_index, temperature = ctx.cfg
        with _on(logits):
            logits, targets, rows = O.prepare_rows(logits, targets, vocab, ignore_index, 1.0 / temperature)
            grad = O.empty_grad(logits)
            O.token_logprobs_grad(rows, kept, kept.data_ptr() + 8 * rows.rows, targets.shape[1], dloss.float(), grad)
        return (grad, *(None,) * 6)


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logp: Optional[torch.Tensor] = None, beta: float = 0.1,
                    kind: str = "sigmoid", label_smoothing: float = 0.0, target_margin: float = 0.0, average: bool = False,
                    temperature: float = 1.0, ignore_index: int = -100, vocab: Optional[int] = None) -> PreferenceLoss:
    """Preference loss over pairs of sequences: logits [2 P, T, V(+pad)] and targets [2 P, T], the P chosen sequences first, then the P
    rejected ones in the same order (padding and prompts marked by `ignore_index`).

    A sequence's log-probability is the sum over its tokens (their mean with ``average``), its log-ratio that minus ``ref_logp`` [2 P]
    (none: without a reference), and with h the chosen log-ratio minus the rejected one and z = beta h - target_margin a pair's loss is
    ``"sigmoid"``: -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z); ``"hinge"``: max(0, 1 - z); ``"ipo"``:
    (h - 1 / (2 beta))^2.  The loss is the mean over the pairs."""
    name = "preference_loss"
    V = _check_logits(name, logits, targets, vocab, temperature, ignore_index)
    if targets.dim() != 2 or targets.shape[0] < 2 or targets.shape[0] % 2:
        raise ValueError(f"{name}: logits must be [2 P, T, V] and targets [2 P, T] with P >= 1 chosen sequences before P rejected ones")
    if kind not in ("sigmoid", "hinge", "ipo"):
        raise ValueError(f"{name}: kind must be 'sigmoid', 'hinge' or 'ipo'")
    if not (math.isfinite(beta) and beta > 0.0):
        raise ValueError(f"{name}: beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing < 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"{name}: label_smoothing must be in [0, 0.5), and belongs to the sigmoid loss")
    if not math.isfinite(target_margin) or (target_margin and kind == "ipo"):
        raise ValueError(f"{name}: target_margin must be finite, and does not belong to the ipo loss")
    pairs = targets.shape[0] // 2
    ref = None if ref_logp is None else _check_values(name, "ref_logp", ref_logp, [(2 * pairs,)], logits.device)
    if targets.numel() and _kernels(logits) and not _dual(logits):
        options = dict(kind=kind, average=bool(average), beta=beta, smoothing=label_smoothing, target_margin=target_margin)
        if _wants(logits):
            return PreferenceLoss(*_PreferenceLoss.apply(logits, targets, V, ignore_index, float(temperature), ref, options))
        return PreferenceLoss(*_preference_forward(logits, targets, V, ignore_index, temperature, ref, options)[2:5])
    keep, lp, logp = _token_parts(logits, targets, ignore_index, temperature, V)
    seq = logp.double().view(targets.shape).sum(-1)
    if average:
        seq = seq / keep.view(targets.shape).sum(-1).clamp(min=1)
    ratio = seq if ref is None else seq - ref.double()
    h = ratio[:pairs] - ratio[pairs:]
    z = beta * h - target_margin
    if kind == "sigmoid":
        each = (label_smoothing - 1.0) * torch.nn.functional.logsigmoid(z)
        if label_smoothing:      # of an infinite z, zero times the other side's logarithm is no number
            each = each - label_smoothing * torch.nn.functional.logsigmoid(-z)
    elif kind == "hinge":
        each = (1.0 - z).clamp(min=0.0)
    else:
        each = (h - 0.5 / beta) ** 2
    return PreferenceLoss(each.mean().to(lp.dtype), seq.detach().to(lp.dtype), h.detach().to(lp.dtype))


# --------------------------------------------------------------------------------------------- gradients of many tensors
def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill their memory without gaps or overlap, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _spans(ts) -> List[tuple]:
    return [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in ts]


def _grad_list(name: str, grads, out):
    """The tensors that count, without None, empty ones and repetitions; with `out`, the tensors their clipped values go to."""
    if out is not None:
        if len(out) != len(grads):
            raise ValueError(f"{name}: {len(grads)} gradients and {len(out)} outputs")
        pairs = [(g, o) for g, o in zip(grads, out) if g is not None]
        grads, out = [g for g, _ in pairs], [o for _, o in pairs]
    else:
        grads = [g for g in grads if g is not None]
    for t in grads if out is None else grads + out:
        if not torch.is_tensor(t) or t.layout != torch.strided or not t.is_floating_point():
            raise ValueError(f"{name}: takes dense floating-point tensors")
        if t.device != grads[0].device:
            raise ValueError(f"{name}: tensors on {t.device} and {grads[0].device}")
    for g in grads:
        if g.element_size() == 1:
            raise ValueError(f"{name}: gradients of {g.dtype} cannot be scaled")
    if out is not None:
        for g, o in zip(grads, out):
            if g.shape != o.shape:
                raise ValueError(f"{name}: output {tuple(o.shape)} of a gradient {tuple(g.shape)}")
    return grads, out


def _separate(name: str, grads, out):
    """Drops tensors listed twice (tied weights: they count and are clipped once); refuses other overlaps of memory."""
    loose = {i for i, g in enumerate(grads) if not _dense(g)}  # views with gaps may interleave: only repetitions are looked for
    seen, twice = {}, set()
    for i in loose:
        g = grads[i]
        if seen.setdefault((g.data_ptr(), g.shape, g.stride(), g.dtype), i) != i:
            twice.add(i)
    spans = _spans(grads)
    order = sorted((i for i in range(len(spans)) if i not in loose), key=spans.__getitem__)
    for a, b in zip(order, order[1:]):
        if spans[b][0] < spans[a][1]:
            if spans[a] != spans[b] or grads[a].stride() != grads[b].stride() or grads[a].dtype != grads[b].dtype:
                raise ValueError(f"{name}: two gradients share a part of their memory")
            twice.add(b)
    if out is not None:
        if twice:
            raise ValueError(f"{name}: a gradient is listed twice, with an output each")
        every = sorted([(s, 0, i) for i, s in enumerate(spans) if i not in loose] + [(s, 1, i) for i, s in enumerate(_spans(out)) if _dense(out[i])])
        for (s, ka, ia), (u, kb, ib) in zip(every, every[1:]):
            if u[0] < s[1] and not (ka != kb and ia == ib and s == u and grads[ia].dtype == out[ia].dtype):
                raise ValueError(f"{name}: an output shares memory with another tensor")
    if twice:
        grads = [g for i, g in enumerate(grads) if i not in twice]
    return grads


def _plain_table(grads, out):
    """The `grad_table` of a list that needs no second look: contiguous, non-empty tensors of one GPU that the kernels take, each with memory of its
    own.  None for every other list, wrong ones among them."""
    every = grads if out is None else grads + out
    try:
        if not every or not _kernels(every[0]) or len(set(map(torch.Tensor.get_device, every))) != 1:
            return None
        if not all(map(torch.Tensor.is_contiguous, every)):
            return None
        if out is not None and list(map(_shape, grads)) != list(map(_shape, out)):
            return None
        if not _KERNEL_SET.issuperset(map(_dtype, every)):     # FP8 has a type code too
            return None
        src, dst, counts, types = table = O.grad_table(grads, out)
    except (AttributeError, NotImplementedError, RuntimeError, TypeError):   # no tensors, or ones without plain memory
        return None
    spans = [(at, n * _BYTES[t & 15]) for at, n, t in zip(src, counts, types)]
    if dst is not None:
        spans += [(at, n * _BYTES[t >> 4]) for at, n, t in zip(dst, counts, types)]
    spans.sort()
    end = 0
    for at, size in spans:
        if at < end or size == 0:
            return None
        end = at + size
    return table


def _square_sum_plain(grads) -> float:
    sq = 0.0
    for g in grads:
        sq += float(g.double().pow(2).sum())
    return sq


def _kernel_list(grads) -> bool:
    return bool(grads) and all(g.dtype in _KERNEL_TYPES for g in grads) and _kernels(grads[0])


def _packed(t: torch.Tensor) -> torch.Tensor:
    return t if _dense(t) else t.contiguous()


def grad_square_sum(grads: Sequence[Optional[torch.Tensor]]) -> float:
    """Sum of squares of all elements in FP64, on the host (one synchronisation): the square of the global gradient norm.  Lists that the kernels do
    not take (sparse tensors, tensors of several devices or of other types) are summed a tensor at a time."""
    grads = [g for g in grads if g is not None]
    if not _kernel_list(grads) or any(g.layout != torch.strided or g.device != grads[0].device for g in grads):
        return _square_sum_plain(grads)
    with _on(grads[0]):
        ts = [_packed(g) for g in grads if g.numel()]
        return float(O.grad_clip(O.grad_table(ts), ts[0].device, None)[0]) if ts else 0.0


def clip_training_grads(grads: Sequence[torch.Tensor], max_norm: float) -> float:
    """Clips the gradients of a training step in place by their global norm and returns the sum of their squares (one synchronisation); where that is
    not finite they stay as they are.  Beside what `clip_grad_norm_` takes, gradients may be sparse, lie on several devices and share memory: such
    lists are summed and scaled a tensor at a time."""
    grads = list(grads)
    table = _plain_table(grads, None)
    if table is not None:
        return float(_clip_table(table, grads, None, max_norm)[0])
    sq = grad_square_sum(grads)
    if math.isfinite(sq):
        coef = min(1.0, max_norm / (math.sqrt(sq) + 1e-6))
        if coef < 1.0:
            with torch.no_grad():
                for g in grads:
                    g.mul_(coef)
    return sq


def _clip_table(table, grads, out, max_norm: float):
    with _on(grads[0]):
        norms = O.grad_clip(table, grads[0].device, max_norm)
    torch.autograd.graph.increment_version(grads if out is None else out)
    return norms


def clip_grads(name: str, grads, max_norm: float, out=None):
    """`clip_grad_norm_` with the FP64 sum of squares beside the FP32 norm."""
    if not max_norm >= 0.0:
        raise ValueError(f"{name}: max_norm must not be negative, got {max_norm}")
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    out = out if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    if forward_ad._current_level >= 0 and _dual(*(t for t in grads + (out or []) if isinstance(t, torch.Tensor))):
        raise NotImplementedError(f"{name}: has no forward-mode derivative")
    table = _plain_table(grads, out)
    if table is not None:
        return _clip_table(table, grads, out, max_norm)
    grads, out = _grad_list(name, grads, out)
    if not grads:
        return torch.zeros((), dtype=torch.float64), torch.zeros((), dtype=torch.float32)
    with torch.no_grad():
        every = [t for t in (grads if out is None else grads + out) if t.numel()]
        for t in every:
            if any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
                raise ValueError(f"{name}: a tensor whose elements share memory (expanded) cannot be clipped")
        if out is not None:
            kept = [(g, o) for g, o in zip(grads, out) if g.numel()]
            full, outs = [g for g, _ in kept], [o for _, o in kept]
        else:
            full, outs = [g for g in grads if g.numel()], None
        if not full:
            return tuple(torch.zeros((), dtype=dt, device=grads[0].device) for dt in (torch.float64, torch.float32))
        full = _separate(name, full, outs)
        if _kernel_list(full) and (outs is None or all(o.dtype in _KERNEL_TYPES for o in outs)):
            with _on(full[0]):
                src = [_packed(g) for g in full]
                if outs is None:
                    norms = O.grad_clip(O.grad_table(src), src[0].device, max_norm)
                    torch.autograd.graph.increment_version(src)
                    for g, s in zip(full, src):
                        if s is not g:
                            g.copy_(s)
                    return norms
                # element order of the memory: an output of another order than its gradient is written through a copy of that order
                dst = [o if o.stride() == s.stride() else torch.empty_like(s, dtype=o.dtype) for o, s in zip(outs, src)]
                norms = O.grad_clip(O.grad_table(src, dst), src[0].device, max_norm)
                torch.autograd.graph.increment_version(dst)
                for o, d in zip(outs, dst):
                    if d is not o:
                        o.copy_(d)
                return norms
        sq = _square_sum_plain(full)
        norm = math.sqrt(sq)
        coef = min(1.0, max_norm / (norm + 1e-6)) if math.isfinite(norm) else 1.0
        for i, g in enumerate(full):
            if outs is not None:
                if coef != 1.0:      # the product in a type that holds both (FP8: of the gradient)
                    g = (g if outs[i].element_size() == 1 else g.to(torch.promote_types(g.dtype, outs[i].dtype))) * coef
                outs[i].copy_(g)
            elif coef != 1.0:
                g.mul_(coef)
        return torch.tensor(sq, dtype=torch.float64), torch.tensor(norm, dtype=torch.float32, device=full[0].device)


def clip_grad_norm_(grads: Sequence[Optional[torch.Tensor]], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Clips gradients by their global norm |g| = sqrt(sum of the squares of all elements): every one times
    ``min(1, max_norm / (|g| + 1e-6))``, in place, or written to the tensors ``out`` (of the same shapes; their type may be another).
    Returns |g| as an FP32 scalar on the tensors' device, without a synchronisation; where it is not finite the gradients stay as they are
    (and are copied to ``out``), for the caller to skip the step.

    ``grads``: BF16, FP16 and FP32 tensors of one device in any mixture; None is left out, a tensor listed twice counts and is clipped once.
    Two launches per 256 tensors; nothing is written in place where the norm is small enough."""
    return clip_grads("clip_grad_norm_", grads, max_norm, out)[1]
