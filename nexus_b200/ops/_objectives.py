"""ctypes bindings of the kernels that fine-tune a language model on rewards and preferences (``nx_api_objectives.h``): log-probabilities
of given tokens, clipped policy loss, preference loss.  Workspaces are allocated per call: calls on several streams and captured graphs
share nothing."""
from __future__ import annotations

import ctypes as C
from array import array
from operator import attrgetter
from typing import Optional, Tuple

import torch

from . import _cuda as K

_functions = {}
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)     # the current stream's handle, without an object around it
_P, _I, _L, _F, _D = C.c_void_p, C.c_int, C.c_int64, C.c_float, C.c_double
_SIGNATURES = {
    "nx_token_logprobs": [_P, _P, _P, _P, _P, _P],
    "nx_token_logprobs_grad": [_P, _P, _P, _L, _P, _P, _P],
    "nx_policy_loss": [_P] * 12 + [_P],
    "nx_policy_loss_grad": [_P] * 5,
    "nx_scale_unless_one": [_P, _P, _I, _L, _P],
    "nx_preference_loss": [_P, _P, _P, _P, _P, _P],
    "nx_head_logprobs": [_P, _P, _P, _P],
    "nx_head_logprobs_grad": [_P, _P, _P],
    "nx_grad_clip": [_P, _D, _I, _P, _P, _P],
}


def _call(name: str, *args) -> None:
    """Calls a C entry point on the current stream with plain integers, floats and structures (their types are declared once: a wrapper per
    argument is a third of a microsecond, and these operators have small forms whose time is the host's)."""
    f = _functions.get(name)
    if f is None:
        f = getattr(K.lib(), name)
        f.argtypes, f.restype = _SIGNATURES[name], C.c_int
        _functions[name] = f
    K._check(f(*args, _stream(torch.cuda.current_device())), name)


KL = {"k1": 0, "k2": 1, "k3": 2}
MEAN = {"token": 0, "sequence": 1, "sum": 2}
PREFERENCE = {"sigmoid": 0, "hinge": 1, "ipo": 2}


class TokenRows(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("targets", C.c_void_p), ("rows", C.c_int64), ("per", C.c_int64), ("stride_outer", C.c_int64),
                ("stride_inner", C.c_int64), ("ignore_index", C.c_int64), ("dtype", C.c_int32), ("targets_wide", C.c_int32),
                ("vocab", C.c_int32), ("width", C.c_int32), ("inv_temp", C.c_float), ("pad_", C.c_int32)]


class PolicyArgs(C.Structure):
    _fields_ = [("old_logp", C.c_void_p), ("ref_logp", C.c_void_p), ("advantages", C.c_void_p), ("adv_per", C.c_int64),
                ("seq_len", C.c_int64), ("clip_low", C.c_float), ("clip_high", C.c_float), ("kl_coef", C.c_float),
                ("entropy_coef", C.c_float), ("scale", C.c_float), ("kl", C.c_int32), ("mean", C.c_int32), ("write_grad", C.c_int32)]


class PreferenceArgs(C.Structure):
    _fields_ = [("logp", C.c_void_p), ("targets", C.c_void_p), ("ref_logp", C.c_void_p), ("pairs", C.c_int64), ("seq_len", C.c_int64),
                ("ignore_index", C.c_int64), ("targets_wide", C.c_int32), ("kind", C.c_int32), ("average", C.c_int32), ("beta", C.c_float),
                ("smoothing", C.c_float), ("target_margin", C.c_float)]


def row_layout(x: torch.Tensor) -> Optional[Tuple[int, int, int]]:
    """(rows of an inner run, stride between runs, stride inside a run) of the rows of x [..., W] in elements; None where the rows are not
    of that form, overlap, or lie so far apart that a gradient of the same layout would waste more than it saves."""
    W = x.shape[-1]
    if x.numel() == 0 or (W > 1 and x.stride(-1) != 1):
        return None
    dims = []
    for size, stride in zip(x.shape[:-1], x.stride()[:-1]):
        if size == 1:
            continue
        if dims and dims[-1][1] == size * stride:
            dims[-1] = (dims[-1][0] * size, stride)
        else:
            dims.append((size, stride))
    if len(dims) > 2:
        return None
    (no, so), (ni, si) = ([(1, 0)] * (2 - len(dims)) + dims)
    if (ni > 1 and si < W) or (no > 1 and so < W):
        return None
    if no > 1 and ni > 1 and so < ni * si and si < no * so:
        return None
    if (no - 1) * so + (ni - 1) * si + W > 2 * no * ni * W:
        return None
    return ni, so, si


def prepare_rows(logits: torch.Tensor, targets: torch.Tensor, vocab: int, ignore_index: int, inv_temp: float):
    """(logits that the kernels read, targets, their description).  The returned tensors must outlive the calls."""
    W, n = logits.shape[-1], targets.numel()
    if logits.is_contiguous():
        lay = n, 0, W
    else:
        lay = row_layout(logits)
        if lay is None:
            logits = logits.contiguous()
            lay = n, 0, W
    if not targets.is_contiguous():
        targets = targets.contiguous()
    return logits, targets, TokenRows(logits.data_ptr(), targets.data_ptr(), n, lay[0], lay[1], lay[2], ignore_index, K._DT[logits.dtype],
                                      targets.dtype == torch.int64, vocab, W, inv_temp)


def empty_grad(logits: torch.Tensor) -> torch.Tensor:
    """A tensor of the layout of `logits` (as `prepare_rows` returned it) that starts at the same place of a 16-byte line."""
    off = logits.data_ptr() % 16 // logits.element_size()
    if off == 0 and logits.is_contiguous():
        return torch.empty_like(logits, requires_grad=False)
    extent = 1 + sum((n - 1) * s for n, s in zip(logits.shape, logits.stride()))
    buf = torch.empty(extent + off, dtype=logits.dtype, device=logits.device)
    return buf.as_strided(logits.shape, logits.stride(), off)


def token_logprobs(rows: TokenRows, like: torch.Tensor):
    """FP32 (logp of the shape of `like` (the contiguous targets), stats: two values per row)."""
    logp = torch.empty_like(like, dtype=torch.float32)
    stats = torch.empty(2 * rows.rows, dtype=torch.float32, device=like.device)
    _call("nx_token_logprobs", C.byref(rows), logp.data_ptr(), stats.data_ptr(), None, K.status_word(like.device).data_ptr())
    return logp, stats


def token_logprobs_grad(rows: TokenRows, stats, coef: int, coef_per: int, factor, grad) -> None:
    """`coef`: an address."""
    _call("nx_token_logprobs_grad", C.byref(rows), stats.data_ptr(), coef, coef_per, None if factor is None else factor.data_ptr(),
          grad.data_ptr())


POLICY_SLOPE = 5                 # FP32 values of a row that its gradient is made of


def policy_loss(rows: TokenRows, args: PolicyArgs, like: torch.Tensor, grad, slopes=None):
    """FP32 (loss, logp, kl, entropy) of the shape of `like` (contiguous FP32, a value per token); `grad` and `slopes` (or None) are written."""
    n, dev = rows.rows, like.device
    loss = like.new_empty(())
    logp, kl, entropy = torch.empty_like(like), torch.empty_like(like), torch.empty_like(like)
    scratch = torch.empty(24 + 4 * (n // args.seq_len) + 4 * n, dtype=torch.uint8, device=dev)   # totals, counts, the rows' losses
    at = scratch.data_ptr()
    args.write_grad = grad is not None
    _call("nx_policy_loss", C.byref(rows), C.byref(args), at, at + 24, logp.data_ptr(), kl.data_ptr(), entropy.data_ptr(),
          at + 24 + 4 * (n // args.seq_len), loss.data_ptr(), None if grad is None else grad.data_ptr(),
          None if slopes is None else slopes.data_ptr(), K.status_word(dev).data_ptr())
    return loss, logp, kl, entropy


def policy_loss_grad(rows: TokenRows, slopes, factor, grad) -> None:
    _call("nx_policy_loss_grad", C.byref(rows), slopes.data_ptr(), factor.data_ptr(), grad.data_ptr())


def scale_unless_one_(x: torch.Tensor, factor: torch.Tensor) -> None:
    """x *= factor in place, factor one FP32 value on the device; where it is 1, nothing is read or written.  x may have gaps, whose memory is its
    own (`empty_grad`): they are multiplied too."""
    n = x.numel() if x.is_contiguous() else 1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    _call("nx_scale_unless_one", x.data_ptr(), factor.data_ptr(), K._DT[x.dtype], n)


def preference_loss(rows: TokenRows, targets, ref_logp, pairs: int, ignore_index: int, *, kind: str, average: bool, beta: float,
                    smoothing: float, target_margin: float):
    """FP32 (loss, logp of the sequences [2 * pairs], margin [pairs]), and what the gradient needs: two values per row, behind them a slope per
    sequence."""
    n, dev = rows.rows, targets.device
    kept = torch.empty(2 * n + 2 * pairs, dtype=torch.float32, device=dev)
    loss, seq_logp, margin = kept.new_empty(()), kept.new_empty(2 * pairs), kept.new_empty(pairs)
    scratch = torch.empty(12 * n, dtype=torch.uint8, device=dev)        # log-probabilities in FP64 and in FP32
    wide, at = scratch.data_ptr(), kept.data_ptr()
    _call("nx_token_logprobs", C.byref(rows), wide + 8 * n, at, wide, K.status_word(dev).data_ptr())
    a = PreferenceArgs(wide, targets.data_ptr(), None if ref_logp is None else ref_logp.data_ptr(), pairs, n // (2 * pairs), ignore_index,
                       targets.dtype == torch.int64, PREFERENCE[kind], average, beta, smoothing, target_margin)
    _call("nx_preference_loss", C.byref(a), seq_logp.data_ptr(), margin.data_ptr(), at + 8 * n, loss.data_ptr())
    return loss, seq_logp, margin, kept


# ------------------------------------------------------------------------------------------- log-probabilities from hidden states
class HeadArgs(C.Structure):
    _fields_ = [("hidden", C.c_void_p), ("weight", C.c_void_p), ("targets", C.c_void_p), ("index", C.c_void_p), ("count", C.c_void_p),
                ("gathered", C.c_void_p), ("stats", C.c_void_p), ("part", C.c_void_p), ("weights", C.c_void_p), ("status", C.c_void_p),
                ("part_rows", C.c_int64), ("ld_weights", C.c_int64), ("rows", C.c_int64), ("ld_hidden", C.c_int64),
                ("ld_weight", C.c_int64), ("ignore_index", C.c_int64), ("vocab", C.c_int32), ("width", C.c_int32), ("dtype", C.c_int32),
                ("targets_wide", C.c_int32), ("inv_temp", C.c_float), ("pad_", C.c_int32)]


class HeadGrad(C.Structure):
    _fields_ = [("coef", C.c_void_p), ("logit_grad", C.c_void_p), ("chunk", C.c_int64), ("ld_logit_grad", C.c_int64), ("scale", C.c_void_p),
                ("d_hidden", C.c_void_p), ("d_weight", C.c_void_p), ("slice_sums", C.c_void_p), ("weight_sums", C.c_void_p),
                ("slices", C.c_int32), ("pad_", C.c_int32)]


HEAD_TILE = 256
HEAD_PARTS = 2                   # maxima and sums of a row that a column tile leaves
HEAD_ROWS = 1 << 16              # rows whose column tiles' maxima and sums are in memory at a time
HEAD_GRAD_ELEMENTS = 1 << 29     # of the logits' gradient at a time: 1 GiB
# From this width on the exponentials are held: writing them and turning them into the gradient is traffic per logit, making the logits again
# work per logit and column.  Forward and backward pass, held and again, us: 4096 x 50257 BF16 at 256 columns 549 and 540, 384 682 and 679, 512 711
# and 741, 1024 1084 and 1207, 2048 2010 and 2327; 380 x 151936 FP16 at 896 columns 435 and 487.
HEAD_KEEP_WIDTH = 512


def head_rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix as the tensor maps take it: contiguous rows on 16-byte boundaries; copied if it is not one."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _head_args(hidden, weight, targets, index, moved, stats: int, part, weights, vocab: int, ignore_index: int, inv_temp: float) -> HeadArgs:
    """`index` (the rows that count and behind them their number), `moved`, `stats`, `part`: addresses."""
    rows, width = hidden.shape
    held, ld = (None, 0) if weights is None else (weights.data_ptr(), weights.stride(0))
    return HeadArgs(hidden.data_ptr(), weight.data_ptr(), targets.data_ptr(), index, None if index is None else index + 4 * rows, moved, stats, part,
                    held, K.status_word(hidden.device).data_ptr(), _part_rows(rows), ld, rows, hidden.stride(0), weight.stride(0), ignore_index,
                    vocab, width, K._DT[hidden.dtype], targets.dtype == torch.int64, inv_temp, 0)


def _part_rows(rows: int) -> int:
    return min(HEAD_ROWS, -(-rows // HEAD_TILE) * HEAD_TILE)


def _head_pitch(vocab: int) -> int:
    return (vocab + 63) // 64 * 64


class _Block:
    """Places of a scratch block: 256-byte boundaries, handed out before the block is allocated."""

    def __init__(self):
        self.size = 0

    def take(self, nbytes: int) -> int:
        at, self.size = self.size, self.size + (nbytes + 255) // 256 * 256
        return at

    def allocate(self, device) -> torch.Tensor:
        return torch.empty(self.size, dtype=torch.uint8, device=device)


def head_logprobs(hidden, weight, targets, vocab: int, ignore_index: int, inv_temp: float, want_grad: bool, recompute: bool = False):
    """FP32 logp (of the shape of `targets`) for hidden [rows, width] and weight [>= vocab, width] (`head_rows` of both), and what the gradient
    needs, None where it is not wanted: a block with the statistics and the rows that count, and the logits' exponentials where these are held
    (the block then has their column tiles' maxima and the gathered rows too)."""
    rows, width = hidden.shape
    dev = hidden.device
    logp = torch.empty_like(targets, dtype=torch.float32)
    full, ld = -(-rows // HEAD_TILE) * HEAD_TILE, _head_pitch(vocab)
    keep = want_grad and not recompute and rows <= HEAD_ROWS and width >= HEAD_KEEP_WIDTH and full * ld <= HEAD_GRAD_ELEMENTS
    parts, gathered = 8 * HEAD_PARTS * -(-vocab // HEAD_TILE) * _part_rows(rows), (rows + 63) // 64 * 64 * width * 2
    kept, scratch = _Block(), _Block()
    stats = kept.take(8 * rows)
    index = kept.take(4 * rows + 4) if want_grad or rows > HEAD_TILE else None
    part = (kept if keep else scratch).take(parts)
    moved = None if index is None else (kept if keep else scratch).take(gathered)
    tlogit = scratch.take(4 * rows)
    if not want_grad:                     # one block
        shift = scratch.take(kept.size)
        block = scratch.allocate(dev)
        at = block.data_ptr()
        base = at + shift
    else:
        block, rest = kept.allocate(dev), scratch.allocate(dev)
        base, at = block.data_ptr(), rest.data_ptr()
    other = base if keep else at
    weights = torch.empty((full, ld), dtype=hidden.dtype, device=dev) if keep else None
    a = _head_args(hidden, weight, targets, None if index is None else base + index, None if moved is None else other + moved, base + stats,
                   other + part, weights, vocab, ignore_index, inv_temp)
    _call("nx_head_logprobs", C.byref(a), logp.data_ptr(), at + tlogit)
    return logp, (block if want_grad else None), weights


def head_slices(rows: int, width: int) -> int:
    """Pieces that the vocabulary may be cut into for a hidden-state gradient [rows, width] (how many it is, the kernels decide by the rows that
    count): none where its tiles alone give every pair of SMs two, else up to 16 whose FP32 sums stay below 128 MiB."""
    tiles = -(-rows // HEAD_TILE) * -(-width // HEAD_TILE)
    if tiles >= 2 * 74:
        return 1
    return max(1, min(16, (1 << 25) // (-(-rows // HEAD_TILE) * HEAD_TILE * width)))


def head_logprobs_grad(hidden, weight, targets, vocab: int, ignore_index: int, inv_temp: float, block, weights, coef, want_hidden: bool,
                       want_weight: bool, again: bool = False):
    """(d_hidden [rows, width], d_weight [all rows of weight, width]), either None where not wanted.  The exponentials become the gradient of the
    logits in place, unless they are needed `again`."""
    rows, width = hidden.shape
    dev, dtype = hidden.device, hidden.dtype
    kept, scratch = _Block(), _Block()
    stats, index = kept.take(8 * rows), kept.take(4 * rows + 4)
    parts, gathered = 8 * HEAD_PARTS * -(-vocab // HEAD_TILE) * _part_rows(rows), (rows + 63) // 64 * 64 * width * 2
    base, ld, chunk = block.data_ptr(), _head_pitch(vocab), -(-rows // HEAD_TILE) * HEAD_TILE
    if weights is not None:
        part, moved = base + kept.take(parts), base + kept.take(gathered)
        grad_at = scratch.take(2 * chunk * ld) if again else None
    else:
        chunk = min(chunk, max(HEAD_TILE, HEAD_GRAD_ELEMENTS // ld // HEAD_TILE * HEAD_TILE))
        part, moved, grad_at = None, scratch.take(gathered), scratch.take(2 * chunk * ld)
    scale = scratch.take(8)
    slices = head_slices(min(rows, chunk), width) if want_hidden else 1
    slice_sums = scratch.take(4 * slices * chunk * width) if slices > 1 else None
    weight_sums = scratch.take(4 * vocab * width) if want_weight and chunk < rows else None
    rest = scratch.allocate(dev)
    at = rest.data_ptr()
    if weights is None:
        moved += at
    dh = torch.empty((rows, width), dtype=dtype, device=dev) if want_hidden else None
    dw = torch.empty((weight.shape[0], width), dtype=dtype, device=dev) if want_weight else None
    if want_weight and weight.shape[0] > vocab:
        dw[vocab:].zero_()
    a = _head_args(hidden, weight, targets, base + index, moved, base + stats, part, weights, vocab, ignore_index, inv_temp)
    g = HeadGrad(coef.data_ptr(), weights.data_ptr() if grad_at is None else at + grad_at, chunk, ld, at + scale,
                 None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr(), None if slice_sums is None else at + slice_sums,
                 None if weight_sums is None else at + weight_sums, slices, 0)
    _call("nx_head_logprobs_grad", C.byref(a), C.byref(g))
    return dh, dw


# ---------------------------------------------------------------------------------------------------- gradients of many tensors
class GradTable(C.Structure):
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("count", C.c_void_p), ("type", C.c_void_p), ("tensors", C.c_int64)]


GRAD_TABLE = 256                 # tensors of a launch, and
GRAD_PARTS = 4 * 148             # partial sums that it leaves, at most


_ptr, _numel, _dtype = torch.Tensor.data_ptr, torch.Tensor.numel, attrgetter("dtype")


def grad_table(grads, out=None):
    """Pointers, numbers of elements and types of dense tensors, as `grad_clip` takes them: (sources, destinations or None, counts, types)."""
    code = K._DT.__getitem__
    src, counts, kinds = list(map(_ptr, grads)), list(map(_numel, grads)), list(map(code, map(_dtype, grads)))
    if out is None:
        return src, None, counts, bytes([17 * c for c in kinds])
    return src, list(map(_ptr, out)), counts, bytes([c | o << 4 for c, o in zip(kinds, map(code, map(_dtype, out)))])


def grad_clip(table, device, max_norm: Optional[float]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(FP64 sum of squares, FP32 norm) of the dense, non-empty tensors of a `grad_table`; with `max_norm` they are clipped, in place or into their
    destinations."""
    src, dst, counts, types = table
    n = len(src)
    src, counts, dst = array("Q", src), array("q", counts), None if dst is None else array("Q", dst)
    buf = torch.empty(2 + -(-n // GRAD_TABLE) * GRAD_PARTS, dtype=torch.float64, device=device)
    a = GradTable(src.buffer_info()[0], None if dst is None else dst.buffer_info()[0], counts.buffer_info()[0],
                  C.cast(C.c_char_p(types), C.c_void_p), n)
    at = buf.data_ptr()
    _call("nx_grad_clip", C.byref(a), 0.0 if max_norm is None else max_norm, max_norm is not None, at + 16, at)
    return buf[0], buf.view(torch.float32)[2]
