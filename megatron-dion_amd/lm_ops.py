"""The training operators around the optimizer: output-layer loss, residual norm, dropout.

The optimizer consumes gradients; these make those of the parameters its elementwise branch updates
(the output layer and the norms), in hand-written HIP kernels (csrc/lm/, C ABI in include/dion_lm.h).
They take the place of what a Megatron model without biases calls there: the vocabulary-parallel cross
entropy after its output layer, the dropout-add before a norm, and the norm itself.

Each operator is a pair of explicit calls, forward and backward, that run on the current HIP stream of
the tensors' device, allocate their results and scratch from torch's caching allocator, never wait for
the GPU and can be captured into a graph.  `lm_autograd.py` wraps them for autograd.

Tensors are float32 or bfloat16 of any leading shape, with unit stride along the last axis, the
leading axes evenly strided and rows that do not overlap (an expanded axis is refused); anything else
raises ``RuntimeError("[DION_...] ...")`` before any work is enqueued.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.distributed as dist

from . import _lib, _lm_lib

__all__ = ["linear_cross_entropy_forward", "linear_cross_entropy_backward", "rms_norm_add_forward",
           "rms_norm_add_backward", "dropout_add_forward", "dropout_add_backward", "RmsNormAdd", "RmsNormAddGrads"]

Rng = Union[Tuple[int, int], torch.Tensor]
_U64 = (1 << 64) - 1
_CODE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_byref = ctypes.byref


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _CODE.get(t.dtype)
    if code is None:
        raise RuntimeError(f"[DION_UNSUPPORTED_DTYPE] {what}: {t.dtype}")
    return code


def _rows(t: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """(rows, cols, row stride) of `t` read as a matrix, without a copy."""
    shape = t.shape
    if not shape:
        raise RuntimeError(f"[DION_BAD_SHAPE] {what} has no axis")
    if not t.is_cuda:
        raise RuntimeError(f"[DION_BAD_DEVICE] {what} is on {t.device}")
    cols = shape[-1]
    if t.is_contiguous():
        return (t.numel() // cols if cols else 0), cols, cols
    strides = t.stride()
    rows, ld, ok = 1, 0, cols <= 1 or strides[-1] == 1
    for n, st in zip(reversed(shape[:-1]), reversed(strides[:-1])):  # the leading axes have to fold into one
        if n != 1:
            ok = ok and (st == rows * ld if ld else st >= cols)
            ld = ld or st
            rows *= n
    if not ok and t.numel():
        raise RuntimeError(f"[DION_NON_ROW_MAJOR] {what}: shape={tuple(shape)} stride={strides}")
    return rows, cols, ld or cols


def _fits(bits: int, **sizes: int) -> None:
    """What goes into a descriptor's field of `bits` bits, which would keep the low ones of a larger number."""
    for what, n in sizes.items():
        if not -(1 << (bits - 1)) <= n < 1 << (bits - 1):
            raise RuntimeError(f"[DION_BAD_SIZE] {what}={n} does not fit {bits} bits")


def _like(t: torch.Tensor, what: str, like: torch.Tensor) -> int:
    """The row stride of `t`, which has to be a tensor like `like`."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] {what}: {tuple(t.shape)} {t.dtype} {t.device}, expected "
                           f"{tuple(like.shape)} {like.dtype} {like.device}")
    return _rows(t, what)[2]


def _empty(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _stream_of(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same without a Stream object in between, where this torch has it: a microsecond of a small call's eight
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream_of)
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(fn, device: torch.device, *args) -> int:
    """`fn(*args, stream)` on the current stream of `device`, which need not be the current device."""
    index = device.index
    if index == _device():
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return fn(*args, _raw_stream(index))


def _workspace(nbytes: int, device) -> torch.Tensor:
    # a call's own memory, from the caching allocator: calls on different streams and captured graphs
    # never share it
    return torch.empty(nbytes if nbytes > 16 else 16, dtype=torch.uint8, device=device)


def _rng(p: float, rng: Optional[Rng], device) -> Optional[_lm_lib.DionRng]:
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"[DION_BAD_DROPOUT] p={p} is not in 0 .. 1")
    if p == 0.0:
        return None
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or rng.numel() != 2 or rng.device != device or not rng.is_contiguous():
            raise RuntimeError(f"[DION_BAD_DROPOUT] rng tensor: two contiguous int64 on {device}, got "
                               f"{tuple(rng.shape)} {rng.dtype} {rng.device}")
        return _lm_lib.DionRng(0, 0, rng.data_ptr())
    if rng is None:
        raise RuntimeError("[DION_BAD_DROPOUT] p > 0 needs rng=(seed, offset)")
    seed, offset = rng
    return _lm_lib.DionRng(int(seed) & _U64, int(offset) & _U64, None)


def _ref(s):
    return None if s is None else _byref(s)


# ------------------------------------------------------------------------------- dropout
def dropout_add_forward(x: torch.Tensor, residual: Optional[torch.Tensor] = None, *, p: float,
                        rng: Optional[Rng] = None) -> torch.Tensor:
    """`residual + dropout(x)` (without `residual`: `dropout(x)`), the mask never stored.

    Philox4x32-10 with key `seed` and counter `(e // 4, offset)`: element e of x (row-major) keeps its
    value, times fp32(1 / (1 - p)), iff word `e % 4` is at least p 2^32, else becomes 0 (also a NaN or an
    infinity).  `rng` is `(seed, offset)`, or an int64 tensor holding them on x's device, which a
    captured graph reads again at each replay.  A (seed, offset) pair is to be used for one mask only:
    count `offset` over layers, steps and ranks."""
    rows, cols, ld = _rows(x, "x")
    ld_r = 0 if residual is None else _like(residual, "residual", x)
    code = _dtype(x, "x")
    device = x.device
    r = _rng(p, rng, device)
    out = _empty(x)
    rc = _call(_lm_lib.load().dion_dropout_add, device, rows, cols, code, x.data_ptr(), ld,
               None if residual is None else residual.data_ptr(), ld_r, out.data_ptr(), cols, p, _ref(r))
    if rc:
        _lm_lib.check(rc, "dion_dropout_add")
    return out


def dropout_add_backward(grad_out: torch.Tensor, *, p: float, rng: Optional[Rng] = None) -> torch.Tensor:
    """Gradient of x: the forward's mask (same `p` and `rng`) on `grad_out`.  The residual's gradient
    is `grad_out` itself."""
    return dropout_add_forward(grad_out, None, p=p, rng=rng)


# ------------------------------------------------------------------------------- residual RMS norm
class RmsNormAdd(NamedTuple):
    y: torch.Tensor                 # x's dtype, or float8_e4m3fn
    h: torch.Tensor                 # the residual stream after the addition (x itself if nothing is added)
    rstd: torch.Tensor              # fp32, one a row
    scale: Optional[torch.Tensor]   # fp32, one a block of columns (8-bit y only)


class RmsNormAddGrads(NamedTuple):
    grad_x: Optional[torch.Tensor]
    grad_residual: Optional[torch.Tensor]  # grad_x's own tensor where there is no dropout
    grad_weight: Optional[torch.Tensor]


@functools.lru_cache(maxsize=512)
def _norm_desc(rows, cols, dtype, w_dtype, gw_dtype, y_dtype, scale_block, accumulate, eps, p, *lds):
    """The descriptor of a call (read only: calls of the same shapes share it) and its scratch."""
    _fits(32, cols=cols)
    d = _lm_lib.DionNormDesc(rows, cols, dtype, w_dtype, gw_dtype, y_dtype, scale_block, accumulate, eps, p, *lds)
    nbytes = ctypes.c_size_t(0)
    _lm_lib.check(_lm_lib.load().dion_rms_norm_add_workspace_bytes(_byref(d), _byref(nbytes)),
                  "dion_rms_norm_add_workspace_bytes")
    return d, int(nbytes.value)


def _norm_weight(weight: torch.Tensor, cols: int, device) -> int:
    if weight.shape != (cols,) or weight.device != device or not weight.is_contiguous():
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] weight: {tuple(weight.shape)} {weight.device}, expected "
                           f"({cols},) on {device}")
    return _dtype(weight, "weight")


def rms_norm_add_forward(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                         eps: float = 1e-5, p: float = 0.0, rng: Optional[Rng] = None,
                         scale_block: int = 0) -> RmsNormAdd:
    """`h = residual + dropout(x)`, rounded to x's dtype; `y = h * rsqrt(mean(h^2) + eps) * weight`.

    Rows of up to 16384 columns.  `scale_block` > 0 (at least 8, or all columns; -1: one block a row): y
    is float8_e4m3fn, each block of that many columns over its own fp32 `scale` = max |y| / 448 (at least
    2^-126), so that `y.float() * scale` restores it.  Dropout as in `dropout_add_forward`."""
    rows, cols, ld = _rows(x, "x")
    ld_r = 0 if residual is None else _like(residual, "residual", x)
    device = x.device
    code, w_code = _dtype(x, "x"), _norm_weight(weight, cols, device)
    r = _rng(p, rng, device)
    stored = residual is not None or r is not None
    shape = x.shape[:-1]
    if scale_block:
        block = cols if scale_block < 0 or scale_block > cols else int(scale_block)
        d, _ = _norm_desc(rows, cols, code, w_code, w_code, _lm_lib.DTYPE_E4M3, block, 0, float(eps), float(p),
                          ld, ld_r, cols, cols)
        scale = torch.empty(shape + (-(-cols // block),), dtype=torch.float32, device=device)
        y = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=device)
    else:
        d, _ = _norm_desc(rows, cols, code, w_code, w_code, code, 0, 0, float(eps), float(p), ld, ld_r, cols, cols)
        scale, y = None, _empty(x)
    h = _empty(x) if stored else x
    rstd = torch.empty(shape, dtype=torch.float32, device=device)
    rc = _call(_lm_lib.load().dion_rms_norm_add, device, _byref(d), x.data_ptr(),
               None if residual is None else residual.data_ptr(), weight.data_ptr(), h.data_ptr() if stored else None,
               y.data_ptr(), None if scale is None else scale.data_ptr(), rstd.data_ptr(), _ref(r))
    if rc:
        _lm_lib.check(rc, "dion_rms_norm_add")
    return RmsNormAdd(y, h, rstd, scale)


def _grad_weight(weight: torch.Tensor, out: Optional[torch.Tensor], accumulate: bool, what: str) -> torch.Tensor:
    if out is None:
        if accumulate:
            raise RuntimeError(f"[DION_BAD_GRAD_OUT] accumulate needs {what}")
        return _empty(weight)
    if out.shape != weight.shape or out.device != weight.device:
        raise RuntimeError(f"[DION_BAD_GRAD_OUT] {what}: {tuple(out.shape)} {out.device}, expected "
                           f"{tuple(weight.shape)} {weight.device}")
    return out


def rms_norm_add_backward(grad_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                          grad_h: Optional[torch.Tensor] = None, *, p: float = 0.0, rng: Optional[Rng] = None,
                          grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                          need_input: bool = True, need_weight: bool = True, need_residual: bool = True
                          ) -> RmsNormAddGrads:
    """Gradients of `rms_norm_add_forward`; `grad_h` is what reaches h past the norm (the residual
    stream's gradient), `p` and `rng` are the forward's.  An 8-bit y passes `grad_y` (x's dtype) as if
    it had not been rounded.  `grad_weight` (fp32 or bf16, e.g. `weight.main_grad`) is written, or with
    `accumulate` added to; without it a new tensor of weight's dtype is returned.  `need_input` asks for
    grad_x and, with `need_residual`, for grad_residual."""
    rows, cols, ld = _rows(h, "h")
    ld_gy = _like(grad_y, "grad_y", h)
    ld_gh = 0 if grad_h is None else _like(grad_h, "grad_h", h)
    device = h.device
    code, w_code = _dtype(h, "h"), _norm_weight(weight, cols, device)
    r = _rng(p, rng, device)
    if rstd.dtype != torch.float32 or rstd.shape != h.shape[:-1] or not rstd.is_contiguous() or rstd.device != device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] rstd: {tuple(rstd.shape)} {rstd.dtype} {rstd.device}")
    gx = gr = gw = ws = None
    gw_code = w_code
    if need_weight:
        gw = _grad_weight(weight, grad_weight, accumulate, "grad_weight")
        if not gw.is_contiguous():
            raise RuntimeError(f"[DION_BAD_GRAD_OUT] grad_weight stride={gw.stride()}")
        gw_code = _dtype(gw, "grad_weight")
    d, nbytes = _norm_desc(rows, cols, code, w_code, gw_code, code, 0, int(bool(accumulate)), 0.0, float(p), 0, 0, ld, 0,
                           ld_gy, ld_gh, cols, cols)
    if need_input:
        gx = _empty(h)
        if r is not None and need_residual:
            gr = _empty(h)
    if need_weight:
        ws = _workspace(nbytes, device)
    rc = _call(_lm_lib.load().dion_rms_norm_add_backward, device, _byref(d), grad_y.data_ptr(), h.data_ptr(),
               weight.data_ptr(), rstd.data_ptr(), None if grad_h is None else grad_h.data_ptr(),
               None if gx is None else gx.data_ptr(), None if gr is None else gr.data_ptr(),
               None if gw is None else gw.data_ptr(), _ref(r), None if ws is None else ws.data_ptr(),
               0 if ws is None else nbytes if nbytes > 16 else 16)
    if rc:
        _lm_lib.check(rc, "dion_rms_norm_add_backward")
    return RmsNormAddGrads(gx, gr if r is not None else gx if need_residual else None, gw)


# ------------------------------------------------------------------------------- linear cross entropy
@functools.lru_cache(maxsize=512)
def _xent_shape(op, tokens, hidden, vocab, dtype, gw_dtype, accumulate, pack_weight, start, total, ignore, ld_hidden,
                ld_weight, ld_grad_weight, piece_bytes):
    """The descriptor of a call (read only: calls of the same shapes share it) and its scratch."""
    _fits(32, hidden=hidden, vocab=vocab)
    _fits(64, vocab_start=start, vocab_size=total, ignore_index=ignore, piece_bytes=piece_bytes)
    d = _lm_lib.DionXentDesc(tokens, hidden, vocab, dtype, gw_dtype, accumulate, pack_weight, start, total, ignore,
                             ld_hidden, ld_weight, hidden, ld_grad_weight, piece_bytes)
    nbytes = ctypes.c_size_t(0)
    _lm_lib.check(_lm_lib.load().dion_xent_workspace_bytes(_byref(d), op, _byref(nbytes)),
                  "dion_xent_workspace_bytes")
    return d, int(nbytes.value)


def _xent_desc(op, hidden, weight, target, vocab_start, vocab_size, ignore_index, grad_weight=None, accumulate=False,
               piece_bytes=0):
    """The descriptor and scratch of a call, None if the weight holds no word of the vocabulary."""
    tokens, cols, ld_h = _rows(hidden, "hidden")
    if weight.dim() != 2 or weight.shape[1] != cols or weight.dtype != hidden.dtype or weight.device != hidden.device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] hidden {tuple(hidden.shape)} {hidden.dtype} {hidden.device}, "
                           f"weight {tuple(weight.shape)} {weight.dtype} {weight.device}")
    rows, _, ld_w = _rows(weight, "weight")
    if target.dtype != torch.int64 or target.shape != hidden.shape[:-1] or target.device != hidden.device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] target: int64 {tuple(hidden.shape[:-1])} on {hidden.device} "
                           f"expected, got {target.dtype} {tuple(target.shape)} {target.device}")
    code = _dtype(hidden, "hidden")
    start = int(vocab_start)
    total = start + rows if vocab_size is None else int(vocab_size)
    if start < 0 or total < 1:
        raise RuntimeError(f"[DION_BAD_VOCAB] weight of {rows} rows from word {start} on, of {total}")
    vocab = min(rows, total - start)  # rows past the vocabulary are padding
    gw_code, ld_gw = code, cols
    if grad_weight is not None:
        gw_code, ld_gw = _dtype(grad_weight, "grad_weight"), _rows(grad_weight, "grad_weight")[2]
    if vocab < 1:
        return None, 0
    return _xent_shape(op, tokens, cols, vocab, code, gw_code, int(bool(accumulate)), int(weight.data_ptr() % 16 != 0),
                       start, total, int(ignore_index), ld_h, ld_w, ld_gw, int(piece_bytes))


def combine_vocab_shards(lse: torch.Tensor, tlogit: torch.Tensor, ignored: torch.Tensor, group):
    """(loss, lse) of the whole vocabulary from each shard's lse and target logit: a maximum and a sum
    over `group` (two small all-reduces)."""
    top = lse.clone()
    dist.all_reduce(top, op=dist.ReduceOp.MAX, group=group)
    safe = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    both = torch.stack((torch.exp(lse - safe), tlogit))
    dist.all_reduce(both, op=dist.ReduceOp.SUM, group=group)
    lse = torch.where(ignored, torch.zeros_like(top), safe + torch.log(both[0]))
    return torch.where(ignored, torch.zeros_like(top), lse - both[1]), lse


def _sum_over_shards(grad_hidden: Optional[torch.Tensor], group) -> Optional[torch.Tensor]:
    if group is not None and grad_hidden is not None:
        with torch.cuda.device(grad_hidden.device):
            dist.all_reduce(grad_hidden, op=dist.ReduceOp.SUM, group=group)
    return grad_hidden


def linear_cross_entropy_forward(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                                 vocab_start: int = 0, vocab_size: Optional[int] = None, ignore_index: int = -100,
                                 group=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, lse), fp32 of target's shape: the cross entropy of `hidden @ weight.T` at each token and
    the logarithm of its softmax's denominator (for the backward pass).  The logits are never stored.

    hidden (..., H) and weight (V, H) are bf16 or fp32 alike, target int64; up to 2^24 tokens, H 2^20, V
    2^21.  An infinity in fp32 inputs makes the logits it meets NaN (they are split into limbs).  A token whose target is
    `ignore_index` costs nothing: its loss and lse are 0 and its hidden state is not read.  Any other
    target outside the vocabulary gives a NaN loss.

    Vocabulary shards (tensor parallel): weight holds the rows from `vocab_start` on of a vocabulary of
    `vocab_size` words (rows past it are padding), `group` the ranks that share it; every rank passes the
    same hidden states and targets and gets the whole vocabulary's loss.  A rank all of whose rows are
    padding takes part as the others do.  A shard without `group` is refused: it has no loss."""
    if group is not None and vocab_size is None:
        raise RuntimeError("[DION_BAD_VOCAB] a vocabulary in shards needs vocab_size, the words of all of them")
    d, nbytes = _xent_desc(_lm_lib.XENT_FORWARD, hidden, weight, target, vocab_start, vocab_size, ignore_index)
    device = hidden.device
    if group is None and (d is None or d.vocab < d.vocab_total):
        raise RuntimeError(f"[DION_BAD_VOCAB] weight of {weight.shape[0]} rows from word {int(vocab_start)} on holds a "
                           "part of the vocabulary: its loss needs group")
    if d is None:
        # the other ranks of the group wait in its reductions
        lse = torch.full(target.shape, float("-inf"), dtype=torch.float32, device=device)
        with torch.cuda.device(device):
            return combine_vocab_shards(lse, torch.zeros_like(lse), target == ignore_index, group)
    target = target.contiguous()
    ws = _workspace(nbytes, device)
    loss = torch.empty(target.shape, dtype=torch.float32, device=device)
    lse = torch.empty_like(loss)
    tlogit = loss if group is not None else None
    rc = _call(_lm_lib.load().dion_xent_forward, device, _byref(d), hidden.data_ptr(), weight.data_ptr(),
               target.data_ptr(), loss.data_ptr() if tlogit is None else None, lse.data_ptr(),
               None if tlogit is None else tlogit.data_ptr(), ws.data_ptr(), ws.numel())
    if rc:
        _lm_lib.check(rc, "dion_xent_forward")
    if group is None:
        return loss, lse
    with torch.cuda.device(device):
        return combine_vocab_shards(lse, tlogit, target == ignore_index, group)


def linear_cross_entropy_backward(grad_loss: torch.Tensor, hidden: torch.Tensor, weight: torch.Tensor,
                                  target: torch.Tensor, lse: torch.Tensor, *, vocab_start: int = 0,
                                  vocab_size: Optional[int] = None, ignore_index: int = -100, group=None,
                                  grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                                  need_hidden: bool = True, need_weight: bool = True, piece_bytes: int = 0
                                  ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(grad_hidden, grad_weight) for the upstream gradient `grad_loss` (fp32, target's shape).

    The logits are made again a piece of the vocabulary at a time; at most `piece_bytes` (0: 1 GiB) of
    their gradient is held.  Tokens that are ignored or whose grad_loss is 0 take no part.
    `grad_weight` (fp32 or bf16, e.g. `weight.main_grad`) is written, or with `accumulate` added to, rows
    past `vocab_size` as zeros; without it a new tensor of weight's dtype is returned.  The logits'
    gradient is rounded to bf16 for the matrix cores where the result is bf16 (for grad_weight of up to 256
    tokens, where few roundings do not average out, to two), and to two fp16 limbs where it is fp32: off by
    2^-22 of itself or by 2^-49 of the token's grad_loss, whichever is more (the gradient of a word of
    probability 1e-12 has 9 bits, below 1e-15 it is 0).  fp32 hidden states and weights are two such limbs: off
    by 2^-22 of the value or 2^-50 of the tensor's largest.  For an fp32 grad_weight a token's hidden states
    take the power of two of its grad_loss along and are off by 2^-39 (bf16) or 2^-50 (fp32) of the largest such
    product: a token whose grad_loss is 2^-39 of the largest adds nothing.  With `group`, grad_hidden is
    summed over the vocabulary's shards."""
    gw = _grad_weight(weight, grad_weight, accumulate, "grad_weight") if need_weight else None
    d, nbytes = _xent_desc(_lm_lib.XENT_BACKWARD, hidden, weight, target, vocab_start, vocab_size, ignore_index, gw,
                           accumulate, piece_bytes)
    device = hidden.device
    for t, what in ((grad_loss, "grad_loss"), (lse, "lse")):
        if t.dtype != torch.float32 or t.shape != target.shape or t.device != device:
            raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] {what}: fp32 {tuple(target.shape)} expected, got "
                               f"{t.dtype} {tuple(t.shape)} {t.device}")
    gh = _empty(hidden) if need_hidden else None
    none = d is None or d.tokens == 0  # no gradient: of no word, or no token's
    if gw is not None and not accumulate and (none or d.vocab < weight.shape[0]):
        (gw if none else gw[d.vocab:]).zero_()
    if none and gh is not None:
        gh.zero_()
    if none or (gh is None and gw is None):
        return _sum_over_shards(gh, group), gw
    target, grad_loss, lse = target.contiguous(), grad_loss.contiguous(), lse.contiguous()
    ws = _workspace(nbytes, device)
    rc = _call(_lm_lib.load().dion_xent_backward, device, _byref(d), hidden.data_ptr(), weight.data_ptr(),
               target.data_ptr(), lse.data_ptr(), grad_loss.data_ptr(), None if gh is None else gh.data_ptr(),
               None if gw is None else gw.data_ptr(), ws.data_ptr(), ws.numel())
    if rc:
        _lm_lib.check(rc, "dion_xent_backward")
    return _sum_over_shards(gh, group), gw
