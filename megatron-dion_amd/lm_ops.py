"""The training operators around the optimizer: output-layer loss, residual norm, dropout.

The optimizer consumes gradients; these make those of the parameters its elementwise branch updates
(the output layer and the norms), in hand-written HIP kernels (csrc/lm/, C ABI in include/dion_lm.h).
They take the place of what a Megatron model calls there: the vocabulary-parallel cross entropy after
its output layer, the bias-dropout-add before a norm, and the norm itself.

Each operator is a pair of explicit calls, forward and backward, that run on the current HIP stream of
the tensors' device, allocate their results and scratch from torch's caching allocator, never wait for
the GPU and can be captured into a graph.  `lm_autograd.py` wraps them for autograd.

Tensors are float32 or bfloat16 of any leading shape, with unit stride along the last axis and the
leading axes evenly strided (what `view(-1, cols)` accepts); anything else raises
``RuntimeError("[DION_...] ...")`` before any work is enqueued.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.distributed as dist

from . import _lib, _lm_lib

__all__ = ["linear_cross_entropy_forward", "linear_cross_entropy_backward", "rms_norm_add_forward",
           "rms_norm_add_backward", "dropout_add_forward", "dropout_add_backward", "RmsNormAdd", "RmsNormAddGrads"]

Rng = Union[Tuple[int, int], torch.Tensor]
_U64 = (1 << 64) - 1
_CODE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _CODE.get(t.dtype)
    if code is None:
        raise RuntimeError(f"[DION_UNSUPPORTED_DTYPE] {what}: {t.dtype}")
    return code


def _matrix(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`t` as (rows, cols) without a copy; its device, shape and dtype checked against `like`."""
    if t.dim() == 0:
        raise RuntimeError(f"[DION_BAD_SHAPE] {what} has no axis")
    if not t.is_cuda:
        raise RuntimeError(f"[DION_BAD_DEVICE] {what} is on {t.device}")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] {what}: {tuple(t.shape)} {t.dtype} {t.device}, expected "
                           f"{tuple(like.shape)} {like.dtype} {like.device}")
    cols = t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or cols <= 1) and (t.stride(0) >= cols or t.shape[0] <= 1):
        return t
    if t.is_contiguous():
        return t.view(t.numel() // cols if cols else 0, cols)
    try:
        v = t.view(-1, cols) if t.numel() else t.reshape(-1, max(cols, 1))
    except RuntimeError:
        v = None
    if v is None or (cols > 1 and v.stride(1) != 1) or (v.shape[0] > 1 and v.stride(0) < cols):
        raise RuntimeError(f"[DION_NON_ROW_MAJOR] {what}: shape={tuple(t.shape)} stride={t.stride()}")
    return v


def _ld(m: torch.Tensor) -> int:
    return int(m.stride(0)) if m.shape[0] > 1 else max(int(m.shape[1]), 1)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


class _on:
    """The device that a call's kernels are launched on (no change when it is the current one)."""

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.guard = None
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _workspace(nbytes: int, device) -> torch.Tensor:
    # a call's own memory, from the caching allocator: calls on different streams and captured graphs
    # never share it
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


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
    return None if s is None else ctypes.byref(s)


# ------------------------------------------------------------------------------- dropout
def dropout_add_forward(x: torch.Tensor, residual: Optional[torch.Tensor] = None, *, p: float,
                        rng: Optional[Rng] = None) -> torch.Tensor:
    """`residual + dropout(x)` (without `residual`: `dropout(x)`), the mask never stored.

    Philox4x32-10 with key `seed` and counter `(e // 4, offset)`: element e of x (row-major) keeps its
    value, times fp32(1 / (1 - p)), iff word `e % 4` is at least p 2^32, else becomes 0 (also a NaN or an
    infinity).  `rng` is `(seed, offset)`, or an int64 tensor holding them on x's device, which a
    captured graph reads again at each replay.  A (seed, offset) pair is to be used for one mask only:
    count `offset` over layers, steps and ranks."""
    xm = _matrix(x, "x")
    rm = None if residual is None else _matrix(residual, "residual", x)
    code = _dtype(x, "x")
    r = _rng(p, rng, x.device)
    lib = _lm_lib.load()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _on(x.device):
        rc = lib.dion_dropout_add(xm.shape[0], xm.shape[1], code, xm.data_ptr(), _ld(xm), _ptr(rm),
                                  0 if rm is None else _ld(rm), out.data_ptr(), max(int(xm.shape[1]), 1), float(p),
                                  _ref(r), _stream(x.device))
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


def _norm_desc(xm: torch.Tensor, weight: torch.Tensor, p: float) -> _lm_lib.DionNormDesc:
    if weight.dim() != 1 or weight.shape[0] != xm.shape[1] or weight.device != xm.device or \
            not weight.is_contiguous():
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] weight: {tuple(weight.shape)} {weight.device}, expected "
                           f"({xm.shape[1]},) on {xm.device}")
    d = _lm_lib.DionNormDesc()
    d.rows, d.cols = int(xm.shape[0]), int(xm.shape[1])
    d.dtype, d.w_dtype = _dtype(xm, "x"), _dtype(weight, "weight")
    d.gw_dtype = d.w_dtype
    d.y_dtype = d.dtype
    d.p = float(p)
    return d


def rms_norm_add_forward(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                         eps: float = 1e-5, p: float = 0.0, rng: Optional[Rng] = None,
                         scale_block: int = 0) -> RmsNormAdd:
    """`h = residual + dropout(x)`, rounded to x's dtype; `y = h * rsqrt(mean(h^2) + eps) * weight`.

    `scale_block` > 0 (at least 8, or all columns; -1: one block a row): y is float8_e4m3fn, each block
    of that many columns over its own fp32 `scale` = max |y| / 448 (at least 2^-126), so that
    `y.float() * scale` restores it.  Dropout as in `dropout_add_forward`."""
    xm = _matrix(x, "x")
    rm = None if residual is None else _matrix(residual, "residual", x)
    d = _norm_desc(xm, weight, p)
    d.eps = float(eps)
    r = _rng(p, rng, x.device)
    rows, cols = int(d.rows), int(d.cols)
    lib = _lm_lib.load()
    stored = rm is not None or p > 0.0
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if stored else x
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    scale = None
    if scale_block:
        d.y_dtype = _lm_lib.DTYPE_E4M3
        d.scale_block = cols if scale_block < 0 or scale_block > cols else int(scale_block)
        scale = torch.empty(tuple(x.shape[:-1]) + (-(-cols // max(d.scale_block, 1)),), dtype=torch.float32,
                            device=x.device)
        y = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d.ld_x, d.ld_residual = _ld(xm), 0 if rm is None else _ld(rm)
    d.ld_h = d.ld_y = cols
    with _on(x.device):
        rc = lib.dion_rms_norm_add(ctypes.byref(d), xm.data_ptr(), _ptr(rm), weight.data_ptr(),
                                   h.data_ptr() if stored else None, y.data_ptr(), _ptr(scale), rstd.data_ptr(),
                                   _ref(r), _stream(x.device))
    _lm_lib.check(rc, "dion_rms_norm_add")
    return RmsNormAdd(y, h, rstd, scale)


def _grad_weight(weight: torch.Tensor, out: Optional[torch.Tensor], accumulate: bool, what: str) -> torch.Tensor:
    if out is None:
        if accumulate:
            raise RuntimeError(f"[DION_BAD_GRAD_OUT] accumulate needs {what}")
        return torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
    if out.shape != weight.shape or out.device != weight.device:
        raise RuntimeError(f"[DION_BAD_GRAD_OUT] {what}: {tuple(out.shape)} {out.device}, expected "
                           f"{tuple(weight.shape)} {weight.device}")
    return out


def rms_norm_add_backward(grad_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                          grad_h: Optional[torch.Tensor] = None, *, p: float = 0.0, rng: Optional[Rng] = None,
                          grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                          need_input: bool = True, need_weight: bool = True) -> RmsNormAddGrads:
    """Gradients of `rms_norm_add_forward`; `grad_h` is what reaches h past the norm (the residual
    stream's gradient), `p` and `rng` are the forward's.  An 8-bit y passes `grad_y` (x's dtype) as if
    it had not been rounded.  `grad_weight` (fp32 or bf16, e.g. `weight.main_grad`) is written, or with
    `accumulate` added to; without it a new tensor of weight's dtype is returned."""
    hm = _matrix(h, "h")
    gm = _matrix(grad_y, "grad_y", h)
    ghm = None if grad_h is None else _matrix(grad_h, "grad_h", h)
    d = _norm_desc(hm, weight, p)
    r = _rng(p, rng, h.device)
    if rstd.dtype != torch.float32 or rstd.shape != h.shape[:-1] or not rstd.is_contiguous() or \
            rstd.device != h.device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] rstd: {tuple(rstd.shape)} {rstd.dtype}")
    cols = int(d.cols)
    gx = gr = gw = ws = None
    if need_input:
        gx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        if p > 0.0:
            gr = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    lib = _lm_lib.load()
    if need_weight:
        gw = _grad_weight(weight, grad_weight, accumulate, "grad_weight")
        if not gw.is_contiguous():
            raise RuntimeError(f"[DION_BAD_GRAD_OUT] grad_weight stride={gw.stride()}")
        d.gw_dtype = _dtype(gw, "grad_weight")
        d.accumulate = int(bool(accumulate))
        nbytes = ctypes.c_size_t(0)
        _lm_lib.check(lib.dion_rms_norm_add_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)),
                      "dion_rms_norm_add_workspace_bytes")
        ws = _workspace(nbytes.value, h.device)
    d.ld_h, d.ld_grad_y, d.ld_grad_h = _ld(hm), _ld(gm), 0 if ghm is None else _ld(ghm)
    d.ld_grad_x = d.ld_grad_residual = cols
    with _on(h.device):
        rc = lib.dion_rms_norm_add_backward(ctypes.byref(d), gm.data_ptr(), hm.data_ptr(), weight.data_ptr(),
                                            rstd.data_ptr(), _ptr(ghm), _ptr(gx), _ptr(gr), _ptr(gw), _ref(r),
                                            _ptr(ws), 0 if ws is None else ws.numel(), _stream(h.device))
    _lm_lib.check(rc, "dion_rms_norm_add_backward")
    return RmsNormAddGrads(gx, gx if gr is None else gr, gw)


# ------------------------------------------------------------------------------- linear cross entropy
def _xent_desc(hidden, weight, target, vocab_start, vocab_size, ignore_index, op):
    hm = _matrix(hidden, "hidden")
    wm = _matrix(weight, "weight")
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or weight.dtype != hidden.dtype or \
            weight.device != hidden.device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] hidden {tuple(hidden.shape)} {hidden.dtype} {hidden.device}, "
                           f"weight {tuple(weight.shape)} {weight.dtype} {weight.device}")
    if target.dtype != torch.int64 or target.shape != hidden.shape[:-1] or target.device != hidden.device:
        raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] target: int64 {tuple(hidden.shape[:-1])} on {hidden.device} "
                           f"expected, got {target.dtype} {tuple(target.shape)} {target.device}")
    d = _lm_lib.DionXentDesc()
    d.dtype = _dtype(hidden, "hidden")
    start, rows = int(vocab_start), int(weight.shape[0])
    total = start + rows if vocab_size is None else int(vocab_size)
    if start < 0 or rows < 1 or total <= start:
        raise RuntimeError(f"[DION_BAD_VOCAB] weight of {rows} rows from word {start} on, of {total}")
    d.tokens, d.hidden = int(hm.shape[0]), int(hm.shape[1])
    d.vocab = min(rows, total - start)  # rows past the vocabulary are padding
    d.vocab_start, d.vocab_total, d.ignore_index = start, total, int(ignore_index)
    d.ld_hidden, d.ld_weight = _ld(hm), _ld(wm)
    d.gw_dtype = d.dtype
    d.pack_weight = int(wm.data_ptr() % 16 != 0)
    return d, hm, wm, target.contiguous().view(-1)


def _xent_workspace(lib, d, op, device):
    nbytes = ctypes.c_size_t(0)
    _lm_lib.check(lib.dion_xent_workspace_bytes(ctypes.byref(d), op, ctypes.byref(nbytes)),
                  "dion_xent_workspace_bytes")
    return _workspace(nbytes.value, device)


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


def linear_cross_entropy_forward(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                                 vocab_start: int = 0, vocab_size: Optional[int] = None, ignore_index: int = -100,
                                 group=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, lse), fp32 of target's shape: the cross entropy of `hidden @ weight.T` at each token and
    the logarithm of its softmax's denominator (for the backward pass).  The logits are never stored.

    hidden (..., H) and weight (V, H) are bf16 or fp32 alike, target int64.  A token whose target is
    `ignore_index` costs nothing: its loss and lse are 0 and its hidden state is not read.  Any other
    target outside the vocabulary gives a NaN loss.

    Vocabulary shards (tensor parallel): weight holds the rows from `vocab_start` on of a vocabulary of
    `vocab_size` words (rows past it are padding), `group` the ranks that share it; every rank passes the
    same hidden states and targets and gets the whole vocabulary's loss."""
    d, hm, wm, tv = _xent_desc(hidden, weight, target, vocab_start, vocab_size, ignore_index, _lm_lib.XENT_FORWARD)
    dev = hidden.device
    lib = _lm_lib.load()
    ws = _xent_workspace(lib, d, _lm_lib.XENT_FORWARD, dev)
    out = torch.empty((2,) + tuple(target.shape), dtype=torch.float32, device=dev)
    loss, lse = out[0], out[1]
    with _on(dev):
        if group is None:
            rc = lib.dion_xent_forward(ctypes.byref(d), hm.data_ptr(), wm.data_ptr(), tv.data_ptr(), loss.data_ptr(),
                                       lse.data_ptr(), None, ws.data_ptr(), ws.numel(), _stream(dev))
            _lm_lib.check(rc, "dion_xent_forward")
            return loss, lse
        tlogit = loss
        rc = lib.dion_xent_forward(ctypes.byref(d), hm.data_ptr(), wm.data_ptr(), tv.data_ptr(), None,
                                   lse.data_ptr(), tlogit.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev))
        _lm_lib.check(rc, "dion_xent_forward")
        return combine_vocab_shards(lse, tlogit, target == ignore_index, group)


def linear_cross_entropy_backward(grad_loss: torch.Tensor, hidden: torch.Tensor, weight: torch.Tensor,
                                  target: torch.Tensor, lse: torch.Tensor, *, vocab_start: int = 0,
                                  vocab_size: Optional[int] = None, ignore_index: int = -100, group=None,
                                  grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                                  need_hidden: bool = True, need_weight: bool = True, piece_bytes: int = 0
                                  ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(grad_hidden, grad_weight) for the upstream gradient `grad_loss` (fp32, target's shape).

    The logits are made again a piece of the vocabulary at a time; at most `piece_bytes` (0:
    1 GiB) of their gradient is held.  Tokens that are ignored or whose grad_loss is 0 take no part.  `grad_weight` (fp32 or bf16,
    e.g. `weight.main_grad`) is written, or with `accumulate` added to, rows past `vocab_size` as zeros;
    without it a new tensor of weight's dtype is returned.  The logits' gradient is rounded to bf16 for
    the matrix cores where the result is bf16, and split into three bf16 limbs (24 bits) where it is fp32.  With `group`, grad_hidden is summed over the vocabulary's shards."""
    d, hm, wm, tv = _xent_desc(hidden, weight, target, vocab_start, vocab_size, ignore_index, _lm_lib.XENT_BACKWARD)
    for t, what in ((grad_loss, "grad_loss"), (lse, "lse")):
        if t.dtype != torch.float32 or t.shape != target.shape or t.device != hidden.device:
            raise RuntimeError(f"[DION_INCONSISTENT_TENSORS] {what}: fp32 {tuple(target.shape)} expected, got "
                               f"{t.dtype} {tuple(t.shape)} {t.device}")
    dev = hidden.device
    gl, ls = grad_loss.contiguous(), lse.contiguous()
    gh = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if need_hidden else None
    gw = None
    if need_weight:
        gw = _grad_weight(weight, grad_weight, accumulate, "grad_weight")
        d.gw_dtype = _dtype(gw, "grad_weight")
        d.ld_grad_weight = _ld(_matrix(gw, "grad_weight"))
        d.accumulate = int(bool(accumulate))
        if not accumulate and (d.tokens == 0 or d.vocab < weight.shape[0]):
            (gw if d.tokens == 0 else gw[d.vocab:]).zero_()
    if d.tokens == 0 or (gh is None and gw is None):
        return gh, gw
    d.ld_grad_hidden = int(d.hidden)
    d.piece_bytes = int(piece_bytes)
    lib = _lm_lib.load()
    ws = _xent_workspace(lib, d, _lm_lib.XENT_BACKWARD, dev)
    with _on(dev):
        rc = lib.dion_xent_backward(ctypes.byref(d), hm.data_ptr(), wm.data_ptr(), tv.data_ptr(), ls.data_ptr(),
                                    gl.data_ptr(), _ptr(gh), _ptr(gw), ws.data_ptr(), ws.numel(), _stream(dev))
        _lm_lib.check(rc, "dion_xent_backward")
        if group is not None and gh is not None:
            dist.all_reduce(gh, op=dist.ReduceOp.SUM, group=group)
    return gh, gw
