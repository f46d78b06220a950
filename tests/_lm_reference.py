"""Plain 64-bit forms of the training operators (CPU), with bounds on what the kernels may be off."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24


def philox(n, seed, offset):
    """The 32-bit words of elements 0 .. n-1 (numpy uint64 arithmetic)."""
    m32 = np.uint64(0xFFFFFFFF)
    g = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [g & m32, g >> np.uint64(32), np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:n]


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    t = math.floor(p * 2.0 ** 32 + 0.5)
    return torch.from_numpy(philox(n, seed, offset) >= np.uint64(t)).view(*shape)


def dropped32(x, keep, p):
    """x in 32 bits times fp32(1 / (1 - p)) where kept, else 0: the operator's own arithmetic."""
    s = torch.tensor(1.0 / (1.0 - p) if p < 1.0 else 0.0, dtype=torch.float32)
    return torch.where(keep, x.float() * s, torch.zeros(()))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def xent(hidden, weight, target, ignore, grad_loss=None, total=None, start=0, out_dtype=None):
    """Loss, lse and gradients in 64 bits, and for each the largest error that the kernels' roundings
    allow.  Sums of k terms run in fp32 in chains of 16: k / 16 + 20 roundings of at most the sum of the
    terms' magnitudes.  An operand of fp32 precision is two fp16 limbs: off by 2^-22 of each value and by
    2^-39 of the largest, and a product of two such leaves out lo lo, 2^-22 again; its sum has three times
    as many terms.  g is rounded to bf16 (2^-8), or to two limbs, and the result once."""
    f32 = hidden.dtype == torch.float32
    x, w = hidden.double(), weight.double()
    t, h = x.shape
    v = w.shape[0]
    valid = target != ignore
    if grad_loss is not None:
        live = valid & (grad_loss != 0)
    x = torch.where(valid[:, None], x, torch.zeros_like(x))  # never read
    z = x @ w.t()
    steps = lambda k: (k / 16 + 20) * (3 if f32 else 1) * U32 + (3 * 2.0 ** -22 if f32 else 0.0)  # noqa: E731
    ez = steps(h) * (x.abs() @ w.abs().t()).amax(1)  # of a logit of each token
    if f32:
        ez = ez + 2 * 2.0 ** -39 * h * x.abs().max() * w.abs().max()
    lse = torch.logsumexp(z, 1)
    at = (target - start).clamp(0, v - 1)
    here = valid & (target >= start) & (target < start + v)
    tl = torch.where(here, z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    zero = torch.zeros_like(lse)
    r = {"lse": torch.where(valid, lse, zero), "loss": torch.where(valid, lse - tl, zero)}
    # exp2 of an argument up to 64 octaves and a sum of positive terms, log, one subtraction
    e_lse = ez + (v / 16 + 120) * U32 + 4 * U32 * (lse.abs() + z.abs().amax(1))
    r["e_loss"] = torch.where(valid, 2 * e_lse, zero)
    if grad_loss is None:
        return r
    gl = torch.where(live, grad_loss.double(), zero)
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p)
    onehot[here, at[here]] = 1.0
    g = (p - onehot) * gl[:, None]
    rel_p = (ez + e_lse + 128 * U32)[:, None]
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    wide = f32 or out_dtype == torch.float32
    # an error of p is at most rel_p of p; g's own rounding is relative to g
    e_p = (rel_p * p + 2 * U32) * gl.abs()[:, None]
    e_x = (2.0 ** -22 if f32 else 2.0 ** -8) * g.abs() + e_p
    e_w = (2.0 ** -22 if wide else 2.0 ** -8) * g.abs() + e_p
    r["grad_hidden"] = g @ w
    tiny = 2.0 ** -148  # the spacing of fp32's least numbers, twice
    floor_w = 2.0 ** -39 * w.abs().max() * g.abs().sum(1, keepdim=True) if f32 else 0.0
    r["e_grad_hidden"] = (e_x @ w.abs() + steps(v) * (g.abs() @ w.abs()) + floor_w + tiny
                          + half_step(hidden.dtype) * r["grad_hidden"].abs())
    r["grad_weight"] = g.t() @ x
    od = out_dtype or weight.dtype
    # X goes in times the power of two below gl, its largest under 2^15
    e2 = torch.where(gl != 0, 2.0 ** torch.floor(torch.log2(gl.abs().clamp_min(1e-300))), torch.ones_like(gl))[:, None]
    floor_x = 2.0 ** -39 * (x.abs() * e2).max() * (g.abs() / e2).sum(0)[:, None] if wide and t else 0.0
    r["e_grad_weight"] = (e_w.t() @ x.abs() + (steps(t) + (2 * (t / 16 + 20) * U32 if wide else 0.0)) * (g.abs().t() @ x.abs())
                          + floor_x + tiny + half_step(od) * r["grad_weight"].abs())
    return r
