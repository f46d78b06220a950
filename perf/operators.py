"""The operators of a training step around the optimizer, as cases that can be timed and compared.

Three operators, each with its gradient:

* ``xent``    the loss of an output layer, cross entropy of ``hidden @ weight.T`` over a large vocabulary,
              without keeping the logits;
* ``norm``    root-mean-square norm of ``residual + dropout(x)``, its result in the input's type or in
              8 bits with one scale for each block of columns;
* ``dropout`` dropout from a counter-based generator (Philox 4x32-10), with or without a residual, its
              mask never stored.

With ``own`` false ``run`` computes them in elementary torch operations, otherwise through this package.
"""
import math

import torch

own = False

IGNORE = -100
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token's loss under a 32000-word output layer: the latency of scoring a candidate
        {"name": "xent one token", "op": "xent", "tokens": 1, "hidden": 4096, "vocab": 32000, "dtype": "bf16",
         "grad": "none", "ignored": 0.0},
        # validation loss of a small model on a ragged tail of tokens, an odd vocabulary, some padding
        {"name": "xent eval ragged", "op": "xent", "tokens": 1023, "hidden": 768, "vocab": 50257, "dtype": "bf16",
         "grad": "none", "ignored": 0.1},
        # GPT-125M training micro-batch: gradients go into fp32 main_grad buffers
        {"name": "xent train 768", "op": "xent", "tokens": 4096, "hidden": 768, "vocab": 50257, "dtype": "bf16",
         "grad": "fp32", "ignored": 0.02},
        # Llama-3-8B training micro-batch: one sequence of 8192, bf16 gradients
        {"name": "xent train 4096", "op": "xent", "tokens": 8192, "hidden": 4096, "vocab": 128256, "dtype": "bf16",
         "grad": "bf16", "ignored": 0.0},
        # fp32 training of an odd-sized model on a batch that is mostly padding (instruction tuning)
        {"name": "xent fp32 padded", "op": "xent", "tokens": 513, "hidden": 1000, "vocab": 5003, "dtype": "fp32",
         "grad": "fp32", "ignored": 0.7},
        # the norm before a layer for one token
        {"name": "norm one token", "op": "norm", "rows": 1, "hidden": 4096, "dtype": "bf16", "p": 0.0,
         "residual": True, "quant": 0, "backward": False},
        # the input of an 8-bit product: one scale for each 128 columns
        {"name": "norm 8 bits", "op": "norm", "rows": 8192, "hidden": 4096, "dtype": "bf16", "p": 0.0,
         "residual": True, "quant": 128, "backward": False},
        # the end of a sublayer in training: dropout, residual, norm, and all gradients
        {"name": "norm train 4096", "op": "norm", "rows": 8192, "hidden": 4096, "dtype": "bf16", "p": 0.1,
         "residual": True, "quant": 0, "backward": True},
        # an odd number of rows of an odd width in fp32, no residual
        {"name": "norm train fp32 odd", "op": "norm", "rows": 1031, "hidden": 1001, "dtype": "fp32", "p": 0.0,
         "residual": False, "quant": 0, "backward": True},
        # one token's activations
        {"name": "dropout small", "op": "dropout", "rows": 1, "cols": 768, "dtype": "bf16", "p": 0.1,
         "residual": False, "backward": False},
        # the activations inside a 14336-wide MLP, forward and backward
        {"name": "dropout mlp", "op": "dropout", "rows": 8192, "cols": 14336, "dtype": "bf16", "p": 0.1,
         "residual": False, "backward": True},
        # fp32 rows of an odd width onto a residual stream, forward and backward
        {"name": "dropout residual odd", "op": "dropout", "rows": 4097, "cols": 1001, "dtype": "fp32", "p": 0.25,
         "residual": True, "backward": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["xent", "norm", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "xent":
        tokens, vocab = _log_int(rng, 1, 8192), _log_int(rng, 1000, 128256)
        hidden = rng.choice([_log_int(rng, 256, 4096), 8 * _log_int(rng, 32, 512)])
        if dtype == "fp32":  # fp32 is the type of small models here
            tokens, vocab, hidden = min(tokens, 1024), min(vocab, 16384), min(hidden, 1024)
        grad = rng.choice(["none", dtype, "fp32"])
        tokens = min(tokens, 4096) if grad == "fp32" else tokens
        return {"op": op, "tokens": tokens, "hidden": hidden, "vocab": vocab, "dtype": dtype, "grad": grad,
                "ignored": rng.choice([0.0, round(rng.uniform(0.0, 0.9), 3)])}
    if op == "norm":
        rows, hidden = _log_int(rng, 1, 8192), rng.choice([_log_int(rng, 128, 8192), 8 * _log_int(rng, 16, 1024)])
        rows = min(rows, (8192 * 4096) // hidden)
        backward = rng.random() < 0.5
        quant = 0 if backward or rng.random() < 0.5 else 128
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "p": rng.choice([0.0, round(rng.uniform(0.01, 0.5), 3)]),
                "residual": rng.random() < 0.7, "quant": quant, "backward": backward}
    rows, cols = _log_int(rng, 1, 8192), rng.choice([_log_int(rng, 64, 14336), 8 * _log_int(rng, 8, 1792)])
    rows = min(rows, (8192 * 14336) // (cols * 4))
    return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "p": round(rng.uniform(0.01, 0.9), 3),
            "residual": rng.random() < 0.5, "backward": rng.random() < 0.5}


def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "xent":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        s["hidden"] = _normal(gen, (t, h), 1.0, dt)
        s["weight"] = _normal(gen, (v, h), 2.0 / math.sqrt(h), dt)  # logits of spread 2, as trained layers have
        target = torch.randint(0, v, (t,), generator=gen, device="cuda")
        drop = torch.rand((t,), generator=gen, device="cuda") < case["ignored"]
        s["target"] = torch.where(drop, torch.full_like(target, IGNORE), target)
        if case["grad"] != "none":
            # the loss mask over the number of tokens, as a mean loss sends it back
            s["grad_loss"] = torch.rand((t,), generator=gen, device="cuda") / t
            s["grad_weight"] = torch.empty((v, h), dtype=DTYPES[case["grad"]], device="cuda")
        return s
    cols = case["hidden"] if case["op"] == "norm" else case["cols"]
    shape = (case["rows"], cols)
    s["x"] = _normal(gen, shape, 1.0, dt)
    s["residual"] = _normal(gen, shape, 2.0, dt) if case["residual"] else None
    s["rng"] = (int(seed) * 7919 + 12345, int(seed) % 1000)  # the generator's key and this layer's offset
    if case["op"] == "norm":
        s["weight"] = 1.0 + _normal(gen, (cols,), 0.1, torch.float32)
    if case["backward"]:
        s["grad_out"] = _normal(gen, shape, 1e-2, dt)
        if case["op"] == "norm":
            s["grad_h"] = _normal(gen, shape, 1e-2, dt) if case["residual"] else None
    return s


# ------------------------------------------------------------------------------- the plain forms
def _product(a, b):
    """a @ b in full 32 bits."""
    return torch.matmul(a, b)


def _plain_xent(s):
    case = s["case"]
    x, w, target = s["hidden"].float(), s["weight"].float(), s["target"]
    valid = target != IGNORE
    at = torch.where(valid, target, torch.zeros_like(target))[:, None]
    logits = _product(x, w.t())
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp().sum(1, keepdim=True).log() + top
    loss = torch.where(valid, (lse - logits.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    if case["grad"] == "none":
        return {"loss": loss}
    scale = torch.where(valid, s["grad_loss"], torch.zeros_like(s["grad_loss"]))[:, None]
    g = (logits - lse).exp() * scale
    g.scatter_add_(1, at, -scale)
    return {"loss": loss, "grad_hidden": _product(g, w).to(s["hidden"].dtype),
            "grad_weight": _product(g.t(), x).to(s["grad_weight"].dtype)}


def _mulhilo(a, m):
    """The high and the low 32 bits of a * m, all held in 64-bit integers."""
    p = a * m  # wraps modulo 2^64, which leaves every bit in place
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _plain_keep(rows, cols, p, rng, device):
    """Philox 4x32-10 with key `seed` and counter (element / 4, offset): element e keeps its value where
    word e % 4 is at least p 2^32."""
    seed, offset = rng
    n = rows * cols
    g = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
    c0, c1 = g & 0xFFFFFFFF, g >> 32
    c2, c3 = torch.full_like(g, offset & 0xFFFFFFFF), torch.full_like(g, (offset >> 32) & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0, c1, c2, c3), 1).view(-1)[:n].view(rows, cols)
    return words >= int(math.floor(p * 4294967296.0 + 0.5))


def _plain_dropped(x, p, keep):
    return torch.where(keep, x * torch.tensor(1.0 / (1.0 - p), dtype=torch.float32, device=x.device), torch.zeros_like(x))


def _plain_norm(s):
    case = s["case"]
    x, dt, w, p = s["x"].float(), s["x"].dtype, s["weight"], case["p"]
    rows, cols = x.shape
    keep = _plain_keep(rows, cols, p, s["rng"], x.device) if p else None
    h = _plain_dropped(x, p, keep) if p else x
    if case["residual"]:
        h = h + s["residual"].float()
    h = h.to(dt)  # the residual stream, which the layers after this one read: the norm is of what they read
    hf = h.float()
    rstd = (hf.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xhat = hf * rstd
    y = xhat * w
    out = {"h": h, "rstd": rstd[:, 0]}
    if case["quant"]:
        pad = -cols % case["quant"]
        blocks = torch.nn.functional.pad(y, (0, pad)).view(rows, -1, case["quant"])
        scale = (blocks.abs().amax(2) / E4M3_MAX).clamp_min(2.0 ** -126)
        q = (blocks / scale[:, :, None]).view(rows, -1)[:, :cols]
        out.update(y=q.to(torch.float8_e4m3fn), scale=scale)
        return out
    out["y"] = y.to(dt)
    if not case["backward"]:
        return out
    dy = s["grad_out"].float()
    wdy = dy * w
    dh = rstd * (wdy - xhat * (wdy * xhat).mean(1, keepdim=True))
    if case["residual"]:
        dh = dh + s["grad_h"].float()
        out["grad_residual"] = dh.to(dt)
    out["grad_x"] = (_plain_dropped(dh, p, keep) if p else dh).to(dt)
    out["grad_weight"] = (dy * xhat).sum(0)
    return out


def _plain_dropout(s):
    case, x = s["case"], s["x"].float()
    keep = _plain_keep(x.shape[0], x.shape[1], case["p"], s["rng"], x.device)
    out = _plain_dropped(x, case["p"], keep)
    if case["residual"]:
        out = out + s["residual"].float()
    out = {"out": out.to(s["x"].dtype)}
    if case["backward"]:
        out["grad_x"] = _plain_dropped(s["grad_out"].float(), case["p"], keep).to(s["x"].dtype)
    return out


# ------------------------------------------------------------------------------- the package's calls
def _own_xent(s):
    import megatron_dion_amd as mda

    loss, lse = mda.linear_cross_entropy_forward(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE)
    if s["case"]["grad"] == "none":
        return {"loss": loss}
    dx, dw = mda.linear_cross_entropy_backward(s["grad_loss"], s["hidden"], s["weight"], s["target"], lse,
                                               ignore_index=IGNORE, grad_weight=s["grad_weight"])
    return {"loss": loss, "grad_hidden": dx, "grad_weight": dw}


def _own_norm(s):
    import megatron_dion_amd as mda

    case = s["case"]
    rng = s["rng"] if case["p"] else None
    f = mda.rms_norm_add_forward(s["x"], s["weight"], s["residual"], eps=1e-5, p=case["p"], rng=rng,
                                 scale_block=case["quant"])
    out = {"h": f.h, "rstd": f.rstd, "y": f.y}
    if case["quant"]:
        out["scale"] = f.scale
    if not case["backward"]:
        return out
    b = mda.rms_norm_add_backward(s["grad_out"], f.h, s["weight"], f.rstd, s["grad_h"], p=case["p"], rng=rng)
    if case["residual"]:
        out["grad_residual"] = b.grad_residual
    out.update(grad_x=b.grad_x, grad_weight=b.grad_weight)
    return out


def _own_dropout(s):
    import megatron_dion_amd as mda

    case = s["case"]
    out = {"out": mda.dropout_add_forward(s["x"], s["residual"], p=case["p"], rng=s["rng"])}
    if case["backward"]:
        out["grad_x"] = mda.dropout_add_backward(s["grad_out"], p=case["p"], rng=s["rng"])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"xent": _own_xent, "norm": _own_norm, "dropout": _own_dropout}[op](state)
    return {"xent": _plain_xent, "norm": _plain_norm, "dropout": _plain_dropout}[op](state)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "xent":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        live = t * (1.0 - case["ignored"])  # a token without a target needs no work
        nbytes, flops = size * (live * h + v * h) + 8 * t + 4 * t, 2.0 * live * h * v
        if case["grad"] != "none":
            gsize = 2 if case["grad"] == "bf16" else 4
            nbytes += 4 * t + size * t * h + gsize * v * h
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "norm":
        n, rows = case["rows"] * case["hidden"], case["rows"]
        stored = case["residual"] or case["p"]  # otherwise h is x itself
        nbytes = n * size * (1 + bool(case["residual"]) + bool(stored)) + 4 * case["hidden"] + 4 * rows
        nbytes += n * (1 if case["quant"] else size) + (4 * rows * -(-case["hidden"] // case["quant"]) if case["quant"] else 0)
        if case["backward"]:
            # grad_y and grad_h are read, grad_x and (where it is another tensor) grad_residual are written
            nbytes += n * size * (2 + bool(case["residual"]) + bool(case["residual"] and case["p"])) + 4 * case["hidden"]
        return {"bytes": nbytes, "flops": 8.0 * n * (3 if case["backward"] else 1)}
    n = case["rows"] * case["cols"]
    return {"bytes": n * size * (2 + bool(case["residual"]) + 2 * bool(case["backward"])), "flops": 2.0 * n}


# ------------------------------------------------------------------------------- in 64 bits
def _keep64(n, p, rng, device):
    """The same generator from its definition, on 16-bit halves so that no product leaves 53 bits."""
    def mul(a, m):
        lo, hi = (a % 65536) * m, (a // 65536) * m  # each below 2^48
        total = lo + (hi % 65536) * 65536
        return hi // 65536 + total // 4294967296, total % 4294967296

    key = [rng[0] % 4294967296, rng[0] // 4294967296 % 4294967296]
    group = torch.arange(-(-n // 4), device=device)
    ctr = [group % 4294967296, group // 4294967296, torch.zeros_like(group) + rng[1] % 4294967296,
           torch.zeros_like(group) + rng[1] // 4294967296 % 4294967296]
    for r in range(10):
        (ha, la), (hb, lb) = mul(ctr[0], 3528531795), mul(ctr[2], 3449720151)
        ka, kb = (key[0] + r * 2654435769) % 4294967296, (key[1] + r * 3144134277) % 4294967296
        ctr = [hb.bitwise_xor(ctr[1]).bitwise_xor(ka), lb, ha.bitwise_xor(ctr[3]).bitwise_xor(kb), la]
    return torch.stack(ctr, 1).reshape(-1)[:n] >= round(p * 4294967296)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "xent":
        x, w, target, t = s["hidden"].double(), s["weight"].double(), s["target"], case["tokens"]
        rows = torch.nonzero(target >= 0)[:, 0]  # only tokens with a target have a loss or a gradient
        x = x[rows]
        at = target[rows]
        z = x @ w.t()
        lse = torch.logsumexp(z, 1)
        loss = torch.zeros(t, dtype=torch.float64, device=z.device)
        loss[rows] = lse - z[torch.arange(len(rows), device=z.device), at]
        if case["grad"] == "none":
            return {"loss": loss}
        z.sub_(lse[:, None]).exp_()
        z[torch.arange(len(rows), device=z.device), at] -= 1
        z.mul_(s["grad_loss"].double()[rows][:, None])
        dx = torch.zeros((t, case["hidden"]), dtype=torch.float64, device=z.device)
        dx[rows] = z @ w
        return {"loss": loss, "grad_hidden": dx, "grad_weight": z.t().contiguous() @ x}
    x, p = s["x"].double(), case["p"]
    scale = 1.0 / (1.0 - p)
    keep = _keep64(x.numel(), p, s["rng"], x.device).view(x.shape) if p else torch.ones_like(x, dtype=torch.bool)
    h = x.mul(scale).masked_fill(~keep, 0.0)
    if case["residual"]:
        h = h + s["residual"].double()
    if case["op"] == "dropout":
        out = {"out": h}
        if case["backward"]:
            out["grad_x"] = s["grad_out"].double().mul(scale).masked_fill(~keep, 0.0)
        return out
    w = s["weight"].double()
    # The norm is of the residual stream as it is stored, which the operator defines as x times the
    # 32-bit scale and the residual, product and sum in 32 bits, rounded to the input's type. From 64
    # bits, sums next to the middle of two bf16 numbers would be stored as the other one.
    kept = torch.where(keep, s["x"].to(torch.float32) * x.new_tensor(scale).to(torch.float32), 0.0)
    hr = (kept + s["residual"].to(torch.float32) if case["residual"] else kept).to(s["x"].dtype).double()
    rstd = 1.0 / torch.sqrt((hr * hr).mean(1) + 1e-5)
    unit = hr * rstd[:, None]
    y = unit * w
    out = {"h": h, "rstd": rstd, "y": y}
    if case["quant"]:
        q, rows = case["quant"], case["rows"]
        n = -(-case["hidden"] // q)
        wide = torch.zeros((rows, n * q), dtype=torch.float64, device=y.device)
        wide[:, :case["hidden"]] = y.abs()
        sc = wide.view(rows, n, q).max(2).values / E4M3_MAX
        out.update(y=y / sc.repeat_interleave(q, 1)[:, :case["hidden"]], scale=sc)
    if case["backward"]:
        dy = s["grad_out"].double()
        dh = (dy * w - unit * (dy * w * unit).mean(1)[:, None]) * rstd[:, None]
        if case["residual"]:
            dh = dh + s["grad_h"].double()
            out["grad_residual"] = dh
        out["grad_x"] = dh.mul(scale).masked_fill(~keep, 0.0)
        out["grad_weight"] = (dy * unit).sum(0)
    return out
