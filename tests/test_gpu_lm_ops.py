"""The training operators on the GPU against their plain forms in 64 bits."""
import itertools

import pytest
import torch

import megatron_dion_amd as mda
from megatron_dion_amd import lm_ops
from tests import _lm_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _randn(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _strided(t, pad):
    """The same values on the GPU with `pad` more elements between rows."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, :t.shape[1]] = t.cuda()
    return wide[:, :t.shape[1]]


def _close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst " \
                          f"{float(((got - want).abs() / (tol + 1e-300)).nan_to_num(1e30).max()):.3g} times the bound"


# ------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 3), (1, 768), (5, 7), (3, 64), (17, 1001), (64, 520)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(dtype, rows, cols, p):
    seed, offset = 0x1234567890ABCDEF, (7 << 32) + 3
    x, res = _randn(1, rows, cols, dtype=dtype), _randn(2, rows, cols, dtype=dtype)
    keep = R.keep_mask((rows, cols), p, seed, offset) if p else torch.ones(rows, cols, dtype=torch.bool)
    kept = R.dropped32(x, keep, p)
    for pad in (0, 3, 8):
        got = mda.dropout_add_forward(_strided(x, pad), p=p, rng=(seed, offset))
        assert torch.equal(got.cpu(), kept.to(dtype))
        got = mda.dropout_add_forward(_strided(x, pad), _strided(res, pad), p=p, rng=(seed, offset))
        assert torch.equal(got.cpu(), (kept + res.float()).to(dtype))
    grad = mda.dropout_add_backward(x.cuda(), p=p, rng=torch.tensor([seed, offset], device="cuda"))
    assert torch.equal(grad.cpu(), kept.to(dtype))


def test_dropout_drops_nan_and_infinity_and_keeps_its_rate():
    n = 1 << 20
    x = torch.full((n,), float("nan"), device="cuda")
    out = mda.dropout_add_forward(x, p=0.3, rng=(5, 9)).cpu()
    dropped = out == 0
    assert torch.equal(dropped, ~R.keep_mask((n,), 0.3, 5, 9))
    assert torch.isnan(out[~dropped]).all()
    # a binomial of n draws: 6 standard deviations
    assert abs(float(dropped.float().mean()) - 0.3) < 6 * (0.3 * 0.7 / n) ** 0.5
    assert (mda.dropout_add_forward(x, p=1.0, rng=(5, 9)) == 0).all()


def test_dropout_past_32_bits_of_elements():
    # 2^32 + 4096 elements: the counter's high word, and offsets of over 4 GiB
    n = (1 << 32) + 4096
    x = torch.ones(n, dtype=BF16, device="cuda")
    out = mda.dropout_add_forward(x, p=0.5, rng=(11, 13))
    tail = out[1 << 32:].cpu()
    g = torch.arange(1024, dtype=torch.int64) + (1 << 30)
    import numpy as np
    c = [np.asarray(g, dtype=np.uint64) & np.uint64(0xFFFFFFFF), np.asarray(g, dtype=np.uint64) >> np.uint64(32)]
    assert c[1].max() == 0  # groups of 4: the high word comes at 2^34 elements
    want = _words_of_groups(g, 11, 13) >= (1 << 31)
    assert torch.equal(tail != 0, want.view(-1))
    assert torch.equal(out[:4096].cpu() != 0, R.keep_mask((4096,), 0.5, 11, 13))


def _words_of_groups(groups, seed, offset):
    first, last = int(groups[0]), int(groups[-1])
    import numpy as np
    m32 = np.uint64(0xFFFFFFFF)
    g = np.arange(first, last + 1, dtype=np.uint64)
    c = [g & m32, g >> np.uint64(32), np.full_like(g, offset), np.zeros_like(g)]
    k0, k1 = seed, 0
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.from_numpy(np.stack(c, 1).astype(np.int64))


# ------------------------------------------------------------------------------- residual RMS norm
def _norm_reference(x, w, res, p, seed, offset, eps):
    keep = R.keep_mask(tuple(x.shape), p, seed, offset) if p else torch.ones(x.shape, dtype=torch.bool)
    h = R.dropped32(x, keep, p)
    h = (h + res.float() if res is not None else h).to(x.dtype)
    hd = h.double()
    rstd = (hd.square().mean(1) + eps).rsqrt()
    return keep, h, rstd, hd * rstd[:, None] * w.double()


NORM_SIZES = [(1, 1), (3, 5), (1, 4096), (5, 64), (2, 512), (9, 520), (4, 768), (3, 1000), (7, 1001), (5, 2048),
              (3, 2056), (2, 4100), (2, 8192), (3, 8200), (2, 16384), (2, 16383)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_norm_forward_and_backward(dtype, rows, cols):
    for k, (p, with_res, wdt, pad) in enumerate([(0.0, True, F32, 0), (0.2, True, F32, 8), (0.2, False, BF16, 3),
                                                 (0.0, False, F32, 0)]):
        seed, offset = 99 + k, 1 << 40
        x = _randn(3, rows, cols, dtype=dtype)
        res = _randn(4, rows, cols, scale=2.0, dtype=dtype) if with_res else None
        w = (1 + _randn(5, cols, scale=0.2)).to(wdt)
        eps = 1e-5
        keep, h, rstd, y = _norm_reference(x, w, res, p, seed, offset, eps)
        f = mda.rms_norm_add_forward(_strided(x, pad), w.cuda(), None if res is None else _strided(res, pad), eps=eps,
                                     p=p, rng=(seed, offset) if p else None)
        assert torch.equal(f.h.cpu(), h)
        e_sum = (cols / 64 + 24) * R.U32  # of the sum of squares: at most cols / 64 terms a thread, then a tree
        _close(f.rstd, rstd, (e_sum / 2 + 4 * R.U32) * rstd, "rstd")
        _close(f.y, y, (e_sum / 2 + 6 * R.U32 + R.half_step(dtype)) * y.abs(), "y")
        # backward
        gy, gh = _randn(6, rows, cols, scale=1e-2, dtype=dtype), _randn(7, rows, cols, scale=1e-2, dtype=dtype)
        gh = gh if with_res else None
        b = mda.rms_norm_add_backward(_strided(gy, pad), f.h, w.cuda(), f.rstd, None if gh is None else _strided(gh, pad),
                                      p=p, rng=(seed, offset) if p else None)
        u = h.double() * rstd[:, None]
        wg = w.double() * gy.double()
        dot = (wg * u).mean(1, keepdim=True)
        d = rstd[:, None] * (wg - u * dot) + (0 if gh is None else gh.double())
        size = rstd[:, None] * (wg.abs() + u.abs() * (wg * u).abs().mean(1, keepdim=True)) + \
            (0 if gh is None else gh.double().abs())
        e_d = (2 * e_sum + 12 * R.U32) * size
        _close(b.grad_residual, d, e_d + R.half_step(dtype) * d.abs(), "grad_residual")
        scale = 1.0 / (1.0 - p)
        gx = torch.where(keep, d * scale, torch.zeros_like(d))
        _close(b.grad_x, gx, (e_d * scale + (R.half_step(dtype) + 3 * R.U32) * gx.abs()), "grad_x")
        gw = (gy.double() * u).sum(0)
        mag = (gy.double() * u).abs().sum(0)
        tol = (e_sum / 2 + (rows + 16) * R.U32) * mag
        _close(b.grad_weight, gw, tol + R.half_step(wdt) * gw.abs(), "grad_weight")
        if p == 0.0:
            assert b.grad_x is b.grad_residual
        only = mda.rms_norm_add_backward(gy.cuda(), f.h, w.cuda(), f.rstd, None if gh is None else gh.cuda(), p=p,
                                         rng=(seed, offset) if p else None, need_weight=False, need_residual=False)
        assert torch.equal(only.grad_x, b.grad_x) and only.grad_residual is None and only.grad_weight is None
        # added to an fp32 and to a bf16 main_grad
        for mdt in (F32, BF16):
            main = _randn(8, cols, dtype=mdt).cuda()
            before = main.double().cpu()
            c = mda.rms_norm_add_backward(gy.cuda(), f.h, w.cuda(), f.rstd, None, grad_weight=main, accumulate=True,
                                          need_input=False)
            assert c.grad_x is None and c.grad_weight is main
            _close(main, before + gw, tol + R.half_step(mdt) * (before + gw).abs() + R.U32 * before.abs(), "main_grad")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols,block", [(1, 1, 1), (3, 128, 128), (5, 200, 128), (4, 768, 32), (2, 1001, 100),
                                             (3, 4096, 128), (2, 4096, -1), (2, 4104, 512), (1, 8192, 8), (2, 16384, 64)])
def test_norm_in_8_bits(dtype, rows, cols, block):
    x, res, w = _randn(1, rows, cols, dtype=dtype), _randn(2, rows, cols, dtype=dtype), 1 + _randn(3, cols, scale=0.3)
    x[0] = 0
    res[0] = 0  # a row of zeros: the least scale, and zeros
    _, h, rstd, y = _norm_reference(x, w, res, 0.0, 0, 0, 1e-5)
    f = mda.rms_norm_add_forward(x.cuda(), w.cuda(), res.cuda(), scale_block=block)
    assert torch.equal(f.h.cpu(), h) and f.y.dtype == torch.float8_e4m3fn
    b = cols if block < 0 else block
    n = -(-cols // b)
    assert f.scale.shape == (rows, n)
    amax = torch.nn.functional.pad(y.abs(), (0, n * b - cols)).view(rows, n, b).amax(2)
    scale = (amax / 448).clamp_min(2.0 ** -126)
    e = (cols / 64 + 24) / 2 * R.U32 + 8 * R.U32
    _close(f.scale, scale, e * scale, "scale")
    got = f.y.float().cpu().double() * f.scale.cpu().double().repeat_interleave(b, 1)[:, :cols]
    # half a step of 3 mantissa bits (2^-4), or of the least subnormal (2^-10 of a unit)
    step = 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale.repeat_interleave(b, 1)[:, :cols]
    _close(got, y, step + 2 * e * y.abs(), "y")
    assert (f.y[0].float() == 0).all()
    top = f.y.float().abs().cpu()
    top = torch.nn.functional.pad(top, (0, n * b - cols)).view(rows, n, b).amax(2)
    assert (top[1:] == 448).all()  # the largest of each block takes the largest code


@pytest.mark.parametrize("rows,cols", [((1 << 26) + 6, 8), ((1 << 21) + 3, 1032)])
def test_norm_of_more_rows_than_one_axis_of_a_grid_holds(rows, cols):
    """64 threads a row make 2^32 of the first; the second fills an axis of 2^21 blocks."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(generator=g)
    w = _randn(4, cols)
    f = mda.rms_norm_add_forward(x, w.cuda(), eps=1e-5)
    for part in (slice(0, 70), slice((1 << 23) - 35, (1 << 23) + 35), slice(rows - 70, rows)):
        part = slice(min(part.start, rows - 70), min(part.stop, rows))
        want = _norm_reference(x[part].cpu(), w, None, 0.0, 0, 0, 1e-5)
        # cols squares added in fp32, a root, a quotient and two products: (cols + 8) half steps; then bf16's
        off = (cols + 8) * R.U32
        _close(f.rstd[part], want[2], off * want[2], "rstd")
        _close(f.y[part], want[3], (off + 2.0 ** -8) * want[3].abs(), "y")


def test_norm_rows_do_not_mix_and_nan_stays_in_its_row():
    x, w = _randn(1, 6, 1024, dtype=BF16), torch.ones(1024)
    x[2, 5], x[4, 7] = float("nan"), float("inf")
    f = mda.rms_norm_add_forward(x.cuda(), w.cuda())
    ok = [0, 1, 3, 5]
    g = mda.rms_norm_add_forward(x[ok].contiguous().cuda(), w.cuda())
    assert torch.equal(f.y[ok], g.y) and torch.isnan(f.y[2]).all() and torch.isnan(f.y[4, 7])
    q = mda.rms_norm_add_forward(x.cuda(), w.cuda(), scale_block=128)
    assert torch.isnan(q.y[2].float()).all() and torch.isfinite(q.y[ok].float()).all()


def test_empty():
    e = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    assert mda.dropout_add_forward(e, p=0.5, rng=(1, 2)).shape == (0, 64)
    f = mda.rms_norm_add_forward(e, w, e)
    assert f.y.shape == (0, 64) and f.rstd.shape == (0,)
    b = mda.rms_norm_add_backward(e, f.h, w, f.rstd, e)
    assert b.grad_x.shape == (0, 64) and (b.grad_weight == 0).all()
    wv = torch.randn(100, 64, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = mda.linear_cross_entropy_forward(e, wv, t)
    assert loss.shape == (0,)
    gh, gw = mda.linear_cross_entropy_backward(loss, e, wv, t, lse)
    assert gh.shape == (0, 64) and (gw == 0).all()
    main = torch.ones_like(wv)
    mda.linear_cross_entropy_backward(loss, e, wv, t, lse, grad_weight=main, accumulate=True)
    assert (main == 1).all()


# ------------------------------------------------------------------------------- linear cross entropy
def _xent_case(tokens, hidden, vocab, dtype, ignored, seed=0):
    x = _randn(seed, tokens, hidden, dtype=dtype)
    w = _randn(seed + 1, vocab, hidden, scale=2 * hidden ** -0.5, dtype=dtype)
    g = torch.Generator().manual_seed(seed + 2)
    t = torch.randint(0, vocab, (tokens,), generator=g)
    t[torch.rand(tokens, generator=g) < ignored] = -100
    gl = torch.rand(tokens, generator=g) / max(tokens, 1)
    return x, w, t, gl


def _xent_check(x, w, t, gl, *, out_dtype=None, pad=0, **kw):
    ref = R.xent(x, w, t, -100, gl, out_dtype=out_dtype)
    xc, wc, tc, gc = _strided(x, pad), _strided(w, pad), t.cuda(), gl.cuda()
    loss, lse = mda.linear_cross_entropy_forward(xc, wc, tc, **kw)
    _close(loss, ref["loss"], ref["e_loss"], "loss")
    _close(lse, ref["lse"], ref["e_loss"], "lse")
    gw = None if out_dtype is None else torch.full(w.shape, float("nan"), dtype=out_dtype, device="cuda")
    dx, dw = mda.linear_cross_entropy_backward(gc, xc, wc, tc, lse, grad_weight=gw, **kw)
    _close(dx, ref["grad_hidden"], ref["e_grad_hidden"], "grad_hidden")
    _close(dw, ref["grad_weight"], ref["e_grad_weight"], "grad_weight")
    return loss, lse, dx, dw, ref


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("tokens,hidden,vocab", [
    (1, 8, 1), (1, 64, 2), (1, 768, 1000), (2, 40, 127), (31, 64, 128), (32, 72, 129), (33, 64, 257), (64, 128, 300),
    (65, 200, 513), (128, 64, 1000), (129, 136, 255), (200, 768, 520), (256, 64, 256), (257, 320, 1003),
    (513, 96, 2001), (40, 1, 50), (40, 7, 50), (2500, 64, 300),
    # every tile: 128 x 128 and 256 x 256 of the logits, 128 x 128 and 256 x 256 of dW
    (300, 72, 20000), (300, 72, 33000), (700, 72, 50000)])
def test_xent(dtype, out_dtype, tokens, hidden, vocab):
    x, w, t, gl = _xent_case(tokens, hidden, vocab, dtype, 0.2 if tokens > 2 else 0.0)
    _xent_check(x, w, t, gl, out_dtype=out_dtype)


@pytest.mark.parametrize("dtype,tokens,hidden,vocab,pad", [
    (BF16, 5, 33, 70, 0), (BF16, 40, 1001, 300, 0), (BF16, 300, 100, 515, 0), (BF16, 70, 64, 200, 3),
    (BF16, 70, 64, 200, 8), (F32, 70, 65, 200, 1), (F32, 300, 250, 515, 0)])
def test_xent_odd_widths_and_strides(dtype, tokens, hidden, vocab, pad):
    x, w, t, gl = _xent_case(tokens, hidden, vocab, dtype, 0.3)
    _xent_check(x, w, t, gl, out_dtype=F32, pad=pad)


def test_xent_misaligned_weight():
    x, w, t, gl = _xent_case(40, 64, 300, BF16, 0.0)
    flat = torch.empty(300 * 64 + 1, dtype=BF16, device="cuda")
    wm = flat[1:].view(300, 64)
    wm.copy_(w)
    loss, lse = mda.linear_cross_entropy_forward(x.cuda(), wm, t.cuda())
    same, _ = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    assert torch.equal(loss, same)


def test_xent_ignored_tokens_are_not_read_and_cost_nothing():
    for dtype, tokens in itertools.product((BF16, F32), (20, 100, 400)):
        x, w, t, gl = _xent_case(tokens, 64, 300, dtype, 0.5)
        gl[3::7] = 0.0
        out = [mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())]
        out.append(mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), out[0][1]))
        bad, badgl = x.clone(), gl.clone()
        bad[t == -100] = float("nan")
        badgl[t == -100] = float("nan")
        loss, lse = mda.linear_cross_entropy_forward(bad.cuda(), w.cuda(), t.cuda())
        assert torch.equal(loss, out[0][0]) and torch.equal(lse, out[0][1])
        bad[gl == 0] = float("inf")
        dx, dw = mda.linear_cross_entropy_backward(badgl.cuda(), bad.cuda(), w.cuda(), t.cuda(), lse)
        assert torch.equal(dx, out[1][0]) and torch.equal(dw, out[1][1])
        off = (t == -100) | (gl == 0)
        assert (dx[off.cuda()] == 0).all()
        _xent_check(x, w, t, gl, out_dtype=F32)


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_xent_no_token_takes_part(tokens):
    x = torch.full((tokens, 64), float("nan"), dtype=BF16, device="cuda")
    w = torch.randn(300, 64, device="cuda").to(BF16)
    t = torch.full((tokens,), -100, device="cuda")
    loss, lse = mda.linear_cross_entropy_forward(x, w, t)
    assert (loss == 0).all() and (lse == 0).all()
    dx, dw = mda.linear_cross_entropy_backward(torch.ones(tokens, device="cuda"), x, w, t, lse)
    assert (dx == 0).all() and (dw == 0).all()
    main = torch.ones(300, 64, device="cuda")
    mda.linear_cross_entropy_backward(torch.ones(tokens, device="cuda"), x, w, t, lse, grad_weight=main, accumulate=True)
    assert (main == 1).all()


def test_xent_targets_outside_the_vocabulary_say_so():
    x, w, t, gl = _xent_case(10, 64, 100, BF16, 0.0)
    t[2], t[5], t[7] = 100, -1, -100
    loss, lse = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    assert torch.isnan(loss).cpu().tolist() == [i in (2, 5) for i in range(10)] and loss[7] == 0
    dx, _ = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), lse)
    assert torch.isnan(dx).all(1).cpu().tolist() == [i in (2, 5) for i in range(10)]


def test_xent_large_logits_and_nan():
    x, w, t, gl = _xent_case(40, 64, 300, F32, 0.0)
    _xent_check(x * 30, w, t, gl, out_dtype=F32)  # logits of hundreds: no overflow of the exponentials
    x[4, 3] = float("nan")
    loss, lse = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    assert torch.isnan(loss).cpu().tolist() == [i == 4 for i in range(40)]


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_xent_vocabulary_shards_and_padding(dtype, out_dtype):
    """Two shards of a vocabulary of 500 in 512 rows, whose last 12 hold NaN: joined as two ranks would."""
    x, w, t, gl = _xent_case(70, 64, 500, dtype, 0.1)
    ref = R.xent(x, w, t, -100, gl, out_dtype=out_dtype)
    pad = torch.full((512, 64), float("nan"), dtype=dtype)
    pad[:500] = w
    lib = lm_ops
    parts = []
    for k in (0, 256):
        hm, wm, tv = x.cuda(), pad[k:k + 256].cuda(), t.cuda()
        d, nbytes = lib._xent_desc(1, hm, wm, tv, k, 500, -100)
        ws = lib._workspace(nbytes, hm.device)
        lse, tl = torch.empty(70, device="cuda"), torch.empty(70, device="cuda")
        import ctypes
        rc = lib._lm_lib.load().dion_xent_forward(ctypes.byref(d), hm.data_ptr(), wm.data_ptr(), tv.data_ptr(), None,
                                                  lse.data_ptr(), tl.data_ptr(), ws.data_ptr(), ws.numel(),
                                                  torch.cuda.current_stream().cuda_stream)
        lib._lm_lib.check(rc, "dion_xent_forward")
        parts.append((lse, tl))
    torch.cuda.synchronize()
    valid = (t != -100).cuda()
    lse = torch.where(valid, torch.logaddexp(parts[0][0], parts[1][0]), torch.zeros(70, device="cuda"))
    loss = torch.where(valid, lse - parts[0][1] - parts[1][1], torch.zeros(70, device="cuda"))
    _close(loss, ref["loss"], ref["e_loss"] + 8 * R.U32 * (1 + ref["lse"].abs()), "loss")
    dx = torch.zeros(70, 64, dtype=torch.float64)
    for k in (0, 256):
        gh, gw = mda.linear_cross_entropy_backward(
            gl.cuda(), x.cuda(), pad[k:k + 256].cuda(), t.cuda(), lse, vocab_start=k, vocab_size=500,
            grad_weight=torch.full((256, 64), float("nan"), dtype=out_dtype, device="cuda"))
        dx += gh.double().cpu()
        n = min(256, 500 - k)
        _close(gw[:n], ref["grad_weight"][k:k + n], 1.01 * ref["e_grad_weight"][k:k + n], "grad_weight")
        assert (gw[n:] == 0).all()
    # each share is rounded once
    _close(dx, ref["grad_hidden"], 1.01 * ref["e_grad_hidden"] + 2 * R.half_step(dtype) * (
        ref["grad_hidden"].abs().amax()), "grad_hidden")


@pytest.mark.parametrize("dtype,mdt", [(BF16, BF16), (BF16, F32), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("hidden", [64, 70])
def test_xent_accumulates_into_main_grad(dtype, mdt, hidden):
    x, w, t, gl = _xent_case(90, hidden, 300, dtype, 0.1)
    ref = R.xent(x, w, t, -100, gl, out_dtype=mdt)
    _, lse = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    main = _randn(9, 300, hidden, scale=1e-2, dtype=mdt).cuda()
    before = main.double().cpu()
    dx, got = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), lse, grad_weight=main,
                                                accumulate=True, need_hidden=False)
    assert dx is None and got is main
    want = before + ref["grad_weight"]
    _close(main, want, ref["e_grad_weight"] + R.half_step(mdt) * (want.abs() + before.abs()) + R.U32 * before.abs(), "main_grad")


def test_xent_gradient_against_differences():
    """fp32: the gradient of the summed loss against central differences of the 64-bit loss."""
    x, w, t, gl = _xent_case(12, 24, 50, F32, 0.2)
    _, lse = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    dx, dw = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), lse)

    def f(xd, wd):
        z = xd @ wd.t()
        ok = t != -100
        per = torch.logsumexp(z, 1) - z.gather(1, t.clamp_min(0)[:, None])[:, 0]
        return float((per * gl.double())[ok].sum())

    xd, wd, e = x.double(), w.double(), 1e-4
    for i, j in [(0, 0), (5, 7), (11, 23)]:
        d = torch.zeros_like(xd)
        d[i, j] = e
        assert abs((f(xd + d, wd) - f(xd - d, wd)) / (2 * e) - float(dx[i, j])) < 1e-6
    for i, j in [(0, 0), (int(t[t >= 0][0]), 3), (49, 23)]:
        d = torch.zeros_like(wd)
        d[i, j] = e
        assert abs((f(xd, wd + d) - f(xd, wd - d)) / (2 * e) - float(dw[i, j])) < 1e-6


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("tokens,hidden,vocab", [(20, 64, 600), (100, 72, 1025), (300, 320, 1300)])
def test_xent_in_pieces_of_256_words(dtype, out_dtype, tokens, hidden, vocab):
    x, w, t, gl = _xent_case(tokens, hidden, vocab, dtype, 0.1)
    ref = R.xent(x, w, t, -100, gl, out_dtype=out_dtype)
    a = (x.cuda(), w.cuda(), t.cuda())
    _, lse = mda.linear_cross_entropy_forward(*a)
    gw = torch.full((vocab, hidden), float("nan"), dtype=out_dtype, device="cuda")
    dx, dw = mda.linear_cross_entropy_backward(gl.cuda(), *a, lse, grad_weight=gw, piece_bytes=1)
    _close(dx, ref["grad_hidden"], ref["e_grad_hidden"], "grad_hidden")
    _close(dw, ref["grad_weight"], ref["e_grad_weight"], "grad_weight")


@pytest.mark.parametrize("tokens", [40, 2500])
def test_xent_fp32_over_many_magnitudes(tokens):
    """Hidden states from 1e-12 to 1e3, weights from 1e-9, upstream gradients from 1e-20: the limbs' scales
    follow the largest, and what a limb cannot hold is 2^-39 of it."""
    x, w, t, gl = _xent_case(tokens, 64, 300, F32, 0.2)
    g = torch.Generator().manual_seed(5)
    x = x * 10.0 ** (torch.rand(tokens, 1, generator=g) * 15 - 12)
    w = w * 10.0 ** (torch.rand(300, 1, generator=g) * 9 - 9)
    gl = gl * 10.0 ** (-20 * torch.rand(tokens, generator=g))
    for scale in (1.0, 1e-25, 1e12):
        _xent_check(x * scale, w / scale, t, gl, out_dtype=F32)


def test_xent_main_grad_in_fp32_precision():
    """bf16 inputs and an fp32 grad_weight: off by no more of its 2-norm than a product in fp32 would be."""
    x, w, t, gl = _xent_case(700, 256, 1500, BF16, 0.1)
    ref = R.xent(x, w, t, -100, gl, out_dtype=F32)["grad_weight"]
    a = (x.cuda(), w.cuda(), t.cuda())
    _, lse = mda.linear_cross_entropy_forward(*a)
    _, dw = mda.linear_cross_entropy_backward(gl.cuda(), *a, lse, grad_weight=torch.empty(1500, 256, device="cuda"))
    assert float((dw.double().cpu() - ref).norm() / ref.norm()) < 1e-6


@pytest.mark.parametrize("tokens", [1, 3, 8, 40, 300, 600])
def test_xent_bf16_gradients_are_near_their_rounding(tokens):
    """bf16 results lose little more than their own rounding to bf16, few tokens or many: dX because what a
    target's g loses is put back, dW of up to 256 tokens because g is an fp16 there.  Of more tokens' dW the
    roundings of g, as large as the result's and independent of them, add as much again: sqrt(2), and 1.6
    leaves room for 300 tokens' scatter."""
    for seed in range(3):
        x, w, t, gl = _xent_case(tokens, 256, 1500, BF16, 0.0, seed=100 * seed + tokens)
        ref = R.xent(x, w, t, -100, gl, out_dtype=BF16)
        a = (x.cuda(), w.cuda(), t.cuda())
        _, lse = mda.linear_cross_entropy_forward(*a)
        got = mda.linear_cross_entropy_backward(gl.cuda(), *a, lse)
        for g, k, most in ((got[0], "grad_hidden", 1.2), (got[1], "grad_weight", 1.2 if tokens <= 256 else 1.6)):
            off = (g.double().cpu() - ref[k]).norm()
            assert float(off) <= most * float((ref[k].to(BF16).double() - ref[k]).norm()), (k, seed)


def test_xent_infinity_stays_in_its_row_and_column():
    x, w, t, gl = _xent_case(50, 64, 300, F32, 0.0)
    clean = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    x[7, 5] = float("inf")
    loss, lse = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    keep = torch.arange(50) != 7
    assert not torch.isfinite(loss[7]) and torch.equal(loss[keep.cuda()], clean[0][keep.cuda()])


def test_xent_is_bitwise_reproducible():
    x, w, t, gl = _xent_case(300, 128, 3000, BF16, 0.1)
    a = (x.cuda(), w.cuda(), t.cuda())
    loss, lse = mda.linear_cross_entropy_forward(*a)
    first = mda.linear_cross_entropy_backward(gl.cuda(), *a, lse)
    for _ in range(3):
        again, lse2 = mda.linear_cross_entropy_forward(*a)
        assert torch.equal(loss, again) and torch.equal(lse, lse2)
        for u, v in zip(first, mda.linear_cross_entropy_backward(gl.cuda(), *a, lse)):
            assert torch.equal(u, v)


def test_leading_axes_and_graph_capture():
    """The step's operators, captured once and replayed with new inputs and a new mask each time."""
    torch.manual_seed(0)
    b, s, h, v = 2, 24, 128, 500
    x = torch.randn(b, s, h, device="cuda").to(BF16)
    res = torch.randn(b, s, h, device="cuda").to(BF16)
    nw = torch.rand(h, device="cuda") + 0.5
    w = (torch.randn(v, h, device="cuda") * 0.1).to(BF16)
    t = torch.randint(0, v, (b, s), device="cuda")
    gl = torch.rand(b, s, device="cuda") / (b * s)
    rng = torch.tensor([7, 0], device="cuda")
    main, nmain = torch.zeros(v, h, device="cuda"), torch.zeros(h, device="cuda")

    def step(r):
        f = mda.rms_norm_add_forward(x, nw, res, p=0.1, rng=r)
        loss, lse = mda.linear_cross_entropy_forward(f.y, w, t)
        gy, _ = mda.linear_cross_entropy_backward(gl, f.y, w, t, lse, grad_weight=main)
        bk = mda.rms_norm_add_backward(gy, f.h, nw, f.rstd, None, p=0.1, rng=r, grad_weight=nmain)
        return loss, bk.grad_x, bk.grad_residual

    step(rng)  # loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(rng)
        rng[1:].add_(1)
    rng[1] = 0
    seen = []
    for k in range(4):
        x.copy_(torch.randn(b, s, h, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out] + [main.clone(), nmain.clone()]
        want = list(step((7, k))) + [main, nmain]
        for u, q in zip(got, want):
            assert torch.equal(u, q), k
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_two_captured_graphs_replayed_together():
    """Large tiles and prepared batches in two graphs, each with its own memory, replayed on two streams."""
    cases = [_xent_case(600, 64, 30000, BF16, 0.1, seed=3), _xent_case(40, 64, 3000, F32, 0.1, seed=4)]
    dev = [tuple(u.cuda() for u in c) for c in cases]

    def step(x, w, t, gl):
        loss, lse = mda.linear_cross_entropy_forward(x, w, t)
        return (loss, *mda.linear_cross_entropy_backward(gl, x, w, t, lse))

    want = [step(*c) for c in dev]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for o in outs:
            for u in o:
                u.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, q in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, q))
        step(*dev[0])  # eager work in between


def test_xent_weight_past_31_bits_of_elements():
    """530000 x 4096 words: offsets of over 2^31 elements in weight and grad_weight."""
    tokens, hidden, vocab = 6, 4096, 530000
    torch.manual_seed(0)
    w = torch.empty(vocab, hidden, dtype=BF16, device="cuda").normal_(0, 0.02)
    x = torch.randn(tokens, hidden, device="cuda").to(BF16)
    t = torch.tensor([0, vocab - 1, vocab - 2, 525000, 262144, -100], device="cuda")
    gl = torch.rand(tokens, device="cuda")
    loss, lse = mda.linear_cross_entropy_forward(x, w, t)
    z = torch.cat([x.float() @ w[k:k + 65536].float().t() for k in range(0, vocab, 65536)], 1).double()
    ref = torch.logsumexp(z, 1)
    live = t >= 0
    want = torch.where(live, ref - z.gather(1, t.clamp_min(0)[:, None])[:, 0], torch.zeros_like(ref))
    # logits of |x||w| sums of 4096 terms of 0.016 on average in fp32, twice
    assert float((loss.double() - want).abs().max()) < 2 * (4096 / 16 + 20) * R.U32 * 66 + 1e-5
    _, dw = mda.linear_cross_entropy_backward(gl, x, w, t, lse, need_hidden=False)
    p = torch.exp(z - ref[:, None])
    p[live.nonzero()[:, 0], t[live]] -= 1
    p *= torch.where(live, gl, torch.zeros_like(gl))[:, None]
    for k in (0, 262144, 524289, 525000, vocab - 2, vocab - 1):
        row = (p[:, k] @ x.double())
        # g is one fp16 here (2^-11 of it), p is off by the logits' 66 (4096 / 16 + 20) 2^-24 = 1.1e-3 at most
        # and measured against fp32 logits, and the sum is rounded once
        tol = (2.0 ** -11 + 1.1e-3) * (p[:, k].abs() @ x.double().abs()) + 2.0 ** -8 * row.abs()
        assert bool(((dw[k].double() - row).abs() <= tol).all()), k


def test_xent_of_more_tiles_than_one_axis_of_a_grid_holds():
    """2^22 tokens x 131072 words are 2^23 tiles of 512 threads: two launches."""
    tokens, hidden, vocab = 1 << 22, 8, 131072
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(tokens, hidden, dtype=BF16, device="cuda").normal_(generator=g)
    w = torch.empty(vocab, hidden, dtype=BF16, device="cuda").normal_(generator=g)
    t = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    loss, lse = mda.linear_cross_entropy_forward(x, w, t)
    some = torch.cat((torch.arange(20), torch.arange(tokens // 2 - 10, tokens // 2 + 10), torch.arange(tokens - 20, tokens)))
    at = some.cuda()
    ref = R.xent(x[at].cpu(), w.cpu(), t[at].cpu(), -100)
    _close(lse[at], ref["lse"], ref["e_loss"], "lse")
    _close(loss[at], ref["loss"], ref["e_loss"], "loss")
    assert bool(torch.isfinite(loss).all())


def test_two_streams_at_once():
    cases = [_xent_case(200 + 50 * k, 128, 1500, BF16, 0.1, seed=10 * k) for k in range(3)]
    dev = [tuple(u.cuda() for u in c) for c in cases]
    alone = []
    for x, w, t, gl in dev:
        loss, lse = mda.linear_cross_entropy_forward(x, w, t)
        alone.append((loss, *mda.linear_cross_entropy_backward(gl, x, w, t, lse)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    for _ in range(3):
        got = []
        for s, (x, w, t, gl) in zip(streams, dev):
            with torch.cuda.stream(s):
                loss, lse = mda.linear_cross_entropy_forward(x, w, t)
                got.append((loss, *mda.linear_cross_entropy_backward(gl, x, w, t, lse)))
        torch.cuda.synchronize()
        for u, q in zip(got, alone):
            assert all(torch.equal(a, b) for a, b in zip(u, q))


# ------------------------------------------------------------------------------- autograd
def test_autograd_step_into_the_optimizer():
    """A small model's end: dropout, residual, norm, loss; gradients by autograd equal those of torch's own
    operations in 64 bits (p = 0), and the optimizer takes them from main_grad."""
    from megatron_dion_amd.optimizer import attach_dp_routing

    torch.manual_seed(1)
    n, h, v = 48, 64, 300
    lin = torch.nn.Parameter((torch.randn(h, h, device="cuda") * 0.1))
    norm = torch.nn.Parameter(torch.ones(h, device="cuda"))
    out = torch.nn.Parameter(torch.randn(v, h, device="cuda") * 0.1)
    x = torch.randn(n, h, device="cuda")
    t = torch.randint(0, v, (n,), device="cuda")
    t[::5] = -100
    out.main_grad = torch.zeros_like(out)
    y, hh = mda.rms_norm_add(x @ lin, norm, x)
    y2, _ = mda.rms_norm_add(y, norm)
    loss = mda.linear_cross_entropy(mda.dropout_add(y2, hh, p=0.0), out, t, into_main_grad=True)
    total = loss.sum() / (t != -100).sum()
    total.backward()
    ld, nd, od, xd = (u.detach().double().cpu().requires_grad_() for u in (lin, norm, out, x))

    def rms(z):
        return z * torch.rsqrt(z.square().mean(1, keepdim=True) + 1e-5) * nd

    hd = xd + xd @ ld
    zd = (rms(rms(hd)) + hd) @ od.t()
    want = torch.nn.functional.cross_entropy(zd, t.cpu(), ignore_index=-100)
    want.backward()
    assert abs(total.item() - want.item()) < 1e-5
    # fp32 through three products and two norms: 1e-5 of the largest gradient is over 100 roundings
    for got, ref in ((lin.grad, ld.grad), (norm.grad, nd.grad), (out.main_grad, od.grad)):
        assert float((got.double().cpu() - ref).abs().max()) < 1e-5 * float(ref.abs().max())
    assert out.grad is None
    lin.main_grad, norm.main_grad = lin.grad, norm.grad
    opt = mda.MegatronDion([lin, norm, out], lr=0.01, rank_fraction=0.25)
    attach_dp_routing(opt, [("linear.weight", lin), ("norm.weight", norm), ("output_layer.weight", out)])
    before = [u.detach().clone() for u in (lin, norm, out)]
    assert mda.dion_grad_norm(opt, [lin.main_grad]) > 0
    opt.step()
    torch.cuda.synchronize()
    for a, b in zip(before, (lin, norm, out)):
        assert torch.isfinite(b).all() and not torch.equal(a, b)


def test_autograd_masks_match_and_unused_outputs():
    x = torch.randn(33, 72, device="cuda", requires_grad=True)
    r = torch.randn(33, 72, device="cuda", requires_grad=True)
    w = torch.rand(72, device="cuda", requires_grad=True)
    rng = torch.tensor([3, 4], device="cuda")
    out = mda.dropout_add(x, r, p=0.4, rng=rng)
    rng.add_(1)  # the state moves on; the backward pass has its own
    out.sum().backward()
    keep = R.keep_mask((33, 72), 0.4, 3, 4).cuda()
    assert torch.equal(x.grad != 0, keep) and (r.grad == 1).all()
    x.grad = r.grad = None
    y, h = mda.rms_norm_add(x, w, r, p=0.4, rng=(3, 4))
    h.sum().backward()  # only the residual stream
    assert torch.equal(x.grad != 0, keep) and (r.grad == 1).all() and w.grad is None
    x.grad = r.grad = None
    y, h = mda.rms_norm_add(x, w, r, p=0.4, rng=(3, 4))
    (2 * y.t()).sum().backward()
    assert torch.equal(x.grad != 0, keep) and w.grad is not None


def test_autograd_is_refused_under_capture():
    x, w, t, gl = _xent_case(8, 64, 100, BF16, 0.0)
    x, w, t = x.cuda(), w.cuda(), t.cuda()
    mda.linear_cross_entropy_forward(x, w, t)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="DION_AUTOGRAD_CAPTURE"):
            mda.linear_cross_entropy(x, w, t)
        with pytest.raises(RuntimeError, match="DION_AUTOGRAD_CAPTURE"):
            mda.dropout_add(x, p=0.1, rng=(1, 1))
        with pytest.raises(RuntimeError, match="DION_AUTOGRAD_CAPTURE"):
            mda.rms_norm_add(x, torch.ones(64, device="cuda"))
        y = x + 1
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x + 1)
