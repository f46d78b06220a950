"""The training operators on the GPU at the ends of their ranges: what each rounding may cost, and no more."""
import pytest
import torch

import megatron_dion_amd as mda
from tests import _lm_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------- norm in 8 bits
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols,block", [(128, 128), (4096, 128), (4096, -1), (4096, 96), (1000, 128), (999, 100), (16, 8)])
def test_norm_in_8_bits_is_the_quotient_rounded(dtype, cols, block):
    """y / s, rounded to fp32 and then to e4m3, code for code.  A row of +-1 with eps = 0 has rstd = 1, so y is +-w
    exactly; the weights are the middles of two codes times a scale that is no power of two, where a rounding more
    changes the code."""
    g = torch.Generator().manual_seed(cols)
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    middles = (codes[1:] + codes[:-1]) / 2
    b = cols if block < 0 else block
    n = -(-cols // b)
    for size in [1.0] * 8 + [2.0 ** -80, 2.0 ** -95, 2.0 ** -115, 2.0 ** 100]:
        top = 448.0 * size * (1.0 + torch.rand(n, generator=g))
        s = (top / 448.0).clamp_min(2.0 ** -126)  # fp32, as the operator takes it from the block's largest
        w = middles[torch.randint(0, len(middles), (n, b), generator=g)] * s[:, None]
        w[:, 0] = top
        w = w.view(-1)[:cols].contiguous()
        x = torch.where(torch.rand(3, cols, generator=g) < 0.5, -1.0, 1.0).to(dtype)
        f = mda.rms_norm_add_forward(x.cuda(), w.cuda(), eps=0.0, scale_block=block)
        assert (f.rstd == 1.0).all()
        assert torch.equal(f.scale.cpu(), s.expand(3, n))
        want = (w / s.repeat_interleave(b)[:cols]).clamp(-448.0, 448.0) * x.float()
        want = want.to(torch.float8_e4m3fn)
        assert torch.equal(f.y.cpu().view(torch.uint8), want.view(torch.uint8)), size


def test_norm_in_8_bits_of_a_block_with_an_infinity():
    """The scale is infinite: the infinity itself becomes NaN, the rest of its block 0."""
    x = torch.ones(1, 256)
    w = torch.ones(256)
    w[3] = float("inf")
    for block in (128, 96):
        f = mda.rms_norm_add_forward(x.cuda(), w.cuda(), eps=0.0, scale_block=block)
        y = f.y.float().cpu()[0]
        assert torch.isnan(y).nonzero()[:, 0].tolist() == [3]
        assert (y[:3] == 0).all() and (y[4:block] == 0).all() and (y[block:] == 448).all()


# ------------------------------------------------------------------------------- linear cross entropy
def _randn(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst " \
                          f"{float(((got - want).abs() / (tol + 1e-300)).nan_to_num(1e30).max()):.3g} times the bound"


def _case(tokens, hidden, vocab, dtype, seed=0):
    x = _randn(seed, tokens, hidden, dtype=dtype)
    w = _randn(seed + 1, vocab, hidden, scale=2 * hidden ** -0.5, dtype=dtype)
    g = torch.Generator().manual_seed(seed + 2)
    t = torch.randint(0, vocab, (tokens,), generator=g)
    return x, w, t, torch.rand(tokens, generator=g) / tokens


def _check(x, w, t, gl, out_dtype):
    ref = R.xent(x, w, t, -100, gl, out_dtype=out_dtype)
    xc, wc, tc = x.cuda(), w.cuda(), t.cuda()
    loss, lse = mda.linear_cross_entropy_forward(xc, wc, tc)
    _close(loss, ref["loss"], ref["e_loss"], "loss")
    gw = torch.full(w.shape, float("nan"), dtype=out_dtype, device="cuda")
    dx, dw = mda.linear_cross_entropy_backward(gl.cuda(), xc, wc, tc, lse, grad_weight=gw)
    # half the spacing of bf16's least numbers, for each g and for the result; fp32's is in the reference's bounds
    low = 2.0 ** -134 if x.dtype == BF16 else 0.0
    _close(dx, ref["grad_hidden"], ref["e_grad_hidden"] + low * (1 + w.double().abs().sum(0)), "grad_hidden")
    low_out = 2.0 ** -134 if out_dtype == BF16 else 0.0
    _close(dw, ref["grad_weight"], ref["e_grad_weight"] + low * x.double().abs().sum(0) + low_out, "grad_weight")


TYPES = [(BF16, BF16), (BF16, F32), (F32, F32)]


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("tokens", [8, 200, 600])
def test_xent_of_tiny_upstream_gradients(dtype, out_dtype, tokens):
    """Tokens whose upstream gradient is tiny or subnormal, among ordinary ones."""
    x, w, t, gl = _case(tokens, 64, 300, dtype)
    gl[1], gl[2], gl[4], gl[5] = 1e-34, -1e-36, 1e-42, 1.5e-45
    _check(x, w, t, gl, out_dtype)


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
def test_xent_of_tiny_upstream_gradients_alone(dtype, out_dtype):
    """All of them far below 1: their powers of two leave the hidden states' limbs all their bits."""
    for scale in (1e-30, 1e-35):
        x, w, t, gl = _case(100, 64, 300, dtype)
        _check(x, w, t, gl * scale, out_dtype)


@pytest.mark.parametrize("tokens", [40, 2500])
@pytest.mark.parametrize("scale", [1e37, 1e36, 1e33, 1e-33, 1e-36, 1e-37])
def test_xent_fp32_to_the_ends_of_its_range(tokens, scale):
    """The largest and the least normal numbers, whose products are ordinary ones."""
    x, w, t, gl = _case(tokens, 64, 300, F32)
    _check(x * scale, w / scale, t, gl, F32)


def test_xent_fp32_large_values_meet_large_gradients():
    """A hidden state times its gradient's power of two is past fp32, the gradient of the weight is not."""
    x, w, t, gl = _case(40, 64, 300, F32)
    x, w = x * 1e30, w * 1e-30
    x[3:] *= 1e-20  # those logits are 0 for any practical purpose
    gl[0] = 1e12
    ref = R.xent(x, w, t, -100, gl, out_dtype=F32)
    _, lse = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    _, dw = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), lse)
    fits = ref["grad_weight"].abs() + ref["e_grad_weight"] < 3.4e38
    assert bool(fits.any())
    _close(torch.where(fits.cuda(), dw, torch.zeros_like(dw)), torch.where(fits, ref["grad_weight"], 0.0),
           ref["e_grad_weight"], "grad_weight")


def _spread_case(tokens, vocab, octaves, dtype):
    """Logits without a rounding, from 0 down to -octaves log(2): column 0 of the hidden states is 1 and of the
    weight the logit (multiples of 1/4), and the weight is 0 under the rest.  Targets are among the first 16
    words, so that every other row of the weight's gradient is a sum of p gl x alone."""
    x = _randn(1, tokens, 24, dtype=dtype)
    x[:, 0] = 1.0
    w = torch.zeros(vocab, 24)
    w[:, 0] = -torch.floor(torch.arange(vocab) / (vocab - 1) * octaves * 0.693147 * 4) / 4
    g = torch.Generator().manual_seed(2)
    t = torch.randint(0, 16, (tokens,), generator=g)
    return x, w.to(dtype), t, (0.5 + torch.rand(tokens, generator=g)) / tokens


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [30, 300, 2100])
def test_xent_rows_of_rare_words_in_fp32_precision(dtype, tokens):
    """The rows of words that are nobody's target, against their own size: g is off by 2^-21 of it or by 2^-48 of
    gl, whichever is more (two fp16 limbs, the low one 2^11 up: each limb off by at most 2^-11 of itself or by
    2^-25 of its unit, g at most 2^13 units)."""
    vocab = 700
    x, w, t, gl = _spread_case(tokens, vocab, 60, dtype)
    xd, z = x.double(), x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    _, lse32 = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    _, dw = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), lse32,
                                              grad_weight=torch.empty(vocab, 24, device="cuda"))
    g = p * gl.double()[:, None]
    want = g.t() @ xd
    # p: an exponent of up to 60 + log2(vocab) in fp32, two roundings of it, the lse's own error (a sum of 700
    # terms in a tree and a logarithm: 64 roundings) and the exponential's; x: 2^-21 of it or 2^-48 of the largest
    rel = (2 * 70 + 64 + 8) * R.U32 + 2.0 ** -21 + (2.0 ** -21 if dtype == F32 else 0.0)
    off = rel * g + 2.0 ** -48 * gl.double()[:, None]
    tol = off.t() @ xd.abs() + 3 * (tokens / 16 + 20) * R.U32 * (g.t() @ xd.abs())
    tol = tol + (2.0 ** -48 * xd.abs().max() * g.sum(0)[:, None] if dtype == F32 else 0.0)
    _close(dw[16:], want[16:], tol[16:], "grad_weight")
    err = (dw.double().cpu() - want).norm(dim=1) / want.norm(dim=1)
    common = p.amin(0) >= 1e-8
    common[:16] = False
    assert int(common.sum()) > 200 and float(err[common].max()) < 2e-5, float(err[common].max())


def test_xent_small_values_of_fp32_inputs_keep_their_bits():
    """Hidden states 2^-30 of the largest: each limb of X and W is off by at most 2^-11 of itself or by 2^-25 of
    its unit, the largest at least 2^14 units and the low limb 2^11 up: 2^-21 of a value or 2^-49 of the largest."""
    x, w, t, _ = _case(40, 64, 300, F32)
    x[:20] *= 2.0 ** -30
    w *= 2.0 ** 30
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    loss, _ = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    size = (x.double().abs() @ w.double().abs().t()).amax(1)
    ez = size * (3 * 2.0 ** -21 + 3 * (64 / 16 + 20) * R.U32) + 2.0 ** -49 * x.double().abs().max() * \
        w.double().abs().sum(1).max()
    tol = 2 * ez + (300 / 16 + 120) * R.U32 + 8 * R.U32 * z.abs().amax(1)
    _close(loss[:20], want[:20], tol[:20], "loss")


@pytest.mark.parametrize("tokens", [1, 40, 256, 300])
def test_xent_bf16_rows_of_rare_words(tokens):
    """bf16 gradients of words down to p = 2^-100, few tokens or many: bf16 has fp32's range, and so has g."""
    vocab = 700
    x, w, t, gl = _spread_case(tokens, vocab, 100, BF16)
    xd, z = x.double(), x.double() @ w.double().t()
    p = torch.softmax(z, 1)
    _, lse32 = mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda())
    _, dw = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), w.cuda(), t.cuda(), lse32)
    g = p * gl.double()[:, None]
    want, size = g.t() @ xd, g.t() @ xd.abs()
    # p as above with exponents of 110; g: one bf16 (2^-8), of up to 256 tokens two (2^-16)
    rel = (2 * 110 + 64 + 8) * R.U32 + (2.0 ** -8 if tokens > 256 else 2.0 ** -16) + (tokens / 16 + 20) * 2 * R.U32
    _close(dw[16:], want[16:], rel * size[16:] + R.half_step(BF16) * want[16:].abs(), "grad_weight")


# ------------------------------------------------------------------------------- dropout
def test_dropout_past_the_low_word_of_the_group():
    """2^34 + 4096 elements: groups of four from 2^32 on have a second counter word that is not 0."""
    n, seed, offset = (1 << 34) + 4096, 11, 13
    x = torch.ones(n, dtype=BF16, device="cuda")
    out = mda.dropout_add_forward(x, p=0.5, rng=(seed, offset))
    m32 = 0xFFFFFFFF
    want = []
    for group in range((1 << 32) - 256, (1 << 32) + 1024):
        c, k = [group & m32, group >> 32, offset, 0], [seed, 0]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & m32, (a >> 32) ^ c[3] ^ k[1], a & m32]
            k = [(k[0] + 0x9E3779B9) & m32, (k[1] + 0xBB67AE85) & m32]
        want += [word >= 1 << 31 for word in c]
    assert (out[(1 << 34) - 1024:].cpu() != 0).tolist() == want
    first = R.keep_mask((4096,), 0.5, seed, offset)
    assert torch.equal(out[:4096].cpu() != 0, first)
    assert not torch.equal(out[1 << 34:].cpu() != 0, first)
