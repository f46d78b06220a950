"""CPU tests of the training operators: the library's exports and refusals, the plain forms, shards over gloo."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import megatron_dion_amd as mda
from megatron_dion_amd import _lib, _lm_lib, lm_ops
from tests import _lm_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_header_symbol():
    lib = _lm_lib.load()
    text = open(os.path.join(ROOT, "include", "dion_lm.h")).read()
    syms = sorted(set(re.findall(r"^(?:int|const char\*)\s+(dion_\w+)\s*\(", text, flags=re.M)))
    assert sorted(_lm_lib.EXPORTED) == syms and all(getattr(lib, s) is not None for s in syms)
    assert lib.dion_lm_abi_version() == _lm_lib.ABI_VERSION
    assert lib.dion_lm_build_id().decode() == _lm_lib.source_build_id()


def test_missing_library_fails_loudly(tmp_path):
    with pytest.raises(_lib.DionLibraryError, match="DION_HIP_LIBRARY_MISSING"):
        _lm_lib.load(str(tmp_path / "missing.so"))


def test_plain_philox_against_published_vectors():
    """Random123's known answers for philox4x32-10 (counter, key -> words)."""
    def one(ctr, key):
        # counter words 0, 1 are the group: element 4 * group
        m = 0xFFFFFFFF
        c, (k0, k1) = list(ctr), key
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k0, b & m, (a >> 32) ^ c[3] ^ k1, a & m]
            k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
        return c

    assert one([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert one([0xFFFFFFFF] * 4, (0xFFFFFFFF,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert one([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    seed, offset = 0x299F31D0A4093822, 0x0370734413198A2E
    words = R.philox(4 * 7, seed, offset)
    for g in range(7):
        want = one([g, 0, offset & 0xFFFFFFFF, offset >> 32], (seed & 0xFFFFFFFF, seed >> 32))
        assert words[4 * g:4 * g + 4].tolist() == want


def test_plain_xent_against_torch():
    torch.manual_seed(0)
    x, w = torch.randn(20, 16, dtype=torch.float64), torch.randn(30, 16, dtype=torch.float64)
    t = torch.randint(0, 30, (20,))
    t[3] = -100
    gl = torch.rand(20, dtype=torch.float64)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = torch.nn.functional.cross_entropy(xr @ wr.t(), t, ignore_index=-100, reduction="none")
    (loss * gl).sum().backward()
    r = R.xent(x.float(), w.float(), t, -100, gl.float())
    assert torch.allclose(r["loss"], loss, atol=1e-5)
    assert torch.allclose(r["grad_hidden"], xr.grad, atol=1e-5) and torch.allclose(r["grad_weight"], wr.grad, atol=1e-5)


def _xent_desc(**kw):
    d = _lm_lib.DionXentDesc()
    base = dict(tokens=4, hidden=64, vocab=100, dtype=_lib.DTYPE_BF16, gw_dtype=_lib.DTYPE_F32, vocab_total=100,
                ignore_index=-100, ld_hidden=64, ld_weight=64, ld_grad_hidden=64, ld_grad_weight=64)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,code", [
    ({}, _lib.DION_OK), ({"tokens": -1}, _lib.DION_E_INVALID), ({"hidden": 0}, _lib.DION_E_INVALID),
    ({"vocab": 0}, _lib.DION_E_INVALID), ({"vocab": 101}, _lib.DION_E_INVALID), ({"vocab_start": -1}, _lib.DION_E_INVALID),
    ({"vocab_start": 1}, _lib.DION_E_INVALID), ({"ld_weight": 63}, _lib.DION_E_INVALID),
    ({"ld_hidden": 63}, _lib.DION_E_INVALID), ({"dtype": 3}, _lib.DION_E_UNSUPPORTED),
    ({"gw_dtype": 0}, _lib.DION_E_UNSUPPORTED), ({"ld_weight": 1 << 22}, _lib.DION_E_UNSUPPORTED),
    ({"tokens": 1 << 25}, _lib.DION_E_UNSUPPORTED),
    ({"vocab_start": (1 << 63) - 1}, _lib.DION_E_INVALID), ({"vocab_total": -(1 << 63)}, _lib.DION_E_INVALID), ({"piece_bytes": -1}, _lib.DION_E_INVALID)])
def test_xent_workspace_query_refuses(kw, code):
    n = ctypes.c_size_t(0)
    assert _lm_lib.load().dion_xent_workspace_bytes(ctypes.byref(_xent_desc(**kw)), _lm_lib.XENT_BACKWARD,
                                                    ctypes.byref(n)) == code


def test_xent_workspace_is_far_from_the_logits():
    """8192 tokens of a 128256-word vocabulary: the fp32 logits would be 4.2 GB."""
    d = _xent_desc(tokens=8192, hidden=4096, vocab=128256, vocab_total=128256, ld_hidden=4096, ld_weight=4096,
                   gw_dtype=_lib.DTYPE_BF16)
    lib, n = _lm_lib.load(), ctypes.c_size_t(0)
    assert lib.dion_xent_workspace_bytes(ctypes.byref(d), _lm_lib.XENT_FORWARD, ctypes.byref(n)) == 0
    assert n.value < 200 << 20
    assert lib.dion_xent_workspace_bytes(ctypes.byref(d), _lm_lib.XENT_BACKWARD, ctypes.byref(n)) == 0
    assert n.value < 1400 << 20
    d.tokens = 0
    for op in (_lm_lib.XENT_FORWARD, _lm_lib.XENT_BACKWARD):
        assert lib.dion_xent_workspace_bytes(ctypes.byref(d), op, ctypes.byref(n)) == 0 and n.value == 0
    d.tokens = 8192
    d.piece_bytes = 64 << 20
    assert lib.dion_xent_workspace_bytes(ctypes.byref(d), _lm_lib.XENT_BACKWARD, ctypes.byref(n)) == 0
    assert n.value < 300 << 20


def test_calls_refuse_before_they_enqueue():
    """None of these reaches the GPU: every pointer is null or never read."""
    lib = _lm_lib.load()
    d, one = _xent_desc(), ctypes.c_void_p(16)
    args = (None, None, None, None, 0, None)
    assert lib.dion_xent_forward(ctypes.byref(d), None, one, one, *args) == _lib.DION_E_INVALID
    assert lib.dion_xent_forward(ctypes.byref(d), one, one, one, one, one, None, None, 0, None) == _lib.DION_E_WORKSPACE
    assert b"workspace" in lib.dion_lm_last_error()
    assert lib.dion_xent_forward(None, one, one, one, *args) == _lib.DION_E_INVALID
    assert lib.dion_xent_forward(ctypes.byref(d), one, ctypes.c_void_p(18), one, *args) == _lib.DION_E_INVALID
    d.tokens = 0
    assert lib.dion_xent_forward(ctypes.byref(d), None, None, None, *args) == _lib.DION_OK
    assert lib.dion_xent_backward(ctypes.byref(d), one, one, one, one, one, one, one, one, 0, None) == _lib.DION_E_INVALID
    rng = _lm_lib.DionRng(1, 2, None)
    drop = lambda rows, cols, dt, p, r, ld=64, x=one: lib.dion_dropout_add(  # noqa: E731
        rows, cols, dt, x, ld, None, 0, x, ld, p, None if r is None else ctypes.byref(r), None)
    assert drop(2, 64, 1, 1.5, rng) == drop(2, 64, 1, -0.1, rng) == drop(2, 64, 1, float("nan"), rng) == -1
    assert drop(2, 64, 1, 0.5, None) == -1 and drop(2, 64, 9, 0.5, rng) == -2 and drop(-1, 64, 1, 0.5, rng) == -1
    assert drop(2, 64, 1, 0.5, rng, ld=63) == -1 and drop(2, 64, 1, 0.5, rng, x=None) == -1
    assert drop(0, 64, 1, 0.5, rng, x=None) == 0
    nd = _lm_lib.DionNormDesc(rows=2, cols=64, dtype=2, w_dtype=1, gw_dtype=1, y_dtype=2, p=0.0, ld_x=64, ld_residual=64,
                              ld_h=64, ld_y=64, ld_grad_y=64, ld_grad_h=64, ld_grad_x=64, ld_grad_residual=64)

    def fwd(x=one, res=None, h=None, scale=None, **kw):
        q = _lm_lib.DionNormDesc.from_buffer_copy(nd)
        for k, v in kw.items():
            setattr(q, k, v)
        return lib.dion_rms_norm_add(ctypes.byref(q), x, res, one, h, one, scale, one, None, None)

    assert fwd(x=None) == fwd(res=one) == fwd(p=0.5, h=one) == fwd(p=2.0) == fwd(cols=0) == fwd(ld_x=63) == -1
    assert fwd(cols=16385, ld_x=16385) == fwd(dtype=3) == fwd(y_dtype=1) == -2
    assert fwd(y_dtype=3, scale_block=4, scale=one) == fwd(y_dtype=3, scale_block=65, scale=one) == -1
    assert fwd(y_dtype=3, scale_block=32) == -1
    assert fwd(rows=0, x=None) == 0
    bwd = lambda ws, n, gw=one: lib.dion_rms_norm_add_backward(  # noqa: E731
        ctypes.byref(nd), one, one, one, one, None, one, None, gw, None, ws, n, None)
    assert bwd(None, 0) == bwd(one, 8) == -4


def test_python_calls_refuse():
    x, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: mda.dropout_add_forward(x, p=0.1, rng=(1, 1)),
                 lambda: mda.rms_norm_add_forward(x, torch.ones(8)),
                 lambda: mda.linear_cross_entropy_forward(x, w, t)):
        with pytest.raises(RuntimeError, match="DION_BAD_DEVICE"):
            call()
    with pytest.raises(RuntimeError, match="DION_BAD_SHAPE"):
        mda.dropout_add_forward(torch.zeros(()), p=0.1, rng=(1, 1))
    dev = torch.device("cpu")
    for p, rng in ((-0.1, (1, 1)), (1.1, (1, 1)), (float("nan"), (1, 1)), (0.5, None), (0.5, torch.zeros(3, dtype=torch.int64)),
                   (0.5, torch.zeros(2))):
        with pytest.raises(RuntimeError, match="DION_BAD_DROPOUT"):
            lm_ops._rng(p, rng, dev)
    assert lm_ops._rng(0.0, None, dev) is None
    r = lm_ops._rng(0.5, (-1, 1 << 64), dev)
    assert (r.seed, r.offset) == ((1 << 64) - 1, 0)
    with pytest.raises(RuntimeError, match="DION_BAD_VOCAB"):
        mda.linear_cross_entropy_forward(x, w, t, group=object())
    with pytest.raises(RuntimeError, match="DION_NO_MAIN_GRAD"):
        mda.linear_cross_entropy(x, w, t, into_main_grad=True)
    with pytest.raises(RuntimeError, match="DION_BAD_GRAD_OUT"):
        lm_ops._grad_weight(w, None, True, "grad_weight")
    with pytest.raises(RuntimeError, match="DION_BAD_GRAD_OUT"):
        lm_ops._grad_weight(w, torch.zeros(4, 8), False, "grad_weight")


def test_sizes_that_a_descriptor_cannot_hold():
    """ctypes would keep the low bits: 2^32 + 8 columns would be taken for 8."""
    big = (1 << 32) + 8
    with pytest.raises(RuntimeError, match="DION_BAD_SIZE.*cols"):
        lm_ops._norm_desc(1, big, 2, 1, 1, 2, 0, 0, 1e-5, 0.0, big, 0, big, big)
    base = dict(op=1, tokens=1, hidden=8, vocab=8, dtype=2, gw_dtype=2, accumulate=0, pack_weight=0, start=0, total=8,
                ignore=-100, ld_hidden=8, ld_weight=8, ld_grad_weight=8, piece_bytes=0)
    assert lm_ops._xent_shape(*base.values())[1] > 0
    for k, v in (("hidden", big), ("vocab", big), ("start", 1 << 63), ("total", 1 << 64), ("ignore", 1 << 63),
                 ("piece_bytes", 1 << 64)):
        with pytest.raises(RuntimeError, match="DION_BAD_SIZE"):
            lm_ops._xent_shape(*{**base, k: v}.values())


def _shards(rank, world, port, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.manual_seed(0)
    z = torch.randn(9, 40, dtype=torch.float32) * 5
    z[4] += 300.0  # the maximum of each token has to come off before the exponentials
    t = torch.randint(0, 40, (9,))
    ignored = torch.zeros(9, dtype=torch.bool)
    ignored[2] = True
    n = 40 // world
    mine = z[:, rank * n:(rank + 1) * n]
    here = (t >= rank * n) & (t < (rank + 1) * n)
    tl = torch.where(here & ~ignored, z.gather(1, t[:, None])[:, 0], torch.zeros(9))
    lse = torch.where(ignored, torch.zeros(9), torch.logsumexp(mine, 1))
    loss, whole = lm_ops.combine_vocab_shards(lse, tl, ignored, dist.group.WORLD)
    ref = torch.nn.functional.cross_entropy(z.double(), torch.where(ignored, -100, t), reduction="none")
    # fp32: a maximum of 300 is held to 300 * 2^-24
    ok = torch.allclose(loss.double(), ref, atol=1e-4) and bool((loss[2] == 0) & (whole[2] == 0))
    ret[rank] = ok
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [1, 2, 4])
def test_vocabulary_shards_join_over_gloo(world):
    with mp.Manager() as m:
        ret = m.dict()
        mp.spawn(_shards, args=(world, 29611 + world, ret), nprocs=world, join=True)
        assert all(ret[r] for r in range(world))
