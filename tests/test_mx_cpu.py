"""Microscaled 4-bit (MXFP4) operators without a GPU: the float64 restatement the GPU tests compare with, packed sizes, and
every refusal of the C entry points and of the Python layer."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as X


def test_oracle_rounds_to_the_nearest_code_with_ties_to_even():
    # one block with scale 1: the largest magnitude lies in [4, 8)
    x = np.zeros((1, 32))
    vals = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 5.5, 7.9, 0.2500001, 0.7499999, -2.4999, 6.0]
    want = [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -4.0, 6.0, 6.0, 0.5, 0.5, -2.0, 6.0]
    x[0, :len(vals)] = vals
    codes, scales = X.quantize(x)
    assert codes.shape == (1, 64) and scales.shape == (1, 4)
    assert scales[0].tolist() == [127, 0, 0, 0]
    assert X.rounded(x)[0, :len(vals)].tolist() == want
    assert (codes[0, 16:] == 0).all()


def test_oracle_scales():
    for v, s in ((1.0, 125), (3.99, 126), (4.0, 127), (2.0 ** -126, 0), (2.0 ** -125, 0), (2.0 ** -124, 1), (2.0 ** -149, 0), (0.0, 0),
                 (3.4e38, 252), (np.inf, 255), (np.nan, 255)):
        codes, scales = X.quantize(np.array([[v]]))
        assert scales[0, 0] == s, v
        if s == 255:
            assert (codes == 0).all() and np.isnan(X.dequantize(codes, scales, 1)).all()


def test_sizes():
    from nerf import _hip
    lib = _hip.lib
    for K, blocks in ((1, 1), (128, 1), (129, 2), (319, 3), (4096, 32)):
        assert lib.nerf_mx_codes_bytes(7, K) == 7 * 64 * blocks and lib.nerf_mx_scales_bytes(7, K) == 7 * 4 * blocks
        assert _hip.mx_packed_shape(7, K) == ((7, 64 * blocks), (7, 4 * blocks))
    assert lib.nerf_mx_codes_bytes(-1, 8) == 0 and lib.nerf_mx_codes_bytes(8, 0) == 0 and lib.nerf_mx_scales_bytes(8, 1 << 23) == 0
    assert lib.nerf_mx_linear_fwd_workspace_bytes(0, 8, 8, 0) == 0 and lib.nerf_mx_linear_fwd_workspace_bytes(8, 0, 8, 0) == 0
    assert lib.nerf_mx_linear_fwd_workspace_bytes(1 << 31, 8, 8, 0) == 0
    assert lib.nerf_mx_linear_bwd_workspace_bytes(9, 0, 8, 8, 8, 1, 1, 1) == 0
    assert lib.nerf_mx_linear_bwd_workspace_bytes(0, 0, 0, 8, 8, 1, 1, 1) == 0
    assert lib.nerf_mx_linear_bwd_workspace_bytes(0, 0, 64, 64, 64, 0, 0, 0) == 0


P = 4096   # a stand-in for a device pointer in calls that are refused before anything could touch it


@pytest.mark.parametrize("args, code, text", [
    ((None, 0, 32, 4, 32, None, None, None), -2, b"x is NULL"),
    ((P, 0, 31, 4, 32, P, P, None), -1, b"ldx=31"),
    ((P, 3, 32, 4, 32, P, P, None), -1, b"unknown type 3"),
    ((P, 0, 32, -1, 32, P, P, None), -1, b"M=-1"),
    ((P, 0, 32, 4, 0, P, P, None), -1, b"K=0"),
    ((P, 0, 32, 4, 32, None, P, None), -2, b"codes is NULL"),
    ((P, 0, 32, 4, 32, P + 8, P, None), -1, b"16-byte"),
    ((P, 0, 32, 4, 32, P, P + 2, None), -1, b"4-byte"),
    ((None, 0, 32, 0, 32, None, None, None), 0, b""),
])
def test_quantize_refusals(args, code, text):
    from nerf import _hip
    assert _hip.lib.nerf_mx_quantize(*args) == code
    assert text in _hip.lib.nerf_last_error() or code == 0


@pytest.mark.parametrize("args, code, text", [
    ((None, P, 4, 32, 0, P, 32, None), -2, b"codes is NULL"),
    ((P, P, 4, 32, 0, None, 32, None), -2, b"out is NULL"),
    ((P, P, 4, 32, 0, P, 31, None), -1, b"ldo=31"),
    ((P, P, 4, 32, -1, P, 32, None), -1, b"unknown type -1"),
    ((P + 4, P, 4, 32, 0, P, 32, None), -1, b"16-byte"),
    ((None, None, 0, 32, 0, None, 32, None), 0, b""),
])
def test_dequantize_refusals(args, code, text):
    from nerf import _hip
    assert _hip.lib.nerf_mx_dequantize(*args) == code
    assert text in _hip.lib.nerf_last_error() or code == 0


def _fwd(**kw):
    a = dict(x=P, dtype=0, ldx=32, wc=P, ws=P, b=None, M=4, K=32, N=8, act=0, pre=1.0, post=1.0, y=P, ldy=8, slope=None, mask=None,
             xc=None, xs=None, work=P, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, code, text", [
    (dict(x=None), -2, b"x is NULL"), (dict(wc=None), -2, b"wcodes is NULL"), (dict(ws=None), -2, b"wscales is NULL"),
    (dict(y=None), -2, b"y is NULL"), (dict(work=None, M=200), -2, b"workspace is NULL"),
    (dict(ldx=31), -1, b"ldx=31"), (dict(ldy=7), -1, b"ldy=7"), (dict(dtype=5), -1, b"unknown type 5"),
    (dict(act=4), -1, b"unknown activation 4"), (dict(M=-1), -1, b"M=-1"), (dict(K=0), -1, b"K=0"), (dict(N=0), -1, b"N=0"),
    (dict(M=(1 << 30) + 1), -1, b"bad shape"), (dict(K=(1 << 22) + 1, ldx=1 << 23), -1, b"bad shape"),
    (dict(M=1 << 30, N=1 << 22, ldy=1 << 22), -1, b"bad shape"), (dict(M=1 << 28), -1, b"bad shape"),
    (dict(M=1 << 19, N=1 << 22, ldy=1 << 22), -1, b"bad shape"),       # 2^32 threads
    (dict(xc=P, xs=P, M=65535 * 64 + 1), -1, b"kept for a backward pass"),
    (dict(xc=P, xs=P, N=65535 * 64 + 1, ldy=1 << 23), -1, b"kept for a backward pass"),
    (dict(xc=P), -1, b"go together"), (dict(wc=P + 4), -1, b"aligned"), (dict(work=P + 8), -1, b"aligned"),
    (dict(M=0, x=None, y=None, work=None), 0, b""),
])
def test_linear_fwd_refusals(kw, code, text):
    from nerf import _hip
    assert _hip.lib.nerf_mx_linear_fwd(*_fwd(**kw)) == code
    assert text in _hip.lib.nerf_last_error() or code == 0


def _bwd(**kw):
    a = dict(dy=P, dtype=0, lddy=8, slope=None, mask=None, act=0, pre=1.0, post=1.0, xc=P, xs=P, wc=P, ws=P, M=4, K=32, N=8, work=P,
             dx=P, lddx=32, dw=P, db=P, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, code, text", [
    (dict(dy=None), -2, b"dy is NULL"), (dict(work=None), -2, b"workspace is NULL"), (dict(act=1), -2, b"mask is NULL"),
    (dict(act=2), -2, b"slope is NULL"), (dict(act=3), -2, b"slope is NULL"), (dict(wc=None), -2, b"wcodes is NULL"),
    (dict(xs=None), -2, b"xscales is NULL"), (dict(lddy=7), -1, b"bad shape"), (dict(lddx=31), -1, b"bad shape"),
    (dict(M=0), -1, b"bad shape"), (dict(dtype=3), -1, b"unknown type 3"), (dict(act=9), -1, b"unknown activation 9"),
    (dict(M=65535 * 64 + 1), -1, b"65535*64"),
    (dict(N=65535 * 64 + 1, lddy=1 << 23), -1, b"65535*64"), (dict(xc=P + 8), -1, b"aligned"),
    (dict(dx=None, dw=None, db=None, dy=None), 0, b""),
])
def test_linear_bwd_refusals(kw, code, text):
    from nerf import _hip
    assert _hip.lib.nerf_mx_linear_bwd(*_bwd(**kw)) == code
    assert text in _hip.lib.nerf_last_error() or code == 0


def test_python_refusals():
    from nerf import mx
    x = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="HIP device only"):
        mx.quantize(x)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        mx.quantize(x.double())
    with pytest.raises(ValueError, match="at least one value"):
        mx.quantize(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="at least one value"):
        mx.quantize(torch.tensor(1.0))
    q = mx.MXTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 32)
    assert q.rows == 4
    with pytest.raises(RuntimeError, match="HIP device only"):
        mx.dequantize(q)
    with pytest.raises(ValueError, match="not packed rows of 200"):
        mx.dequantize(q._replace(K=200))
    with pytest.raises(ValueError, match="32 values per row"):
        mx.linear(torch.zeros(4, 33), q)
    with pytest.raises(ValueError, match="unknown activation"):
        mx.linear(x, q, act=7)
    with pytest.raises(TypeError, match="like x"):
        mx.linear(x, torch.zeros(8, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match=r"\[N,K\]"):
        mx.linear(x, torch.zeros(32))
    with pytest.raises(RuntimeError, match="HIP device only"):
        mx.linear(x, torch.zeros(8, 32))


def test_models_and_commands_know_the_mode():
    from nerf.models import NeRF, Siren
    for m in (NeRF(), NeRF(hidden_dim=64), Siren(), Siren(num_layers=3, hidden_dim=96)):
        assert not m.runs_mxfp4()
        m.set_training_precision("mxfp4")
        assert m.runs_mxfp4()
        with torch.no_grad():
            assert not m.runs_mxfp4()
        m.set_inference_precision("mxfp4")
        with torch.no_grad():
            assert m.runs_mxfp4()
        with pytest.raises(ValueError):
            m.set_training_precision("fp4")
        with pytest.raises(ValueError):
            m.set_inference_precision("fp8")
        m.set_training_precision("fp32").set_inference_precision("fp32")
        assert not m.runs_mxfp4()
    from nerf.rendering import _fused_model
    m = NeRF()
    assert _fused_model(m)
    m.set_training_precision("mxfp4")
    assert not _fused_model(m)


@pytest.mark.parametrize("packed, dual", [(False, "x"), (False, "weight"), (False, "bias"), (True, "x"), (True, "bias")])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(monkeypatch, packed, dual, grad):
    """A tangent on any operand is refused, whether or not gradients are recorded: it would be lost without a word.  (The
    kernels are replaced: this runs without a GPU, and nothing may reach them.)"""
    import torch.autograd.forward_ad as fwd
    from nerf import _hip, mx
    calls = []
    monkeypatch.setattr(_hip, "mx_linear_fwd", lambda x, wc, *a: calls.append("fwd") or x.new_zeros(x.shape[0], wc.shape[0]))
    monkeypatch.setattr(_hip, "mx_quantize", lambda w: (torch.zeros(w.shape[0], 64, dtype=torch.uint8), None))
    monkeypatch.setattr(mx.MXLinearFunction, "apply", lambda x, w, *a: calls.append("train") or x.new_zeros(x.shape[0], 8))
    t = {"x": torch.ones(4, 32, requires_grad=grad), "weight": torch.ones(8, 32), "bias": torch.ones(8)}
    q = mx.MXTensor(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8), 32)
    with fwd.dual_level():
        plain = dict(t)
        t[dual] = fwd.make_dual(t[dual], torch.ones_like(t[dual]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    mx.linear(t["x"], q if packed else t["weight"], t["bias"])
        assert not calls
        mx.linear(plain["x"], q if packed else plain["weight"], plain["bias"])      # no tangent: the level alone changes nothing
        assert calls == ["train" if grad else "fwd"]
    mx.linear(plain["x"], q if packed else plain["weight"], None)
    assert calls[1:] == ["train" if grad else "fwd"]


def test_large_tile_reads_its_scales_inside_lds(tmp_path):
    """The addresses of the large packed tile's scales (csrc/mx_large.h), followed on the host for all lengths of a row."""
    import os
    import subprocess
    exe = tmp_path / "lds"
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host", "mx_large_lds.cpp")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-o", str(exe), source], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


@pytest.mark.parametrize("K, rows", [(1, 268435440), (128, 268435440), (129, 134217720), (1 << 22, 8191)])
def test_most_rows_that_are_taken(K, rows):
    """rows * 16 ceil(K / 128) groups of eight values, at most 2^32 - 256: accepted up to there (a NULL pointer is all that is
    wrong then), refused behind."""
    from nerf import _hip
    lib = _hip.lib
    assert rows * 16 * -(-K // 128) <= 2 ** 32 - 256 < (rows + 1) * 16 * -(-K // 128)
    assert lib.nerf_mx_codes_bytes(rows, K) == rows * 64 * -(-K // 128) and lib.nerf_mx_codes_bytes(rows + 1, K) == 0
    assert lib.nerf_mx_scales_bytes(rows, K) == rows * 4 * -(-K // 128) and lib.nerf_mx_scales_bytes(rows + 1, K) == 0
    assert lib.nerf_mx_quantize(None, 0, K, rows, K, P, P, None) == -2
    assert lib.nerf_mx_quantize(None, 0, K, rows + 1, K, P, P, None) == -1
    assert lib.nerf_mx_linear_fwd(*_fwd(M=rows, K=K, ldx=K, x=None)) == -2
    assert lib.nerf_mx_linear_fwd(*_fwd(M=rows + 1, K=K, ldx=K, x=None)) == -1 and b"bad shape" in lib.nerf_last_error()


def test_most_outputs_that_are_taken():
    """Up to 2^22 rows of W and fewer than 2^24 tiles of 128 x 128 in y."""
    from nerf import _hip
    lib, n = _hip.lib, 1 << 22
    assert lib.nerf_mx_linear_fwd(*_fwd(N=n, ldy=n, x=None)) == -2
    assert lib.nerf_mx_linear_fwd(*_fwd(N=n + 1, ldy=n + 1, x=None)) == -1 and b"bad shape" in lib.nerf_last_error()
    assert lib.nerf_mx_linear_fwd(*_fwd(M=128 * 511, N=n, ldy=n, x=None)) == -2
    assert lib.nerf_mx_linear_fwd(*_fwd(M=128 * 511 + 1, N=n, ldy=n, x=None)) == -1 and b"bad shape" in lib.nerf_last_error()
