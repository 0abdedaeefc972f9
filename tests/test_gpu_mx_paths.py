"""Microscaled 4-bit (MXFP4) operators: the borders of each way to multiply, which the cases of tests/test_gpu_mx.py pass by.
Oracle and tolerances are that file's; where a result has to be the same sums in the same order, its bits are compared."""
import pytest
import torch

from test_gpu_mx import ACTS, DEV, TYPES, check_backward, check_forward, randn, run_training

pytestmark = pytest.mark.gpu


def training_case(M, K, N, act, dtype):
    """Inputs whose ReLU decisions are not the rounding's: a bias of +-30 keeps the sums off zero."""
    x, w = randn(M, K, seed=31, dtype=dtype), randn(N, K, seed=32, dtype=dtype, scale=K ** -0.5)
    b = (torch.sign(randn(N, seed=33)) * 30).to(dtype) if act == "relu" else randn(N, seed=33, dtype=dtype)
    return x, w, b, randn(M, N, seed=34, dtype=dtype)


def backward_entry(kept, dy, ld, need, fill=None):
    """The C entry on what a training forward kept: ([dx, dw, db], workspace), the workspace filled with a byte first."""
    from nerf import _hip
    lib, M, K, N, dtype = _hip.lib, kept.M, kept.K, kept.N, dy.dtype
    base, extra = kept.buffer.data_ptr(), None if kept.extra is None else kept.buffer.data_ptr() + kept.extra
    out = [torch.full(s, 7.0, dtype=dtype, device=DEV) if n else None for s, n in zip(((M, K), (N, K), (N,)), need)]
    nbytes = lib.nerf_mx_linear_bwd_workspace_bytes(_hip.MX_DTYPES[dtype], kept.act, M, K, N, *need)
    ws = torch.full((nbytes,), 0x5a if fill is None else fill, dtype=torch.uint8, device=DEV)
    ptr = [None if o is None else o.data_ptr() for o in out]
    rc = lib.nerf_mx_linear_bwd(dy.data_ptr(), _hip.MX_DTYPES[dtype], ld, extra, extra, kept.act, kept.pre, kept.post, base + kept.xcodes,
                                base + kept.xscales, base + kept.wcodes, base + kept.wscales, M, K, N, ws.data_ptr(), ptr[0], K, ptr[1],
                                ptr[2], torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.nerf_last_error()
    return out, ws


def is_narrow(kept, dy, ld):
    """Whether these gradients take the one pass for narrow layers: dx alone needs no workspace there; the general way lays dz
    and W out in it."""
    _, ws = backward_entry(kept, dy, ld, (1, 0, 0))
    return bool((ws == 0x5a).all())


# ------------------------------------------------------------------------------------------------ narrow layers, gradients
# what a pass for up to 256 x 256 takes by its alignment: rows of dy and slopes in whole 16 bytes; K free
NARROW = [(4101, 255, 248), (4500, 132, 8), (5003, 129, 128), (6001, 200, 256), (4100, 100, 96), (16390, 161, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, K, N", NARROW + [(4300, 130, 252), (4097, 250, 20)])
def test_narrow_gradients_end_inside_a_step(dtype, act, M, K, N):
    from nerf import _hip, mx
    x, w, b, dy = training_case(M, K, N, act, dtype)
    _, kept = _hip.mx_linear_train(x, w, None, b, mx.ACTIVATIONS[act], 1.5, 2.0)
    assert is_narrow(kept, dy, N) == (N * dtype.itemsize % 16 == 0)
    y, grads = run_training(x, w, b, dy, act, 1.5, 2.0)
    check_forward(y, x, w, b, act, 1.5, 2.0)
    check_backward(grads, dy, x, w, b, act, 1.5, 2.0, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, K, N", [(4101, 255, 248), (4500, 60, 64), (700, 200, 72)])
def test_each_gradient_alone(dtype, act, M, K, N):
    """Any subset of the gradients: the same bits as all three, whatever the workspace held; what lies between rows of dy (NaN
    here) is not read."""
    from nerf import _hip, mx
    x, w, b, dy = training_case(M, K, N, act, dtype)
    _, kept = _hip.mx_linear_train(x, w, None, b, mx.ACTIVATIONS[act], 1.5, 2.0)
    full, _ = backward_entry(kept, dy, N, (1, 1, 1))
    check_backward(full, dy, x, w, b, act, 1.5, 2.0, dtype)
    wide = torch.full((M, N + 24), float("nan"), dtype=dtype, device=DEV)
    wide[:, :N] = dy
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1), (1, 1, 1)):
        for g, ld in ((dy, N), (wide, N + 24)):
            got, _ = backward_entry(kept, g, ld, need, fill=0xff)
            for a, c, n in zip(got, full, need):
                assert a is None if not n else torch.equal(a, c)


def test_bf16_rows_of_dy_are_read_in_place():
    """bf16 without an activation goes into the product as it lies: any pitch and address, NaN between the rows."""
    from nerf import _hip, mx
    for M, K, N in ((300, 300, 128), (4200, 300, 128), (3400, 3601, 192)):
        x, w, _, dy = training_case(M, K, N, "none", torch.bfloat16)
        _, kept = _hip.mx_linear_train(x, w, None, None, mx.ACT_NONE, 1.0, 1.0)
        want, _ = backward_entry(kept, dy, N, (1, 1, 1))
        for pitch, shift in ((N + 8, 0), (N + 8, 8), (N + 8, 3), (N + 1, 0), (2 * N, 0)):
            buf = torch.full((M * pitch + shift,), float("nan"), dtype=torch.bfloat16, device=DEV)
            rows = buf[shift:].view(M, pitch)
            rows[:, :N] = dy
            got, _ = backward_entry(kept, rows, pitch, (1, 1, 1))
            assert all(torch.equal(a, c) for a, c in zip(got, want)), (M, pitch, shift)
