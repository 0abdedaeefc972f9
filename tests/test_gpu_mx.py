"""Microscaled 4-bit (MXFP4) operators on the GPU against their float64 restatement (oracle/mx_oracle.py).

Rounding to codes is a discrete result and has to match exactly.  Tolerances of sums, element by element: a sum of n
products in fp32, in whatever order, is off by at most n 2^-24 times the sum of the products' magnitudes (S); a smooth
activation passes an error of z on with its largest slope and adds 4 2^-24 of its own scale (a few fp32 operations); the
result is rounded to its type by half a step, eps/2 of the value."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as X

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
ACTS = ["none", "relu", "sin", "sigmoid"]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def np64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def randn(*shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def check_packed(q, x):
    codes, scales = X.quantize(np64(x))
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    got, want = q.codes.cpu().numpy(), codes
    # the sign of a zero is kept by both; compare the codes themselves
    assert np.array_equal(got, want)


# ----------------------------------------------------------------------------------------------- quantise, read back
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value(dtype):
    """All 65536 values, in blocks with a shared scale: neighbours in value, and shuffled (mixed magnitudes)."""
    from nerf import mx
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    for order in (torch.arange(65536), torch.randperm(65536, generator=torch.Generator().manual_seed(0))):
        x = bits[order].view(dtype).view(512, 128).to(DEV)
        check_packed(mx.quantize(x), x)


def test_fp32_bit_patterns():
    from nerf import mx
    g = torch.Generator().manual_seed(1)
    raw = torch.randint(-2 ** 31, 2 ** 31, (256, 128), generator=g).to(torch.int32)          # any exponent, some NaN / infinity
    near = (torch.randint(-2 ** 19, 2 ** 19, (256, 128), generator=g).to(torch.int32) & 0x3) + torch.tensor(
        [0x3E800000, 0x3F400000, 0x3FA00000, 0x3FE00000, 0x40200000, 0x40600000, 0x40A00000, 0x40FFFFFC], dtype=torch.int32).repeat(256, 16) - 2
    for bits in (raw, near):                                                                # one step around each rounding border
        x = bits.view(torch.float32).to(DEV)
        check_packed(mx.quantize(x), x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K, pad, shift", [(1, 1, 0, 0), (1, 128, 0, 0), (2, 31, 0, 0), (3, 32, 5, 0), (5, 33, 0, 1), (257, 127, 1, 0),
                                              (2, 129, 7, 3), (64, 256, 8, 0), (1031, 100, 24, 0), (3, 1000, 0, 2), (1, 8192, 0, 1)])
def test_quantize_shapes_pitches_and_offsets(dtype, M, K, pad, shift):
    from nerf import mx
    buf = randn(M * (K + pad) + shift, seed=M * K + pad, dtype=dtype, scale=3.0)
    x = buf[shift:].view(M, K + pad)[:, :K]
    q = mx.quantize(x)
    assert q.K == K and q.rows == M
    check_packed(q, x)
    back = mx.dequantize(q, dtype)
    assert back.shape == (M, K) and back.dtype == dtype
    want = torch.from_numpy(X.rounded(np64(x))).to(dtype)      # one rounding of the exact value
    assert torch.equal(back.cpu(), want)


def test_blocks_with_nan_infinity_zero_and_subnormals():
    from nerf import mx
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(3))
    x[0, 5] = float("nan")
    x[1, 40] = float("inf")
    x[2, 95] = -float("inf")
    x[3] = 0.0
    x[4] = 2.0 ** -140 * torch.arange(96)
    x[5, :32] = 3.4e38
    x[5, 32:64] = -0.0
    x = x.to(DEV)
    q = mx.quantize(x)
    check_packed(q, x)
    back = mx.dequantize(q).cpu()
    assert torch.isnan(back[0, :32]).all() and torch.isfinite(back[0, 32:]).all()
    assert torch.isnan(back[1, 32:64]).all() and torch.isnan(back[2, 64:]).all() and torch.isfinite(back[2, :64]).all()
    assert (back[3] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_scale_and_code_reads_back(dtype):
    from nerf import mx
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).repeat(256, 1)             # 512 codes a row
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None].repeat(1, 16)
    got = mx.dequantize(mx.MXTensor(codes.to(DEV), scales.to(DEV), 512), dtype).cpu()
    want = torch.from_numpy(X.dequantize(codes.numpy(), scales.numpy(), 512)).to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(want, nan=0.0, posinf=1.0, neginf=-1.0))


def test_offsets_beyond_31_bits():
    """More than 2^31 values: the last rows are those of a small call."""
    from nerf import mx
    M, K = (1 << 24) + 5, 130
    x = torch.empty(M, K, dtype=torch.bfloat16, device=DEV)
    tail = randn(7, K, seed=9, dtype=torch.bfloat16)
    x[:7] = tail
    x[-7:] = tail
    q, small = mx.quantize(x), mx.quantize(tail)
    assert torch.equal(q.codes[-7:], small.codes) and torch.equal(q.scales[-7:], small.scales)
    back = mx.dequantize(q, torch.bfloat16)
    assert torch.equal(back[-7:], mx.dequantize(small, torch.bfloat16)) and torch.equal(back[:7], back[-7:])


def test_empty_rows_and_leading_dimensions():
    from nerf import mx
    q = mx.quantize(torch.zeros(0, 40, device=DEV))
    assert q.codes.shape == (0, 64) and mx.dequantize(q).shape == (0, 40)
    w = mx.quantize(randn(24, 40, seed=1))
    assert mx.linear(torch.zeros(0, 40, device=DEV), w).shape == (0, 24)
    x = randn(2, 3, 5, 40, seed=2)
    assert torch.equal(mx.linear(x, w), mx.linear(x.view(30, 40), w).view(2, 3, 5, 24))
    t = randn(40, 9, seed=4).t()                                   # transposed: copied
    assert torch.equal(mx.linear(t, w), mx.linear(t.contiguous(), w))
    e = randn(1, 40, seed=5).expand(6, 40)                         # rows that overlap: copied
    assert torch.equal(mx.linear(e, w), mx.linear(e.contiguous(), w))


# ----------------------------------------------------------------------------------------------------------- product
def tolerance_z(xq, wq, b):
    S = np.abs(xq) @ np.abs(wq).T + (0.0 if b is None else np.abs(np64(b)))
    return xq.shape[1] * U * S + U * S


def check_forward(y, x, w, b, act, pre, post, wq=None):
    xq = X.rounded(np64(x))
    wq = X.rounded(np64(w)) if wq is None else wq
    want, slope, z = X.linear(xq, wq, None if b is None else np64(b), act, pre, post)
    tz = tolerance_z(xq, wq, b)
    steepest = abs(pre * post)
    top = np.abs(want) if act in ("none", "relu") else abs(post)
    tol = steepest * tz + 4 * U * top + np.abs(steepest * z) * 4 * U + torch.finfo(y.dtype).eps / 2 * np.abs(want) + 2.0 ** -24 * (y.dtype == torch.float16)
    err = np.abs(np64(y) - want)
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


SHAPES = [(1, 32, 16), (1, 256, 256), (1, 1000, 33), (2, 129, 300), (5, 4096, 512), (13, 500, 257), (16, 512, 64), (17, 96, 129), (33, 640, 160),
          (64, 1024, 1000), (100, 63, 7), (128, 256, 128), (129, 257, 130), (300, 319, 257), (1000, 128, 1), (257, 2048, 600), (3, 8200, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K, N", SHAPES)
def test_linear_shapes(dtype, M, K, N):
    from nerf import mx
    x, w = randn(M, K, seed=1, dtype=dtype), randn(N, K, seed=2, dtype=dtype, scale=K ** -0.5)
    b = randn(N, seed=3, dtype=dtype)
    y = mx.linear(x, w, b)
    assert y.shape == (M, N) and y.dtype == dtype
    check_forward(y, x, w, b, "none", 1.0, 1.0)
    q = mx.quantize(w)
    assert torch.equal(mx.linear(x, q, b), y)            # packed or float weight: the same call underneath
    assert torch.equal(mx.linear(x, q, b), y)            # and the same bits again


@pytest.mark.parametrize("dtype, act, M, K, N", [
    (torch.float32, "sin", 3500, 100, 3600), (torch.bfloat16, "none", 3301, 300, 4001), (torch.float16, "relu", 3400, 1030, 3333),
    (torch.float32, "relu", 50000, 256, 256), (torch.bfloat16, "sigmoid", 12600, 700, 1025), (torch.float16, "none", 130, 513, 100000)])
def test_linear_many_tiles(dtype, act, M, K, N):
    """Outputs of some 200 tiles of 256 x 256 and more, one to nine steps along the rows, ragged at both edges."""
    from nerf import mx
    x, w, b = randn(M, K, seed=1, dtype=dtype), randn(N, K, seed=2, dtype=dtype, scale=K ** -0.5), randn(N, seed=3, dtype=dtype)
    check_forward(mx.linear(x, w, b, mx.ACTIVATIONS[act]), x, w, b, act, 1.0, 1.0)


FEW = [(16, 8192, 8192), (17, 8192, 8192), (26, 256, 300), (28, 256, 300), (64, 4096, 4096), (64, 4100, 4096), (65, 512, 512), (8, 40, 33000), (16, 130, 17000), (17, 130, 17000), (1, 130, 300000)]


@pytest.mark.parametrize("M, K, N", FEW)
def test_rows_of_a_batch_agree_with_single_rows(M, K, N):
    """Both sides of the choice between the ways to multiply: every row as if it came alone, but for the order of its sums."""
    from nerf import mx
    x, q = randn(M, K, seed=1), mx.quantize(randn(N, K, seed=2, scale=K ** -0.5))
    y = mx.linear(x, q)
    assert torch.equal(y, mx.linear(x, q))
    ax, aw = mx.dequantize(mx.quantize(x)).double(), mx.dequantize(q).double()
    S = (ax.abs() @ aw.abs().t())
    tol = 2 * (K * U * S + U * S) + 2.0 ** -23 * y.double().abs()
    for m in {0, M // 2, M - 1}:
        assert ((mx.linear(x[m:m + 1], q) - y[m:m + 1]).abs() <= tol[m:m + 1]).all()
    assert ((y - ax @ aw.t()).abs() <= tol / 2).all()


NARROW_FWD = [(16384, 256, 256), (16389, 100, 33), (16400, 31, 16), (17001, 255, 250), (16500, 132, 1), (20003, 128, 129), (16385, 1, 200)]
NARROW = [(4096, 256, 256), (4111, 100, 33), (4097, 31, 16), (6001, 255, 250), (4500, 132, 1), (5003, 128, 129), (9000, 64, 64), (4099, 1, 200)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, K, N", NARROW_FWD)
def test_linear_narrow(dtype, act, M, K, N):
    """Up to 256 inputs and outputs over many rows, ragged everywhere; then rows with a pitch and at an odd address."""
    from nerf import mx
    x, w, b = randn(M, K, seed=1, dtype=dtype), randn(N, K, seed=2, dtype=dtype, scale=K ** -0.5), randn(N, seed=3, dtype=dtype)
    y = mx.linear(x, w, b, mx.ACTIVATIONS[act], 1.5, 2.0)
    check_forward(y, x, w, b, act, 1.5, 2.0)
    buf = randn(M * (K + 8) + 5, seed=4, dtype=dtype)
    for shift, width in ((0, K + 8), (5, K + 3)):
        x2 = buf[shift:shift + M * width].view(M, width)[:, :K]
        assert torch.equal(mx.linear(x2, w, b, mx.ACTIVATIONS[act]), mx.linear(x2.contiguous(), w, b, mx.ACTIVATIONS[act]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, K, N", [(1, 300, 50), (40, 200, 70), (700, 256, 256)])
def test_linear_activations(dtype, act, M, K, N):
    from nerf import mx
    x, w, b = randn(M, K, seed=4, dtype=dtype), randn(N, K, seed=5, dtype=dtype, scale=K ** -0.5), randn(N, seed=6, dtype=dtype)
    for pre, post, bias in ((1.0, 1.0, b), (3.0, 0.5, None), (-2.0, 10.0, b)):
        y = mx.linear(x, w, bias, mx.ACTIVATIONS[act], pre, post)
        check_forward(y, x, w, bias, act, pre, post)


def test_linear_takes_a_pitch_and_an_odd_address():
    from nerf import mx
    buf = randn(50 * 210 + 3, seed=7, dtype=torch.bfloat16)
    x = buf[3:].view(50, 210)[:, 4:204]
    w = randn(48, 200, seed=8, dtype=torch.bfloat16)
    check_forward(mx.linear(x, w), x, w, None, "none", 1.0, 1.0)


@pytest.mark.parametrize("M", [5, 40, 300, 16400])
@pytest.mark.parametrize("far", [0.0, 0.01, 0.5])
def test_sines_of_large_arguments(M, far):
    """Sums that are exact (codes times powers of two, small integers), times a power of two up to 2^20: sine and cosine of the
    exact argument, a few, half or none of them beyond the short reduction's range, some infinite."""
    from nerf import mx
    K, N, g = 32, 40, torch.Generator().manual_seed(M)
    x = torch.randint(0, 3, (M, K), generator=g).float()
    x[torch.rand(M, generator=g) < far] *= 2.0 ** 8
    w = torch.randint(-2, 3, (N, K), generator=g).float()
    x, w = x.to(DEV), w.to(DEV)
    assert torch.equal(mx.dequantize(mx.quantize(x)), x) and torch.equal(mx.dequantize(mx.quantize(w)), w)
    pre = 2.0 ** 10
    t = np64(x) @ np64(w).T * pre
    assert (np.abs(t) < 2 ** 30).all() and (np.abs(t[0]) > 0).any()
    xl = x.clone().requires_grad_(True)
    y = mx.linear(xl, w, None, mx.ACT_SIN, pre, 2.0)
    assert (np.abs(np64(y) - 2 * np.sin(t)) <= 2 * 8 * U).all()
    (dx,) = torch.autograd.grad(y, xl, torch.ones_like(y))
    want = (2 * pre * np.cos(t)) @ np64(w)
    assert (np.abs(np64(dx) - want) <= 2 * pre * (8 + N) * U * np.abs(np64(w)).sum(0)).all()
    x[1] = 2.0 ** 120
    b = mx.linear(x, w, None, mx.ACT_SIN, 2.0 ** 20, 1.0)
    over = np.abs(np64(x) @ np64(w).T) * 2.0 ** 20 > torch.finfo(torch.float32).max
    assert torch.isnan(b)[torch.from_numpy(over).to(DEV)].all() and not torch.isnan(b[0]).any()


def test_far_scales():
    """Blocks of very different magnitude: 2^-60 to 2^60 in one row (the products of the small ones vanish beside the sum)."""
    from nerf import mx
    e = torch.randint(-60, 60, (20, 8, 1), generator=torch.Generator().manual_seed(1)).double()
    x = (randn(20, 256, seed=10).cpu().double().view(20, 8, 32) * torch.pow(2.0, e)).view(20, 256).float().to(DEV)
    w = randn(30, 256, seed=11)
    check_forward(mx.linear(x, w), x, w, None, "none", 1.0, 1.0)


@pytest.mark.parametrize("M", [1, 7, 300])
def test_nan_stays_in_its_row_or_column(M):
    from nerf import mx
    x, w = randn(M, 200, seed=12), randn(40, 200, seed=13)
    for act in ACTS:
        clean = mx.linear(x, w, None, mx.ACTIVATIONS[act])
        xn = x.clone()
        xn[M - 1, 150] = float("inf")
        y = mx.linear(xn, w, None, mx.ACTIVATIONS[act])
        assert torch.isnan(y[M - 1]).all() and torch.equal(y[:M - 1], clean[:M - 1])
        wn = w.clone()
        wn[3, 0] = float("nan")
        y = mx.linear(x, wn, None, mx.ACTIVATIONS[act])
        assert torch.isnan(y[:, 3]).all()
        keep = [n for n in range(40) if n != 3]
        assert torch.equal(y[:, keep], clean[:, keep])


@pytest.mark.parametrize("M, K, N", [(37, 160, 45), (300, 160, 45), (300, 1200, 45), (3400, 600, 3601), (16390, 160, 45)])
@pytest.mark.parametrize("act", ["relu", "sin"])
def test_outputs_beside_the_rows_are_left_alone(act, M, K, N):
    """The C entries with a pitch wider than the row: what lies between the rows, and behind the last, keeps its contents."""
    from nerf import _hip, mx
    lib, ld, A = _hip.lib, N + 19, mx.ACTIVATIONS[act]
    st = torch.cuda.current_stream().cuda_stream
    x, q = randn(M, K, seed=14), mx.quantize(randn(N, K, seed=15))
    y = torch.full((M + 3, ld), 7.0, device=DEV)
    ws = torch.empty(lib.nerf_mx_linear_fwd_workspace_bytes(M, K, N, 0) + 16, dtype=torch.uint8, device=DEV)
    rc = lib.nerf_mx_linear_fwd(x.data_ptr(), 0, K, q.codes.data_ptr(), q.scales.data_ptr(), None, M, K, N, A, 1.0, 1.0, y.data_ptr(), ld,
                                None, None, None, None, ws.data_ptr(), st)
    assert rc == 0
    assert torch.equal(y[:M, :N], mx.linear(x, q, None, A)) and (y[:, N:] == 7.0).all() and (y[M:] == 7.0).all()
    want, kept = _hip.mx_linear_train(x, None, (q.codes, q.scales), None, A, 1.0, 1.0)
    dy = randn(M, N, seed=16)
    dx, dw, db = _hip.mx_linear_bwd(dy, kept, kept.buffer, (q.codes, q.scales), True, True, True)
    base = kept.buffer.data_ptr()
    wide, dw2, db2 = torch.full((M + 3, K + 5), 7.0, device=DEV), torch.full((N + 3, K), 7.0, device=DEV), torch.full((N + 9,), 7.0, device=DEV)
    nbytes = lib.nerf_mx_linear_bwd_workspace_bytes(0, A, M, K, N, 1, 1, 1)
    ws = torch.full((nbytes + 256,), 7, dtype=torch.uint8, device=DEV)
    rc = lib.nerf_mx_linear_bwd(dy.data_ptr(), 0, N, base + kept.extra, base + kept.extra, A, 1.0, 1.0, base + kept.xcodes, base + kept.xscales,
                                q.codes.data_ptr(), q.scales.data_ptr(), M, K, N, ws.data_ptr(), wide.data_ptr(), K + 5, dw2.data_ptr(),
                                db2.data_ptr(), st)
    assert rc == 0
    assert torch.equal(wide[:M, :K], dx) and (wide[:, K:] == 7.0).all() and (wide[M:] == 7.0).all()
    assert torch.equal(dw2[:N], dw) and (dw2[N:] == 7.0).all() and torch.equal(db2[:N], db) and (db2[N:] == 7.0).all()
    assert (ws[nbytes:] == 7).all()


# --------------------------------------------------------------------------------------------------------- gradients
def terms_error(dtype, act):
    """Relative error of dz as bf16 terms: exact, or cut behind the last term (half a step of a bf16 remainder)."""
    if dtype == torch.float32:
        return 2.0 ** -25
    return 2.0 ** -17 if act in ("sin", "sigmoid") else 0.0


def check_backward(grads, dy, x, w, b, act, pre, post, dtype):
    xq, wq = X.rounded(np64(x)), X.rounded(np64(w))
    _, slope, z = X.linear(xq, wq, None if b is None else np64(b), act, pre, post)
    g = np64(dy)
    M, N = g.shape
    # relu: decisions of sums that the fp32 rounding could turn are left out by the callers' seeds (asserted here)
    tz = tolerance_z(xq, wq, b)
    if act == "relu":
        assert (np.abs(z) > tz).all()
    # d slope / d z is at most |post| pre^2 for the three others' derivatives; a few fp32 operations on top
    ts = np.zeros_like(z) if act in ("none", "relu") else abs(post) * pre * pre * tz + 8 * U * abs(pre * post) * (1 + np.abs(pre * z))
    dz = g * slope
    tdz = np.abs(g) * ts + np.abs(dz) * (terms_error(dtype, act) + 2 * U)
    for name, got, want, S, t, n in (
            ("dx", grads[0], dz @ wq, np.abs(dz) @ np.abs(wq), tdz @ np.abs(wq), N * 3),
            ("dw", grads[1], dz.T @ xq, np.abs(dz).T @ np.abs(xq), tdz.T @ np.abs(xq), M * 3),
            ("db", grads[2], dz.sum(0), np.abs(dz).sum(0), tdz.sum(0), M)):
        if got is None:
            continue
        assert got.dtype == dtype and got.shape == want.shape, name
        tol = (n + 4) * U * S + t + torch.finfo(dtype).eps / 2 * np.abs(want) * (1 + 2.0 ** -7) + 2.0 ** -24 * (dtype == torch.float16)
        err = np.abs(np64(got) - want)
        assert (err <= tol).all(), (name, float((err - tol).max()), float(err.max()))


def run_training(x, w, b, dy, act, pre=1.0, post=1.0):
    from nerf import mx
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    y = mx.linear(*leaves, mx.ACTIVATIONS[act], pre, post)
    return y.detach(), torch.autograd.grad(y, leaves, dy)


GRAD_SHAPES = [(1, 1, 1), (1, 32, 16), (3, 130, 40), (64, 64, 64), (65, 33, 129), (100, 319, 257), (700, 96, 200), (513, 256, 256), (2500, 40, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K, N", GRAD_SHAPES)
def test_gradient_shapes(dtype, M, K, N):
    x, w = randn(M, K, seed=21, dtype=dtype), randn(N, K, seed=22, dtype=dtype, scale=K ** -0.5)
    b, dy = randn(N, seed=23, dtype=dtype), randn(M, N, seed=24, dtype=dtype)
    y, grads = run_training(x, w, b, dy, "none")
    check_forward(y, x, w, b, "none", 1.0, 1.0)
    check_backward(grads, dy, x, w, b, "none", 1.0, 1.0, dtype)
    again = run_training(x, w, b, dy, "none")[1]
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gradient_activations(dtype, act):
    M, K, N = 150, 100, 90
    x, w = randn(M, K, seed=31, dtype=dtype), randn(N, K, seed=32, dtype=dtype, scale=K ** -0.5)
    dy = randn(M, N, seed=34, dtype=dtype)
    # the bias keeps ReLU sums away from zero, where the decision would be the rounding's
    b = (torch.sign(randn(N, seed=33)) * 30).to(dtype) if act == "relu" else randn(N, seed=33, dtype=dtype)
    for pre, post in ((1.0, 1.0), (0.5, 3.0), (-1.5, 2.0)):
        y, grads = run_training(x, w, b, dy, act, pre, post)
        check_forward(y, x, w, b, act, pre, post)
        check_backward(grads, dy, x, w, b, act, pre, post, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, K, N", NARROW + [(16390, 256, 256), (16387, 64, 40), (16500, 100, 129)])
def test_gradients_narrow(dtype, act, M, K, N):
    x, w = randn(M, K, seed=31, dtype=dtype), randn(N, K, seed=32, dtype=dtype, scale=K ** -0.5)
    b = (torch.sign(randn(N, seed=33)) * 30).to(dtype) if act == "relu" else randn(N, seed=33, dtype=dtype)
    dy = randn(M, N, seed=34, dtype=dtype)
    y, grads = run_training(x, w, b, dy, act, 1.5, 2.0)
    check_forward(y, x, w, b, act, 1.5, 2.0)
    check_backward(grads, dy, x, w, b, act, 1.5, 2.0, dtype)
    again = run_training(x, w, b, torch.cat([dy, dy], 1)[:, N:], act, 1.5, 2.0)[1]      # dy with a pitch
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


@pytest.mark.parametrize("dtype, act, M, K, N", [
    (torch.float32, "sin", 3400, 3500, 90), (torch.bfloat16, "none", 3333, 3601, 130), (torch.float16, "sigmoid", 90, 3400, 3600),
    (torch.float32, "none", 45, 3601, 3400), (torch.bfloat16, "sin", 130, 3400, 3700)])
def test_gradients_many_tiles(dtype, act, M, K, N):
    """dx or dW of more than 192 tiles of 256 x 256, one to twelve steps along the reduction."""
    x, w = randn(M, K, seed=31, dtype=dtype), randn(N, K, seed=32, dtype=dtype, scale=K ** -0.5)
    b, dy = randn(N, seed=33, dtype=dtype), randn(M, N, seed=34, dtype=dtype)
    y, grads = run_training(x, w, b, dy, act)
    check_forward(y, x, w, b, act, 1.0, 1.0)
    check_backward(grads, dy, x, w, b, act, 1.0, 1.0, dtype)


def test_relu_mask_is_the_forward_decision():
    """Mixed decisions in every sixteen-bit word, at widths that end inside one: the gradient is open where y > 0."""
    from nerf import mx
    for N in (1, 15, 16, 17, 50):
        x, w = randn(70, 64, seed=35), randn(N, 64, seed=36)
        x.requires_grad_(True)
        b = torch.zeros(N, device=DEV, requires_grad=True)
        y = mx.linear(x, w, b, mx.ACT_RELU)
        (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
        assert torch.equal(db, (y > 0).float().sum(0))


def test_gradients_match_differences():
    """Directional differences of the float64 product at the rounded operands: <grad, v> = (L(h) - L(-h)) / 2h up to h^2."""
    M, K, N = 60, 70, 50
    x, w, b, dy = randn(M, K, seed=41), randn(N, K, seed=42, scale=K ** -0.5), randn(N, seed=43), randn(M, N, seed=44)
    for act in ("none", "sin", "sigmoid"):
        _, grads = run_training(x, w, b, dy, act, 1.5, 2.0)
        xq, wq, b64, g = X.rounded(np64(x)), X.rounded(np64(w)), np64(b), np64(dy)
        loss = lambda a, c, d: float((g * X.linear(a, c, d, act, 1.5, 2.0)[0]).sum())
        rng = np.random.default_rng(5)
        v = [rng.standard_normal(t.shape) for t in (xq, wq, b64)]
        for i in range(3):
            h = 1e-5
            plus = [t + h * d if j == i else t for j, (t, d) in enumerate(zip((xq, wq, b64), v))]
            minus = [t - h * d if j == i else t for j, (t, d) in enumerate(zip((xq, wq, b64), v))]
            want = (loss(*plus) - loss(*minus)) / (2 * h)
            got = float((np64(grads[i]) * v[i]).sum())
            # differences: third derivative times h^2 and 1e-16 / h of the loss; gradients: 1e-5 of their norm
            assert abs(got - want) <= 1e-5 * np.linalg.norm(np64(grads[i])) * np.linalg.norm(v[i]) / np.sqrt(v[i].size) + 1e-6 * abs(want) + 1e-5


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_unfinite_upstream_gradients(dtype):
    """Values whose bf16 rounding would overflow stay finite; infinities and NaN reach the gradients they feed."""
    from nerf import _hip, mx
    x, w, b = randn(70, 64, seed=51, dtype=dtype), randn(32, 64, seed=52, dtype=dtype), randn(32, seed=53, dtype=dtype)
    dy = randn(70, 32, seed=54, dtype=dtype)
    top = torch.finfo(dtype).max
    dy[2, 3] = top
    _, (dx, dw, db) = run_training(x, w, b, dy, "none")
    if dtype == torch.float32:
        assert torch.isfinite(db).all() and float(db[3]) > 0.99 * top
    dy[2, 3] = float("inf")
    dy[5, 6] = float("nan")
    _, (dx, dw, db) = run_training(x, w, b, dy, "none")
    assert not torch.isfinite(db[3]) and torch.isnan(db[6]) and torch.isfinite(db[[i for i in range(32) if i not in (3, 6)]]).all()
    assert torch.isnan(dx[5]).all() and not torch.isfinite(dx[2]).any()
    assert torch.isfinite(dx[[i for i in range(70) if i not in (2, 5)]]).all()


def test_gradient_layouts_and_subsets():
    from nerf import mx
    x, w, b = randn(40, 64, seed=61), randn(48, 64, seed=62), randn(48, seed=63)
    dy = randn(40, 48, seed=64)
    full = run_training(x, w, b, dy, "none")[1]
    xl = x.clone().requires_grad_(True)
    q = mx.quantize(w)
    (dx,) = torch.autograd.grad(mx.linear(xl, q, b), xl, dy)          # frozen packed weight
    assert torch.equal(dx, full[0])
    wl = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(mx.linear(x, wl), wl, dy)
    assert torch.equal(dw, full[1])
    bl = b.clone().requires_grad_(True)
    (db,) = torch.autograd.grad(mx.linear(x, w, bl), bl, dy)
    assert torch.equal(db, full[2])
    # upstream gradients that are expanded (a sum's), transposed or cut out of something wider
    ones = torch.ones(40, 48, device=DEV)
    want = run_training(x, w, b, ones, "none")[1]
    xl = x.clone().requires_grad_(True)
    mx.linear(xl, w, b).sum().backward()
    assert torch.equal(xl.grad, want[0])
    for view in (dy.t().contiguous().t(), torch.cat([dy, dy], 1)[:, :48], torch.cat([dy[:, :1], dy], 1)[:, 1:]):
        assert all(torch.equal(a, c) for a, c in zip(run_training(x, w, b, view, "none")[1], full))
    # leading dimensions
    x3 = x.view(5, 8, 64).clone().requires_grad_(True)
    (d3,) = torch.autograd.grad(mx.linear(x3, w, b), x3, dy.view(5, 8, 48))
    assert torch.equal(d3.view(40, 64), full[0])
    # no rows
    x0 = torch.zeros(0, 64, device=DEV, requires_grad=True)
    d0, dw0 = torch.autograd.grad(mx.linear(x0, wl, b).sum(), (x0, wl))
    assert d0.shape == (0, 64) and (dw0 == 0).all()
    # the same tensor as input and weight
    s = randn(48, 64, seed=65).requires_grad_(True)
    (ds,) = torch.autograd.grad(mx.linear(s, s), s, dy[:40].new_ones(48, 48))
    a, c = s.detach().clone().requires_grad_(True), s.detach().clone().requires_grad_(True)
    da, dc = torch.autograd.grad(mx.linear(a, c), (a, c), dy.new_ones(48, 48))
    assert torch.equal(ds, da + dc)
    # first order only
    xl = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(mx.linear(xl, w, b, mx.ACT_SIN), xl, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# ------------------------------------------------------------------------------------------------- streams, graphs, runs
def test_other_stream():
    from nerf import mx
    x, w, dy = randn(300, 256, seed=71), randn(128, 256, seed=72), randn(300, 128, seed=74)
    b = randn(128, seed=73)
    want = run_training(x, w, b, dy, "sin")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_training(x, w, b, dy, "sin")
        q = mx.dequantize(mx.quantize(x))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, c) for a, c in zip(got[1], want[1]))
    assert torch.equal(q, mx.dequantize(mx.quantize(x)))


def test_gradients_at_odd_addresses():
    """dy, slopes and decisions anywhere their types allow: the same bits as at aligned addresses."""
    from nerf import _hip, mx
    lib, M, K, N = _hip.lib, 4100, 64, 64
    st = torch.cuda.current_stream().cuda_stream
    x, w, dy = randn(M, K, seed=1), randn(N, K, seed=2), randn(M, N, seed=3)
    for act in (mx.ACT_SIN, mx.ACT_RELU):
        _, kept = _hip.mx_linear_train(x, w, None, None, act, 1.0, 1.0)
        base = kept.buffer.data_ptr()
        size = 4 * M * N if act == mx.ACT_SIN else 2 * M * (N // 16)
        extra = torch.zeros(size + 16, dtype=torch.uint8, device=DEV)
        at = 4 if act == mx.ACT_SIN else 2
        extra[at:at + size] = kept.buffer[kept.extra:kept.extra + size]
        odd = torch.zeros(M * N + 1, device=DEV)
        odd[1:] = dy.view(-1)
        ws = torch.empty(lib.nerf_mx_linear_bwd_workspace_bytes(0, act, M, K, N, 1, 1, 1), dtype=torch.uint8, device=DEV)
        want = _hip.mx_linear_bwd(dy, kept, kept.buffer, None, True, True, True)
        x64 = (np64(dy), np64(mx.dequantize(mx.quantize(x))), np64(mx.dequantize(mx.quantize(w))))
        for dptr, eptr in ((odd.data_ptr() + 4, base + kept.extra), (dy.data_ptr(), extra.data_ptr() + at)):
            dx, dw, db = torch.empty(M, K, device=DEV), torch.empty(N, K, device=DEV), torch.empty(N, device=DEV)
            rc = lib.nerf_mx_linear_bwd(dptr, 0, N, eptr, eptr, act, 1.0, 1.0, base + kept.xcodes, base + kept.xscales, base + kept.wcodes,
                                        base + kept.wscales, M, K, N, ws.data_ptr(), dx.data_ptr(), K, dw.data_ptr(), db.data_ptr(), st)
            assert rc == 0
            slope = np64(kept.buffer[kept.extra:kept.extra + size].view(torch.float32).view(M, N)) if act == mx.ACT_SIN else \
                (np.unpackbits(kept.buffer[kept.extra:kept.extra + size].cpu().numpy().view(np.uint8), bitorder="little").reshape(M, N))
            dz = x64[0] * slope
            for got, same, exact, S, n in ((dx, want[0], dz @ x64[2], np.abs(dz) @ np.abs(x64[2]), N),
                                           (dw, want[1], dz.T @ x64[1], np.abs(dz).T @ np.abs(x64[1]), M),
                                           (db, want[2], dz.sum(0), np.abs(dz).sum(0), M)):
                tol = (n + 4) * U * S + 2.0 ** -24 * np.abs(exact) + 2.0 ** -25 * S
                assert (np.abs(np64(got) - exact) <= tol).all() and (np.abs(np64(same) - exact) <= tol).all()


def test_products_beyond_32_bits():
    """Outputs and operands of more than 2^32 bytes and 2^31 values: the last rows are those of a small call."""
    from nerf import _hip, mx
    # tiles: 2.3e9 outputs with their slopes (one step along the rows, so the order of the sums is the same everywhere)
    M, K, N = 70000, 40, 32800
    x, w = randn(M, K, seed=1, dtype=torch.bfloat16), randn(N, K, seed=2, dtype=torch.bfloat16)
    y, kept = _hip.mx_linear_train(x, w, None, None, mx.ACT_SIN, 1.0, 1.0)
    small, few = _hip.mx_linear_train(x[-300:], w, None, None, mx.ACT_SIN, 1.0, 1.0)
    assert torch.equal(y[-300:], small)
    assert torch.equal(kept.buffer[kept.extra + 4 * (M - 300) * N:kept.extra + 4 * M * N], few.buffer[few.extra:few.extra + 4 * 300 * N])
    del y, kept, small, few, x, w
    # narrow and general gradients at the most rows a call trains; only the last rows have an upstream gradient
    M, tail = 65535 * 64, 16384
    for K, N, dtype in ((256, 256, torch.float32), (40, 300, torch.float32), (40, 300, torch.bfloat16)):
        x = torch.zeros(M, K, dtype=dtype, device=DEV)
        x[-tail:] = randn(tail, K, seed=3, dtype=dtype)
        dy = torch.zeros(M, N, dtype=dtype, device=DEV)
        dy[-tail:] = randn(tail, N, seed=4, dtype=dtype)
        w = randn(N, K, seed=5, dtype=dtype)
        y, kept = _hip.mx_linear_train(x, w, None, None, mx.ACT_SIN, 1.0, 1.0)
        dx, dw, db = _hip.mx_linear_bwd(dy, kept, kept.buffer, None, True, True, True)
        assert not dx[:-tail].any()
        xt, dyt = x[-tail:].clone(), dy[-tail:].clone()
        del x, dy, kept
        ys, kept = _hip.mx_linear_train(xt, w, None, None, mx.ACT_SIN, 1.0, 1.0)
        dxs, dws, dbs = _hip.mx_linear_bwd(dyt, kept, kept.buffer, None, True, True, True)
        eps = torch.finfo(dtype).eps
        X64, W64 = mx.dequantize(mx.quantize(xt)).double().abs(), mx.dequantize(mx.quantize(w)).double().abs()
        z = X64 @ W64.t()
        # |dz| <= |dy|; the two calls sum in other orders, in y's case inside the argument of the sine as well
        assert ((y[-tail:] - ys).double().abs() <= 2 * (K + 2) * U * z + 8 * U + eps * ys.double().abs()).all()
        dz, ez = dyt.double().abs(), dyt.double().abs() * (2 * (K + 2) * U * z + 8 * U)
        for got, want, S, E, n in ((dx[-tail:], dxs, dz @ W64, ez @ W64, N), (dw, dws, dz.t() @ X64, ez.t() @ X64, tail),
                                   (db, dbs, dz.sum(0), ez.sum(0), tail)):
            assert ((got - want).double().abs() <= E + (2 * (3 * n + 8) * U + 2.0 ** -16) * S + eps * want.double().abs()).all()
        del y, dx, ys, kept


def test_two_calls_at_once():
    """The same layers forward and backward on two streams that run side by side, several times over."""
    sets = [(randn(m, k, seed=1), randn(n, k, seed=2), randn(n, seed=3), randn(m, n, seed=4))
            for m, k, n in ((20, 512, 300), (700, 256, 256), (17000, 256, 256), (3400, 300, 3601))]
    want = [run_training(*s, "sin") for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for st, order in zip(streams, (sets, sets[::-1])):
            with torch.cuda.stream(st):
                got.append([run_training(*s, "sin") for s in order][::1 if order is sets else -1])
    torch.cuda.synchronize()
    for run in got:
        for a, c in zip(run, want):
            assert torch.equal(a[0], c[0]) and all(torch.equal(g, h) for g, h in zip(a[1], c[1]))


@pytest.mark.parametrize("M, K, N", [(1, 512, 256), (40, 512, 256), (700, 512, 256), (5000, 128, 256), (16390, 256, 200), (3400, 520, 3601)])
def test_captured_and_replayed(M, K, N):
    """Two captured graphs (a layer's product, and a product with its gradients), replayed alternately with new inputs
    and eager work between, against the eager results."""
    from nerf import _hip, mx
    w, b = randn(N, K, seed=81), randn(N, seed=82)
    q = mx.quantize(w)
    x, dy = randn(M, K, seed=83), randn(M, N, seed=84)

    def serve():
        return mx.linear(x, q, b, mx.ACT_RELU)

    def train():
        y, kept = _hip.mx_linear_train(x, w, None, b, mx.ACT_SIN, 1.0, 1.0)
        return (y, *_hip.mx_linear_bwd(dy, kept, kept.buffer, None, True, True, True))

    with torch.no_grad():
        serve(), train()
        torch.cuda.synchronize()
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1):
            out1 = serve()
        with torch.cuda.graph(g2):
            out2 = train()
        for i in range(4):
            x.copy_(randn(M, K, seed=90 + i))
            dy.copy_(randn(M, N, seed=190 + i))
            g1.replay()
            g2.replay()
            g1.replay()
            torch.cuda.synchronize()
            assert torch.equal(out1, serve())
            assert all(torch.equal(a, c) for a, c in zip(out2, train()))


@pytest.mark.parametrize("M, K, N", [(30, 96, 64), (5000, 96, 64)])
def test_captured_through_autograd(M, K, N):
    """Forward and torch.autograd.grad inside one capture (warmed up on another stream), replayed with new inputs."""
    from nerf import mx
    x, w, b, dy = randn(M, K, seed=1), randn(N, K, seed=2), randn(N, seed=3), randn(M, N, seed=4)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = mx.linear(*leaves, mx.ACT_SIN)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(randn(M, K, seed=20 + i))
            leaves[1].copy_(randn(N, K, seed=30 + i))
            dy.copy_(randn(M, N, seed=40 + i))
        graph.replay()
        torch.cuda.synchronize()
        y, grads = run_training(*leaves, dy, "sin")
        assert torch.equal(out[0], y) and all(torch.equal(a, c) for a, c in zip(out[1:], grads))


def test_a_run_of_layers_as_a_model_uses_them():
    """Three layers forward and backward through autograd: every layer's output and gradients against the float64
    restatement at the inputs that layer saw."""
    from nerf import mx
    M, dims, acts = 200, [96, 128, 64, 40], ["sin", "sin", "none"]
    ws = [randn(o, i, seed=100 + i, scale=i ** -0.5).requires_grad_(True) for i, o in zip(dims, dims[1:])]
    bs = [randn(o, seed=200 + o, scale=0.3).requires_grad_(True) for o in dims[1:]]
    x = randn(M, dims[0], seed=99)
    hs = [x.clone().requires_grad_(True)]
    for w, b, act in zip(ws, bs, acts):
        h = mx.linear(hs[-1], w, b, mx.ACTIVATIONS[act])
        h.retain_grad()
        hs.append(h)
    (hs[-1].square().mean()).backward()
    for i, act in enumerate(acts):
        check_forward(hs[i + 1], hs[i], ws[i], bs[i], act, 1.0, 1.0)
        check_backward((hs[i].grad, ws[i].grad, bs[i].grad), hs[i + 1].grad, hs[i], ws[i], bs[i], act, 1.0, 1.0, torch.float32)


@pytest.mark.parametrize("tag", ["nerf", "nerf64", "siren", "siren3"])
def test_models_in_the_mxfp4_mode(tag):
    """The modes of the models: the layers between hidden activations are mx.linear calls, everything else is unchanged;
    training and rendering run the same network, and every parameter gets a finite gradient."""
    from nerf import mx
    from nerf.encoding import positional_encoding
    from nerf.models import NeRF, Siren
    from nerf.rendering import render_nerf, render_nerf_hierarchical
    torch.manual_seed(3)
    model = {"nerf": NeRF, "nerf64": lambda: NeRF(hidden_dim=64), "siren": Siren, "siren3": lambda: Siren(num_layers=3, hidden_dim=96)}[tag]().to(DEV)
    pts, dirs = randn(200, 3, seed=1, scale=0.4), torch.nn.functional.normalize(randn(200, 3, seed=2), dim=1)
    with torch.no_grad():
        c32, d32 = model(pts, dirs)
        model.set_inference_precision("mxfp4")
        c4, d4 = model(pts, dirs)
        assert not torch.equal(c32, c4)
    model.set_training_precision("mxfp4")
    ct, dt = model(pts, dirs)
    assert torch.equal(ct, c4) and torch.equal(dt, d4)
    seen, real = [], mx.linear          # what the 4-bit product is given: hidden activations alone
    mx.linear = lambda *a: seen.append(a[0].detach()) or real(*a)
    try:
        model(pts, dirs)
    finally:
        mx.linear = real
    lin = torch.nn.functional.linear
    if tag.startswith("nerf"):
        first = torch.relu(lin(positional_encoding(pts, 10), model.block1[0].weight, model.block1[0].bias))
    else:
        first = torch.sin(30.0 * lin(pts, model.block1[0].layer.weight, model.block1[0].layer.bias))
    width = first.shape[1]
    assert len(seen) == {"nerf": 8, "nerf64": 8, "siren": 8, "siren3": 3}[tag] and all(t.shape == (200, width) for t in seen)
    assert torch.allclose(seen[0], first.detach(), atol=2e-4)
    o, d = randn(50, 3, seed=5), torch.nn.functional.normalize(randn(50, 3, seed=6), dim=1)
    u = torch.rand(32, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    rgb = render_nerf(model, o, d, 2.0, 6.0, num_samples=32, device=DEV, u=[u])
    with torch.no_grad():
        assert torch.equal(rgb, render_nerf(model, o, d, 2.0, 6.0, num_samples=32, device=DEV, u=[u]))
    rgb.square().mean().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    with pytest.raises(TypeError, match="mxfp4"):
        render_nerf_hierarchical(model, model, o, d, 2.0, 6.0)


@pytest.mark.parametrize("model_type, optimizer", [("nerf", "fused"), ("siren", "torch")])
def test_train_resume_eval_in_the_mxfp4_mode(tmp_path, model_type, optimizer):
    """train.py with train_precision = mxfp4, resumed, then eval.py --precision mxfp4; a coarse + fine pair is refused."""
    import os
    import sys
    from test_callers import make_dataset, write_config
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nerf-pytorch_amd"))
    import eval as eval_script
    import train
    root, save = make_dataset(str(tmp_path / "ds")), str(tmp_path / "models")
    cfg = str(tmp_path / "c.txt")
    write_config(cfg, root, save, model_type, "train_precision = mxfp4")
    train.main(["--config", cfg, "--optimizer", optimizer, "--max-iters", "4"])
    files = sorted(os.listdir(save))
    train.main(["--config", cfg, "--optimizer", optimizer, "--resume", os.path.join(save, files[0])])
    last = os.path.join(save, sorted(os.listdir(save))[-1])
    frames = str(tmp_path / "frames")
    eval_script.main(["--config", cfg, "--checkpoint", last, "--output", frames, "--precision", "mxfp4"])
    assert len(os.listdir(frames)) == 2
    write_config(cfg, root, save, model_type, "train_precision = mxfp4\nnum_fine_samples = 8")
    with pytest.raises(ValueError, match="single network"):
        train.main(["--config", cfg])
