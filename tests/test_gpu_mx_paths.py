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


# ------------------------------------------------------------------------------------ the ends of the range, NaN, infinities
@pytest.mark.parametrize("act", ["none", "relu", "sin"])
@pytest.mark.parametrize("M, K, N", [(70, 64, 32), (4200, 64, 32), (4200, 200, 256), (700, 300, 320)])
def test_upstream_gradients_at_the_end_of_the_range(act, M, K, N):
    """Values above the largest bf16, whose first term would round to infinity: dx and dW, which are made of the terms, against
    float64.  x and w are small enough for the true results to stay finite."""
    from nerf import _hip, mx
    top = torch.finfo(torch.float32).max
    x, w = randn(M, K, seed=51, scale=2.0 ** -10), randn(N, K, seed=52, scale=2.0 ** -12)
    b = torch.sign(randn(N, seed=53)).clamp(min=0 if act == "relu" else -1) * (30.0 if act == "relu" else 0.0)
    if act == "relu":
        b[b == 0] = -30.0
        b[[3, 5, N - 1]] = 30.0
    dy = randn(M, N, seed=54)
    for m, n, v in ((2, 3, top), (M - 1, N - 1, -top), (M // 2, 5, 0.9985 * top), (33, 0, -0.9999 * top)):
        dy[m, n] = v
    assert (dy.abs() > 3.3895e38).sum() == 4 and torch.isinf(dy.to(torch.bfloat16)).sum() == 4
    y, grads = run_training(x, w, b, dy, act)
    assert all(torch.isfinite(g).all() for g in grads)
    assert float(grads[0][2].abs().max()) > 1e33 and float(grads[1][3].abs().max()) > 1e33
    check_backward(grads, dy, x, w, b, act, 1.0, 1.0, torch.float32)
    _, kept = _hip.mx_linear_train(x, w, None, b, mx.ACTIVATIONS[act], 1.0, 1.0)
    assert is_narrow(kept, dy, N) == (M >= 4096)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K, N", [(70, 200, 64), (4200, 200, 64), (4101, 255, 248)])
def test_unfinite_upstream_gradients_stay_in_their_row_and_column(dtype, M, K, N):
    for act in ("none", "sin"):
        x, w, b, dy = training_case(M, K, N, act, dtype)
        clean = run_training(x, w, b, dy, act)[1]
        bad = dy.clone()
        bad[2, 3], bad[M - 1, N - 1], bad[40, 6] = float("inf"), float("nan"), float("-inf")
        dx, dw, db = run_training(x, w, b, bad, act)[1]
        rows, cols = torch.ones(M, dtype=torch.bool), torch.ones(N, dtype=torch.bool)
        rows[[2, M - 1, 40]], cols[[3, N - 1, 6]] = False, False
        assert torch.equal(dx[rows], clean[0][rows]) and torch.equal(dw[cols], clean[1][cols]) and torch.equal(db[cols], clean[2][cols])
        assert not torch.isfinite(dx[~rows]).any() and not torch.isfinite(dw[~cols]).any() and not torch.isfinite(db[~cols]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K, N", [(70, 200, 64), (4200, 200, 64), (3400, 900, 200)])
def test_nan_blocks_reach_the_gradients_they_feed(dtype, M, K, N):
    """A block of x that is NaN: its 32 columns of dW, nothing else.  A block of W: its 32 columns of dx."""
    x, w, b, dy = training_case(M, K, N, "none", dtype)
    dx, dw, db = run_training(x, w, b, dy, "none")[1]
    k0 = K // 32 * 32          # the last, incomplete block
    assert k0 < K
    xn, wn = x.clone(), w.clone()
    xn[M - 1, K - 1], wn[5, 40] = float("inf"), float("nan")
    ex, ew, eb = run_training(xn, w, b, dy, "none")[1]
    assert torch.equal(ex, dx) and torch.equal(eb, db) and torch.equal(ew[:, :k0], dw[:, :k0]) and torch.isnan(ew[:, k0:]).all()
    ex, ew, eb = run_training(x, wn, b, dy, "none")[1]
    assert torch.equal(ew, dw) and torch.equal(eb, db) and torch.isnan(ex[:, 32:64]).all()
    keep = [k for k in range(K) if not 32 <= k < 64]
    assert torch.equal(ex[:, keep], dx[:, keep])


@pytest.mark.parametrize("M, K, N", [(16400, 200, 40), (16390, 100, 130), (3400, 1100, 3601), (3400, 520, 3601), (4000, 900, 2200)])
@pytest.mark.parametrize("act", ACTS)
def test_nan_stays_in_its_row_or_column_of_many_rows(act, M, K, N):
    """The pass for narrow layers, and tiles: the large one with nine and five steps has the poisoned blocks in the last stage,
    half of which does not exist."""
    from nerf import mx
    x, w = randn(M, K, seed=12), randn(N, K, seed=13, scale=K ** -0.5)
    clean = mx.linear(x, w, None, mx.ACTIVATIONS[act])
    xn, wn = x.clone(), w.clone()
    xn[M - 1, K - 1] = float("inf")
    y = mx.linear(xn, w, None, mx.ACTIVATIONS[act])
    assert torch.isnan(y[M - 1]).all() and torch.equal(y[:M - 1], clean[:M - 1])
    wn[3, K - 1], wn[N - 1, 0] = float("nan"), float("-inf")
    y = mx.linear(x, wn, None, mx.ACTIVATIONS[act])
    keep = [n for n in range(N) if n not in (3, N - 1)]
    assert torch.isnan(y[:, [3, N - 1]]).all() and torch.equal(y[:, keep], clean[:, keep])


# ------------------------------------------------------------------------------------------------------------ the large tile
@pytest.mark.parametrize("dtype, act, K", [
    (torch.float32, "relu", 512), (torch.bfloat16, "none", 512), (torch.float32, "sin", 385), (torch.float16, "sigmoid", 400),
    (torch.float32, "relu", 800), (torch.bfloat16, "relu", 897), (torch.float16, "none", 897), (torch.float32, "none", 1024),
    (torch.bfloat16, "sin", 1024), (torch.float32, "relu", 1153)])
def test_large_tile_from_four_steps(dtype, act, K):
    """14 x 15 tiles of 256 x 256, ragged at both edges, four to ten steps of 128 values along the rows: two stages with one window
    of scales, windows moved back to the row's end, last stages that exist by half."""
    from nerf import mx
    M, N = 3400, 3601
    x, w, b, _ = training_case(M, K, N, "none", dtype)
    y = mx.linear(x, w, b, mx.ACTIVATIONS[act])
    check_forward(y, x, w, b, act, 1.0, 1.0)


@pytest.mark.parametrize("M, K, N", [(3400, 512, 3601), (3400, 650, 3601), (16400, 200, 250), (16387, 70, 33), (300, 200, 75), (4000, 900, 2200)])
def test_relu_masks_of_every_tile(M, K, N):
    """Mixed decisions: the gradient is open exactly where y > 0 (column sums of ones: whole numbers, exact)."""
    from nerf import mx
    x, w = randn(M, K, seed=35), randn(N, K, seed=36)
    b = torch.zeros(N, device=DEV, requires_grad=True)
    y = mx.linear(x, w, b, mx.ACT_RELU)
    (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
    assert torch.equal(db, (y > 0).float().sum(0)) and 0 < float(db.min()) and float(db.max()) < M


def test_training_relu_through_the_large_tile():
    x, w, b, dy = training_case(3400, 512, 3601, "relu", torch.float32)
    y, grads = run_training(x, w, b, dy, "relu", 0.5, 3.0)
    check_forward(y, x, w, b, "relu", 0.5, 3.0)
    check_backward(grads, dy, x, w, b, "relu", 0.5, 3.0, torch.float32)


# ---------------------------------------------------------------------------------------------------------------- layouts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K, N", [(1, 1000, 40), (13, 500, 40), (40, 4100, 300), (300, 319, 257), (16400, 200, 40), (3400, 650, 3601)])
def test_what_lies_between_rows_is_not_read(dtype, M, K, N):
    """x with NaN between its rows, at an odd address, in every way to multiply and in the rounding."""
    from nerf import mx
    x, w = randn(M, K, seed=1, dtype=dtype), randn(N, K, seed=2, dtype=dtype)
    buf = torch.full((M * (K + 7) + 3,), float("nan"), dtype=dtype, device=DEV)
    rows = buf[3:].view(M, K + 7)
    rows[:, :K] = x
    q = mx.quantize(w)
    assert torch.equal(mx.linear(rows[:, :K], q), mx.linear(x, q))
    a, c = mx.quantize(rows[:, :K]), mx.quantize(x)
    assert torch.equal(a.codes, c.codes) and torch.equal(a.scales, c.scales)
    part = slice(N // 3, N)     # some of the rows of a packed weight are packed rows
    some = mx.MXTensor(q.codes[part], q.scales[part], K)
    want = mx.linear(x, mx.quantize(w[part]))
    assert torch.equal(mx.linear(x, some), want) and torch.equal(mx.dequantize(some), mx.dequantize(q)[part])


# ------------------------------------------------------------------------------------------------------------ data parallel
@pytest.mark.parametrize("tag", ["nerf", "siren"])
def test_flat_bucket_holds_the_mean_over_ranks(tag, monkeypatch):
    """Data-parallel training in the mxfp4 mode: the layers' gradients land in the flat bucket that the ranks reduce.  Two
    ranks' halves of a batch, one after the other in this process; the collective is replaced by their sum."""
    from nerf import parallel
    from nerf.models import NeRF, Siren
    from nerf.rendering import render_nerf
    torch.manual_seed(7)
    model = {"nerf": NeRF, "siren": Siren}[tag]().to(DEV).set_training_precision("mxfp4")
    if tag == "nerf":      # some density everywhere: an empty volume has no gradients
        with torch.no_grad():
            model.block2[-1].bias[model.hidden_dim] = 1.0
    R, S = 64, 32
    o, d = randn(R, 3, seed=5), torch.nn.functional.normalize(randn(R, 3, seed=6), dim=1)
    tgt = torch.rand(R, 3, device=DEV, generator=torch.Generator(DEV).manual_seed(2))
    u = torch.rand(S, device=DEV, generator=torch.Generator(DEV).manual_seed(1))

    def loss(sl):
        rgb = render_nerf(model, o[sl], d[sl], 2.0, 6.0, num_samples=S, device=DEV, u=[u])
        return torch.nn.functional.mse_loss(rgb, tgt[sl])

    shards = [parallel.shard_slice(R, r, 2) for r in range(2)]
    want = [torch.cat([g.reshape(-1) for g in torch.autograd.grad(loss(sl), list(model.parameters()))]) for sl in shards]
    assert float(want[0].norm()) > 0 and not torch.equal(want[0], want[1])
    flat = parallel.FlatParameters(model)
    buckets = []
    for sl in shards:
        flat.zero_grad()
        loss(sl).backward()
        buckets.append(flat.grad.clone())
    monkeypatch.setattr(parallel, "world", lambda: (0, 2))
    monkeypatch.setattr(parallel.dist, "all_reduce", lambda t, op=None: t.copy_(buckets[0] + buckets[1]))
    flat.all_reduce_mean()
    mean = (want[0].double() + want[1].double()) / 2
    # the same shard twice: the kernels' sums are the same, those that atomics may reorder differ by their rounding
    assert float((flat.grad.double() - mean).norm() / mean.norm()) < 1e-6
    opt, before = parallel.FusedAdam(flat, lr=5e-4), flat.flat.clone()
    opt.step()
    assert not torch.equal(flat.flat, before) and all(p.data_ptr() >= flat.flat.data_ptr() for p in model.parameters())


# ---------------------------------------------------------------------------------------------------- the ends of the sizes
def whole(*shape, seed):
    """-1, 0 and 1: exact in every block, and sums of up to 2^24 of their products are exact in fp32 in any order."""
    g = torch.Generator(DEV).manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device=DEV, dtype=torch.int8).float()


def product64(a, b):
    """a [m,k] b [n,k]^T in float64, a piece of k at a time."""
    out = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device=DEV)
    for k in range(0, a.shape[1], 1 << 18):
        out += a[:, k:k + (1 << 18)].double() @ b[:, k:k + (1 << 18)].double().t().contiguous()
    return out


@pytest.mark.parametrize("M, K, N", [(3, 1 << 22, 17), (40, 1 << 22, 17), (40, (1 << 22) - 129, 9)])
def test_longest_rows(M, K, N):
    x, w, b, dy = whole(M, K, seed=1), whole(N, K, seed=2), whole(N, seed=3), whole(M, N, seed=4)
    y, (dx, dw, db) = run_training(x, w, b, dy, "none")
    assert torch.equal(y.double(), product64(x, w) + b.double())
    assert torch.equal(dx, dy @ w) and torch.equal(dw, dy.t().contiguous() @ x) and torch.equal(db, dy.sum(0))


def test_most_rows_of_a_weight():
    from nerf import mx
    for M, K, N in ((1, 40, 1 << 22), (130, 40, 1 << 22)):
        x, w = whole(M, K, seed=1), whole(N, K, seed=2)
        y = mx.linear(x, w)
        for n in range(0, N, 1 << 20):
            assert torch.equal(y[:, n:n + (1 << 20)], x @ w[n:n + (1 << 20)].t().contiguous())
        del y
    M, K, N = 5, 33, 65535 * 64
    x, w, b, dy = whole(M, K, seed=1), whole(N, K, seed=2), whole(N, seed=3), whole(M, N, seed=4)
    y, (dx, dw, db) = run_training(x, w, b, dy, "none")
    assert torch.equal(y, x @ w.t().contiguous() + b) and torch.equal(dx.double(), product64(dy, w.t().contiguous()))
    assert torch.equal(dw, dy.t().contiguous() @ x) and torch.equal(db, dy.sum(0))


def test_most_rows():
    """2^28 - 16 rows: rounded, read back and multiplied."""
    from nerf import mx
    rows = 268435440
    x = whole(rows, 1, seed=1)
    q = mx.quantize(x)
    assert torch.equal(mx.dequantize(q), x)
    del q
    w, b = torch.full((1, 1), 2.0, device=DEV), torch.ones(1, device=DEV)
    y = mx.linear(x, w, b, mx.ACT_RELU)
    assert torch.equal(y, torch.relu(2 * x + 1))


# ------------------------------------------------------------------------------------------------------------- calls in turn
@pytest.mark.parametrize("act", ACTS)
def test_backward_twice_and_after_other_calls(act):
    """What a forward keeps is its own: other layers' calls in between and a second backward change nothing."""
    from nerf import mx
    cases = [training_case(M, K, N, act, torch.float32) for M, K, N in ((30, 200, 72), (700, 200, 72), (4200, 200, 72))]
    want = [run_training(*c, act) for c in cases]
    runs = []
    for x, w, b, dy in cases:
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        runs.append((mx.linear(*leaves, mx.ACTIVATIONS[act]), leaves, dy))
    for _ in range(2):
        for (y, leaves, dy), (wy, wg) in list(zip(runs, want))[::-1]:
            got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            assert torch.equal(y, wy) and all(torch.equal(a, c) for a, c in zip(got, wg))


def test_two_threads():
    """Two host threads, each on a stream of its own."""
    import threading
    cases = [training_case(M, K, N, "sin", torch.float32) for M, K, N in ((20, 300, 72), (700, 256, 256), (5000, 200, 72), (3400, 300, 3601))]
    want = [run_training(*c, "sin") for c in cases]
    torch.cuda.synchronize()
    results = {}

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            results[k] = [[run_training(*c, "sin") for c in cases[::1 if k else -1]][::1 if k else -1] for _ in range(3)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k in range(2):
        for run in results[k]:
            for a, c in zip(run, want):
                assert torch.equal(a[0], c[0]) and all(torch.equal(g, h) for g, h in zip(a[1], c[1]))


@pytest.mark.parametrize("tag", ["nerf", "siren"])
def test_gradients_of_the_points_alone(tag):
    """A frozen network in the mxfp4 mode: the same outputs as without gradients, and d out / d points from the layers' dx."""
    from nerf.models import NeRF, Siren
    torch.manual_seed(3)
    model = {"nerf": NeRF, "siren": Siren}[tag]().to(DEV).set_inference_precision("mxfp4")
    if tag == "nerf":
        with torch.no_grad():
            model.block2[-1].bias[model.hidden_dim] = 1.0
    model.requires_grad_(False)
    pts, dirs = randn(5000, 3, seed=1, scale=0.4), torch.nn.functional.normalize(randn(5000, 3, seed=2), dim=1)
    with torch.no_grad():
        c, d = model(pts, dirs)
    leaf = pts.clone().requires_grad_(True)
    ce, de = model(leaf, dirs)
    assert torch.equal(c, ce) and torch.equal(d, de)
    (g,) = torch.autograd.grad(ce.sum() + de.sum(), leaf)
    assert torch.isfinite(g).all() and float(g.abs().max()) > 0
