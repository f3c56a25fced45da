"""ops.linear_cross_entropy (csrc/linear_xent.hip) against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0") if torch.cuda.is_available() else None
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24


def _case(n, v, d, dtype, bias=True, ignored=0.2, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, d, generator=g) * (2.0 * spread / math.sqrt(d))).to(dtype)
    x = torch.randn(n, d, generator=g).to(dtype)
    b = torch.randn(v, generator=g).to(dtype) if bias else None
    t = torch.randint(0, v, (n,), generator=g)
    t = torch.where(torch.rand(n, generator=g) < ignored, torch.full_like(t, -100), t)
    return x, w, b, t


def _formula(x, w, b, t, reduction, up, ignore=-100):
    """Loss, gradients and a bound for each of their elements, all in 64 bits.

    Logits: exact products of the inputs added in fp32, d + 1 roundings of at most 2^-24 of the sum of magnitudes A (for fp32 inputs the
    split's dropped terms add 3 * 2^-25 A and there are six sums: 7 (d + 1) + 2 in all is above it).  exp: relative error of the argument's error
    plus 2^-24 (|argument| + 4) of its own rounding.  d g / max |g| is rounded to the operand type (half a step; fp16's are stored times 2^14,
    so their subnormal half step is 2^-25 / 2^14; fp32 is split to 2^-25).  A gradient is a sum of K products in fp32: K roundings of 2^-24 of the sum
    of magnitudes (six sums for fp32 inputs), a few more of the scales, and the rounding to its type."""
    X, W = x.double(), w.double()
    n, d = X.shape
    v = W.shape[0]
    wide = x.dtype == torch.float32
    sums = 7 if wide else 1
    z = X @ W.t() + (0 if b is None else b.double())
    A = X.abs() @ W.abs().t() + (0 if b is None else b.double().abs().nan_to_num(posinf=0.0))
    ez = A * (sums * (d + 1) + 2) * U32
    lse = torch.logsumexp(z, dim=1)
    kept = t != ignore
    at = torch.where(kept, t, torch.zeros_like(t))
    zt = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(kept, lse - zt, torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    # lse moves by at most the probability-weighted logit errors; its own sums, exp and log round relative to the sum (v + 4 roundings)
    spread = (z - z.max(dim=1, keepdim=True).values).clamp(min=-110).abs()
    e_lse = (p * (ez + (spread + 4) * U32)).sum(dim=1) + (v / 64 + 40) * U32 + lse.abs() * 2 * U32
    e_loss = torch.where(kept, e_lse + ez.gather(1, at[:, None])[:, 0] + (lse.abs() + zt.abs()) * 2 * U32, torch.zeros_like(lse))
    count = kept.sum().double()
    if reduction == "none":
        out, e_out = loss, e_loss
        g = up.double()
    elif reduction == "sum":
        out, e_out = loss.sum(), e_loss.sum() + loss.abs().sum() * 2 * U32
        g = up.double().expand(n)
    else:
        out, e_out = loss.sum() / count, e_loss.sum() / count + loss.abs().sum() / count * 2 * U32
        g = (up.double() / count).expand(n)
    g = torch.where(kept, g, torch.zeros_like(g))
    D = p.clone()
    D[torch.arange(n, device=D.device), at] -= 1.0
    D[~kept] = 0
    half = torch.finfo(x.dtype).eps / 2 if not wide else 2.0 ** -25
    tiny = 2.0 ** -39 if x.dtype == torch.float16 else 2.0 ** -130
    e_d = p * (ez + e_lse[:, None] + ((z - lse[:, None]).abs().clamp(max=110) + 6) * U32) + D.abs() * (half + 4 * U32)
    e_dg = e_d * g.abs()[:, None] + (D * g[:, None]).abs() * 4 * U32 + tiny * g.abs().max()
    e_dg[~kept] = 0
    final = torch.finfo(x.dtype).eps / 2
    ftiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}[x.dtype]
    DG = D * g[:, None]
    dx, dw, db = DG @ W, DG.t() @ X, DG.sum(dim=0)
    b_dx = e_dg @ W.abs() + DG.abs() @ W.abs() * (sums * (v + 2) + 8) * U32 + dx.abs() * final * 1.01 + ftiny
    b_dw = e_dg.t() @ X.abs() + DG.t().abs() @ X.abs() * (sums * (n + 2) + 8) * U32 + dw.abs() * final * 1.01 + ftiny
    b_db = e_dg.sum(dim=0) + DG.abs().sum(dim=0) * (n + 8) * U32 + db.abs() * final * 1.01 + ftiny
    return (out, dx, dw, db), (e_out * 1.01, b_dx * 1.01, b_dw * 1.01, b_db * 1.01)


def _run(x, w, b, t, reduction, up, piece=0):
    from phc_gnn_amd import ops
    xs, ws, bs = (None if q is None else q.to(DEV).detach().requires_grad_() for q in (x, w, b))
    loss = ops.linear_cross_entropy(xs, ws, t.to(DEV), bias=bs, reduction=reduction, piece=piece)
    grads = torch.autograd.grad(loss, [q for q in (xs, ws, bs) if q is not None], up.to(DEV))
    return (loss.detach(), *grads)


def _check(n, v, d, dtype, bias=True, reduction="mean", ignored=0.2, piece=0, seed=0, spread=1.0):
    x, w, b, t = _case(n, v, d, dtype, bias, ignored, seed, spread)
    if reduction == "mean" and not bool((t != -100).any()):
        t[0] = v - 1
    g = torch.Generator().manual_seed(seed + 99)
    up = torch.randn(n, generator=g) if reduction == "none" else torch.tensor(1.0 if reduction == "mean" else -0.5)
    exact, bound = _formula(x, w, b, t, reduction, up)
    got = _run(x, w, b, t, reduction, up, piece)
    for what, a, e, m in zip(("loss", "dx", "dW", "db"), got, exact, bound):
        err = (a.cpu().double() - e).abs()
        assert a.dtype == (torch.float32 if what == "loss" else dtype)
        assert bool((err <= m).all()), (what, float(err.max()), float((err / m).max()))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 2, 3), (2, 17, 8), (5, 1000, 64), (1, 5003, 72), (63, 127, 65), (64, 128, 64), (65, 129, 128),
                                   (130, 300, 7), (129, 257, 200), (257, 1000, 180), (300, 40, 260), (16, 4099, 64), (17, 4100, 128)])
def test_loss_and_gradients(n, v, d, dtype):
    _check(n, v, d, dtype, bias=n % 2 == 1, reduction=("mean", "sum", "none")[(n + v + d) % 3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("piece", [64, 200, 256])
def test_vocabulary_in_pieces(piece, reduction, dtype):
    """Pieces that end inside a tile and a last one that is nearly empty."""
    _check(150, 513, 96, dtype, reduction=reduction, piece=piece, seed=3)
    _check(70, 449, 64, dtype, reduction=reduction, piece=piece, seed=4, bias=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(1100, 2500, 320), (640, 3001, 576), (2000, 700, 136)])
def test_more_tiles_and_splits(n, v, d, dtype):
    _check(n, v, d, dtype, reduction="mean", ignored=0.05, seed=7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(40, 66003, 64), (150, 33100, 300), (256, 50000, 70), (33100, 150, 300), (2700, 7000, 130)])
def test_more_tiles_than_the_card_holds(n, v, d, dtype):
    """More output tiles than workgroups fit at once, in each of the products (256 of the large tiles, 512 of the small ones).  The formula
    and its bounds on the GPU, in 64 bits."""
    x, w, b, t = (q.to(DEV) for q in _case(n, v, d, dtype, seed=9))
    up = torch.tensor(1.0, device=DEV)
    exact, bound = _formula(x, w, b, t, "mean", up)
    for what, a, e, m in zip(("loss", "dx", "dW", "db"), _run(x, w, b, t, "mean", up), exact, bound):
        err = (a.double() - e).abs()
        assert bool((err <= m).all()), (what, float(err.max()), float((err / m).max()))


@pytest.mark.parametrize("dtype", TYPES)
def test_sharp_and_flat_distributions(dtype):
    """Logits of +-100 (all exponentials but one underflow) and of nearly 0."""
    _check(90, 600, 64, dtype, spread=20.0, reduction="sum", seed=5)
    _check(90, 600, 64, dtype, spread=1e-3, bias=False, reduction="sum", seed=6)


def test_rows_that_do_not_count():
    from phc_gnn_amd import ops
    for dtype in TYPES:
        x, w, b, t = _case(70, 300, 64, dtype)
        t[:] = -100
        loss, dx, dw, db = _run(x, w, b, t, "mean", torch.tensor(1.0))
        assert math.isnan(float(loss))
        assert all(int(torch.count_nonzero(q)) == 0 for q in (dx, dw, db))
        loss, dx, dw, db = _run(x, w, b, t, "sum", torch.tensor(1.0))
        assert float(loss) == 0.0 and all(int(torch.count_nonzero(q)) == 0 for q in (dx, dw, db))
        # what lies in such rows does not matter: the others' results are the same bits
        x, w, b, t = _case(70, 300, 64, dtype, ignored=0.4, seed=2)
        want = _run(x, w, b, t, "mean", torch.tensor(1.0))
        y = x.clone()
        y[t == -100] = float("nan")
        y[int((t == -100).nonzero()[0])] = float("inf")
        got = _run(y, w, b, t, "mean", torch.tensor(1.0))
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        xs = torch.zeros(0, 64, dtype=dtype, device=DEV, requires_grad=True)
        ws = w.to(DEV).requires_grad_()
        none = torch.zeros(0, dtype=torch.int64, device=DEV)
        assert math.isnan(float(ops.linear_cross_entropy(xs, ws, none)))
        assert tuple(ops.linear_cross_entropy(xs, ws, none, reduction="none").shape) == (0,)
        loss = ops.linear_cross_entropy(xs, ws, none, reduction="sum")
        loss.backward()
        assert float(loss) == 0.0 and tuple(xs.grad.shape) == (0, 64) and int(torch.count_nonzero(ws.grad)) == 0


def test_other_ignore_index():
    from phc_gnn_amd import ops
    x, w, b, t = _case(40, 50, 32, torch.float32, ignored=0.0)
    t[::3] = 7
    got = ops.linear_cross_entropy(x.to(DEV), w.to(DEV), t.to(DEV), ignore_index=7, reduction="none")
    assert int(torch.count_nonzero(got[::3])) == 0 and bool((got[t.to(DEV) != 7] > 0).all())


def test_columns_taken_out_by_their_bias():
    """A bias of -inf (and of the type's lowest value): probability 0, gradient 0, whole tiles of them too."""
    for dtype in TYPES:
        for low in (-math.inf, torch.finfo(dtype).min):
            x, w, b, t = _case(50, 700, 64, dtype, ignored=0.1, seed=11)
            b[130:420] = low
            b[600:] = low
            t = torch.where((t >= 130) & (t < 420) | (t >= 600), t % 100, t)
            t = torch.where(t < -100, torch.full_like(t, -100), t)
            loss, dx, dw, db = _run(x, w, b, t, "mean", torch.tensor(1.0))
            keep = torch.cat([torch.arange(130), torch.arange(420, 600)])
            place = torch.full((700,), -1)
            place[keep] = torch.arange(len(keep))
            t2 = torch.where(t == -100, t, place[t.clamp(min=0)])
            (e, ex, ew, eb), (m, mx, mw, mb) = _formula(x, w[keep], b[keep], t2, "mean", torch.tensor(1.0))
            assert abs(float(loss) - float(e)) <= float(m)
            assert bool(((dx.cpu().double() - ex).abs() <= mx).all())
            assert bool(((dw.cpu().double()[keep] - ew).abs() <= mw).all()) and bool(((db.cpu().double()[keep] - eb).abs() <= mb).all())
            gone = torch.ones(700, dtype=torch.bool)
            gone[keep] = False
            assert int(torch.count_nonzero(dw.cpu()[gone])) == 0 and int(torch.count_nonzero(db.cpu()[gone])) == 0


def test_target_in_a_column_taken_out():
    x, w, b, t = _case(10, 200, 64, torch.float32, ignored=0.0)
    b[5] = -math.inf
    t[3] = 5
    loss, dx, dw, db = _run(x, w, b, t, "none", torch.ones(10))
    assert float(loss[3]) == math.inf and bool(loss[torch.arange(10) != 3].isfinite().all())
    assert bool(dx.isfinite().all()) and bool(dw.isfinite().all())              # p - 1 = -1 in that column


def test_logits_that_are_not_finite_stay_in_their_rows():
    for dtype in (torch.bfloat16, torch.float16):
        x, w, b, t = _case(40, 300, 64, dtype, ignored=0.0, seed=13)
        want = _run(x, w, b, t, "none", torch.ones(40))
        y = x.clone()
        y[7, 3] = math.inf
        y[9, 0] = math.nan
        got = _run(y, w, b, t, "none", torch.ones(40))
        rest = torch.ones(40, dtype=torch.bool)
        rest[[7, 9]] = False
        assert torch.equal(want[0].cpu()[rest], got[0].cpu()[rest]) and torch.equal(want[1].cpu()[rest], got[1].cpu()[rest])
        assert bool(got[0].cpu()[~rest].isnan().all())


def test_bad_targets_count_as_zero_and_are_reported():
    from phc_gnn_amd import check_indices, ops
    x, w, b, t = _case(30, 100, 64, torch.float32, ignored=0.0)
    ok = t.clone()
    for i, bad in ((0, 100), (5, -1), (29, 1 << 40)):
        t[i] = bad
        ok[i] = 0
    got = ops.linear_cross_entropy(x.to(DEV), w.to(DEV), t.to(DEV), reduction="none")
    with pytest.raises(IndexError, match="target outside"):
        check_indices(DEV)
    want = ops.linear_cross_entropy(x.to(DEV), w.to(DEV), ok.to(DEV), reduction="none")
    check_indices(DEV)
    assert torch.equal(got, want)
    a, b_ = _run(x, w, b, t, "mean", torch.tensor(1.0)), _run(x, w, b, ok, "mean", torch.tensor(1.0))
    with pytest.raises(IndexError):
        check_indices(DEV)
    assert all(torch.equal(p, q) for p, q in zip(a, b_))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_alignment_and_shapes(dtype):
    from phc_gnn_amd import ops
    g = torch.Generator().manual_seed(1)
    xb, wb = torch.randn(4, 9, 150, generator=g).to(dtype).to(DEV), torch.randn(203, 150, generator=g).to(dtype).to(DEV)
    t = torch.randint(0, 200, (4, 9), generator=g).to(DEV)
    for lo, d in ((0, 64), (8, 64), (3, 64), (1, 128), (16, 128), (2, 70)):
        xs, ws = xb[..., lo:lo + d].detach().requires_grad_(), wb[:200, lo:lo + d].detach().requires_grad_()
        loss = ops.linear_cross_entropy(xs, ws, t.to(torch.int32), reduction="none")
        assert tuple(loss.shape) == (4, 9)
        up = torch.rand(4, 9, generator=g).to(DEV)
        got = (loss.detach(), *torch.autograd.grad(loss, [xs, ws], up))
        xc, wc = xs.detach().reshape(36, d).clone().requires_grad_(), ws.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        ref = ops.linear_cross_entropy(xc, wc, t.reshape(-1), reduction="none")
        want = (ref.detach(), *torch.autograd.grad(ref, [xc, wc], up.reshape(-1)))
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want)), (lo, d)
    # rows in another order in memory, one row repeated for all, a scalar target
    xt = torch.randn(64, 20, device=DEV).to(dtype).t()
    assert torch.equal(ops.linear_cross_entropy(xt, wb[:, :64], t.reshape(-1)[:20]), ops.linear_cross_entropy(xt.contiguous(), wb[:, :64], t.reshape(-1)[:20]))
    one = xb[0, 0, :64]
    rep = ops.linear_cross_entropy(one.expand(5, 64), wb[:, :64], t.reshape(-1)[:5], reduction="none")
    assert torch.equal(rep, torch.stack([ops.linear_cross_entropy(one, wb[:, :64], t.reshape(-1)[i], reduction="none") for i in range(5)]))


def test_gradient_of_a_part_only():
    from phc_gnn_amd import ops
    x, w, b, t = (q.to(DEV) for q in _case(60, 300, 64, torch.bfloat16, seed=21))
    full = _run(x, w, b, t, "mean", torch.tensor(1.0))
    for k in range(3):
        leaves = [q.detach().clone().requires_grad_(i == k) for i, q in enumerate((x, w, b))]
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        (g,) = torch.autograd.grad(loss, [leaves[k]])
        assert torch.equal(g, full[1 + k])
    assert not ops.linear_cross_entropy(x, w, t, bias=b).requires_grad


def test_large_upstream_gradients_of_fp16():
    """A scaled loss: the gradients of 16-bit inputs are not lost below the type's range, and scale exactly with powers of two."""
    x, w, b, t = _case(200, 900, 64, torch.float16, seed=8)
    a = _run(x, w, b, t, "mean", torch.tensor(1024.0))
    c = _run(x, w, b, t, "mean", torch.tensor(4096.0))
    for p, q in zip(a[1:], c[1:]):
        normal = p.abs() >= 2.0 ** -14
        assert bool(normal.any()) and torch.equal(p[normal].float() * 4, q[normal].float())


def test_against_differences():
    """Along a direction the loss's derivative is <gradient, direction>.  The central difference is off by h^2 / 6 times the third
    derivative, at most (2 a_i)^3 for a row whose logits move by at most a_i, plus the forward's bound twice over 2h."""
    from phc_gnn_amd import ops
    x, w, b, t = _case(40, 200, 64, torch.float32, seed=17)
    up = torch.tensor(1.0)
    (_, *_), (m, *_) = _formula(x, w, b, t, "sum", up)
    _, dx, dw, db = _run(x, w, b, t, "sum", up)
    g = torch.Generator().manual_seed(2)
    h = 2.0 ** -5
    for which, grad, base in (("x", dx, x), ("w", dw, w), ("b", db, b)):
        v = torch.randn(base.shape, generator=g) / math.sqrt(base.shape[-1] if which != "b" else 1.0)
        moved = {"x": lambda s: (x + s * v, w, b), "w": lambda s: (x, w + s * v, b), "b": lambda s: (x, w, b + s * v)}[which]
        ends = []
        for s in (h, -h):
            xx, ww, bb = (q.to(DEV) for q in moved(s))
            ends.append(float(ops.linear_cross_entropy(xx, ww, t.to(DEV), bias=bb, reduction="sum").double()))
        diff = (ends[0] - ends[1]) / (2 * h)
        dz = {"x": lambda: v.double() @ w.double().t(), "w": lambda: x.double() @ v.double().t(), "b": lambda: v.double().expand(40, 200)}[which]()
        a = dz.abs().max(dim=1).values
        kept = t != -100
        # (the moved inputs are themselves rounded: half a step of 2^-24 of |value| each, over 2h)
        moved_by = {"x": lambda: (x.double().abs() + v.abs() * h) @ w.double().abs().t(), "w": lambda: x.double().abs() @ (w.double().abs() + v.abs() * h).t(),
                    "b": lambda: (b.double().abs() + v.abs() * h).expand(40, 200)}[which]().max(dim=1).values * U32
        slack = float(((2 * a) ** 3 * h * h / 6)[kept].sum() + 2 * (float(m) + 4 * float(moved_by[kept].sum())) / (2 * h))
        inner = float((grad.cpu().double() * v.double()).sum())
        assert abs(diff - inner) <= slack + abs(inner) * 1e-5, (which, diff, inner, slack)
        assert slack < 0.2 * float((grad.cpu().double().norm() * v.double().norm())), (which, slack)       # (the test says something)


def test_bitwise_reproducible():
    for dtype in TYPES:
        x, w, b, t = _case(300, 1500, 192, dtype, seed=31)
        want = _run(x, w, b, t, "mean", torch.tensor(1.0))
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(want, _run(x, w, b, t, "mean", torch.tensor(1.0))))


def test_graph_replay_and_streams():
    from phc_gnn_amd import ops
    x, w, b, t = (q.to(DEV) for q in _case(200, 1100, 128, torch.bfloat16, seed=41))
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()

    def step():
        loss = ops.linear_cross_entropy(x, w, t, bias=b, piece=384)
        return (loss.detach(), *torch.autograd.grad(loss, [x, w, b]))
    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cap = step()
    s.synchronize()
    for k in range(4):
        with torch.no_grad():
            x.mul_(1.25)
            w.add_(0.01)
            t.copy_(torch.roll(t, 3))
        want = step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(cap, want)), k


def test_two_streams_at_once():
    from phc_gnn_amd import ops
    cases = []
    for k in range(2):
        x, w, b, t = (q.to(DEV) for q in _case(300, 2000, 128, torch.bfloat16, seed=50 + k))
        x.requires_grad_(), w.requires_grad_()
        cases.append((x, w, b, t, torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b), [x, w])))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(4):
        for k, (x, w, b, t, _) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b), [x, w]))
    torch.cuda.synchronize()
    for (*_, want), gs in zip(cases, got):
        assert all(torch.equal(p, q) for pair in gs for p, q in zip(want, pair))


def test_changed_inputs_are_noticed():
    from phc_gnn_amd import ops
    x, w, b, t = (q.to(DEV) for q in _case(20, 100, 64, torch.float32))
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_embedding_loss_and_clipping_together():
    """One step as they are used: tokens -> embedding -> PHM layer -> loss against the same (tied) table -> clipped gradients -> Adam.
    Gradients against autograd of the same step in 64 bits."""
    from phc.hypercomplex.layers import PHMLinear
    from phc_gnn_amd import ops, optim
    torch.manual_seed(0)
    v, d, n = 601, 64, 300
    table = torch.nn.Parameter((torch.randn(v, d) * 0.2).to(DEV))
    lin = PHMLinear(d, d, phm_dim=4).to(DEV)
    params = [table, *lin.parameters()]
    opt = torch.optim.Adam(params, lr=1e-3)
    tokens, target = torch.randint(0, v, (n,)), torch.randint(0, v, (n,))
    target[::7] = -100
    for step in range(3):
        before = [p.detach().cpu().double().requires_grad_() for p in params]
        opt.zero_grad(set_to_none=True)
        h = lin(ops.embedding(tokens.to(DEV), table, scale=8.0))
        loss = ops.linear_cross_entropy(h, table, target.to(DEV))
        loss.backward()
        names = dict(zip(["table"] + [k for k, _ in lin.named_parameters()], before))
        H = torch.einsum("iac,ikp->akcp", names["phm_rule"], names["W"]).reshape(d, d)
        logits = (names["table"][tokens] * 8.0 @ H + names["b"]) @ names["table"].t()
        ref = torch.nn.functional.cross_entropy(logits, target, ignore_index=-100)
        grads = torch.autograd.grad(ref, before)
        # sums of at most 601 products in fp32 chained three deep: 3 * 601 * 2^-24 of the largest magnitude is above 1e-4
        assert abs(float(loss.detach()) - float(ref)) <= 1e-4 * abs(float(ref))
        for p, g in zip(params, grads):
            assert float((p.grad.cpu().double() - g).abs().max()) <= 2e-4 * float(g.abs().max())
        norm = optim.clip_grad_norm_(params, 0.05)
        want = math.sqrt(sum(float(g.pow(2).sum()) for g in grads))
        assert abs(float(norm) - want) <= 2e-4 * want and want > 0.05
        assert abs(float(optim.grad_norm([p.grad for p in params])) - 0.05) <= 1e-5 * 0.05 + 0.05 * 1e-6 / want * 1.01
        opt.step()
    from phc_gnn_amd import check_indices
    check_indices(DEV)


def test_more_tiles_than_a_line_of_the_launch():
    """2^21 tiles of 256 x 256 and more: the launch is laid out in two dimensions.  |x . w| <= 8 * 3 * 3 (clipped), accumulated in fp32 over
    8 terms: an error of at most 8 * 72 * 2^-24 = 3.5e-5 in a logit, in the target's and, weighted, in the logarithm's.  Three more
    roundings at that size (l - max, max + log, the loss: 3 * 72 * 2^-24 = 1.3e-5) and the sum (below 100 additions to a term, an
    exponential of 2^-20: 0.7e-5) stay below 2^-15."""
    from phc_gnn_amd import ops
    n, v, d = (1 << 19) + 300, (1 << 18) + 77, 8
    x = torch.randn(n, d, device=DEV).clamp_(-3, 3).bfloat16()
    w = torch.randn(v, d, device=DEV).clamp_(-3, 3).bfloat16()
    t = torch.randint(0, v, (n,), device=DEV)
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    for rows in (torch.arange(0, 40), torch.arange(n // 2, n // 2 + 40), torch.arange(n - 40, n)):
        rows = rows.to(DEV)
        logits = x[rows].double() @ w.double().T
        want = torch.logsumexp(logits, 1) - logits.gather(1, t[rows][:, None])[:, 0]
        assert float((loss[rows].double() - want).abs().max()) <= 2 * 3.5e-5 + 2.0 ** -15


def test_no_row_counts_whatever_the_upstream_gradient():
    from phc_gnn_amd import ops
    for n in (3, 100):
        x = torch.randn(n, 16, device=DEV, requires_grad=True)
        w = torch.randn(50, 16, device=DEV, requires_grad=True)
        b = torch.zeros(50, device=DEV, requires_grad=True)
        t = torch.full((n,), -100, device=DEV)
        for reduction in ("mean", "sum"):
            loss = ops.linear_cross_entropy(x, w, t, b, reduction=reduction)
            for g in torch.autograd.grad(loss, [x, w, b], torch.tensor(float("inf"), device=DEV)):
                assert float(g.abs().max()) == 0.0


def test_capture_beside_a_live_eager_graph_of_x_is_refused():
    """x is flattened on the way: its gradient node stands behind a view."""
    from phc_gnn_amd import ops
    from phc_gnn_amd.lib import PhcError
    x = torch.randn(2, 70, 8, device=DEV, requires_grad=True)
    w = torch.randn(40, 8, device=DEV)
    t = torch.randint(0, 40, (2, 70), device=DEV)
    alive = ops.linear_cross_entropy(x, w, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            with pytest.raises(PhcError, match="captured into a graph"):
                ops.linear_cross_entropy(x, w, t)
            out = ops.linear_cross_entropy(x.detach(), w, t)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive.detach())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(1, 33001, 129), (3, 32769, 1), (20, 40007, 67), (50, 35000, 33), (64, 70001, 31), (16, 5000, 255), (64, 3000, 513)])
def test_few_rows_of_odd_lengths(n, v, d, dtype):
    """Rows that begin at odd elements, alone and inside wider buffers (the last element of a buffer is the last of a row), and more columns than
    one round of the workgroups takes."""
    from phc_gnn_amd import ops
    x, w, b, t = (q.to(DEV) for q in _case(n, v, d, dtype, seed=11))
    for bias in (None, b):
        exact, bound = _formula(x, w, bias, t, "none", torch.ones(n, device=DEV))
        runs = []
        for pad in (0, 1, 2):
            xs = torch.zeros(n * (d + pad), device=DEV, dtype=dtype).view(n, d + pad)[:, pad:].copy_(x)
            ws = torch.zeros(v * (d + pad), device=DEV, dtype=dtype).view(v, d + pad)[:, pad:].copy_(w)
            runs.append(ops.linear_cross_entropy(xs, ws, t, bias, reduction="none"))
        assert all(torch.equal(r, runs[0]) for r in runs)
        err = (runs[0].double() - exact[0]).abs()
        assert bool((err <= bound[0]).all()), float((err / bound[0]).max())


def test_few_rows_with_groups_of_columns_taken_out():
    """Whole groups of columns at -inf, at the beginning, for one workgroup's every round, and for all but the last column."""
    from phc_gnn_amd import ops
    n, v, d = 30, 70000, 16
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(n, d, generator=g).to(DEV), torch.randn(v, d, generator=g).to(DEV)
    for kept in (torch.arange(64, v), torch.arange(v)[(torch.arange(v) // 64) % 512 != 3], torch.tensor([v - 1])):
        b = torch.full((v,), float("-inf"))
        b[kept] = 0.0
        b, k = b.to(DEV), kept.to(DEV)
        t = k[torch.arange(n, device=DEV) * 7 % len(kept)]
        got = ops.linear_cross_entropy(x, w, t, b, reduction="none")
        logits = x.double() @ w[k].double().T
        want = torch.logsumexp(logits, 1) - (x.double() * w[t].double()).sum(1)
        # 16 products in fp32 (4 steps of 4): 16 * 2^-24 of sum |x w| <= 40 here; 8 roundings at the logits' size in what follows
        bound = (16 + 8) * 2.0 ** -24 * (2 * (x.abs() @ w[k].abs().T).max().double() + 20)
        assert float((got.double() - want).abs().max()) <= float(bound)


def test_refusals_of_the_engine_are_phc_errors():
    from phc_gnn_amd import ops
    from phc_gnn_amd.lib import PhcError
    w = torch.zeros(1, (1 << 20) + 1, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    t = torch.zeros(1, device=DEV, dtype=torch.int64)
    with pytest.raises(PhcError, match="beyond"):
        ops.embedding(t, w)
    with pytest.raises(PhcError, match="beyond"):
        ops.linear_cross_entropy(w.detach(), w, t)


def test_leaves_of_any_shape_get_gradients_of_theirs():
    from phc_gnn_amd import ops
    x = torch.randn(2, 3, 16, device=DEV, requires_grad=True)
    w = torch.randn(40, 16, device=DEV, requires_grad=True)
    b = torch.zeros(40, device=DEV, requires_grad=True)
    t = torch.randint(0, 40, (2, 3), device=DEV)
    ops.linear_cross_entropy(x, w, t, b).backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape and b.grad.shape == b.shape
    flat = x.detach().reshape(6, 16).requires_grad_()
    got = torch.autograd.grad(ops.linear_cross_entropy(flat, w, t.reshape(-1), b), [flat, w, b])
    assert torch.equal(got[0].reshape(2, 3, 16), x.grad) and torch.equal(got[1], w.grad) and torch.equal(got[2], b.grad)
    v = torch.randn(16, device=DEV, requires_grad=True)                       # one row, no batch dimension; no bias
    (dv,) = torch.autograd.grad(ops.linear_cross_entropy(v, w, t[0, 0]), [v])
    assert dv.shape == v.shape
    p = torch.softmax(v.detach().double() @ w.detach().double().T, 0)
    p[t[0, 0]] -= 1
    # 16 products and 40 terms in fp32: below 100 roundings of 2^-24 at the size of |p| |w| sums (at most 2 * 5)
    assert float((dv.double() - p @ w.detach().double()).abs().max()) <= 100 * 2.0 ** -24 * 10


@pytest.mark.parametrize("kept", [0, 1, 63, 64, 65, 128, 129, 192, 193, 250])
def test_fp32_rows_that_count_choose_the_tile(kept):
    """fp32 on its own matrix instructions: the logits' tile size goes by the rows that count, known on the device alone."""
    n, v, d = 250, 12500, 40
    x, w, b, t = (q.to(DEV) for q in _case(n, v, d, torch.float32, ignored=0.0, seed=13))
    gone = torch.randperm(n, generator=torch.Generator().manual_seed(kept))[kept:].to(DEV)
    t = t.index_fill(0, gone, -100)
    up = torch.tensor(1.0, device=DEV)
    exact, bound = _formula(x, w, b, t, "sum", up)
    for piece in (0, 6300):
        for what, a, e, m in zip(("loss", "dx", "dW", "db"), _run(x, w, b, t, "sum", up, piece=piece), exact, bound):
            err = (a.double() - e).abs()
            assert bool((err <= m).all()), (what, float(err.max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(70, 300, 8), (150, 13000, 72), (300, 1000, 200), (129, 260, 344), (600, 26000, 136)])
def test_rows_of_w_inside_wider_ones(n, v, d, dtype):
    """W is read where it lies; what stands behind its rows' ends (NaN here) is not, nor is anything behind its last row."""
    x, w, b, t = (q.to(DEV) for q in _case(n, v, d, dtype, seed=17))
    up = torch.tensor(1.0, device=DEV)
    want = _run(x, w.clone(), b, t, "mean", up)
    for extra in (8, 64):
        buf = torch.full((v * (d + extra) - extra,), float("nan"), device=DEV, dtype=dtype)
        wide = torch.as_strided(buf, (v, d), (d + extra, 1))
        wide.copy_(w)
        from phc_gnn_amd import ops
        xs, bs = x.clone().requires_grad_(), b.clone().requires_grad_()
        ws = wide.requires_grad_()
        loss = ops.linear_cross_entropy(xs, ws, t, bs)
        got = (loss.detach(), *torch.autograd.grad(loss, [xs, ws, bs], up))
        assert all(torch.equal(a, e) for a, e in zip(got, want)), extra


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(1, 17, 700), (16, 8128, 40), (16, 8129, 40), (17, 2496, 40), (33, 2497, 40), (64, 15, 600), (64, 1000, 264)])
def test_few_rows_of_small_vocabularies(n, v, d, dtype):
    """Groups of 16 columns and of 64, and the sizes where one gives way to the other."""
    _check(n, v, d, dtype, bias=n % 2 == 1, reduction="none" if n > 16 else "sum", seed=19)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [12, 150, 300])
def test_an_infinite_upstream_gradient_stays_in_its_row(n, dtype):
    """dx_i = g_i sum_v d_iv w_v: an infinite or NaN g_i leaves the other rows' dx as they are with g_i = 0, to the bit.  dW and db have a
    term of it in every element."""
    x, w, b, t = _case(n, 500, 72, dtype, ignored=0.0, seed=23)
    t[4] = -100
    g = torch.Generator().manual_seed(24)
    up = torch.rand(n, generator=g) + 0.5
    bad = {7: math.inf, 9: -math.inf, 11: math.nan}
    up[list(bad)] = 0.0
    want = _run(x, w, b, t, "none", up)
    exact, bound = _formula(x, w, b, t, "none", up)
    for a, e, m in zip(want, exact, bound):
        assert bool(((a.cpu().double() - e).abs() <= m).all())
    for rows in ([7], [9], [7, 9, 11]):
        part = up.clone()
        for i in rows:
            part[i] = bad[i]
        part[4] = math.inf                                           # (a row that does not count)
        loss, dx, dw, db = _run(x, w, b, t, "none", part)
        rest = torch.ones(n, dtype=torch.bool)
        rest[rows] = False
        assert torch.equal(loss, want[0])
        assert torch.equal(dx.cpu()[rest], want[1].cpu()[rest])
        assert not bool(dx.cpu()[~rest].isfinite().any())
        assert not bool(dw.isfinite().any()) and not bool(db.isfinite().any())
    part = torch.zeros(n)                                            # no other row has a gradient
    part[7] = math.inf
    _, dx, dw, _ = _run(x, w, b, t, "none", part)
    rest = torch.arange(n) != 7
    assert int(torch.count_nonzero(dx.cpu()[rest])) == 0 and not bool(dx[7].isfinite().any()) and not bool(dw.isfinite().any())


def test_a_penalty_on_gradients_is_refused():
    """The gradients depend on x, weight and bias whatever the upstream gradient is: a second derivative that would leave their terms out is refused,
    also when the sum has other terms that autograd can go through."""
    from phc_gnn_amd import ops
    for n in (5, 90):
        x, w, b, t = (q.to(DEV) for q in _case(n, 60, 16, torch.float32, ignored=0.0))
        leaves = [q.requires_grad_() for q in (x, w, b)]
        plain = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b), leaves)
        for k in range(3):
            loss = ops.linear_cross_entropy(x, w, t, bias=b)
            grads = torch.autograd.grad(loss, leaves, create_graph=True)
            assert all(torch.equal(p, q.detach()) for p, q in zip(plain, grads))
            with pytest.raises(RuntimeError, match="once_differentiable"):
                (loss + grads[k].pow(2).sum()).backward()
        # only one of them asks for a gradient
        x1 = x.detach().requires_grad_()
        loss = ops.linear_cross_entropy(x1, w.detach(), t)
        (dx,) = torch.autograd.grad(loss, [x1], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (loss + dx.pow(2).sum()).backward()
        # a graph that is kept and not used again is no second derivative  (the refused call may have added its first term already)
        x1.grad = None
        ops.linear_cross_entropy(x1, w.detach(), t).backward(create_graph=True)
        assert torch.equal(x1.grad.detach(), dx.detach())
        x1.grad = None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [50, 150, 300])
def test_all_columns_as_one_piece(n, dtype):
    x, w, b, t = _case(n, 513, 96, dtype, seed=3)
    up = torch.tensor(1.0)
    want = _run(x, w, b, t, "mean", up, piece=513)
    for piece in (514, 1 << 40, (1 << 63) - 64, (1 << 63) - 1):
        assert all(torch.equal(p, q) for p, q in zip(want, _run(x, w, b, t, "mean", up, piece=piece))), piece


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [66, 150, 300])
@pytest.mark.parametrize("piece", [64, 200, 256, 1024])
def test_forward_in_pieces(piece, n, dtype):
    """Rows of W that are laid out anew (97 columns; fp32 of 300 rows): the forward's statistics are carried from piece to piece.  Targets in the
    first and last columns of pieces, whole pieces at -inf, one value that is far above all others in the first or the last piece."""
    from phc_gnn_amd import ops
    v = 1300
    _check(n, v, 97, dtype, bias=n % 4 == 0, reduction=("mean", "sum", "none")[n % 3], piece=piece, seed=29)
    x, w, b, t = _case(n, v, 97, dtype, ignored=0.1, seed=31)
    edges = torch.tensor([0, piece - 1, piece, v - 1, v - 2]).clamp(max=v - 1)
    t[:40] = edges[torch.arange(40) % 5]
    for at in (None, 0, v - 1):
        bias = b.clone()
        bias[piece + 1:min(3 * piece, v - 2)] = -math.inf
        if at is not None:
            bias[at] = 60.0
        keep = bias.isfinite().nonzero()[:, 0]
        place = torch.full((v,), -1)
        place[keep] = torch.arange(len(keep))
        t1 = torch.where((t >= 0) & ~bias.isfinite()[t.clamp(min=0)], torch.zeros_like(t), t)
        t2 = torch.where(t1 == -100, t1, place[t1.clamp(min=0)])
        (e, *_), (m, *_) = _formula(x, w[keep], bias[keep], t2, "none", torch.ones(n))
        got = ops.linear_cross_entropy(x.to(DEV), w.to(DEV), t1.to(DEV), bias=bias.to(DEV), reduction="none", piece=piece)
        err = (got.cpu().double() - e).abs()
        assert bool((err <= m).all()), float((err / m).max())


def test_forward_scratch_is_what_is_taken():
    """The memory a forward takes at its peak stays near half a GiB where the statistics or W's layout of the whole vocabulary would take several."""
    from phc_gnn_amd import ops
    for n, v, d, dtype, all_at_once in ((1 << 17, 1 << 19, 16, torch.bfloat16, 4 << 30), (300, 131072, 2049, torch.float32, 3 << 29)):
        x, w = torch.zeros(n, d, device=DEV, dtype=dtype), torch.zeros(v, d, device=DEV, dtype=dtype)
        t = torch.zeros(n, device=DEV, dtype=torch.int64)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = ops.linear_cross_entropy(x, w, t, reduction="none")
        torch.cuda.synchronize()
        taken = torch.cuda.max_memory_allocated() - before
        assert taken <= (640 << 20) < all_at_once
        # v equal logits: log v, an exact sum of ones (v is a power of two), one logarithm
        assert float((loss.double() - math.log(v)).abs().max()) <= 4 * U32 * math.log(v)
        del x, w, loss


@pytest.mark.parametrize("dtype", TYPES)
def test_pieces_that_the_layout_of_w_asks_for(dtype):
    """Rows of W that are laid out anew and fill the scratch before d does: several pieces in both directions without being asked for."""
    n, v, d = 300, 131072, 2049
    x, w, b, t = (q.to(DEV) for q in _case(n, v, d, dtype, seed=43))
    up = torch.tensor(1.0, device=DEV)
    exact, bound = _formula(x, w, b, t, "mean", up)
    for what, a, e, m in zip(("loss", "dx", "dW", "db"), _run(x, w, b, t, "mean", up), exact, bound):
        err = (a.double() - e).abs()
        assert bool((err <= m).all()), (what, float(err.max()), float((err / m).max()))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_lie_far_apart(dtype):
    """The last position of long sequences, hidden[:, -1]; a table with rows far apart; a single row of any stride."""
    from phc_gnn_amd import ops
    far = (1 << 22) + 24
    for n, v in ((3, 90), (70, 130)):
        x, w, b, t = (q.to(DEV) for q in _case(n, v, 64, dtype, seed=37))
        up = torch.tensor(1.0, device=DEV)
        want = _run(x, w, b, t, "mean", up)
        buf = torch.empty((max(n, v) - 1) * far + 64, device=DEV, dtype=dtype)
        for which in ("x", "w"):
            src = x if which == "x" else w
            wide = torch.as_strided(buf, src.shape, (far, 1)).copy_(src).requires_grad_()
            xs, ws = (wide, w.clone().requires_grad_()) if which == "x" else (x.clone().requires_grad_(), wide)
            loss = ops.linear_cross_entropy(xs, ws, t, b)
            got = (loss.detach(), *torch.autograd.grad(loss, [xs, ws]))
            assert all(torch.equal(p, q) for p, q in zip(got, want)), (n, which)
        del buf, wide
    x, w, b, t = (q.to(DEV) for q in _case(5, 1, 64, dtype, ignored=0.0))
    one = torch.as_strided(w, (1, 64), (1 << 40, 1))
    assert torch.equal(ops.linear_cross_entropy(x, one, t), ops.linear_cross_entropy(x, w, t))
    one = torch.as_strided(x, (1, 64), (1 << 40, 1))
    assert torch.equal(ops.linear_cross_entropy(one, w, t[:1]), ops.linear_cross_entropy(x[:1], w, t[:1]))
    assert torch.equal(ops.embedding(torch.zeros(2, dtype=torch.int64, device=DEV), torch.as_strided(w, (1, 64), (1 << 40, 1))), w.expand(2, 64))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ignored", [0.0, 0.85])
@pytest.mark.parametrize("piece", [0, 1024])
def test_large_tiles_of_dx_and_dw_with_splits(piece, ignored, dtype):
    """256 x 256 tiles of both gradient products with their k loops split (7 and 5 ways; more where few rows count), and dx added up over pieces at the
    same time.  The formula and its bounds on the GPU, in 64 bits."""
    n, v, d = 2300, 3000, 1024
    x, w, b, t = (q.to(DEV) for q in _case(n, v, d, dtype, ignored=ignored, seed=47))
    for reduction in ("mean", "none"):
        up = torch.tensor(1.0, device=DEV) if reduction == "mean" else torch.rand(n, generator=torch.Generator().manual_seed(3)).to(DEV) - 0.3
        exact, bound = _formula(x, w, b, t, reduction, up)
        for what, a, e, m in zip(("loss", "dx", "dW", "db"), _run(x, w, b, t, reduction, up, piece=piece), exact, bound):
            err = (a.double() - e).abs()
            assert bool((err <= m).all()), (what, reduction, float(err.max()), float((err / m).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(4, 2180), (16, 900), (20, 1500), (32, 2400), (50, 1000), (5, 20000), (30, 9000), (60, 6000)])
def test_few_rows_of_many_columns(n, v, dtype):
    """Rows longer than one round of the k loop, ending at every step of the next: the wavefronts' last rounds are partly empty, each differently."""
    from phc_gnn_amd import ops
    x, w, b, t = (q.to(DEV) for q in _case(n, v, 2600, dtype, ignored=0.1, seed=53))
    for d in (*range(500, 1600, 37), *range(1024, 1600, 32), 1343, 2048, 2065, 2577, 2600):
        xs, ws = x[:, :d].contiguous(), w[:, :d].contiguous()
        exact, bound = _formula(xs, ws, b, t, "none", torch.ones(n, device=DEV))
        err = (ops.linear_cross_entropy(xs, ws, t, b, reduction="none").double() - exact[0]).abs()
        assert bool((err <= bound[0]).all()), (d, float((err / bound[0]).max()))


def test_graph_replay_of_a_forward_in_pieces():
    """Rows of W that are laid out anew, several pieces in both directions, a g for each row, the number of rows that count changing from replay to
    replay."""
    from phc_gnn_amd import ops
    x, w, b, t = (q.to(DEV) for q in _case(200, 1100, 97, torch.bfloat16, seed=61))
    up = torch.rand(200, device=DEV)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()

    def step():
        loss = ops.linear_cross_entropy(x, w, t, bias=b, piece=256, reduction="none")
        return (loss.detach(), *torch.autograd.grad(loss, [x, w, b], up))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cap = step()
    s.synchronize()
    for k in range(4):
        with torch.no_grad():
            x.mul_(1.25)
            t.copy_(torch.where(torch.arange(200, device=DEV) % 5 == k, torch.full_like(t, -100), torch.roll(t, 3)))
            up.mul_(-0.5)
        want = step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(cap, want)), k
