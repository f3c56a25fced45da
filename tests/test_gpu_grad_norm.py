"""optim.grad_norm / clip_grads / clip_grad_norm_ (csrc/grad_norm.hip) against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0") if torch.cuda.is_available() else None
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(4, 32, 32), (1,), (0,), (119, 32), (8192,), (8193,), (5,), (3, 5, 7), (20000,), (2, 0, 3)]


def _tensors(shapes, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    types = TYPES if dtype == "mixed" else [dtype]
    return [(torch.randn(s, generator=g) * scale).to(types[i % len(types)]) for i, s in enumerate(shapes)]


def _norm(ts, p):
    flat = torch.cat([t.detach().cpu().double().flatten() for t in ts])
    return float(flat.abs().max() if p == math.inf else flat.abs().pow(p).sum().pow(1 / p))


def _close(got, exact, coef, max_norm):
    """c in fp32 (one rounding of an fp64 quotient), one fp32 product, one rounding to the type: two roundings of 2^-24 and half a step."""
    want = exact.double() * coef
    eps = torch.finfo(got.dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}[got.dtype]
    err = (got.cpu().double() - want).abs()
    assert bool((err <= want.abs() * (eps + 2.0 ** -23) * 1.01 + tiny).all()), float(err.max())


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES + ["mixed"])
def test_norm_and_clip(dtype, p):
    from phc_gnn_amd import optim
    ts = _tensors(SHAPES, dtype)
    dev = [t.to(DEV) for t in ts]
    exact = _norm(ts, p)
    norm = optim.grad_norm(dev, p)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    # fp64 sums: what is left is the rounding of the result
    assert abs(float(norm) - exact) <= exact * 2.0 ** -23
    for bound in (0.3 * exact, 3.0 * exact, 0.0):
        coef = min(1.0, bound / (exact + 1e-6))
        got_norm, out = optim.clip_grads(dev, bound, p)
        assert float(got_norm) == float(norm)
        out32 = [torch.full(t.shape, 7.0, device=DEV) for t in dev]
        optim.clip_grads(dev, bound, p, out=out32)
        for t, d, o, q in zip(ts, dev, out, out32):
            assert o.dtype == t.dtype and torch.equal(d.cpu(), t)                # the inputs stay
            _close(o, t, coef, bound)
            _close(q, t, coef, bound)
        params = [torch.nn.Parameter(torch.empty_like(d)) for d in dev] + [torch.nn.Parameter(torch.ones(3, device=DEV))]
        for q, d in zip(params, dev):
            q.grad = d.clone()
        assert float(optim.clip_grad_norm_(params, bound, p)) == float(norm)
        for q, o in zip(params, out):
            assert torch.equal(q.grad, o)                                        # in place and not: the same bits
        assert params[-1].grad is None


def test_many_tensors():
    """More tensors than one launch takes, empty ones among them, the last ones alone in a group."""
    from phc_gnn_amd import optim
    for n in (1, 127, 128, 129, 256, 300):
        ts = _tensors([((i * 37) % 11,) for i in range(n)], "mixed", seed=n)
        ts[0] = torch.ones(3)
        dev = [t.to(DEV) for t in ts]
        exact = _norm(ts, 2.0)
        norm, out = optim.clip_grads(dev, 0.5 * exact)
        assert abs(float(norm) - exact) <= exact * 2.0 ** -23
        for t, o in zip(ts, out):
            _close(o, t, 0.5 * exact / (exact + 1e-6), 0.5 * exact)


def test_views_of_one_buffer_at_odd_addresses():
    from phc_gnn_amd import optim
    for dtype in TYPES:
        sizes = [1, 7, 8191, 3, 20001, 64, 5]
        flat = torch.randn(sum(sizes) + 1, device=DEV).to(dtype)[1:]
        keep = flat.clone()
        parts = list(flat.split(sizes))
        exact = _norm([keep], 2.0)
        params = [torch.nn.Parameter(torch.empty_like(p)) for p in parts]
        for q, p in zip(params, parts):
            q.grad = p
        norm = optim.clip_grad_norm_(params, 0.25 * exact)
        assert abs(float(norm) - exact) <= exact * 2.0 ** -23
        _close(flat, keep.cpu(), 0.25 * exact / (exact + 1e-6), 0.25 * exact)


def test_dense_and_strided_gradients():
    from phc_gnn_amd import optim
    base = torch.randn(6, 10, 8, device=DEV)
    views = [base.permute(2, 0, 1), torch.randn(9, 9, device=DEV)[:, ::2], torch.randn(5, 1, device=DEV).expand(5, 4).clone().t()]
    before = [v.clone() for v in views]
    exact = _norm(before, 2.0)
    assert abs(float(optim.grad_norm(views)) - exact) <= exact * 2.0 ** -23
    params = [torch.nn.Parameter(torch.empty(v.shape, device=DEV)) for v in views]
    for q, v in zip(params, views):
        q.grad = v
    optim.clip_grad_norm_(params, 0.5 * exact)
    for v, b in zip(views, before):
        _close(v.contiguous(), b.cpu(), 0.5 * exact / (exact + 1e-6), 0.5 * exact)


def test_large_values_do_not_overflow():
    """Squares beyond the largest fp32 value."""
    from phc_gnn_amd import optim
    t = torch.full((5000,), 1e30, device=DEV)
    exact = 1e30 * math.sqrt(5000)
    assert abs(float(optim.grad_norm([t])) - exact) <= exact * 1e-6
    small = torch.full((5000,), 1e-30, device=DEV)
    # 1e-30 is no fp32 value (2^-24 of it off), and the norm is rounded once: 2^-23 of 7e-29 = 8.4e-36 in all
    assert abs(float(optim.grad_norm([small])) - 1e-30 * math.sqrt(5000)) <= 1e-30 * math.sqrt(5000) * 2.0 ** -23
    norm, (out,) = optim.clip_grads([t], 1.0)
    assert abs(float(out[0]) * math.sqrt(5000) - 1.0) <= 1e-5


def test_values_that_are_not_finite():
    from phc_gnn_amd import optim
    for p in (2.0, 1.0, math.inf):
        a, b = torch.ones(9000, device=DEV), torch.ones(4, device=DEV)
        a[8500] = math.inf
        norm, out = optim.clip_grads([a, b], 1.0, p)
        # coefficient 0: zeros, and inf * 0
        assert float(norm) == math.inf and float(out[1].abs().max()) == 0.0
        assert bool(out[0][8500].isnan()) and float(out[0][:8500].abs().max()) == 0.0
        b[2] = math.nan
        norm, out = optim.clip_grads([a, b], 1.0, p)
        assert math.isnan(float(norm)) and bool(out[1].isnan().all())
        q = torch.nn.Parameter(torch.zeros(4, device=DEV))
        q.grad = b.clone()
        keep = b.clone()
        with pytest.raises(RuntimeError, match="total norm"):
            optim.clip_grad_norm_([q], 1.0, p, error_if_nonfinite=True)
        assert torch.equal(q.grad.isnan(), keep.isnan()) and float(q.grad[0]) == 1.0        # nothing was scaled


def test_in_place_below_the_bound_changes_nothing():
    from phc_gnn_amd import optim
    ts = [t.to(DEV) for t in _tensors(SHAPES, "mixed", seed=3)]
    params = [torch.nn.Parameter(torch.empty_like(t)) for t in ts]
    for q, t in zip(params, ts):
        q.grad = t.clone()
    norm = optim.clip_grad_norm_(params, 1e9)
    assert all(torch.equal(q.grad, t) for q, t in zip(params, ts))
    assert float(norm) == float(optim.grad_norm(ts))


def test_shared_memory_is_refused():
    from phc_gnn_amd import optim
    from phc_gnn_amd.lib import PhcError
    g = torch.ones(10, device=DEV)
    a, b = torch.nn.Parameter(torch.zeros(10, device=DEV)), torch.nn.Parameter(torch.zeros(10, device=DEV))
    a.grad = b.grad = g
    with pytest.raises(PhcError, match="share memory"):
        optim.clip_grad_norm_([a, b], 1.0)
    with pytest.raises(PhcError, match="share memory"):
        optim.clip_grad_norm_([a, a], 1.0)
    assert abs(float(optim.grad_norm([g, g])) - math.sqrt(20.0)) < 1e-5                     # reading one tensor twice is fine
    assert float(g[0]) == 1.0


def test_same_result_as_torch_and_reproducible():
    from phc_gnn_amd import optim
    ts = [t.to(DEV) for t in _tensors(SHAPES * 3, torch.float32, seed=8)]
    mine, ref = [], []
    for t in ts:
        for out in (mine, ref):
            out.append(torch.nn.Parameter(torch.zeros_like(t)))
            out[-1].grad = t.clone()
    n1, n2 = optim.clip_grad_norm_(mine, 2.0), torch.nn.utils.clip_grad_norm_(ref, 2.0)
    torch.testing.assert_close(n1, n2, rtol=1e-6, atol=0)
    for p, q in zip(mine, ref):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)
    assert len({float(optim.grad_norm(ts)) for _ in range(5)}) == 1


def test_graph_replay():
    from phc_gnn_amd import optim
    ts = [t.to(DEV) for t in _tensors(SHAPES, "mixed", seed=4)]
    optim.clip_grads(ts, 1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            norm, out = optim.clip_grads(ts, 1.0)
    s.synchronize()
    for k in range(4):
        for t in ts:
            t.mul_(0.5 + k)
        want_norm, want = optim.clip_grads(ts, 1.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want_norm) and all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_scaled_tensors_count_as_changed():
    """Autograd has to notice that a tensor it saved was scaled."""
    from phc_gnn_amd import optim
    a = torch.ones(5, device=DEV)
    x = torch.ones(5, device=DEV, requires_grad=True)
    y = (x * a).sum()
    p = torch.nn.Parameter(torch.zeros(5, device=DEV))
    p.grad = a
    optim.clip_grad_norm_([p], 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_expanded_gradients_are_refused_before_anything_is_scaled():
    from phc_gnn_amd import optim
    from phc_gnn_amd.lib import PhcError
    p = [torch.nn.Parameter(torch.zeros(4, device=DEV)), torch.nn.Parameter(torch.zeros(6, device=DEV))]
    p[0].grad = torch.full((4,), 3.0, device=DEV)
    p[1].grad = torch.full((1,), 2.0, device=DEV).expand(6)
    with pytest.raises(PhcError, match="in place"):
        optim.clip_grad_norm_(p, 1.0)
    assert torch.equal(p[0].grad.cpu(), torch.full((4,), 3.0)) and torch.equal(p[1].grad.cpu(), torch.full((6,), 2.0))
    assert float(optim.grad_norm([q.grad for q in p])) == pytest.approx((4 * 9 + 6 * 4) ** 0.5, rel=2.0 ** -23)


def test_inference_mode():
    from phc_gnn_amd import optim
    g = [torch.full((5,), 2.0, device=DEV), torch.full((3,), 4.0, device=DEV, dtype=torch.bfloat16)]
    with torch.inference_mode():
        norm, out = optim.clip_grads(g, 1.0)
        again, _ = optim.clip_grads(out, 10.0, out=out)
    assert float(norm) == pytest.approx(68 ** 0.5, rel=2.0 ** -23) and 0.99 < float(again) < 1.01


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_norm_that_is_not_finite_is_raised_before_anything_is_written(bad):
    from phc_gnn_amd import optim
    grads = [torch.ones(100, device=DEV), torch.ones(7, device=DEV, dtype=torch.bfloat16)]
    grads[0][3] = bad
    kept = [g.clone() for g in grads]
    for out in (grads, [torch.full((100,), 7.0, device=DEV), torch.full((7,), 7.0, device=DEV)]):
        before = [o.clone() for o in out]
        with pytest.raises(RuntimeError, match="total norm"):
            optim.clip_grads(grads, 1.0, out=out, error_if_nonfinite=True)
        assert all(torch.equal(o.isnan(), q.isnan()) and torch.equal(o.nan_to_num(), q.nan_to_num()) for o, q in zip(out, before))
    with pytest.raises(RuntimeError, match="total norm"):
        optim.clip_grads(grads, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(g.nan_to_num(), k.nan_to_num()) for g, k in zip(grads, kept))
    grads[0][3] = 2.0
    norm, _ = optim.clip_grads(grads, 1.0, out=grads, error_if_nonfinite=True)
    # 106 ones and one 2: sqrt(110), rounded once
    assert abs(float(norm) - math.sqrt(110.0)) <= math.sqrt(110.0) * 2.0 ** -23 and float(grads[0][0]) < 1.0
