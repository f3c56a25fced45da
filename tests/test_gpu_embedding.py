"""ops.embedding (csrc/embedding.hip) against the formulas in 64 bits: out = scale W[t], dW[v] = scale sum of dy over t = v."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0") if torch.cuda.is_available() else None
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tokens(n, v, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, v, (n,), generator=g)
    if kind == "falling":                                    # frequencies fall with the token's number
        return ((float(v + 1) ** torch.rand(n, generator=g, dtype=torch.float64)).long() - 1).clamp_(0, v - 1)
    if kind == "one":
        return torch.full((n,), v // 2)
    return torch.where(torch.rand(n, generator=g) < 0.5, torch.full((n,), v - 1), torch.randint(0, v, (n,), generator=g))     # "half"


def _bound(tokens, dy, v, scale, exact, dtype):
    """c terms of one row are added in fp32 (c - 1 roundings of partial sums, each at most 2^-24 of the sum of magnitudes), times the fp32
    scale (one rounding, and one of the scale itself), then rounded to the type (half a step; fp16 has subnormal steps of 2^-24)."""
    mag = torch.zeros(v, dy.shape[1], dtype=torch.float64).index_add_(0, tokens, dy.abs()) * abs(scale)
    count = torch.bincount(tokens, minlength=v).double()[:, None]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}[dtype]
    return mag * (count + 2) * 2.0 ** -24 * 1.01 + exact.abs() * torch.finfo(dtype).eps / 2 * 1.01 + tiny


def _check(n, v, d, dtype, kind="falling", scale=1.0, pad=None, seed=0):
    from phc_gnn_amd import ops
    g = torch.Generator().manual_seed(seed + 1)
    t = _tokens(n, v, kind, seed)
    w = torch.randn(v, d, generator=g).to(dtype)
    dy = torch.randn(n, d, generator=g).to(dtype)
    wd = w.to(DEV).requires_grad_()
    out = ops.embedding(t.to(DEV), wd, scale=scale, padding_idx=pad)
    assert out.dtype == dtype and tuple(out.shape) == (n, d)
    # one fp32 product, one rounding: the same bits
    assert torch.equal(out.detach().cpu(), (w[t].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype))
    (dw,) = torch.autograd.grad(out, [wd], dy.to(DEV))
    exact = torch.zeros(v, d, dtype=torch.float64).index_add_(0, t, dy.double()) * scale
    if pad is not None:
        exact[pad] = 0
    assert dw.dtype == dtype
    err = (dw.cpu().double() - exact).abs()
    assert bool((err <= _bound(t, dy.double(), v, scale, exact, dtype)).all()), float(err.max())
    if pad is not None:
        assert int(torch.count_nonzero(dw[pad])) == 0
    return dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(0, 7, 8), (1, 1, 1), (1, 5000, 64), (31, 9, 5), (32, 9, 8), (33, 300, 130), (64, 1, 16), (2047, 119, 32),
                                   (2049, 257, 24), (5000, 70000, 36), (300, 65536, 8), (100, 300000, 8), (17000, 600001, 4), (4100, 1000, 257), (513, 40, 2056)])
def test_lookup_and_gradient(n, v, d, dtype):
    _check(n, v, d, dtype, scale=0.75, pad=0 if v > 1 else None)


@pytest.mark.parametrize("kind", ["uniform", "one", "half"])
@pytest.mark.parametrize("n,v,d", [(97, 50, 12), (4000, 700, 40), (20000, 300, 16)])
def test_token_distributions(n, v, d, kind):
    """Runs inside a chunk, over many chunks, and all positions one token; sort tiles that end inside."""
    for dtype in (torch.float32, torch.bfloat16):
        _check(n, v, d, dtype, kind=kind, scale=2.0, pad=v - 1 if kind == "uniform" else None)


def test_gradient_of_a_run_is_its_sum_across_chunks():
    """One token with integer gradients: the sum is exact whatever the order, so a lost or doubled part shows."""
    from phc_gnn_amd import ops
    for n in (31, 32, 33, 63, 64, 65, 96, 1000, 4097):
        w = torch.zeros(3, 8, device=DEV, requires_grad=True)
        t = torch.ones(n, dtype=torch.int64, device=DEV)
        t[:5] = 0
        dy = torch.arange(n * 8, device=DEV, dtype=torch.float32).reshape(n, 8) % 97
        (dw,) = torch.autograd.grad(ops.embedding(t, w), [w], dy)
        want = torch.zeros(3, 8, dtype=torch.float64).index_add_(0, t.cpu(), dy.cpu().double())
        assert torch.equal(dw.cpu().double(), want), n


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_alignment_and_shapes(dtype):
    from phc_gnn_amd import ops
    g = torch.Generator().manual_seed(5)
    base = torch.randn(41, 50, generator=g).to(dtype)
    t = torch.randint(0, 40, (6, 7), generator=g)
    dy_base = torch.randn(6, 7, 64, generator=g).to(dtype)
    # a column slice that starts at an odd element, a transposed table, int32 tokens of two dimensions and a strided gradient
    for make in (lambda b: b[:40, 3:36], lambda b: b[1:41, 2:34], lambda b: b[:40, :48].t().contiguous().t()):
        w = make(base.to(DEV)).detach().requires_grad_()
        d = w.shape[1]
        out = ops.embedding(t.to(DEV).to(torch.int32), w, scale=3.0)
        assert torch.equal(out.detach().cpu(), (make(base)[t].float() * 3.0).to(dtype))
        dy = dy_base.to(DEV)[..., 1:1 + d]
        (dw,) = torch.autograd.grad(out, [w], dy)
        ref = ops.embedding(t.to(DEV), w.detach().clone().contiguous().requires_grad_(), scale=3.0)
        (dw2,) = torch.autograd.grad(out := ops.embedding(t.to(DEV), (w2 := w.detach().clone().contiguous().requires_grad_()), scale=3.0), [w2], dy.contiguous())
        assert torch.equal(dw, dw2) and tuple(ref.shape) == (6, 7, d)
    tt = t.to(DEV).t()                                       # tokens that are no contiguous tensor
    assert torch.equal(ops.embedding(tt, base.to(DEV)), base.to(DEV)[tt])


def test_expanded_gradient():
    """The gradient of a sum arrives with zero strides."""
    from phc_gnn_amd import ops
    w = torch.randn(5, 6, device=DEV, requires_grad=True)
    t = torch.tensor([1, 1, 4], device=DEV)
    ops.embedding(t, w, scale=0.5).sum().backward()
    assert torch.equal(w.grad.cpu(), torch.tensor([0.0, 1.0, 0, 0, 0.5])[:, None].expand(5, 6))


def test_bad_tokens_read_row_zero_and_are_reported():
    from phc_gnn_amd import check_indices, ops
    w = torch.randn(5, 8, device=DEV, requires_grad=True)
    t = torch.tensor([2, 5, -1, 1 << 40], device=DEV)
    out = ops.embedding(t, w)
    with pytest.raises(IndexError, match="embedding table"):
        check_indices(DEV)
    check_indices(DEV)
    assert torch.equal(out.detach(), w.detach()[torch.tensor([2, 0, 0, 0], device=DEV)])
    (dw,) = torch.autograd.grad(out, [w], torch.ones_like(out))
    assert torch.equal(dw.cpu()[:, 0], torch.tensor([3.0, 0, 1, 0, 0]))


def test_inf_and_nan_stay_in_their_rows():
    from phc_gnn_amd import ops
    w = torch.randn(6, 8, device=DEV, requires_grad=True)
    t = torch.tensor([3, 1, 3, 0], device=DEV)
    dy = torch.ones(4, 8, device=DEV)
    dy[1] = float("nan")
    dy[0, 2] = float("inf")
    (dw,) = torch.autograd.grad(ops.embedding(t, w, padding_idx=0), [w], dy)
    assert bool(dw[1].isnan().all()) and float(dw[3, 2]) == float("inf")
    ok = dw.clone()
    ok[1] = 0
    ok[3, 2] = 0
    assert bool(ok.isfinite().all()) and int(torch.count_nonzero(dw[[0, 2, 4, 5]])) == 0


def test_gradient_is_bitwise_reproducible():
    for dtype in (torch.float32, torch.bfloat16):
        a = _check(9000, 500, 72, dtype, kind="half", scale=1.5)
        for _ in range(3):
            assert torch.equal(a, _check(9000, 500, 72, dtype, kind="half", scale=1.5))


def test_other_stream_and_graph_replay():
    from phc_gnn_amd import ops
    w = torch.randn(400, 96, device=DEV, requires_grad=True)
    t = torch.randint(0, 400, (3000,), device=DEV)
    dy = torch.randn(3000, 96, device=DEV)

    def step():
        out = ops.embedding(t, w, scale=2.0)
        return out.detach(), torch.autograd.grad(out, [w], dy)[0]
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cap = step()
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for k in range(4):
        with torch.no_grad():
            w.mul_(1.25)
            dy.add_(0.5)
            t.copy_(torch.randint(0, 400, (3000,), device=DEV))
        want = step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(cap[0], want[0]) and torch.equal(cap[1], want[1]), k


def test_two_streams_at_once():
    from phc_gnn_amd import ops
    cases = []
    for k in range(2):
        w = torch.randn(700, 64, device=DEV, requires_grad=True)
        t = torch.randint(0, 700, (6000,), device=DEV)
        dy = torch.randn(6000, 64, device=DEV)
        cases.append((w, t, dy, torch.autograd.grad(ops.embedding(t, w), [w], dy)[0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for k, (w, t, dy, _) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(torch.autograd.grad(ops.embedding(t, w), [w], dy)[0])
    torch.cuda.synchronize()
    for (_, _, _, want), gs in zip(cases, got):
        assert all(torch.equal(want, x) for x in gs)


def test_capture_beside_a_live_eager_graph_is_refused():
    """The parameter's gradient node belongs to the eager result's stream: a backward captured elsewhere would end the process."""
    from phc_gnn_amd import ops
    from phc_gnn_amd.lib import PhcError
    w = torch.randn(40, 8, device=DEV, requires_grad=True)
    t = torch.randint(0, 40, (30,), device=DEV)
    alive = ops.embedding(t, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    x = torch.ones(8, device=DEV)
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = x + 1.0                                       # (the capture is not empty)
            with pytest.raises(PhcError, match="captured into a graph"):
                ops.embedding(t, w)
            with pytest.raises(PhcError, match="captured into a graph"):
                ops.linear_cross_entropy(torch.ones(2, 8, device=DEV), w, t[:2])
            out = ops.embedding(t, w.detach())               # no gradient, no objection
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive.detach()) and float(y[0]) == 2.0
    del alive
    with torch.cuda.stream(s):
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=s):
            (dw,) = torch.autograd.grad(ops.embedding(t, w), [w], torch.ones(30, 8, device=DEV))
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(dw[:, 0].cpu(), torch.bincount(t.cpu(), minlength=40).float())


def test_second_derivatives_are_refused():
    from phc_gnn_amd import ops
    w = torch.randn(10, 4, device=DEV, requires_grad=True)
    t = torch.tensor([1, 2, 2], device=DEV)
    dy = torch.ones(3, 4, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(ops.embedding(t, w), [w], dy, create_graph=True)
    assert torch.equal(dw.detach().cpu()[:, 0], torch.tensor([0.0, 1, 2, 0, 0, 0, 0, 0, 0, 0]))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dw.sum().backward()
    x = torch.randn(3, 4, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(x, w.detach(), t), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="does not require grad"):
        dx.sum().backward()


def test_more_rows_than_one_launch_takes():
    """2^25 rows of an odd length need 2^31 threads; the lookup goes on in a second launch.  All sums are of ones and exact: no partial sum
    passes 2^24."""
    from phc_gnn_amd import ops
    n, v, d = (1 << 25) + 37, 9, 33
    w = torch.randn(v, d, device=DEV, requires_grad=True)
    t = torch.randint(0, v, (n,), device=DEV)
    out = ops.embedding(t, w, scale=0.5)
    for at in (0, (1 << 25) - 100, n - 1000):
        s = slice(at, at + 1000)
        assert torch.equal(out[s], 0.5 * w.detach()[t[s]])
    dy = torch.ones(n, d, device=DEV)
    (dw,) = torch.autograd.grad(out, [w], dy)
    assert torch.equal(dw, 0.5 * torch.bincount(t, minlength=v).float()[:, None].expand(v, d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 9, 63, 64, 65])
def test_few_positions(n, dtype):
    """Up to 64 positions are not sorted: every token's first position adds its rows, in order.  One token for all, two in turn, all
    different ones, the padding row among them, out-of-range ones; several column slabs and an odd length."""
    from phc_gnn_amd import check_indices, ops
    g = torch.Generator().manual_seed(n)
    for v, d in ((130, 1032), (65, 129), (64, 4)):
        w = torch.randn(v, d, generator=g).to(dtype).to(DEV).requires_grad_()
        dy = torch.randn(n, d, generator=g).to(dtype).to(DEV)
        for t in (torch.full((n,), v - 1), torch.arange(n) % 2, torch.randperm(v, generator=g).repeat(2)[:n], torch.full((n,), 5)):
            (dw,) = torch.autograd.grad(ops.embedding(t.to(DEV), w, scale=0.5, padding_idx=5), [w], dy)
            want = torch.zeros(v, d, dtype=torch.float64).index_add_(0, t, dy.cpu().double()) * 0.5
            mag = torch.zeros(v, d, dtype=torch.float64).index_add_(0, t, dy.cpu().double().abs()) * 0.5
            want[5], mag[5] = 0, 0
            # n roundings of 2^-24 of the sum of magnitudes, and the rounding to the type
            bound = mag * n * 2.0 ** -24 + want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -10) + 2.0 ** -24 * (dtype == torch.float16)
            assert bool(((dw.cpu().double() - want).abs() <= bound).all())
    t = torch.randint(0, 30, (n,), generator=g)
    t[0] = 64
    w = torch.randn(64, 8, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(ops.embedding(t.to(DEV), w), [w], torch.ones(n, 8, device=DEV))
    with pytest.raises(IndexError):
        check_indices()
    t[0] = 0
    assert torch.equal(dw.cpu()[:, 0], torch.bincount(t, minlength=64).float())


def test_capture_beside_a_live_graph_of_other_operators_is_refused():
    """The eager graph may be anybody's; one made on the capture's own stream is no obstacle."""
    from phc_gnn_amd import ops
    from phc_gnn_amd.lib import PhcError
    w = torch.randn(40, 8, device=DEV, requires_grad=True)
    t = torch.randint(0, 40, (30,), device=DEV)
    alive = w * 2.0
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = ops.embedding(t, w.detach())
            with pytest.raises(PhcError, match="captured into a graph"):
                ops.embedding(t, w)
            with pytest.raises(PhcError, match="captured into a graph"):
                ops.linear_cross_entropy(torch.ones(2, 8, device=DEV), w, t[:2])
    del alive
    with torch.cuda.stream(s):
        here = ops.embedding(t, w)                              # its node is this stream's
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=s):
            (dw,) = torch.autograd.grad(ops.embedding(t, w), [w], torch.ones(30, 8, device=DEV))
    g.replay()
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, here.detach())
    assert torch.equal(dw[:, 0].cpu(), torch.bincount(t.cpu(), minlength=40).float())
