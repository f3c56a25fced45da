"""Embedding, linear cross entropy and gradient norm without a GPU: what they refuse, and their workspace queries."""
import ctypes as C

import pytest
import torch


def _lib():
    from phc_gnn_amd import lib
    return lib, lib.load()


def test_cpu_tensors_are_refused():
    from phc_gnn_amd import ops, optim
    from phc_gnn_amd.lib import PhcError
    w, t = torch.randn(5, 4), torch.tensor([0, 1])
    p = torch.nn.Parameter(torch.randn(3))
    p.grad = torch.randn(3)
    for call in (lambda: ops.embedding(t, w), lambda: ops.linear_cross_entropy(torch.randn(2, 4), w, t), lambda: optim.grad_norm([w]),
                 lambda: optim.clip_grad_norm_([p], 1.0), lambda: optim.clip_grads([w], 1.0)):
        with pytest.raises(PhcError, match="no CPU fallback"):
            call()


def test_nothing_to_clip():
    from phc_gnn_amd import optim
    assert float(optim.grad_norm([])) == 0.0
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0       # no gradients
    norm, out = optim.clip_grads([], 1.0)
    assert float(norm) == 0.0 and out == []


def test_norm_arguments():
    from phc_gnn_amd import optim
    from phc_gnn_amd.lib import PhcError
    g = [torch.ones(2)]
    for norm_type in (0.0, 3.0, -1.0, float("nan")):
        with pytest.raises(PhcError, match="norm_type"):
            optim.grad_norm(g, norm_type)
    for bad in (-1.0, float("nan")):
        with pytest.raises(PhcError, match="max_norm"):
            optim.clip_grads(g, bad)
    with pytest.raises(PhcError, match="results"):
        optim.clip_grads(g, 1.0, out=[])
    with pytest.raises(PhcError, match="contiguous tensor of shape"):
        optim.clip_grads(g, 1.0, out=[torch.ones(3)])


def test_embedding_entry_points_check_their_arguments():
    lib, h = _lib()
    ok = 1 << 20                                       # an address: nothing is dereferenced before the checks are through
    assert h.phc_embedding_fwd(ok, ok, 3, 5, 4, 4, 7, 1.0, ok, None) == -1 and b"dtype" in h.phc_last_error()
    assert h.phc_embedding_fwd(None, ok, 3, 5, 4, 4, 0, 1.0, ok, None) == -1
    assert h.phc_embedding_fwd(ok, ok, -1, 5, 4, 4, 0, 1.0, ok, None) == -1
    assert h.phc_embedding_fwd(ok, ok, 3, 0, 4, 4, 0, 1.0, ok, None) == -1
    assert h.phc_embedding_fwd(ok, ok, 3, 5, 4, 3, 0, 1.0, ok, None) == -1 and b"row stride" in h.phc_last_error()
    assert h.phc_embedding_fwd(ok, ok, 3, 1 << 31, 4, 4, 0, 1.0, ok, None) == -2
    assert h.phc_embedding_fwd(None, None, 0, 5, 4, 4, 0, 1.0, None, None) == 0                # nothing to do
    need = h.phc_embedding_bwd_ws_bytes(1000, 50, 16)
    assert need >= 2 * 4 * 1000 and h.phc_embedding_bwd_ws_bytes(-1, 50, 16) == 0
    assert h.phc_embedding_bwd(ok, ok, 1000, 50, 16, 16, 0, 1.0, -1, ok, ok, need - 1, None) == -3
    assert h.phc_embedding_bwd(ok, ok, 1000, 50, 16, 16, 0, 1.0, -1, ok, None, need, None) == -3
    assert h.phc_embedding_bwd(ok, ok, 1000, 50, 16, 16, 0, 1.0, -1, ok, ok + 4, need, None) == -3
    assert h.phc_embedding_bwd(ok, None, 1000, 50, 16, 16, 0, 1.0, -1, ok, ok, need, None) == -1


def _desc(lib, **kw):
    d = lib.LinearXentDesc()
    ok = 1 << 20
    for k, v in dict(dict(N=10, V=300, D=64, ldx=64, ldw=64, ignore_index=-100, piece=0, dtype=1, reduction=2, x=ok, W=ok, target=ok, loss=ok,
                          state=ok, ws=ok, ws_bytes=1 << 40), **kw).items():
        setattr(d, k, v)
    return d


def test_linear_xent_entry_points_check_their_arguments():
    lib, h = _lib()
    for kw, code in ((dict(dtype=3), -1), (dict(reduction=3), -1), (dict(N=0), -1), (dict(V=0), -1), (dict(D=0), -1), (dict(ldx=63), -1),
                     (dict(ldw=63), -1), (dict(N=1 << 23), -2), (dict(V=1 << 23), -2), (dict(ldw=1 << 23), -2), (dict(piece=-1), -1),
                     (dict(x=None), -1), (dict(W=None), -1), (dict(target=None), -1), (dict(state=None), -1), (dict(state=(1 << 20) + 8), -1),
                     (dict(loss=None), -1), (dict(ws=None), -3), (dict(ws=(1 << 20) + 16), -3), (dict(ws_bytes=8), -3)):
        assert h.phc_linear_xent_fwd(C.byref(_desc(lib, **kw)), None) == code, kw
    assert h.phc_linear_xent_fwd(None, None) == -1
    for kw, code in ((dict(), -1), (dict(dloss=1 << 20, db=1 << 20), -1), (dict(dloss=1 << 20, ws_bytes=8), -3)):
        assert h.phc_linear_xent_bwd(C.byref(_desc(lib, **kw)), None) == code, kw
    assert h.phc_linear_xent_bwd(C.byref(_desc(lib, dloss=1 << 20)), None) == 0                # no gradient wanted


def test_linear_xent_workspace_does_not_hold_the_logits():
    lib, h = _lib()
    d = _desc(lib, N=16384, V=131072, D=1024, ldx=1024, ldw=1024, dloss=1 << 20, dx=1 << 20, dW=1 << 20)
    logits = 16384 * 131072 * 2
    assert 0 < h.phc_linear_xent_ws_bytes(C.byref(d), 0) < logits // 8
    assert 0 < h.phc_linear_xent_ws_bytes(C.byref(d), 1) < logits // 4
    d.piece = 1024
    assert h.phc_linear_xent_ws_bytes(C.byref(d), 1) < logits // 16
    d.V = 0
    assert h.phc_linear_xent_ws_bytes(C.byref(d), 1) == 0


def _norm_call(h, lib, src, numel, dt, dst=None, odt=None, kind=0, max_norm=1.0, ws=1 << 20, ws_bytes=1 << 20, res=1 << 20):
    n = len(src)
    arr = lambda ty, v: None if v is None else (ty * n)(*v)
    return h.phc_grad_norm_clip(n, arr(C.c_void_p, src), arr(C.c_int64, numel), arr(C.c_int32, dt), kind, max_norm, arr(C.c_void_p, dst),
                                arr(C.c_int32, odt), res, ws, ws_bytes, None)


def test_grad_norm_entry_point_checks_its_arguments():
    lib, h = _lib()
    a, b = 1 << 24, 1 << 25
    assert _norm_call(h, lib, [a], [4], [5]) == -1
    assert _norm_call(h, lib, [a], [4], [0], kind=3) == -1
    assert _norm_call(h, lib, [a], [-4], [0]) == -1
    assert _norm_call(h, lib, [None], [4], [0]) == -1
    assert _norm_call(h, lib, [a + 2], [4], [0]) == -1 and b"aligned" in h.phc_last_error()
    assert _norm_call(h, lib, [a], [4], [0], max_norm=-1.0) == -1
    assert _norm_call(h, lib, [a], [4], [0], max_norm=float("nan")) == -1
    assert _norm_call(h, lib, [a], [4], [0], res=None) == -1
    assert _norm_call(h, lib, [a], [4], [0], ws_bytes=8) == -3
    assert _norm_call(h, lib, [a], [4], [0], dst=[b]) == -1                                  # results without types
    # results that share memory, results over another gradient, a result over its own gradient in another type or at another place
    assert _norm_call(h, lib, [a, a + 8], [4, 4], [0, 0], [a, a + 8], [0, 0]) == -1 and b"share memory" in h.phc_last_error()
    assert _norm_call(h, lib, [a, a], [4, 4], [0, 0], [a, a], [0, 0]) == -1
    assert _norm_call(h, lib, [a, b], [4, 4], [0, 0], [b, b + 64], [0, 0]) == -1 and b"reads memory" in h.phc_last_error()
    assert _norm_call(h, lib, [a], [4], [1], [a], [0]) == -1
    assert _norm_call(h, lib, [a], [4], [0], [a + 4], [0]) == -1


def test_grad_norm_workspace_is_small():
    lib, h = _lib()
    n = (C.c_int64 * 4)(10, 0, 1 << 30, 5000)
    assert 8 * 2 <= h.phc_grad_norm_ws_bytes(4, n) <= 8 * 2100
    assert h.phc_grad_norm_ws_bytes(0, None) == 8
    many = (C.c_int64 * 1000)(*([1 << 20] * 1000))
    assert h.phc_grad_norm_ws_bytes(1000, many) <= 8 * (8 * 2048 + 1)


def test_shape_checks_of_the_python_layer(monkeypatch):
    """The refusals that come before a launch, with the device check taken out of the way."""
    from phc_gnn_amd import lib, ops, vocab
    monkeypatch.setattr(vocab.L, "require_device", lambda *t: torch.device("cpu"))
    w, x, t = torch.randn(5, 4), torch.randn(2, 4), torch.tensor([0, 1])
    for args, kw, what in (((x, w, t[:1]), {}, "target"), ((x[:, :3], w, t), {}, "does not fit weight"), ((x, w.half(), t), {}, "one type"),
                           ((x, w, t), dict(bias=torch.zeros(4)), "bias"), ((x, w, t), dict(bias=torch.zeros(5).half()), "one type"),
                           ((x, w, t), dict(reduction="max"), "reduction"), ((x.double(), w.double(), t), {}, "float32"),
                           ((x, w, t.float()), {}, "int64"), ((x, w, t), dict(piece=-1), "piece"), ((x, w[0], t), {}, "does not fit")):
        with pytest.raises(lib.PhcError, match=what):
            ops.linear_cross_entropy(*args, **kw)
    for args, kw, what in (((t, w.double()), {}, "float32"), ((t.float(), w), {}, "int64"), ((t, w[0]), {}, "V, D"), ((t, w[:0]), {}, "V, D"),
                           ((t, w), dict(padding_idx=5), "padding_idx"), ((t, w), dict(padding_idx=-6), "padding_idx")):
        with pytest.raises(lib.PhcError, match=what):
            ops.embedding(*args, **kw)


def test_sizes_beyond_one_launch_are_refused():
    """The hardware counts a launch's threads in 32 bits: sizes that would need more are refused before anything is launched."""
    lib, h = _lib()
    ok = 1 << 20
    assert h.phc_embedding_bwd_ws_bytes(10, (1 << 29) + 1, 4) == 0
    assert h.phc_embedding_fwd(ok, ok, 3, (1 << 29) + 1, 4, 4, 0, 1.0, ok, None) == -2
    n, d = 1 << 28, (1 << 20) - 1                       # an odd row length: a lane for each column
    need = h.phc_embedding_bwd_ws_bytes(n, 10, d)
    assert h.phc_embedding_bwd(ok, ok, n, 10, d, d, 1, 1.0, -1, ok, ok, need, None) == -2 and b"one launch" in h.phc_last_error()


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_pieces_of_more_columns_than_there_are(dtype):
    """`piece` up to the largest int64 ("all at once") is all the columns: the same scratch, and no size that wrapped around."""
    lib, h = _lib()
    for n in (100, 8192):
        d = _desc(lib, N=n, V=131071, D=96, ldx=96, ldw=96, dtype=dtype, dloss=1 << 20, dx=1 << 20, dW=1 << 20)
        for backward in (0, 1):
            d.piece = d.V
            want = h.phc_linear_xent_ws_bytes(C.byref(d), backward)
            assert backward == 0 or want >= n * d.V * 2
            for piece in (d.V + 1, 1 << 22, 1 << 40, (1 << 63) - 65, (1 << 63) - 64, (1 << 63) - 63, (1 << 63) - 1):
                d.piece = piece
                assert h.phc_linear_xent_ws_bytes(C.byref(d), backward) == want, piece


def _x_copy(n, d, dtype):
    """x as the products read it: rows and columns rounded up to whole steps; fp32 of more than 256 rows in three 16-bit terms."""
    wide = dtype == 0 and n > 256
    size = 6 if wide else 4 if dtype == 0 else 2
    line = 32 if dtype == 0 and not wide else 64
    return (n + 63) // 64 * 64 * ((d + line - 1) // line * line) * size


@pytest.mark.parametrize("n,v,d,dtype", [(257, 131072, 4096, 0), (1 << 20, 262144, 64, 1), (1 << 22, 1 << 22, 64, 2), (8192, 131072, 2048, 1),
                                         (300, 131072, 4097, 1), (100, 1 << 22, 1023, 0), (65, 131072, 4097, 2), (1 << 18, 50000, 256, 0), (5, 1 << 22, 4097, 0)])
def test_linear_xent_forward_scratch_is_bounded(n, v, d, dtype):
    """Half a GiB for a piece of the vocabulary (its row statistics, its rows of W where they are laid out), and beside it x laid out and a few
    words for each row.  An explicit piece bounds the layout of W."""
    lib, h = _lib()
    beside = _x_copy(n, d, dtype) + n * 16 + 8192
    q = _desc(lib, N=n, V=v, D=d, ldx=d, ldw=d, dtype=dtype)
    assert 0 < h.phc_linear_xent_ws_bytes(C.byref(q), 0) <= (512 << 20) + beside
    q.piece = 2048
    stats = (v + 63) // 64 * n * 8 if n <= 12288 else 512 << 20
    assert 0 < h.phc_linear_xent_ws_bytes(C.byref(q), 0) <= min(stats, 512 << 20) + 2048 * ((d + 63) // 64 * 64) * 6 + beside


@pytest.mark.parametrize("n,v,d,dtype", [(257, 131072, 4096, 0), (300, 131072, 4097, 1), (8192, 131072, 2048, 1), (100, 1 << 22, 1023, 0), (3000, 131072, 2050, 2),
                                         (1, 1 << 22, 4097, 1), (1 << 18, 50000, 256, 0), (1 << 20, 32000, 64, 1)])
def test_linear_xent_backward_scratch_is_what_is_documented(n, v, d, dtype):
    """Half a GiB, or 2048 columns, for a piece's d and its rows of W where they are laid out; N / 8 bytes a column (rounded up) for db; x laid out; dx
    in fp32 if there are several pieces; 128 MiB for split products."""
    lib, h = _lib()
    wide = dtype == 0 and n > 256
    size = 4 if dtype == 0 else 2
    column = (6 if wide else size) * ((n + 63) // 64 * 64) + ((d + 63) // 64 * 64 * (6 if wide else size) if wide or d * size % 16 else 0)
    columns = min(v + 63, max(2048, (512 << 20) // column + 256))
    beside = _x_copy(n, d, dtype) + n * d * 4 + (128 << 20) + ((n + 63) // 64 * 8 + 8) * columns + n * 16 + 16384
    q = _desc(lib, N=n, V=v, D=d, ldx=d, ldw=d, dtype=dtype, dloss=1 << 20, dx=1 << 20, dW=1 << 20, bias=1 << 20, db=1 << 20)
    assert 0 < h.phc_linear_xent_ws_bytes(C.byref(q), 1) <= columns * column + beside
    q.piece = 2048
    assert 0 < h.phc_linear_xent_ws_bytes(C.byref(q), 1) <= 2048 * column + beside
