"""token_logprob forward and backward against its definition in 64 bits: row lengths from one to many trips,
unaligned and strided rows, masks that leave a row empty, ties, NaN and infinities, padding tokens, graphs, streams."""
import ctypes as C

import numpy as np
import pytest

import lm_reference as R
import plast_b200 as pb

pytestmark = pytest.mark.gpu
U = R.U


def run(x, token, temperature=1.0, top=0, view=None, optional=True):
    """Forward on [rows, C] values; `view` makes the logits tensor from the array."""
    rows, cols = x.shape
    t = {"x": view(x) if view else pb.Tensor.from_numpy(x), "token": pb.Tensor.from_numpy(token.astype(np.int32))}
    for k in ("logprob", "entropy", "log_norm"):
        t[k] = pb.Tensor((rows,))
    t["stats"] = pb.Tensor((rows, 2))
    t["top_logprob"] = pb.Tensor((rows, top)) if top else None
    t["top_index"] = pb.Tensor((rows, top), dtype=pb.INT32) if top else None
    pb.token_logprob(t["x"], t["token"], t["logprob"], t["entropy"] if optional else None,
                     t["log_norm"] if optional else None, t["stats"] if optional else None, t["top_logprob"], t["top_index"], temperature=temperature)
    return t


def check(t, x, token, temperature=1.0, top=0):
    ref = R.token_logprob(x, token, temperature, top)
    bound = R.log_sum_bound(ref, x.shape[1])
    for k in ("logprob", "log_norm"):
        np.testing.assert_allclose(t[k].numpy(), ref[k], rtol=2 * U, atol=bound, err_msg=k)
    # H = log S - ln 2 U / S: U carries S's relative error and is at most H
    h = np.nan_to_num(ref["entropy"])
    got = t["entropy"].numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref["entropy"]))
    assert (np.abs(np.nan_to_num(got) - h) <= bound * (1 + 2 * h) + 2 * U * h).all()
    if top:
        assert np.array_equal(t["top_index"].numpy(), ref["top_index"])
        np.testing.assert_allclose(t["top_logprob"].numpy(), ref["top_logprob"], rtol=2 * U, atol=bound)
    return ref


@pytest.mark.parametrize("cols", [1, 2, 3, 4, 5, 31, 64, 100, 1023, 1024, 4097, 8192, 20001, 65536, 131073])
@pytest.mark.parametrize("rows", [1, 3])
def test_row_lengths(rows, cols):
    rs = np.random.RandomState(cols + rows)
    x = (rs.randn(rows, cols) * 3).astype(np.float32)
    token = rs.randint(0, cols, rows)
    for top in (0, min(cols, 1), min(cols, 7), min(cols, 32)):
        check(run(x, token, top=top), x, token, top=top)


@pytest.mark.parametrize("rows,cols,top", [(700, 513, 5), (300, 3001, 20), (160, 32768, 8)])
def test_many_rows(rows, cols, top):
    rs = np.random.RandomState(1)
    x = (rs.randn(rows, cols) * 2 + 5).astype(np.float32)
    token = rs.randint(0, cols, rows)
    check(run(x, token, 0.7, top), x, token, 0.7, top)


def test_optional_outputs_may_be_missing():
    rs = np.random.RandomState(2)
    x, token = rs.randn(4, 50).astype(np.float32), np.arange(4)
    t = run(x, token, optional=False)
    np.testing.assert_allclose(t["logprob"].numpy(), R.token_logprob(x, token)["logprob"], atol=1e-5)


def test_masks_empty_rows_and_lowest_values():
    rs = np.random.RandomState(3)
    low = np.finfo(np.float32).min
    x = rs.randn(9, 4100).astype(np.float32)
    x[0] = -np.inf                                  # empty
    x[1, 5:] = -np.inf                              # five tokens left
    x[2] = low                                      # every logit the lowest value: uniform
    x[3, ::2] = low
    x[4, :] = -np.inf; x[4, 4099] = -3.0            # one token left: certain
    x[5, 17] = 3e38                                 # far above the rest
    x[6, 4000:] = -np.inf
    token = np.array([3, 2, 9, 1, 4099, 17, 4050, 0, -1])   # 4050 of row 6 is masked
    t = run(x, token, top=8)
    ref = check(t, x, token, top=8)
    assert ref["logprob"][0] == -np.inf and t["logprob"].numpy()[0] == -np.inf and t["entropy"].numpy()[0] == 0.0
    assert t["logprob"].numpy()[6] == -np.inf and t["logprob"].numpy()[8] == 0.0
    assert np.array_equal(t["top_index"].numpy()[0], np.arange(8))


def test_nan_and_infinity_stay_in_their_rows():
    rs = np.random.RandomState(4)
    x = rs.randn(6, 700).astype(np.float32)
    x[1, 30] = np.nan
    x[2, 600] = np.inf
    x[3, :695] = np.nan                             # fewer numbers than alternatives
    x[4, :] = np.nan
    token = np.array([1, 2, 3, 4, 5, 6])
    t = run(x, token, top=8)
    ref = R.token_logprob(x, token, 1.0, 8)
    for k in ("logprob", "entropy", "log_norm"):
        assert np.array_equal(np.isnan(t[k].numpy()), np.isnan(ref[k])), k
    assert np.array_equal(t["top_index"].numpy(), ref["top_index"])
    assert np.array_equal(np.isnan(t["top_logprob"].numpy()), np.isnan(ref["top_logprob"]))
    good = [0, 5]
    np.testing.assert_allclose(t["logprob"].numpy()[good], ref["logprob"][good], atol=1e-5)


@pytest.mark.parametrize("cols", [900, 30000])
@pytest.mark.parametrize("kind", ["equal", "two_values", "ascending", "descending", "zeros", "blocks"])
def test_ties_and_orders_of_alternatives(kind, cols):
    """The list of candidates overflows in most of these: any order has to end with the exact answer."""
    i = np.arange(cols)
    row = {"equal": np.full(cols, 1.5), "two_values": (i * 7919 % 3 == 0) * 1.0, "ascending": i * 1e-3,
           "descending": -i * 1e-3, "zeros": np.where(i % 2, 0.0, -0.0), "blocks": (i // 700) * 1.0}[kind]
    x = np.stack([row, row[::-1]]).astype(np.float32)
    token = np.array([0, cols - 1])
    for top in (1, 5, 32):
        t = run(x, token, top=top)
        assert np.array_equal(t["top_index"].numpy(), R.token_logprob(x, token, 1.0, top)["top_index"]), (kind, top)


def strided(x):       # every second row, columns from the third on, of a larger tensor
    rows, cols = x.shape
    big = pb.Tensor((2 * rows, cols + 5), requires_grad=False)
    host = np.full((2 * rows, cols + 5), 7.0, dtype=np.float32)
    host[::2, 3:3 + cols] = x
    big.copy_from(host)
    return big.view((rows, cols), (2 * (cols + 5), 1), offset=3)


def transposed(x):    # the vocabulary is not the contiguous axis
    return pb.Tensor.from_numpy(np.ascontiguousarray(x.T)).transpose(0, 1)


@pytest.mark.parametrize("view", [strided, transposed])
@pytest.mark.parametrize("cols", [33, 5000])
def test_views(view, cols):
    rs = np.random.RandomState(5)
    x, token = rs.randn(6, cols).astype(np.float32), rs.randint(0, cols, 6)
    check(run(x, token, 1.3, 4, view=view), x, token, 1.3, 4)


def test_leading_dims_and_strided_tokens():
    rs = np.random.RandomState(6)
    x = rs.randn(3, 4, 65).astype(np.float32)
    token = rs.randint(0, 65, (4, 3)).astype(np.int32)
    tx = pb.Tensor.from_numpy(np.ascontiguousarray(x.transpose(1, 0, 2))).transpose(0, 1)   # [3, 4, 65], batch inside
    tt = pb.Tensor.from_numpy(token).transpose(0, 1)
    lp = pb.Tensor((3, 4))
    pb.token_logprob(tx, tt, lp)
    ref = R.token_logprob(x.reshape(12, 65), token.T.reshape(12))
    np.testing.assert_allclose(lp.numpy().reshape(12), ref["logprob"], rtol=2 * U, atol=R.log_sum_bound(ref, 65))
    one, tok, out = pb.Tensor.from_numpy(x[0, 0]), pb.Tensor.from_numpy(np.array([5], np.int32)), pb.Tensor((1,))
    pb.token_logprob(one, tok, out)                    # a single distribution
    ref = R.token_logprob(x[0, :1], np.array([5]))
    np.testing.assert_allclose(out.numpy(), ref["logprob"], rtol=2 * U, atol=R.log_sum_bound(ref, 65))
    empty = pb.Tensor((0, 7))
    pb.token_logprob(empty, pb.Tensor((0,), dtype=pb.INT32), pb.Tensor((0,)))


def values(t):
    """A view's values, read through the tensor that owns the memory."""
    if t._base is None:
        return t.numpy()
    flat = t._base.numpy().ravel()
    at = (int(t.c.data) - int(t._base.c.data)) // 4
    return np.lib.stride_tricks.as_strided(flat[at:], shape=t.shape, strides=[4 * s for s in t.strides]).copy()


def backward(x, token, temperature, g, start, view=None, grad_view=None):
    t = run(x, token, temperature, view=view)
    rows = x.shape[0]
    for k, v in g.items():
        if v is not None:
            t[k].attach_grad().copy_from(v)
    dx = grad_view(start) if grad_view else pb.Tensor.from_numpy(start)
    t["x"].set_grad(dx)
    pb.token_logprob_backward(t["x"], t["token"], t["stats"], t["logprob"], t["entropy"], t["log_norm"], temperature)
    return t, values(dx)


def grad_bound(ref, want, start, x, token, temperature, g):
    """With t = (x - m) log2(e) / T: three roundings of t (3 U |t| ln 2 relative in p_j), the exponential's 2^-22, the
    sum's own error, four more roundings; the bracket p_j multiplies sums terms of at most |gn| + |gl| +
    |gh| (|t| ln 2 + log S + H) with 6 U, and carries the error of log S and H; two roundings of the sum with the
    former gradient."""
    p, lp = ref["p"], np.where(ref["p"] > 0, ref["logp"], 0.0)
    s = R.log_sum_bound(ref, x.shape[1])
    log_s = np.where(np.isfinite(ref["log_norm"]), ref["log_norm"] - ref["shift"], 0.0)[:, None]
    t = np.abs(lp) + log_s                                      # |x - m| / T
    rel = U * 3 * t + 2.0 ** -22 + s + 4 * U
    H = ref["entropy"][:, None]
    gl, gh, gn = (np.abs(g[k])[:, None] if g[k] is not None else 0.0 for k in ("logprob", "entropy", "log_norm"))
    bracket = gn + gl + gh * (t + log_s + H)
    own = p * (bracket * (rel + 6 * U) + gh * s * (2 + 2 * H))
    one_hot = gl * (np.arange(x.shape[1])[None] == token[:, None]) * 4 * U
    return (own + one_hot) / temperature + 4 * U * (np.abs(want) + np.abs(start)) + 1e-30


def upstream(rs, rows, which=("logprob", "entropy", "log_norm")):
    return {k: rs.randn(rows).astype(np.float32) if k in which else None for k in ("logprob", "entropy", "log_norm")}


def want_grad(ref, token, temperature, g, start):
    z = [np.zeros(len(token)) if g[k] is None else g[k].astype(np.float64) for k in ("logprob", "entropy", "log_norm")]
    return start.astype(np.float64) + R.token_logprob_grad(ref, token, temperature, *z)


@pytest.mark.parametrize("cols", [1, 2, 5, 33, 1000, 4099, 40000])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_gradient(cols, temperature):
    rs = np.random.RandomState(cols)
    rows = 7
    x, token = (rs.randn(rows, cols) * 3).astype(np.float32), rs.randint(0, cols, rows)
    token[2] = -1
    if cols > 4:
        x[1, : cols // 2] = -np.inf
        x[3] = -np.inf
        token[1] = 0                                 # a masked token
        token[4] = cols                              # outside: padding
    start = rs.randn(rows, cols).astype(np.float32)
    for which in (("logprob", "entropy", "log_norm"), ("logprob",), ("entropy",), ("log_norm",)):
        g = upstream(rs, rows, which)
        ref = R.token_logprob(x, token, temperature)
        want = want_grad(ref, token, temperature, g, start)
        _, got = backward(x, token, temperature, g, start)
        bound = grad_bound(ref, want, start, x, token, float(np.float32(temperature)), g)
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= bound).all(), (which, np.max(np.abs(got - want) / bound))
        if cols > 4:
            assert np.array_equal(got[3], start[3])   # the empty row's gradient stays as it was


@pytest.mark.parametrize("view,grad_view", [(strided, strided), (strided, None), (transposed, transposed), (None, strided)])
@pytest.mark.parametrize("cols", [301, 40001])
def test_gradient_of_views(view, grad_view, cols):
    rs = np.random.RandomState(8)
    x, token = rs.randn(5, cols).astype(np.float32), rs.randint(0, cols, 5)
    g, start = upstream(rs, 5), rs.randn(5, cols).astype(np.float32)
    ref = R.token_logprob(x, token, 1.0)
    want = want_grad(ref, token, 1.0, g, start)
    _, got = backward(x, token, 1.0, g, start, view, grad_view)
    assert (np.abs(got - want) <= grad_bound(ref, want, start, x, token, 1.0, g)).all()


def test_gradient_of_many_long_rows():
    """Enough rows for the longer pieces; a few of them against the formula."""
    torch = pytest.importorskip("torch")
    rows, cols = 2500, 65533
    torch.manual_seed(4)
    x, dx = torch.randn(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
    rs = np.random.RandomState(4)
    token, g = rs.randint(0, cols, rows).astype(np.int32), upstream(rs, rows)
    torch.cuda.synchronize()
    X = pb.Tensor.wrap_pointer(x.data_ptr(), [rows, cols], owner=x)
    X.c.requires_grad = True
    X.set_grad(pb.Tensor.wrap_pointer(dx.data_ptr(), [rows, cols], owner=dx))
    lp, H, L, st = (pb.Tensor(s) for s in ((rows,), (rows,), (rows,), (rows, 2)))
    T = pb.Tensor.from_numpy(token)
    pb.token_logprob(X, T, lp, entropy=H, log_norm=L, stats=st)
    for t, k in ((lp, "logprob"), (H, "entropy"), (L, "log_norm")):
        t.set_grad(pb.Tensor.from_numpy(g[k]))
    pb.token_logprob_backward(X, T, st, lp, entropy=H, log_norm=L)
    pb.synchronize()
    pick = np.r_[0, 1, 2, 1250, rows - 1]
    xs, ts, gs = x[pick].cpu().numpy(), token[pick], {k: v[pick] for k, v in g.items()}
    ref, start = R.token_logprob(xs, ts, 1.0), np.zeros((len(pick), cols), np.float32)
    want = want_grad(ref, ts, 1.0, gs, start)
    got = dx[pick].cpu().numpy()
    assert (np.abs(got - want) <= grad_bound(ref, want, start, xs, ts, 1.0, gs)).all()


def test_gradient_matches_differences():
    """Central differences of the forward in 64 bits."""
    rs = np.random.RandomState(9)
    x, token = rs.randn(3, 40).astype(np.float32), np.array([1, 5, 39])
    g = upstream(rs, 3)
    _, got = backward(x, token, 0.8, g, np.zeros_like(x))

    def value(v):
        r = R.token_logprob(v, token, 0.8)
        return sum((r[k] * g[k]).sum() for k in g)

    h, x64 = 1e-5, x.astype(np.float64)
    for r, c in [(0, 1), (0, 7), (1, 5), (2, 0), (2, 39)]:
        d = np.zeros_like(x64); d[r, c] = h
        assert abs((value(x64 + d) - value(x64 - d)) / (2 * h) - got[r, c]) < 1e-5


def test_gradient_far_from_zero():
    """Rows whose logits are all the lowest value, or lie around 10^6: softmax does not see the shift."""
    low = np.finfo(np.float32).min
    rs = np.random.RandomState(12)
    x = np.stack([np.full(300, low), 1e6 + np.round(rs.randn(300) * 8) / 4, np.where(np.arange(300) % 3, low, 1.0)]).astype(np.float32)
    token = np.array([4, 7, 9])
    g, start = upstream(rs, 3), rs.randn(3, 300).astype(np.float32)
    ref = R.token_logprob(x, token, 1.0)
    want = want_grad(ref, token, 1.0, g, start)
    _, got = backward(x, token, 1.0, g, start)
    assert (np.abs(got - want) <= grad_bound(ref, want, start, x, token, 1.0, g)).all()


def test_nothing_outside_the_rows_is_written():
    rs = np.random.RandomState(10)
    x, token = rs.randn(4, 77).astype(np.float32), np.arange(4)
    host = rs.randn(8, 82).astype(np.float32)
    big = pb.Tensor.from_numpy(host)
    dx = big.view((4, 77), (2 * 82, 1), offset=3)
    t = run(x, token)
    for k in ("logprob", "entropy", "log_norm"):
        t[k].attach_grad().copy_from(np.ones(4, np.float32))
    t["x"].set_grad(dx)
    pb.token_logprob_backward(t["x"], t["token"], t["stats"], t["logprob"], t["entropy"], t["log_norm"])
    after = big.numpy()
    mask = np.ones_like(host, bool); mask[::2, 3:80] = False
    assert np.array_equal(after[mask], host[mask])


def test_same_bits_on_every_run_on_another_stream_and_in_a_graph():
    torch = pytest.importorskip("torch")
    rs = np.random.RandomState(11)
    x, token = (rs.randn(40, 50001) * 2).astype(np.float32), rs.randint(0, 50001, 40)
    first = run(x, token, 0.9, 16)
    want = {k: first[k].numpy() for k in ("logprob", "entropy", "log_norm", "top_logprob", "top_index")}
    stream = torch.cuda.Stream()
    pb.synchronize()
    t = {k: first[k] for k in ("x", "token")}
    out = {k: pb.Tensor(v.shape, dtype=pb.INT32 if v.dtype == np.int32 else pb.FLOAT32) for k, v in want.items()}
    pb.synchronize()
    pb.lib.plast_b200_set_stream(C.c_void_p(stream.cuda_stream))
    try:
        call = lambda: pb.token_logprob(t["x"], t["token"], out["logprob"], out["entropy"], out["log_norm"],  # noqa: E731
                                        None, out["top_logprob"], out["top_index"], temperature=0.9)
        call()
        stream.synchronize()
        for k, v in want.items():
            assert np.array_equal(out[k].numpy(), v), k
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        x2 = (rs.randn(40, 50001) * 2).astype(np.float32)
        t["x"].copy_from(x2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = {k: out[k].numpy() for k in want}
    finally:
        pb.lib.plast_b200_set_stream(None)
    ref = R.token_logprob(x2, token, 0.9, 16)
    assert np.array_equal(got["top_index"], ref["top_index"])
    np.testing.assert_allclose(got["logprob"], ref["logprob"], rtol=2 * U, atol=R.log_sum_bound(ref, 50001))


def test_offsets_beyond_32_bits():
    torch = pytest.importorskip("torch")
    rows, cols = 3, 1 << 30                     # the third row starts at element 2^31
    x = torch.full((rows, cols), -30.0, device="cuda")
    x[2, 5], x[2, cols - 1], x[1, 7] = 2.0, 4.0, 3.0
    torch.cuda.synchronize()
    tx = pb.Tensor.wrap_pointer(x.data_ptr(), (rows, cols))
    tok = pb.Tensor.from_numpy(np.array([0, 7, cols - 1], np.int32))
    lp, tl, ti = pb.Tensor((rows,)), pb.Tensor((rows, 2)), pb.Tensor((rows, 2), dtype=pb.INT32)
    pb.token_logprob(tx, tok, lp, top_logprob=tl, top_index=ti)
    assert ti.numpy().tolist() == [[0, 1], [7, 0], [cols - 1, 5]]
    rest = np.exp(-30.0) * cols
    # about 2^12 additions in a thread
    np.testing.assert_allclose(lp.numpy()[1:], [3 - np.log(np.exp(3) + rest), 4 - np.log(np.exp(4) + np.exp(2) + rest)],
                               atol=2.0 ** -12 + 1e-5)


@pytest.mark.parametrize("cols", [8192, 16387, 50001, 70000])
@pytest.mark.parametrize("kind", ["random", "equal", "two_values", "late_ties", "zeros", "ascending", "descending", "masked"])
def test_many_long_rows(kind, cols):
    """More rows than resident CTAs: the persistent kernel, several rows per CTA, lists that overflow, empty rows."""
    rs = np.random.RandomState(cols)
    rows, i = 1300 if cols < 20000 else 620, np.arange(cols)
    x = {"random": lambda: rs.randn(rows, cols) * 3, "equal": lambda: np.broadcast_to(rs.randn(rows, 1), (rows, cols)),
         "two_values": lambda: np.broadcast_to((i * 7919 % 3 == 0) * 1.0, (rows, cols)),
         "late_ties": lambda: np.broadcast_to((i >= cols - 700) * 1.0, (rows, cols)),
         "zeros": lambda: np.broadcast_to(np.where(i % 3 == 1, -0.0, 0.0), (rows, cols)),
         "ascending": lambda: np.broadcast_to(i * 1e-3, (rows, cols)),
         "descending": lambda: np.broadcast_to(-i * 1e-3, (rows, cols)),
         "masked": lambda: np.where(rs.rand(rows, cols) < 0.999, -np.inf, rs.randn(rows, cols))}[kind]().astype(np.float32)
    x = np.array(x)
    x[5] = -np.inf
    x[7, 3] = np.nan
    token = rs.randint(-1, cols + 1, rows)
    for top in (0, 1, 5, 16) if cols < 16384 else (0, 1, 20, 32):
        t = run(x, token, 0.8, top)
        assert pb.last_kernel() == ("token_logprob_rows_top" if top else "token_logprob_rows")
        pick = np.r_[0:12, rs.randint(0, rows, 20), rows - 3:rows]
        ref = R.token_logprob(x[pick], token[pick], 0.8, top)
        # the merges and a thread's additions as in log_sum_bound, with up to cols / 256 additions
        bound = R.log_sum_bound(ref, cols) + cols / 256 * U
        for k in ("logprob", "log_norm", "entropy"):
            got = t[k].numpy()[pick]
            np.testing.assert_allclose(got, ref[k], rtol=2 * U, atol=bound * (1 if k != "entropy" else 1 + 2 * np.log(cols)), err_msg=k)
        if top:
            assert np.array_equal(t["top_index"].numpy()[pick], ref["top_index"])
            np.testing.assert_allclose(t["top_logprob"].numpy()[pick], ref["top_logprob"], rtol=2 * U, atol=bound)


def test_many_long_rows_of_a_view():
    rs = np.random.RandomState(3)
    x, token = rs.randn(620, 8201).astype(np.float32), rs.randint(0, 8201, 620)
    for view in (strided, transposed):
        check(run(x, token, 1.3, 6, view=view), x, token, 1.3, 6)
        assert pb.last_kernel() == "token_logprob_rows_top"


@pytest.mark.parametrize("rows, cols, top", [(591, 16384, 8), (600, 4096, 0), (600, 4095, 0), (600, 8191, 1), (1300, 16383, 32), (1300, 300, 3),
                                             (297, 8192, 0), (296, 8192, 0), (300, 8191, 5), (74, 16384, 1), (73, 16384, 1), (80, 65537, 4),
                                             (1, 8192, 17), (3, 40960, 32), (3, 40961, 32), (2, 8191, 20)])
def test_on_both_sides_of_the_rule(rows, cols, top):
    rs = np.random.RandomState(rows + cols)
    x, token = rs.randn(rows, cols).astype(np.float32), rs.randint(0, cols, rows)
    check(run(x, token, 1.0, top), x, token, 1.0, top)


@pytest.mark.parametrize("rows, cols, top, by_rows", [
    (1, 8192, 17, False), (1, 40960, 32, False), (24, 24000, 32, False), (148, 16384, 16, False), (148, 16384, 23, False),
    (7, 16384, 20, False), (8, 24576, 17, True), (8, 24577, 17, False), (148, 32768, 22, True), (148, 32769, 22, False),
    (149, 8192, 9, True), (149, 8192, 8, False), (200, 65536, 24, True), (200, 65537, 24, False), (296, 8192, 25, False),
    (297, 8192, 32, True), (297, 8191, 32, False)])
def test_few_rows_go_where_they_are_measured_to_be_faster(rows, cols, top, by_rows):
    """The borders of the rule on a GPU of 148 SMs; the results on both sides."""
    torch = pytest.importorskip("torch")
    rs = np.random.RandomState(rows + cols)
    x, token = rs.randn(rows, cols).astype(np.float32), rs.randint(0, cols, rows)
    t = run(x, token, 1.0, top)
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert pb.last_kernel() == ("token_logprob_rows_top" if by_rows else "token_logprob_top")
    check(t, x, token, 1.0, top)
