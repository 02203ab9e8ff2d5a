"""rotary and qk_norm_rotary against their definitions in 64 bits: head sizes from two to 1024, both pair layouts,
parts of a head, layouts of the dims, far positions, weights shared by queries and keys, in place, graphs."""
import ctypes as C

import numpy as np
import pytest

import lm_reference as R
import plast_b200 as pb

pytestmark = pytest.mark.gpu
U = R.U
# cos and sin of an angle reduced to [-pi/4, pi/4] in 64 bits: the argument's rounding (U), the functions'
# 2 ulp (4 U), the amplitude (U); then a product and a sum: at most 8 U of |a| + |b|
TURN = 8 * U


def data(rs, *shape):
    return rs.randn(*shape).astype(np.float32)


def pair_sum(x, n, interleaved):
    """|a| + |b| of every element's pair (its own magnitude where it is not turned)."""
    return R.rotate(np.abs(x), np.zeros(x.shape[:-1]), np.zeros(n, np.float32), interleaved) + \
        np.abs(R.rotate(np.abs(x), np.ones(x.shape[:-1]) * 1.0, np.full(n, np.pi / 2, np.float32), interleaved))


SHAPES = [((2, 3, 4, 128), 64), ((1, 1, 1, 2), 1), ((2, 5, 3, 80), 40), ((3, 2, 2, 96), 24), ((2, 2, 2, 64), 1),
          ((2, 3, 5, 7), 2), ((1, 4, 2, 257), 100), ((2, 1, 3, 1024), 512), ((1, 2, 1, 1023), 511), ((2, 2, 2, 512), 256),
          ((1, 300, 9, 256), 128), ((4, 2, 16, 72), 20)]


@pytest.mark.parametrize("shape,n", SHAPES)
@pytest.mark.parametrize("layout", [pb.ROTARY_HALVES, pb.ROTARY_INTERLEAVED])
def test_forward_and_backward(shape, n, layout):
    rs = np.random.RandomState(n)
    x, dy, start = data(rs, *shape), data(rs, *shape), data(rs, *shape)
    pos = rs.randint(0, 100000, shape[:2] + (1,)).astype(np.int32)
    freq = (10000.0 ** (-np.arange(n) / n)).astype(np.float32)
    tx, tp, tf, ty = pb.Tensor.from_numpy(x, requires_grad=True), pb.Tensor.from_numpy(pos), pb.Tensor.from_numpy(freq), \
        pb.Tensor(shape, requires_grad=True)
    tx.grad.copy_from(start)
    ty.grad.copy_from(dy)
    pb.forward("rotary", [tx, tp, tf], ty, dim=layout, fval=1.25)
    pb.backward("rotary", [tx, tp, tf], ty, dim=layout, fval=1.25)
    want = R.rotate(x.astype(np.float64), pos, freq, layout == 1, 1.25)
    assert (np.abs(ty.numpy() - want) <= 1.25 * TURN * pair_sum(x, n, layout == 1) + U * np.abs(want)).all()
    back = R.rotate(dy.astype(np.float64), pos, freq, layout == 1, 1.25, sign=-1.0)
    bound = 1.25 * TURN * pair_sum(dy, n, layout == 1) + 2 * U * (np.abs(back) + np.abs(start))
    assert (np.abs(tx.grad.numpy() - (start + back)) <= bound).all()
    if 2 * n < shape[-1]:
        assert np.array_equal(ty.numpy()[..., 2 * n:], x[..., 2 * n:])      # passed on unchanged


@pytest.mark.parametrize("position", [0, 1, -5, 1 << 20, 2**31 - 1, -2**31])
def test_far_positions_keep_their_angle(position):
    x = np.ones((1, 1, 128), np.float32)
    freq = (500000.0 ** (-np.arange(64) / 64)).astype(np.float32)
    pos = np.array([[position]], np.int32)
    out = pb.Tensor(x.shape)
    pb.forward("rotary", [pb.Tensor.from_numpy(x), pb.Tensor.from_numpy(pos), pb.Tensor.from_numpy(freq)], out, fval=1.0)
    want = R.rotate(x.astype(np.float64), pos, freq)
    # numpy's own angle is rounded to 64 bits: 2^31 * 2^-53
    assert np.abs(out.numpy() - want).max() <= 2 * TURN + 2.0 ** -21


@pytest.mark.parametrize("dims", ["bthd", "bhtd", "packed", "unaligned", "head_strided", "positions_of_batch"])
def test_layouts_of_the_dims(dims):
    rs = np.random.RandomState(3)
    B, T, H, D, n = 2, 5, 3, 32, 16
    freq = (100.0 ** (-np.arange(n) / n)).astype(np.float32)
    x = data(rs, B, T, H, D)
    pos = rs.randint(0, 1000, (B, T, 1)).astype(np.int32)
    tp, tf = pb.Tensor.from_numpy(pos), pb.Tensor.from_numpy(freq)
    want = R.rotate(x.astype(np.float64), pos, freq)
    if dims == "bthd":
        tx, ty = pb.Tensor.from_numpy(x), pb.Tensor(x.shape)
    elif dims == "bhtd":                                   # stored heads first, seen as [B, T, H, D]
        tx = pb.Tensor.from_numpy(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).transpose(1, 2)
        ty = pb.Tensor((B, H, T, D)).transpose(1, 2)
    elif dims == "packed":                                 # queries inside a row that also holds other things
        host = np.zeros((B, T, 5 * D * H), np.float32)
        host[..., D * H:2 * D * H] = x.reshape(B, T, -1)
        tx = pb.Tensor.from_numpy(host).view(x.shape, (T * 5 * D * H, 5 * D * H, D, 1), offset=D * H)
        ty = pb.Tensor(x.shape)
    elif dims == "unaligned":
        host = np.concatenate([np.zeros(1, np.float32), x.ravel()])
        tx = pb.Tensor.from_numpy(host).view(x.shape, pb.contiguous_strides(x.shape), offset=1)
        ty = pb.Tensor(x.shape)
    elif dims == "head_strided":                           # the head's elements are not adjacent
        tx = pb.Tensor.from_numpy(np.ascontiguousarray(x.transpose(3, 0, 1, 2))).view(x.shape, (T * H, H, 1, B * T * H))
        ty = pb.Tensor(x.shape)
    else:                                                  # one position per time step, all batches alike
        pos = pos[:1]
        tp = pb.Tensor.from_numpy(pos[0])
        want = R.rotate(x.astype(np.float64), pos, freq)
        tx, ty = pb.Tensor.from_numpy(x), pb.Tensor(x.shape)
    pb.forward("rotary", [tx, tp, tf], ty, dim=0, fval=1.0)
    assert (np.abs(ty.numpy() - want) <= TURN * pair_sum(x, n, False) + U * np.abs(want)).all()


def test_in_place_and_empty():
    rs = np.random.RandomState(4)
    x, pos, freq = data(rs, 6, 2, 64), np.arange(6, dtype=np.int32)[:, None], np.array([0.5, 0.25], np.float32)
    tx, tp, tf = pb.Tensor.from_numpy(x), pb.Tensor.from_numpy(pos), pb.Tensor.from_numpy(freq)
    out = pb.Tensor(x.shape)
    pb.forward("rotary", [tx, tp, tf], out, fval=1.0)
    pb.forward("rotary", [tx, tp, tf], tx, fval=1.0)
    assert np.array_equal(tx.numpy(), out.numpy())
    pb.forward("rotary", [pb.Tensor((0, 2, 64)), pb.Tensor((0, 1), dtype=pb.INT32), tf], pb.Tensor((0, 2, 64)), fval=1.0)


def qk_case(rs, qs, ks, n, weights=True):
    D = qs[-1]
    v = {"q": data(rs, *qs), "k": data(rs, *ks) if ks else None, "n": n, "pos": rs.randint(0, 4096, qs[:-2] + (1,)).astype(np.int32),
         "freq": (10000.0 ** (-np.arange(n) / n)).astype(np.float32)}
    for s in ("q", "k"):
        v[s + "w"] = (1 + 0.3 * data(rs, D)) if weights and v[s] is not None else None
        if v[s] is not None:
            v["d" + s] = data(rs, *v[s].shape)
            v["start_" + s] = data(rs, *v[s].shape)
            v["start_" + s + "w"] = data(rs, D)
    return v


def qk_run(v, layout, epsilon, amplitude=1.0):
    t = {"pos": pb.Tensor.from_numpy(v["pos"]), "freq": pb.Tensor.from_numpy(v["freq"])}
    for s in ("q", "k"):
        t[s] = t[s + "w"] = t[s + "o"] = None
        if v[s] is None:
            continue
        t[s] = pb.Tensor.from_numpy(v[s], requires_grad=True)
        t[s].grad.copy_from(v["start_" + s])
        t[s + "o"] = pb.Tensor(v[s].shape, requires_grad=True)
        t[s + "o"].grad.copy_from(v["d" + s])
        if v[s + "w"] is not None:
            t[s + "w"] = pb.Tensor.from_numpy(v[s + "w"], requires_grad=True)
            t[s + "w"].grad.copy_from(v["start_" + s + "w"])
    args = [t[k] for k in ("q", "k", "qw", "kw", "pos", "freq", "qo", "ko")]
    pb.qk_norm_rotary(*args, epsilon=epsilon, layout=layout, amplitude=amplitude)
    pb.qk_norm_rotary_backward(*args, epsilon=epsilon, layout=layout, amplitude=amplitude)
    return t


def qk_check(v, t, layout, epsilon, amplitude=1.0):
    inter = layout == pb.ROTARY_INTERLEAVED
    for s in ("q", "k"):
        if v[s] is None:
            continue
        x, D = v[s].astype(np.float64), v[s].shape[-1]
        w = np.ones(D) if v[s + "w"] is None else v[s + "w"].astype(np.float64)
        n, r, u = R.qk_norm(x, w, epsilon)
        want = R.rotate(u, v["pos"], v["freq"], inter, amplitude)
        # r: the sum of squares (D / lanes + 5 additions, all positive: at most 40 U), halved by the root, and four
        # roundings; n and u one each
        norm = 28 * U
        got = t[s + "o"].numpy()
        assert (np.abs(got - want) <= amplitude * (TURN + norm) * pair_sum(u, v["n"], inter) + U * np.abs(want)).all()
        du = R.rotate(v["d" + s].astype(np.float64), v["pos"], v["freq"], inter, amplitude, sign=-1.0)
        dx, dw = R.qk_norm_rotary_grad(x, w, epsilon, du)
        du_err = amplitude * TURN * pair_sum(v["d" + s], v["n"], inter) + U * np.abs(du)
        dot = np.abs(du * w * n).mean(axis=-1, keepdims=True)            # bounds |mean(dn n)| and carries its error
        dot_err = (du_err * np.abs(w * n)).mean(axis=-1, keepdims=True) + dot * (40 * U + norm)
        bound = r * (du_err * np.abs(w) + np.abs(n) * (dot_err + dot * (norm + 4 * U)) + np.abs(du * w) * (norm + 4 * U))
        start = v["start_" + s]
        assert (np.abs(t[s].grad.numpy() - (start + dx)) <= bound + 2 * U * (np.abs(dx) + np.abs(start))).all()
        if v[s + "w"] is not None:
            heads = x.reshape(-1, D).shape[0]
            each = np.abs(du * n).reshape(-1, D)
            bound = (du_err * np.abs(n)).reshape(-1, D).sum(axis=0) + each.sum(axis=0) * (norm + (min(heads, 200) + 80) * U)
            start = v["start_" + s + "w"]
            assert (np.abs(t[s + "w"].grad.numpy() - (start + dw)) <= bound + 2 * U * (np.abs(dw) + np.abs(start))).all()


QK = [((2, 3, 4, 128), (2, 3, 2, 128), 64), ((1, 1, 1, 2), (1, 1, 1, 2), 1), ((2, 7, 3, 80), (2, 7, 1, 80), 20),
      ((3, 5, 5, 33), (3, 5, 2, 33), 11), ((2, 2, 2, 256), (2, 2, 2, 256), 128), ((1, 3, 2, 1024), (1, 3, 1, 1024), 512),
      ((1, 2, 3, 1023), (1, 2, 2, 1023), 300), ((2, 40, 16, 64), (2, 40, 2, 64), 32), ((2, 9, 6, 512), None, 100),
      ((2, 700, 8, 128), (2, 700, 2, 128), 64)]


@pytest.mark.parametrize("qs,ks,n", QK)
@pytest.mark.parametrize("layout", [pb.ROTARY_HALVES, pb.ROTARY_INTERLEAVED])
def test_qk_norm(qs, ks, n, layout):
    v = qk_case(np.random.RandomState(n), qs, ks, n)
    qk_check(v, qk_run(v, layout, 1e-6), layout, 1e-6)


def test_qk_norm_without_weights_and_with_amplitude():
    v = qk_case(np.random.RandomState(5), (3, 4, 6, 64), (3, 4, 2, 64), 16, weights=False)
    qk_check(v, qk_run(v, 0, 1e-3, 0.75), 0, 1e-3, 0.75)


def test_rows_of_zeros_and_of_large_values():
    v = qk_case(np.random.RandomState(6), (2, 2, 2, 128), (2, 2, 1, 128), 64)
    v["q"][0, 0, 0] = 0.0
    v["q"][0, 1, 0] *= 1e15
    v["k"][1, 0, 0] *= 1e-15
    qk_check(v, qk_run(v, 0, 1e-6), 0, 1e-6)
    v["q"][1, 1, 1, 3] = np.nan                                 # one head's business only
    out = qk_run(v, 0, 1e-6)["qo"].numpy()
    bad = np.isnan(out).any(axis=-1)
    assert bad[1, 1, 1] and bad.sum() == 1


def test_one_weight_for_queries_and_keys_receives_both_gradients():
    rs = np.random.RandomState(7)
    v = qk_case(rs, (2, 6, 4, 64), (2, 6, 2, 64), 32)
    v["kw"] = v["qw"]
    t = qk_run(v, 0, 1e-6)                                      # separate tensors: the two parts
    parts = (t["qw"].grad.numpy() - v["start_qw"]) + (t["kw"].grad.numpy() - v["start_kw"])
    w = pb.Tensor.from_numpy(v["qw"], requires_grad=True)
    args = [t["q"], t["k"], w, w, t["pos"], t["freq"], t["qo"], t["ko"]]
    pb.qk_norm_rotary_backward(*args)
    scale = np.abs(v["dq"]).sum() + np.abs(v["dk"]).sum()
    assert np.abs(w.grad.numpy() - parts).max() <= 20 * U * scale


def test_weight_gradient_alone():
    v = qk_case(np.random.RandomState(10), (2, 6, 4, 64), (2, 6, 2, 64), 32)
    t = qk_run(v, 0, 1e-6)
    q, w = pb.Tensor.from_numpy(v["q"]), pb.Tensor.from_numpy(v["qw"], requires_grad=True)
    w.grad.copy_from(v["start_qw"])
    pb.qk_norm_rotary_backward(q, None, w, None, t["pos"], t["freq"], t["qo"], None)
    assert np.array_equal(w.grad.numpy(), t["qw"].grad.numpy())


def test_gradients_match_differences():
    rs = np.random.RandomState(8)
    v = qk_case(rs, (1, 2, 2, 16), (1, 2, 1, 16), 8)
    for s in ("q", "k"):
        v["start_" + s][:], v["start_" + s + "w"][:] = 0, 0
    t = qk_run(v, 1, 1e-6)

    def value(q, w):
        u = R.qk_norm(q, w, 1e-6)[2]
        return (R.rotate(u, v["pos"], v["freq"], True) * v["dq"]).sum()

    q, w, h = v["q"].astype(np.float64), v["qw"].astype(np.float64), 1e-5
    for at in [(0, 0, 0, 0), (0, 1, 1, 15), (0, 0, 1, 8)]:
        d = np.zeros_like(q); d[at] = h
        assert abs((value(q + d, w) - value(q - d, w)) / (2 * h) - t["q"].grad.numpy()[at]) < 1e-4
    for i in (0, 7, 15):
        d = np.zeros_like(w); d[i] = h
        assert abs((value(q, w + d) - value(q, w - d)) / (2 * h) - t["qw"].grad.numpy()[i]) < 1e-4


def test_same_bits_again_and_in_a_graph():
    torch = pytest.importorskip("torch")
    rs = np.random.RandomState(9)
    v = qk_case(rs, (2, 300, 8, 128), (2, 300, 2, 128), 64)
    t = qk_run(v, 0, 1e-6)
    first = {k: t[k].grad.numpy() for k in ("q", "k", "qw", "kw")}
    again = qk_run(v, 0, 1e-6)
    for k, g in first.items():
        assert np.array_equal(again[k].grad.numpy(), g), k
    args = [t[k] for k in ("q", "k", "qw", "kw", "pos", "freq", "qo", "ko")]
    stream = torch.cuda.Stream()
    pb.synchronize()
    pb.lib.plast_b200_set_stream(C.c_void_p(stream.cuda_stream))
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            pb.qk_norm_rotary(*args)
            pb.qk_norm_rotary_backward(*args)
        for _ in range(2):
            for s in ("q", "k"):
                t[s].grad.copy_from(v["start_" + s])
                t[s + "w"].grad.copy_from(v["start_" + s + "w"])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for k, g in first.items():
                assert np.array_equal(t[k].grad.numpy(), g), k
    finally:
        pb.lib.plast_b200_set_stream(None)


def test_offsets_beyond_32_bits():
    torch = pytest.importorskip("torch")
    x = torch.zeros((3, 1 << 24, 64), device="cuda")          # the third slab starts at element 2^31
    x[2, -1] = torch.arange(64, device="cuda")
    torch.cuda.synchronize()
    tx = pb.Tensor.wrap_pointer(x.data_ptr(), (3, 1 << 24, 64))
    pos = pb.Tensor.from_numpy(np.array([[0], [1], [3]], np.int32))
    freq = np.array([1.0, 0.1], np.float32)
    pb.forward("rotary", [tx, pos, pb.Tensor.from_numpy(freq)], tx, dim=1, fval=1.0)
    pb.synchronize()
    want = R.rotate(np.arange(64.0)[None], np.array([3]), freq, True)[0]
    np.testing.assert_allclose(x[2, -1].cpu().numpy(), want, atol=1e-5)


def test_heads_of_one_fused_row():
    """Queries, keys and values side by side in a row, as one product gives them: normed and rotated in place, and the
    gradients added into the slices of one row of gradients. The same bits as with buffers of their own."""
    rs = np.random.RandomState(12)
    v = qk_case(rs, (2, 30, 6, 64), (2, 30, 2, 64), 32)
    t = qk_run(v, 0, 1e-6)
    B, T, H, K, D = 2, 30, 6, 2, 64
    row = (H + 2 * K) * D

    def fused(q, k):
        host = data(rs, B, T, row)
        host[..., :H * D], host[..., H * D:(H + K) * D] = q.reshape(B, T, -1), k.reshape(B, T, -1)
        whole = pb.Tensor.from_numpy(host)
        return host, whole, [whole.view((B, T, n, D), (T * row, row, D, 1), offset=o) for n, o in ((H, 0), (K, H * D))]

    def same(whole, host, q, k):
        got = whole.numpy()
        assert np.array_equal(got[..., :H * D], q.reshape(B, T, -1)) and np.array_equal(got[..., H * D:(H + K) * D], k.reshape(B, T, -1))
        assert np.array_equal(got[..., (H + K) * D:], host[..., (H + K) * D:])      # the values

    host, whole, (q, k) = fused(v["q"], v["k"])
    dhost, dwhole, (dq, dk) = fused(v["start_q"], v["start_k"])
    q.set_grad(dq)
    k.set_grad(dk)
    weights = [pb.Tensor.from_numpy(v[s], requires_grad=True) for s in ("qw", "kw")]
    pb.qk_norm_rotary_backward(q, k, *weights, t["pos"], t["freq"], t["qo"], t["ko"], epsilon=1e-6)
    same(dwhole, dhost, t["q"].grad.numpy(), t["k"].grad.numpy())
    pb.qk_norm_rotary(q, k, t["qw"], t["kw"], t["pos"], t["freq"], q, k, epsilon=1e-6)
    same(whole, host, t["qo"].numpy(), t["ko"].numpy())
    # the rotation alone, of the keys in place, and its gradient over the gradient of its output
    _, _, (_, k) = fused(v["q"], v["k"])
    out = pb.Tensor((B, T, K, D))
    pb.forward("rotary", [pb.Tensor.from_numpy(v["k"]), t["pos"], t["freq"]], out, fval=1.0)
    pb.forward("rotary", [k, t["pos"], t["freq"]], k, fval=1.0)
    assert np.array_equal(k._base.numpy()[..., H * D:(H + K) * D], out.numpy().reshape(B, T, -1))
    x, y = pb.Tensor.from_numpy(v["k"], requires_grad=True), pb.Tensor((B, T, K, D), requires_grad=True)
    y.grad.copy_from(v["dk"])
    x.grad.copy_from(v["dk"])
    pb.backward("rotary", [x, t["pos"], t["freq"]], y, fval=1.0)
    want = x.grad.numpy()
    x.set_grad(y.grad)
    pb.backward("rotary", [x, t["pos"], t["freq"]], y, fval=1.0)
    assert np.array_equal(x.grad.numpy(), want)


def test_a_side_without_gradients_is_not_looked_at():
    """Keys that want no gradient: what their output's gradient lies over is of no matter."""
    v = qk_case(np.random.RandomState(13), (2, 5, 4, 64), (2, 5, 4, 64), 32)
    t = qk_run(v, 0, 1e-6)
    want = t["q"].grad.numpy()
    q, k, ko = pb.Tensor.from_numpy(v["q"], requires_grad=True), pb.Tensor.from_numpy(v["k"]), pb.Tensor(v["k"].shape)
    q.grad.copy_from(v["start_q"])
    ko.set_grad(q.grad)
    qw, kw = pb.Tensor.from_numpy(v["qw"]), pb.Tensor.from_numpy(v["kw"])
    pb.qk_norm_rotary_backward(q, k, qw, kw, t["pos"], t["freq"], t["qo"], ko)
    assert np.array_equal(q.grad.numpy(), want)
