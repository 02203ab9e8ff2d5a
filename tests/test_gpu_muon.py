"""orthogonalise and muon_step against the Newton-Schulz definition in 64 bits: sizes around the tiles, wide and tall,
many matrices in a call, zeros, NaN, extreme scales, any number of steps, momenta of either owner, graphs."""
import ctypes as C

import numpy as np
import pytest

import lm_reference as R
import plast_b200 as pb
from plast_b200 import optim as O

pytestmark = pytest.mark.gpu
U = R.U


@pytest.fixture(autouse=True, params=["built_in", "fused", "pairs"])
def route(request):
    """Every test by the built-in choice, by the fused steps and by the pairs of CTAs."""
    pb.lib.plast_b200_tune(12, {"built_in": -1, "fused": 0, "pairs": 1}[request.param])
    yield request.param
    pb.lib.plast_b200_tune(12, -1)
    assert pb.lib.plast_b200_muon_status() == 0


def tolerance(m, steps=5):
    """Frobenius error relative to the result's. A product whose terms carry 2^-22 adds at most about 20 * 2^-22 of
    |X|_F per step (3.4 + 4.8 * 1.45 + 2 * 2.03 * 2.1, times 1.2, rounded up); an error grows at most by
    max |f'| = 4 in a step (divided differences of the odd polynomial on [-1.21, 1.21]); |X|_F starts at 1 and ends
    above 0.6 sqrt(rank) where the singular values have been lifted. The errors of five steps: (4^5 - 1) / 3 * 20."""
    return 20 * (4.0 ** steps - 1) / 3 * 2.0 ** -22 / (0.6 * np.sqrt(m)) + 4 * U


def orth(xs, steps=5, epsilon=1e-7, in_place=False):
    ins = [pb.Tensor.from_numpy(x) for x in xs]
    outs = ins if in_place else [pb.Tensor(x.shape) for x in xs]
    O.orthogonalise(ins, outs, steps, epsilon)
    return [t.numpy() for t in outs]


def rel(got, want):
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 5), (16, 16), (64, 64), (65, 63), (127, 129), (128, 128), (129, 128),
          (130, 260), (257, 100), (33, 1000), (1000, 33), (300, 520), (256, 512), (640, 384)]


@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalise(shape):
    rs = np.random.RandomState(shape[0])
    x = rs.randn(*shape).astype(np.float32)
    got = orth([x])[0]
    want = R.orthogonalise(x)
    assert rel(got, want) <= tolerance(min(shape)), rel(got, want)


@pytest.mark.parametrize("shape", [(128, 128), (256, 640), (700, 300), (512, 512), (100, 4000)])
def test_as_exact_as_products_in_fp32(shape):
    """The same steps in numpy fp32 (products with fp32 operands and sums) are the yardstick."""
    rs = np.random.RandomState(1)
    x = rs.randn(*shape).astype(np.float32)
    a, b, c = np.float32(3.4445), np.float32(-4.7750), np.float32(2.0315)
    y = (x.T if shape[0] > shape[1] else x) / np.float32(np.linalg.norm(x.astype(np.float64)))
    for _ in range(5):
        g = y @ y.T
        y = a * y + (b * g + c * (g @ g)) @ y
    y = y.T if shape[0] > shape[1] else y
    want = R.orthogonalise(x)
    assert rel(orth([x])[0], want) <= 2 * rel(y, want) + 2.0 ** -21


def test_orthogonal_rows():
    x = np.random.RandomState(2).randn(96, 400).astype(np.float32)
    s = np.linalg.svd(orth([x])[0].astype(np.float64), compute_uv=False)
    assert s.min() > 0.6 and s.max() < 1.2026


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 9])
def test_number_of_steps(steps):
    rs = np.random.RandomState(steps)
    xs = [rs.randn(40, 70).astype(np.float32), rs.randn(70, 40).astype(np.float32)]
    for x, got in zip(xs, orth(xs, steps)):
        want = R.orthogonalise(x, steps)
        # beyond five steps the values stay in the polynomial's attractor: one more factor of 4 each
        assert rel(got, want) <= 20 * (4.0 ** steps) * 2.0 ** -22 + 4 * U, steps


def test_more_than_two_dims_count_as_rows_times_the_rest():
    x = np.random.RandomState(3).randn(24, 3, 5, 5).astype(np.float32)
    got = orth([x])[0]
    want = R.orthogonalise(x.reshape(24, 75)).reshape(x.shape)
    assert rel(got, want) <= tolerance(24)


@pytest.mark.parametrize("in_place", [False, True])
def test_many_matrices_in_one_call(in_place):
    rs = np.random.RandomState(4)
    xs = [rs.randn(int(r), int(c)).astype(np.float32) for r, c in rs.randint(1, 200, (75, 2))]
    xs.insert(10, np.zeros((0, 5), np.float32))
    xs.insert(20, rs.randn(400, 300).astype(np.float32))
    for x, got in zip(xs, orth(xs, in_place=in_place)):
        assert got.shape == x.shape
        if x.size:
            assert rel(got, R.orthogonalise(x)) <= tolerance(min(x.shape))


def test_zeros_nan_and_scales_stay_in_their_matrices():
    rs = np.random.RandomState(5)
    base = rs.randn(60, 90).astype(np.float32)
    bad = base.copy(); bad[3, 4] = np.nan
    inf = base.copy(); inf[3, 4] = np.inf
    one = np.outer(rs.randn(60), rs.randn(90)).astype(np.float32)
    xs = [base, np.zeros((60, 90), np.float32), bad, inf, base * np.float32(1e-25), base * np.float32(1e30), one]
    got = orth(xs, epsilon=0.0)
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all() and np.isnan(got[3]).all()   # 0 / 0, NaN, inf
    want = R.orthogonalise(base, epsilon=0.0)
    for i in (0, 4, 5):
        assert rel(got[i], want) <= tolerance(60), i
    assert rel(got[6], R.orthogonalise(one, epsilon=0.0)) <= tolerance(1)
    got = orth(xs[:2] + [base * np.float32(1e-25)])
    assert not got[1].any()
    assert rel(got[2], R.orthogonalise(xs[4])) <= tolerance(1) * 1e7   # far below epsilon: stays tiny
    assert np.abs(got[2]).max() < 1e-12


def test_the_same_call_gives_the_same_bits():
    rs = np.random.RandomState(6)
    xs = [rs.randn(r, c).astype(np.float32) for r, c in [(200, 300), (130, 128), (500, 90), (64, 2500)]]
    first = orth(xs)
    for _ in range(3):
        for a, b in zip(first, orth(xs)):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("shape", [(64, 4096), (2000, 100), (300, 3000), (512, 512), (130, 1920)])
def test_long_products_whose_k_is_split(shape):
    rs = np.random.RandomState(shape[1])
    x = rs.randn(*shape).astype(np.float32)
    want = R.orthogonalise(x)
    assert rel(orth([x])[0], want) <= tolerance(min(shape))


SETS = {"mixed": [(64, 64), (100, 300), (300, 100), (33, 65)], "tall": [(257, 64)], "image": [(16, 3, 5, 5), (8, 8)]}


def step_reference(w, v, g, lr, mu, wd, nesterov, scale):
    v = mu * v + g
    u = g + mu * v if nesterov else v
    r, c = w.shape[0], w[0].size
    s = {0: np.sqrt(max(1.0, r / c)), 1: 0.2 * np.sqrt(max(r, c)), 2: 1.0}[scale]
    o = R.orthogonalise(u.reshape(r, c)).reshape(w.shape)
    return w * (1 - lr * wd) - lr * s * o, v, lr * s * np.linalg.norm(o)


@pytest.mark.parametrize("kind", sorted(SETS))
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", [O.MUON_SCALE_ASPECT, O.MUON_SCALE_RMS, O.MUON_SCALE_NONE])
def test_three_steps(kind, nesterov, scale):
    rs = np.random.RandomState(7)
    shapes = SETS[kind]
    ws = [rs.randn(*s).astype(np.float32) for s in shapes]
    params = [pb.Tensor.from_numpy(w, requires_grad=True) for w in ws] + [None, pb.Tensor.from_numpy(np.ones((4, 4), np.float32))]
    lr, mu, wd = (float(np.float32(v)) for v in (0.05, 0.9, 0.1))
    opt = O.Muon.create(lr=lr, momentum=mu, weight_decay=wd, nesterov=nesterov, scale=scale)
    want = [(w.astype(np.float64), np.zeros(w.shape)) for w in ws]
    off = [0.0] * len(ws)
    for _ in range(3):
        for i, p in enumerate(params[:-2]):
            g = rs.randn(*ws[i].shape).astype(np.float32)
            p.grad.copy_from(g)
            w, v, size = step_reference(*want[i], g.astype(np.float64), lr, mu, wd, nesterov, scale)
            want[i] = (w, v)
            # the update's error, three roundings of the weight, and the momentum's rounding through the step
            off[i] += size * (tolerance(min(ws[i].shape[0], ws[i][0].size)) + 4 * U) + 3 * U * np.linalg.norm(w)
        O.step(opt, params)
    for i, p in enumerate(params[:-2]):
        assert np.linalg.norm(p.numpy() - want[i][0]) <= off[i], i
        m = pb.Tensor.wrap_pointer(opt.m[i].contents.data, ws[i].shape)
        m._storage_elems = ws[i].size
        np.testing.assert_allclose(m.numpy(), want[i][1], rtol=0, atol=8 * U * np.abs(want[i][1]).max())
    assert np.array_equal(params[-1].numpy(), np.ones((4, 4), np.float32))       # no gradient: untouched
    O.release_state(opt)


def test_momenta_of_the_caller():
    rs = np.random.RandomState(8)
    w, v, g = (rs.randn(70, 50).astype(np.float32) for _ in range(3))
    p, m = pb.Tensor.from_numpy(w, requires_grad=True), pb.Tensor.from_numpy(v)
    p.grad.copy_from(g)
    opt = O.Muon.create(lr=0.1, momentum=0.5, moments=[m])
    O.step(opt, [p])
    want_w, want_v, size = step_reference(w.astype(np.float64), v.astype(np.float64), g.astype(np.float64), 0.1, 0.5, 0.0, True, 0)
    assert np.linalg.norm(p.numpy() - want_w) <= size * (tolerance(50) + 4 * U) + 3 * U * np.linalg.norm(w)
    np.testing.assert_allclose(m.numpy(), want_v, rtol=0, atol=4 * U * 8)


def test_graph_replays_match_eager_steps():
    torch = pytest.importorskip("torch")
    rs = np.random.RandomState(9)
    shapes = [(96, 160), (200, 64), (130, 130)]
    ws, gs = [rs.randn(*s).astype(np.float32) for s in shapes], [rs.randn(*s).astype(np.float32) for s in shapes]

    def make():
        ps = [pb.Tensor.from_numpy(w, requires_grad=True) for w in ws]
        for p, g in zip(ps, gs):
            p.grad.copy_from(g)
        ms = [pb.Tensor(s) for s in shapes]
        for m in ms:
            m.zero_()
        return ps, O.Muon.create(lr=0.1, moments=ms)

    ps, opt = make()
    for _ in range(3):
        O.step(opt, ps)
    want = [p.numpy() for p in ps]
    qs, opt2 = make()
    stream = torch.cuda.Stream()
    pb.synchronize()
    pb.lib.plast_b200_set_stream(C.c_void_p(stream.cuda_stream))
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            O.step(opt2, qs)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        got = [q.numpy() for q in qs]
    finally:
        pb.lib.plast_b200_set_stream(None)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


def test_two_streams_and_two_graphs_at_once():
    """Calls on two streams, then two captured calls replayed on two streams, neither waiting for the other."""
    torch = pytest.importorskip("torch")
    rs = np.random.RandomState(19)
    xs = [[pb.Tensor.from_numpy(rs.randn(*s).astype(np.float32)) for s in shapes]
          for shapes in ([(520, 900), (130, 70)], [(1000, 600)])]
    want = []
    for group in xs:
        outs = [pb.Tensor(x.shape) for x in group]
        O.orthogonalise(group, outs)
        want.append([o.numpy() for o in outs])
    outs = [[pb.Tensor(x.shape) for x in group] for group in xs]
    streams, graphs = [torch.cuda.Stream() for _ in xs], []

    def check():
        torch.cuda.synchronize()
        for group, w in zip(outs, want):
            for o, v in zip(group, w):
                assert np.array_equal(o.numpy(), v)
                o.zero_()
        torch.cuda.synchronize()

    pb.synchronize()
    try:
        for _ in range(5):
            for stream, group, out in zip(streams, xs, outs):
                pb.lib.plast_b200_set_stream(C.c_void_p(stream.cuda_stream))
                O.orthogonalise(group, out)
        check()
        for stream, group, out in zip(streams, xs, outs):
            pb.lib.plast_b200_set_stream(C.c_void_p(stream.cuda_stream))
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                O.orthogonalise(group, out)
        for _ in range(5):
            for stream, graph in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
        check()
    finally:
        pb.lib.plast_b200_set_stream(None)


def test_nothing_outside_the_matrices_is_written():
    rs = np.random.RandomState(10)
    host = rs.randn(3000).astype(np.float32)
    big = pb.Tensor.from_numpy(host)
    x = pb.Tensor.from_numpy(rs.randn(35, 61).astype(np.float32))
    O.orthogonalise([x], [big.view((35, 61), (61, 1), offset=101)])
    after = big.numpy()
    assert np.array_equal(after[:101], host[:101]) and np.array_equal(after[101 + 35 * 61:], host[101 + 35 * 61:])
    assert rel(after[101:101 + 35 * 61].reshape(35, 61), R.orthogonalise(x.numpy())) <= tolerance(35)


def test_one_training_step_of_a_small_language_model():
    """The operators as one step uses them: queries and keys are normed and rotated, the scores are softmaxed into a
    mixture, its logits give token log probabilities, and the gradients that come back through all of it move the
    weights with Muon. Products between them in 64 bits on the host; the same step in 64 bits is the reference."""
    rs = np.random.RandomState(11)
    T, H, D, E, V = 12, 2, 16, 32, 50
    x = rs.randn(T, E).astype(np.float32)
    wq, wk, wo = (rs.randn(*s).astype(np.float32) * 0.3 for s in [(E, H * D), (E, H * D), (E, V)])
    gq, gk = (1 + 0.1 * rs.randn(D)).astype(np.float32), (1 + 0.1 * rs.randn(D)).astype(np.float32)
    pos, freq = np.arange(T, dtype=np.int32)[:, None], (100.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
    token = rs.randint(0, V, T).astype(np.int32)
    dev = pb.Tensor.from_numpy

    def product(a, b):
        return (a.astype(np.float64) @ b.astype(np.float64)).astype(np.float32)

    # ---- the library
    q, k = dev(product(x, wq).reshape(T, H, D), requires_grad=True), dev(product(x, wk).reshape(T, H, D), requires_grad=True)
    qw, kw = dev(gq, requires_grad=True), dev(gk, requires_grad=True)
    qo, ko = pb.Tensor((T, H, D), requires_grad=True), pb.Tensor((T, H, D), requires_grad=True)
    tp, tf = dev(pos), dev(freq)
    pb.qk_norm_rotary(q, k, qw, kw, tp, tf, qo, ko)
    scores = np.einsum("thd,shd->hts", qo.numpy().astype(np.float64), ko.numpy().astype(np.float64)) / np.sqrt(D)
    s, a = dev(scores.astype(np.float32), requires_grad=True), pb.Tensor((H, T, T), requires_grad=True)
    pb.forward("softmax", [s], a, dim=2)
    mixed = (a.numpy().mean(axis=0).astype(np.float64) @ x).astype(np.float32)
    logits = dev(product(mixed, wo), requires_grad=True)
    lp, ent, st = pb.Tensor((T,), requires_grad=True), pb.Tensor((T,), requires_grad=True), pb.Tensor((T, 2))
    tt = dev(token)
    pb.token_logprob(logits, tt, lp, ent, stats=st)
    lp.grad.copy_from(np.full(T, -1.0 / T, np.float32))
    ent.grad.copy_from(np.full(T, -0.01 / T, np.float32))
    pb.token_logprob_backward(logits, tt, st, lp, ent)
    dlogits = logits.grad.numpy()
    dmixed = product(dlogits, wo.T)
    a.grad.copy_from(np.broadcast_to((dmixed.astype(np.float64) @ x.T / H).astype(np.float32), (H, T, T)))
    pb.backward("softmax", [s], a, dim=2)
    ds = s.grad.numpy().astype(np.float64) / np.sqrt(D)
    qo.grad.copy_from(np.einsum("hts,shd->thd", ds, ko.numpy().astype(np.float64)).astype(np.float32))
    ko.grad.copy_from(np.einsum("hts,thd->shd", ds, qo.numpy().astype(np.float64)).astype(np.float32))
    pb.qk_norm_rotary_backward(q, k, qw, kw, tp, tf, qo, ko)
    grads = [product(x.T, q.grad.numpy().reshape(T, -1)), product(x.T, k.grad.numpy().reshape(T, -1)), product(mixed.T, dlogits)]
    params = [dev(w, requires_grad=True) for w in (wq, wk, wo)]
    for p, g in zip(params, grads):
        p.grad.copy_from(g)
    opt = O.Muon.create(lr=0.02, momentum=0.95)
    O.step(opt, params)
    O.release_state(opt)

    # ---- the same in 64 bits
    def forward(wq, wk, wo, gq, gk):
        qr = R.rotate(R.qk_norm((x @ wq).reshape(T, H, D), gq, 1e-6)[2], pos, freq)
        kr = R.rotate(R.qk_norm((x @ wk).reshape(T, H, D), gk, 1e-6)[2], pos, freq)
        sc = np.einsum("thd,shd->hts", qr, kr) / np.sqrt(D)
        e = np.exp(sc - sc.max(axis=2, keepdims=True))
        at = e / e.sum(axis=2, keepdims=True)
        z = at.mean(axis=0) @ x @ wo
        lsm = z - z.max(axis=1, keepdims=True)
        lsm = lsm - np.log(np.exp(lsm).sum(axis=1, keepdims=True))
        entropy = -(np.exp(lsm) * lsm).sum(axis=1)
        return -(lsm[np.arange(T), token].mean()) - 0.01 * entropy.mean()

    w64 = [w.astype(np.float64) for w in (wq, wk, wo, gq, gk)]
    found = grads + [qw.grad.numpy(), kw.grad.numpy()]
    h = 1e-5
    for i, (w, g) in enumerate(zip(w64, found)):
        for at in [tuple(rs.randint(0, n) for n in w.shape) for _ in range(6)]:
            up, down = [v.copy() for v in w64], [v.copy() for v in w64]
            up[i][at] += h
            down[i][at] -= h
            want = (forward(*up) - forward(*down)) / (2 * h)
            # six fp32 stages of about 2^-18 each, and the difference's own h^2
            assert abs(want - g[at]) <= 1e-4 * np.abs(g).max() + 1e-8, (i, at, want, g[at])
    for p, w, g in zip(params, w64, grads):
        r, c = w.shape
        o = R.orthogonalise(1.95 * g.astype(np.float64))
        want = w - 0.02 * np.sqrt(max(1.0, r / c)) * o
        # the gradient has at most 12 directions of T tokens: fewer than min(r, c), so compare where the values are lifted
        assert np.linalg.norm(p.numpy() - want) <= 0.03 * np.linalg.norm(o) * tolerance(1) + 4 * U * np.linalg.norm(w)


def same_bits_and_right(xs, times):
    """Against 64 bits, and the same bits from `times` calls."""
    ins, outs = [pb.Tensor.from_numpy(x) for x in xs], [pb.Tensor(x.shape) for x in xs]
    O.orthogonalise(ins, outs)
    first = [o.numpy() for o in outs]
    for x, got in zip(xs, first):
        assert rel(got, R.orthogonalise(x)) <= tolerance(min(x.shape)), x.shape
    for _ in range(times):
        for o in outs:
            o.zero_()
        O.orthogonalise(ins, outs)
        for o, want in zip(outs, first):
            assert np.array_equal(o.numpy(), want), want.shape


@pytest.mark.parametrize("shape", [(64, 32768), (32768, 40), (128, 20001), (250, 12000)])
def test_many_tiles_of_few_k_blocks_in_a_cta(shape):
    """A tile of one or two K blocks and its linear term fill the ring of stages once or not at all: terms and operands
    take turns on the same stage from one tile to the next."""
    same_bits_and_right([np.random.RandomState(shape[1]).randn(*shape).astype(np.float32)], 10)


@pytest.mark.parametrize("shapes", [[(64, 4672)] * 32, [(64, 4672), (33, 4650), (128, 4700)] * 10])
def test_warps_of_a_cta_on_different_tiles(shapes):
    """Tiles of one K block from many matrices: some of the warps that read a tile's linear term are a tile ahead of
    the others, those that have nothing to store among them."""
    rs = np.random.RandomState(len(shapes[0]))
    same_bits_and_right([rs.randn(*s).astype(np.float32) for s in shapes], 10)


@pytest.mark.parametrize("shapes", [[(100, 1000 + 70 * i) for i in range(28)], [(128, 128), (40, 2100), (60, 61), (64, 700)] * 8,
                                    [(200 + i, 290) for i in range(30)]])
def test_warps_that_have_nothing_to_store_run_ahead(shapes):
    """More tiles than CTAs, at ragged right edges, of matrices whose products follow each other closely: a tile may be
    told of when every warp has stored its part of this very tile."""
    rs = np.random.RandomState(len(shapes))
    same_bits_and_right([rs.randn(*s).astype(np.float32) for s in shapes], 10)


def test_parts_of_a_split_k_are_added_in_one_order():
    rs = np.random.RandomState(23)
    same_bits_and_right([rs.randn(*s).astype(np.float32) for s in [(64, 9000), (120, 4000), (300, 3000)]], 20)


def test_a_wait_that_runs_out_leaves_nan_and_a_status():
    """A limit of no cycles: the waits for a product of many microseconds give up at their first look. What was not
    computed is NaN, the rest is right, the next call works."""
    rs = np.random.RandomState(29)
    xs = [rs.randn(2048, 2500).astype(np.float32), rs.randn(1900, 1500).astype(np.float32)]
    ins, outs = [pb.Tensor.from_numpy(x) for x in xs], [pb.Tensor(x.shape) for x in xs]
    ws = [rs.randn(*x.shape).astype(np.float32) for x in xs]

    def orthogonalised():
        O.orthogonalise(ins, outs)
        return [o.numpy() for o in outs]

    def stepped():
        ps, ms = [pb.Tensor.from_numpy(w) for w in ws], [pb.Tensor.from_numpy(x) for x in xs]
        for p, x in zip(ps, ins):
            p.set_grad(x)
        O.step(O.Muon.create(lr=0.1, momentum=0.5, moments=ms), ps)
        return [p.numpy() for p in ps], [m.numpy() for m in ms]

    want, (want_w, want_m) = orthogonalised(), stepped()
    assert not O.muon_status()
    for call in (orthogonalised, lambda: stepped()):
        for o in outs:
            o.copy_from(np.full(o.shape, 7.0, np.float32))
        pb.lib.plast_b200_tune(13, 0)
        try:
            got = call()
        finally:
            pb.lib.plast_b200_tune(13, -1)
        assert O.muon_status() and not O.muon_status()          # told once
        if call is not orthogonalised:
            got, moments = got
            for g, w in zip(moments, want_m):
                assert np.array_equal(g, w)
        assert any(np.isnan(g).any() for g in got)
        for g, w in zip(got, want if call is orthogonalised else want_w):
            assert np.array_equal(g[~np.isnan(g)], w[~np.isnan(g)])
    for g, w in zip(orthogonalised(), want):
        assert np.array_equal(g, w)


def test_a_product_may_take_longer_than_the_limit_of_a_wait():
    """8192 x 8192: a tile takes up to 0.25 million cycles and a product 2 million and more. What is waited for is a
    tile at a time, so a limit of 1.2 million is not reached."""
    torch = pytest.importorskip("torch")
    x, out = torch.randn(8192, 8192, device="cuda"), torch.empty(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    pb.lib.plast_b200_tune(13, 1200)
    try:
        O.orthogonalise([pb.Tensor.wrap_pointer(x.data_ptr(), x.shape)], [pb.Tensor.wrap_pointer(out.data_ptr(), x.shape)], steps=2)
    finally:
        pb.lib.plast_b200_tune(13, -1)
    assert not O.muon_status()
    assert torch.isfinite(out).all()


# ---- accuracy ------------------------------------------------------------------------------------------
# What a panel cannot hold: 2^-39 of a value below 2^-14. The elements of X are stored after every step and carried on by
# the following ones, which multiply them by at most a = 3.4445 where X is small: 1 + a + ... + a^5 = 685.
FLOOR, CARRIED = 2.0 ** -39, sum(3.4445 ** s for s in range(6))


@pytest.mark.parametrize("scale", [1e-25, 1e-18, 1e-15, 1e-13])
def test_far_below_epsilon_an_absolute_error_is_left(scale):
    """X begins with |x| / epsilon, so the steps are linear to first order: X <- a X. Per step an element carries twice
    2^-22 of it for its storage, and 8 * 2^-22 for the diagonal of the moved polynomial (2.3 and 0.7 * 1.93 and 2.03 *
    0.49 with 2^-22 each, rounded up); off the diagonal the polynomial's 2^-39 times the sum of a column, below one more
    2^-39."""
    base = np.random.RandomState(31).randn(60, 90).astype(np.float32)
    x = base * np.float32(scale)
    want = R.orthogonalise(x)
    bound = 2 * CARRIED * FLOOR + 5 * 12 * 2.0 ** -22 * np.abs(want)
    got = orth([x])[0]
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
    assert np.abs(want).max() < 2 * CARRIED * FLOOR or got.any()


def fp32_steps(x, steps=5):
    """The same steps with products of fp32 operands and fp32 sums, on the GPU (torch, no TF32)."""
    torch = pytest.importorskip("torch")
    assert not torch.backends.cuda.matmul.allow_tf32
    a, b, c = R.COEFFICIENTS
    y = torch.from_numpy(x).cuda()
    y = y.t() if x.shape[0] > x.shape[1] else y
    y = (y / torch.linalg.norm(y.double()).float())
    for _ in range(steps):
        g = y @ y.t()
        y = a * y + (b * g + c * (g @ g)) @ y
    y = y.t() if x.shape[0] > x.shape[1] else y
    return y.cpu().numpy()


def exact_steps(x, steps=5):
    """R.orthogonalise on the GPU."""
    torch = pytest.importorskip("torch")
    a, b, c = (float(np.float32(v)) for v in R.COEFFICIENTS)
    y = torch.from_numpy(x).cuda().double()
    y = y.t() if x.shape[0] > x.shape[1] else y
    y = y / (torch.linalg.norm(y) + float(np.float32(1e-7)))
    for _ in range(steps):
        g = y @ y.t()
        y = a * y + (b * g + c * (g @ g)) @ y
    y = y.t() if x.shape[0] > x.shape[1] else y
    return y.cpu().numpy()


@pytest.mark.parametrize("shape", [(512, 2048), (2048, 300), (700, 700)])
@pytest.mark.parametrize("small", [1.0, 1e-3, 1e-5, 1e-6, 1e-8])
def test_rows_of_two_sizes(shape, small):
    """Row by row (of the shorter side), relative to the row: as the same steps in fp32, and the 2^-39 of a row's n
    elements, of its m elements of the polynomial (times |X| <= 1.21) and of X X^T (times 1.93 + 2 * 2.03 * 0.75 <= 5
    in the polynomial: 7.3 sqrt(m) together), carried on by the following steps."""
    rs = np.random.RandomState(32)
    x = rs.randn(*shape)
    tall = shape[0] > shape[1]
    rows = x.T if tall else x                       # a view
    rows[::2] *= small
    x = x.astype(np.float32)
    got, want, plain = (v.T if tall else v for v in (orth([x])[0].astype(np.float64), exact_steps(x), fp32_steps(x).astype(np.float64)))
    m, n = want.shape
    size = np.linalg.norm(want, axis=1)
    error, fp32 = (np.linalg.norm(v - want, axis=1) / size for v in (got, plain))
    bound = 4 * max(fp32.max(), 2.0 ** -22) + CARRIED * FLOOR * (np.sqrt(n) + 7.3 * np.sqrt(m)) / size
    assert (error <= bound).all(), (error.max(), np.max(error / bound))


@pytest.mark.parametrize("shapes", [[(1024, 1024)] * 4 + [(1024, 4096)], [(2048, 3000)], [(4096, 2048)], [(1500, 3100), (1600, 900)]])
def test_large_matrices_are_as_exact_as_products_in_fp32(shapes):
    """Sizes at which the built-in choice takes pairs of CTAs: twice the error of the same steps in fp32, and the 22 bits
    of the operands."""
    rs = np.random.RandomState(33)
    xs = [rs.randn(*s).astype(np.float32) for s in shapes]
    for x, got in zip(xs, orth(xs)):
        want = exact_steps(x)
        assert rel(got, want) <= 2 * rel(fp32_steps(x), want) + 2.0 ** -21


@pytest.mark.parametrize("kind", ["identity", "permutation", "blocks", "wide"])
def test_sums_that_truncate_nothing(kind):
    """One or two terms to a sum, so that nothing is truncated when it is added up, while the drained sums are raised by one
    or three units of 2^-23 (the average truncation of full sums). The singular values are all alike and go one way x ->
    f(x); every product adds at most 6 * 2^-23 of its terms (three units, an operand's 2^-23 each, lo lo), in units of x:
    the gram matrix through 1.93 + 2 * 2.03 |s|, s = x^2 - 0.7; the polynomial 2.03 s^2 + 1.93 |s| + 3; apply 2.3 + 1.15 + |q|.
    f' carries it on."""
    rs, n = np.random.RandomState(34), 256
    x = {"identity": np.eye(n), "permutation": np.eye(n)[rs.permutation(n)] * np.where(rs.rand(n) < 0.5, 1, -1)[:, None],
         "blocks": np.kron(np.eye(n // 2), np.array([[1.0, 1.0], [1.0, -1.0]])), "wide": np.eye(n, 4 * n, 37)}[kind].astype(np.float32)
    got, want = orth([x])[0], R.orthogonalise(x)
    a, b, c = R.COEFFICIENTS
    v, off = 1.0 / np.sqrt(n), 2.0 ** -22 / np.sqrt(n)
    for _ in range(5):
        s, eta = v * v - 0.7, 6 * 2.0 ** -23
        poly = b * v * v + c * v ** 4
        off = abs(a + 3 * b * v * v + 5 * c * v ** 4) * off + eta * v * (v * v * (1.93 + 4.06 * abs(s)) + 2.03 * s * s + 1.93 * abs(s) + 3
                                                                   + 3.45 + abs(poly + 2.3))
        v = v * (a + poly)
    assert rel(got, want) <= off / abs(v), (rel(got, want), off / abs(v))


@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_one_infinity_or_nan_makes_its_matrix_nan(steps, value):
    x = np.random.RandomState(35).randn(70, 50).astype(np.float32)
    bad = x.copy()
    bad[40, 20] = value
    got = orth([bad, x], steps)
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
def test_a_first_step_and_the_status_are_refused_in_a_capture(mode):
    """Neither spoils the capture: what else it holds replays, and the momenta's zero-fill is not part of it."""
    torch = pytest.importorskip("torch")
    rs = np.random.RandomState(36)
    x, out = pb.Tensor.from_numpy(rs.randn(50, 60).astype(np.float32)), pb.Tensor((50, 60))
    want = orth([x.numpy()])[0]
    p = pb.Tensor.from_numpy(rs.randn(50, 60).astype(np.float32), requires_grad=True)
    opt, stream, codes = O.Muon.create(), torch.cuda.Stream(), []
    pb.synchronize()
    pb.lib.plast_b200_set_stream(C.c_void_p(stream.cuda_stream))
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode=mode):
            for call in (lambda: O.step(opt, [p]), O.muon_status):
                try:
                    call()
                except pb.PlastError as e:
                    codes.append(pb.ERROR_NAMES[e.code])
            O.orthogonalise([x], [out])
        assert codes == ["UNSUPPORTED"] * 2 and not opt.m
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.numpy(), want)
    finally:
        pb.lib.plast_b200_set_stream(None)
