"""What token_logprob, rotary and qk_norm_rotary refuse, and the host-side frequency tables: no GPU needed, a
refused call launches nothing."""
import numpy as np
import pytest

import plast_b200 as pb
from plast_b200 import optim as O

F, I = pb.FLOAT32, pb.INT32


def T(*shape, dtype=F, **kw):
    return pb.Tensor(shape, device="cpu", dtype=dtype, **kw)


def refused(code, fn, *args, **kw):
    with pytest.raises(pb.PlastError) as e:
        fn(*args, **kw)
    assert pb.ERROR_NAMES[e.value.code] == code, str(e.value)


def expanded(t, shape, strides):
    return t.view(shape, strides)


def test_token_logprob_refusals():
    x, tok, row = T(4, 10), T(4, dtype=I), T(4)
    f = pb.token_logprob
    refused("NULL", f, None, tok, row)
    refused("NULL", f, x, None, row)
    refused("NULL", f, x, tok, None)
    refused("DTYPE", f, T(4, 10, dtype=I), tok, row)
    refused("DTYPE", f, x, T(4), row)
    refused("DTYPE", f, x, tok, T(4, dtype=I))
    refused("SHAPE", f, x, T(3, dtype=I), row)
    refused("SHAPE", f, x, T(2, 2, dtype=I), row)
    refused("SHAPE", f, T(4, 0), tok, row)
    refused("SHAPE", f, T(), T(dtype=I), T(1))
    refused("SHAPE", f, x, tok, T(5))
    refused("SHAPE", f, x, tok, row, entropy=T(3))
    refused("UNSUPPORTED", f, x, tok, T(8).view((4,), (2,)))
    refused("SHAPE", f, x, tok, row, stats=T(4))
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-38):
        refused("UNSUPPORTED", f, x, tok, row, temperature=bad)
    refused("NULL", f, x, tok, row, top_logprob=T(4, 3))
    refused("NULL", f, x, tok, row, top_index=T(4, 3, dtype=I))
    refused("SHAPE", f, x, tok, row, top_logprob=T(4, 11), top_index=T(4, 11, dtype=I))
    refused("SHAPE", f, x, tok, row, top_logprob=T(4, 3), top_index=T(3, 3, dtype=I))
    refused("DTYPE", f, x, tok, row, top_logprob=T(4, 3), top_index=T(4, 3))
    refused("LIMIT", f, T(4, 50), tok, row, top_logprob=T(4, 33), top_index=T(4, 33, dtype=I))
    big = T(1).view((1 << 28, 2), (0, 0))
    refused("LIMIT", f, big, T(1, dtype=I).view((1 << 28,), (0,)), row)


def test_token_logprob_backward_refusals():
    b = pb.token_logprob_backward
    tok, st, row, H, L = T(4, dtype=I), T(4, 2), T(4), T(4), T(4)
    x = T(4, 10)
    b(x, tok, st, row, H, L)                             # no gradient wanted: nothing to do
    x = T(4, 10, requires_grad=True)
    refused("NULL", b, x, tok, None, row, H, L)
    refused("SHAPE", b, x, tok, T(4), row, H, L)
    refused("UNSUPPORTED", b, x, tok, T(10).view((4, 2), (2, 1), offset=1), row, H, L)
    lp = T(4)
    lp.set_grad(T(3))
    refused("SHAPE", b, x, tok, st, lp, H, L)
    ent = T(4, requires_grad=True)
    ent.c.data = None
    refused("NULL", b, x, tok, st, row, ent, L)
    x.set_grad(T(4, 9))
    refused("SHAPE", b, x, tok, st, row, H, L)
    x.set_grad(T(4, 10, dtype=I))
    refused("DTYPE", b, x, tok, st, row, H, L)
    x.set_grad(T(10).view((4, 10), (0, 1)))              # an expanded gradient
    refused("UNSUPPORTED", b, x, tok, st, row, H, L)
    x.c.grad = None
    refused("NULL", b, x, tok, st, row, H, L)


def test_rotary_refusals():
    x, pos, freq, out = T(2, 3, 4, 16), T(2, 3, 1, dtype=I), T(8), T(2, 3, 4, 16)

    def f(x=x, pos=pos, freq=freq, out=out, dim=0, fval=1.0):
        pb.forward("rotary", [x, pos, freq], out, dim=dim, fval=fval)

    refused("DTYPE", f, x=T(2, 3, 4, 16, dtype=I))
    refused("DTYPE", f, pos=T(2, 3, 1))
    refused("DTYPE", f, freq=T(8, dtype=I))
    refused("SHAPE", f, pos=T(2, 5, 1, dtype=I))
    refused("SHAPE", f, pos=T(2, 3, 4, 16, dtype=I))
    refused("SHAPE", f, freq=T(9))
    refused("SHAPE", f, freq=T(0))
    refused("SHAPE", f, freq=T(2, 4))
    refused("SHAPE", f, out=T(2, 3, 4, 8))
    refused("SHAPE", f, x=T(), out=T())
    refused("LIMIT", f, x=T(2, 1, 1, 1025), pos=T(2, 1, 1, dtype=I), out=T(2, 1, 1, 1025))
    refused("UNSUPPORTED", f, dim=2)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        refused("UNSUPPORTED", f, fval=bad)
    refused("UNSUPPORTED", f, out=T(16).view((2, 3, 4, 16), (0, 0, 0, 1)))
    refused("UNSUPPORTED", f, out=x.view((2, 3, 4, 16), (12 * 16, 16, 48, 1)))   # in place with other strides
    refused("UNSUPPORTED", f, freq=T(8, requires_grad=True))
    wide = T(1).view((1 << 16, 1 << 15, 2), (0, 0, 0))
    refused("LIMIT", f, x=wide, pos=T(1, 1, dtype=I), freq=T(1), out=T(1).view((1 << 16, 1 << 15, 2), (2 << 15, 2, 1)))
    x.set_grad(T(2, 3, 4, 16))
    with pytest.raises(pb.PlastError):                                           # no upstream gradient
        pb.backward("rotary", [x, pos, freq], out, fval=1.0)
    x.set_grad(T(16).view((2, 3, 4, 16), (0, 0, 0, 1)))
    out.attach_grad()
    refused("UNSUPPORTED", pb.backward, "rotary", [x, pos, freq], out, fval=1.0)


def test_qk_norm_refusals():
    base = dict(q=T(2, 3, 4, 16), k=T(2, 3, 2, 16), qw=T(16), kw=T(16), pos=T(2, 3, 1, dtype=I), freq=T(8),
                qo=T(2, 3, 4, 16), ko=T(2, 3, 2, 16))

    def f(call=pb.qk_norm_rotary, epsilon=1e-6, layout=0, amplitude=1.0, **kw):
        a = {**base, **kw}
        call(*[a[n] for n in ("q", "k", "qw", "kw", "pos", "freq", "qo", "ko")], epsilon=epsilon, layout=layout,
           amplitude=amplitude)

    refused("NULL", f, q=None)
    refused("NULL", f, qo=None)
    refused("NULL", f, k=None)
    refused("NULL", f, k=None, kw=None)
    refused("DTYPE", f, k=T(2, 3, 2, 16, dtype=I))
    refused("SHAPE", f, k=T(2, 3, 2, 8))
    refused("SHAPE", f, ko=T(2, 3, 4, 16))
    refused("SHAPE", f, qw=T(8))
    refused("SHAPE", f, kw=T(2, 16))
    refused("SHAPE", f, k=T(2, 4, 2, 16), ko=T(2, 4, 2, 16))           # positions do not fit the keys
    refused("UNSUPPORTED", f, epsilon=-1.0)
    refused("UNSUPPORTED", f, epsilon=float("nan"))
    refused("UNSUPPORTED", f, layout=3)
    refused("UNSUPPORTED", f, layout=-1)
    refused("UNSUPPORTED", f, amplitude=0.0)
    same = T(2, 3, 4, 16)
    refused("UNSUPPORTED", f, k=T(2, 3, 4, 16), qo=same, ko=same)
    back = pb.qk_norm_rotary_backward
    f(call=back)                                                          # no gradient wanted
    refused("NULL", f, call=back, qw=T(16, requires_grad=True))         # no upstream gradient
    refused("NULL", f, call=back, q=T(2, 3, 4, 16, requires_grad=True))
    g = T(2, 3, 4, 16)
    q, k = T(2, 3, 4, 16), T(2, 3, 4, 16)
    q.set_grad(g)
    k.set_grad(g)
    refused("UNSUPPORTED", f, call=back, q=q, k=k, qo=T(2, 3, 4, 16, requires_grad=True), ko=T(2, 3, 4, 16, requires_grad=True))


def test_frequency_tables():
    n, base = 64, 10000.0
    i = np.arange(n)
    plain = base ** (-2.0 * i / 128)
    table, amplitude = pb.rotary_frequencies(128, base)
    np.testing.assert_allclose(table, plain, rtol=2.0 ** -24)
    assert amplitude == 1.0
    np.testing.assert_allclose(pb.rotary_frequencies(128, base, "linear", factor=4.0)[0], plain / 4, rtol=2.0 ** -23)
    slow, _ = pb.rotary_frequencies(128, base, "base", factor=8.0)
    np.testing.assert_allclose([slow[0], slow[-1]], [1.0, plain[-1] / 8], rtol=1e-6)
    parts, amplitude = pb.rotary_frequencies(128, base, "parts", factor=16.0, slow=1, fast=32, context=4096)
    turns = 4096 * plain / (2 * np.pi)
    assert np.allclose(parts[turns > 40], plain[turns > 40], rtol=1e-6)
    assert np.allclose(parts[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-6)
    assert ((parts <= plain * 1.000001) & (parts >= plain / 16 * 0.999999)).all()
    assert (np.diff(parts) < 0).all()
    np.testing.assert_allclose(amplitude, 0.1 * np.log(16.0) + 1.0, rtol=2.0 ** -24)
    bands, _ = pb.rotary_frequencies(128, base, "bands", factor=8.0, slow=1, fast=4, context=8192)
    turns = 8192 * plain / (2 * np.pi)
    keep = np.clip((turns - 1) / 3, 0, 1)
    np.testing.assert_allclose(bands, plain * keep + plain / 8 * (1 - keep), rtol=2.0 ** -23)
    for bad in (dict(rotated=3), dict(rotated=0), dict(rotated=2048)):
        refused("SHAPE", pb.rotary_frequencies, base=base, **bad)
    for bad in (dict(base=1.0), dict(base=float("inf")), dict(scaling="linear", factor=0.5),
                dict(scaling="parts", factor=2.0, slow=32, fast=1, context=4096),
                dict(scaling="bands", factor=2.0, slow=1, fast=4, context=0), dict(scaling="base", factor=2.0, rotated=2)):
        refused("UNSUPPORTED", pb.rotary_frequencies, **{"rotated": 8, "base": base, **bad})


def test_muon_refusals_change_nothing():
    def params(*shapes):
        return [T(*s, requires_grad=True) for s in shapes]

    def f(ps, moments=None, **kw):
        opt = O.Muon.create(moments=moments, **{k: v for k, v in kw.items()})
        try:
            O.step(opt, ps)
        finally:
            assert moments is not None or not opt.m          # nothing was created

    f([])
    f([None, T(3, 3)])                                        # nothing to update
    refused("SHAPE", f, params((4, 4), (5,)))
    refused("SHAPE", f, params(()))
    refused("LIMIT", f, params((1, 262145)))
    refused("UNSUPPORTED", f, params((4, 4)), ns_steps=-1)
    refused("UNSUPPORTED", f, params((4, 4)), ns_steps=33)
    refused("UNSUPPORTED", f, params((4, 4)), epsilon=-1e-7)
    refused("UNSUPPORTED", f, params((4, 4)), epsilon=float("nan"))
    refused("UNSUPPORTED", f, params((4, 4)), scale=3)
    p = params((4, 4))[0]
    refused("UNSUPPORTED", f, [p, p])
    refused("UNSUPPORTED", f, params((4, 4), (4, 4)), moments=[T(4, 4)] * 2)
    refused("NULL", f, params((4, 4), (4, 4)), moments=[T(4, 4), None])
    base = T(12, 4)
    halves = [base.view((8, 4), (4, 1)), base.view((8, 4), (4, 1), offset=16)]     # rows 0 to 7 and 4 to 11
    for t in halves:
        t.set_grad(T(8, 4))
    refused("UNSUPPORTED", f, halves)
    refused("UNSUPPORTED", f, params((8, 4), (8, 4)), moments=halves)
    t = base.view((8, 4), (4, 1))
    t.set_grad(base.view((8, 4), (4, 1), offset=4))
    refused("UNSUPPORTED", f, [t])                            # its own gradient, a row on
    t.set_grad(T(8, 4))
    refused("UNSUPPORTED", f, [t], moments=[base.view((8, 4), (4, 1))])
    refused("SHAPE", f, params((4, 4)), moments=[T(4, 3)])
    refused("DTYPE", f, params((4, 4)), moments=[T(4, 4, dtype=I)])
    t = T(8, 8).transpose(0, 1)
    t.set_grad(T(8, 8))
    refused("UNSUPPORTED", f, [t])
    t = T(8, 8)
    t.set_grad(T(8, 8).transpose(0, 1))
    refused("UNSUPPORTED", f, [t])
    t.set_grad(T(8, 7))
    refused("SHAPE", f, [t])
    t = T(8, 8, dtype=I)
    t.set_grad(T(8, 8))
    refused("DTYPE", f, [t])
    t = T(8, 8, requires_grad=True)
    t.c.data = None
    refused("NULL", f, [t])


def test_orthogonalise_refusals():
    x, y, o = T(4, 6), T(4, 6), T(4, 6)
    O.orthogonalise([], [])
    O.orthogonalise([T(0, 4)], [T(0, 4)])
    refused("NULL", O.orthogonalise, [None], [o])
    refused("NULL", O.orthogonalise, [x], [None])
    refused("SHAPE", O.orthogonalise, [T(4)], [T(4)])
    refused("SHAPE", O.orthogonalise, [x], [T(6, 4)])
    refused("DTYPE", O.orthogonalise, [T(4, 6, dtype=I)], [o])
    refused("DTYPE", O.orthogonalise, [x], [T(4, 6, dtype=I)])
    refused("UNSUPPORTED", O.orthogonalise, [x.transpose(0, 1)], [T(6, 4)])
    refused("UNSUPPORTED", O.orthogonalise, [x, y], [o, o])
    refused("UNSUPPORTED", O.orthogonalise, [x, y], [y, o])
    base = T(8, 6)
    refused("UNSUPPORTED", O.orthogonalise, [base.view((4, 6), (6, 1))], [base.view((4, 6), (6, 1), offset=6)])
    refused("UNSUPPORTED", O.orthogonalise, [x, y], [base.view((4, 6), (6, 1)), base.view((4, 6), (6, 1), offset=18)])
    refused("UNSUPPORTED", O.orthogonalise, [x], [o], 40)
    refused("UNSUPPORTED", O.orthogonalise, [x], [o], 5, -1.0)


def test_rotary_refuses_buffers_that_overlap():
    base, pos, freq = T(1000), T(2, 3, 1, dtype=I), T(8)
    shape, dense = (2, 3, 4, 16), (192, 64, 16, 1)

    def at(offset, strides=dense):
        return base.view(shape, strides, offset=offset)

    def f(x, out, pos=pos, freq=freq):
        refused("UNSUPPORTED", pb.forward, "rotary", [x, pos, freq], out, fval=1.0)

    f(at(0), at(16))                                          # a head on
    f(at(17), at(0))
    f(at(0), at(0, (192, 16, 48, 1)))                        # the same memory in another order
    f(at(0), at(3, (384, 128, 32, 2)))                       # every second element
    f(at(400), at(0), freq=base.view((8,), (1,), offset=383))
    f(at(400), at(0), freq=base.view((8,), (2,), offset=100))
    f(at(400), at(0), pos=pb.Tensor((2, 3, 1), device="cpu", dtype=I, _base=base, _storage_elems=1000))
    x, out = at(0), T(*shape)
    x.set_grad(at(400))
    out.set_grad(at(401))
    refused("UNSUPPORTED", pb.backward, "rotary", [x, pos, freq], out, fval=1.0)
    out.set_grad(at(400, (192, 16, 48, 1)))
    refused("UNSUPPORTED", pb.backward, "rotary", [x, pos, freq], out, fval=1.0)


def test_qk_norm_refuses_buffers_that_overlap():
    base, pos, freq = T(4000), T(2, 3, 1, dtype=I), T(8)

    def q_at(offset):
        return base.view((2, 3, 4, 16), (192, 64, 16, 1), offset=offset)

    def k_at(offset):
        return base.view((2, 3, 2, 16), (96, 32, 16, 1), offset=offset)

    def f(q, k, qo, ko, qw=None, kw=None, call=pb.qk_norm_rotary):
        refused("UNSUPPORTED", call, q, k, qw, kw, pos, freq, qo, ko)

    f(q_at(0), k_at(500), k_at(500).view((2, 3, 4, 16), (192, 64, 16, 1)), k_at(1000))    # q_out begins where k does
    f(q_at(0), k_at(500), q_at(595), k_at(1000))                                          # one element of k
    f(q_at(0), k_at(500), q_at(1000), k_at(383))                                          # k_out over the end of q
    f(q_at(0), k_at(500), q_at(1000), k_at(1100))                                         # over q_out
    f(q_at(0), k_at(500), q_at(16), k_at(1000))                                           # over its own input, a head on
    f(q_at(0), k_at(500), q_at(1000), k_at(508))
    f(q_at(0), k_at(500), q_at(1000), k_at(2000), qw=base.view((16,), (1,), offset=2090))
    f(q_at(0), None, q_at(1000), None, qw=base.view((16,), (1,), offset=1000))

    back = pb.qk_norm_rotary_backward
    q, k, qo, ko = q_at(0), k_at(500), T(2, 3, 4, 16), T(2, 3, 2, 16)

    def grads(dq, dk, dqo, dko):
        for t, g in ((q, dq), (k, dk), (qo, dqo), (ko, dko)):
            t.set_grad(g)

    grads(q_at(1000), k_at(1383), q_at(2000), k_at(2500))     # dq and dk
    f(q, k, qo, ko, call=back)
    grads(q_at(1000), k_at(1500), q_at(2000), k_at(1000))     # dq and the gradient of k_out
    f(q, k, qo, ko, call=back)
    grads(q_at(1000), k_at(1500), q_at(1004), k_at(2500))     # dq, four elements off the gradient of q_out
    f(q, k, qo, ko, call=back)
    grads(q_at(1000), k_at(100), q_at(2000), k_at(2500))      # dk and q
    f(q, k, qo, ko, call=back)
    grads(q_at(1000), k_at(1500), q_at(2000), k_at(2500))
    qw, kw = T(16), T(16)
    qw.set_grad(base.view((16,), (1,), offset=3000))
    kw.set_grad(base.view((16,), (1,), offset=3004))          # the gradients of the weights
    f(q, k, qo, ko, qw=qw, kw=kw, call=back)
    kw.set_grad(base.view((16,), (2,), offset=3000))
    f(q, k, qo, ko, qw=qw, kw=kw, call=back)


def test_outputs_and_gradients_with_an_element_at_two_indices():
    """Rows that run into each other, without a stride of 0: several threads would write one element."""
    base, pos, freq = T(1000), T(6, 1, dtype=I), T(4)
    x, ok = T(6, 3, 8), T(6, 3, 8)
    for strides in ((23, 8, 1), (24, 7, 1), (1, 24, 3)):
        out = base.view((6, 3, 8), strides)
        refused("UNSUPPORTED", pb.forward, "rotary", [x, pos, freq], out, fval=1.0)
        refused("UNSUPPORTED", pb.qk_norm_rotary, x, None, None, None, pos, freq, out, None)
        x.set_grad(out)
        ok.attach_grad()
        refused("UNSUPPORTED", pb.backward, "rotary", [x, pos, freq], ok, fval=1.0)
        refused("UNSUPPORTED", pb.qk_norm_rotary_backward, x, None, None, None, pos, freq, ok, None)
    logits, tok, st, lp = T(6, 40), T(6, dtype=I), T(6, 2), T(6, requires_grad=True)
    logits.set_grad(base.view((6, 40), (39, 1)))
    refused("UNSUPPORTED", pb.token_logprob_backward, logits, tok, st, lp)


def test_token_logprob_refuses_buffers_that_overlap():
    base = T(400)
    x, tok = base.view((4, 10), (10, 1)), base.view((4,), (1,), offset=40)
    tok.c.dtype = I

    def at(offset, *shape, dtype=F):
        t = base.view(shape, pb.contiguous_strides(shape), offset=offset)
        t.c.dtype = dtype
        return t

    f = pb.token_logprob
    refused("UNSUPPORTED", f, x, tok, at(39, 4))                                    # the last logit
    refused("UNSUPPORTED", f, x, tok, at(40, 4))                                    # the tokens
    refused("UNSUPPORTED", f, x, tok, at(50, 4), entropy=at(53, 4))
    refused("UNSUPPORTED", f, x, tok, at(50, 4), log_norm=at(50, 4))
    refused("UNSUPPORTED", f, x, tok, at(50, 4), stats=at(36, 4, 2))
    refused("UNSUPPORTED", f, x, tok, at(50, 4), top_logprob=at(60, 4, 3), top_index=at(71, 4, 3, dtype=I))
    refused("UNSUPPORTED", f, x, tok, at(50, 4), top_logprob=at(60, 4, 3), top_index=at(42, 4, 3, dtype=I))
    b = pb.token_logprob_backward
    lp, ent, norm = at(50, 4), at(54, 4), at(58, 4)
    stats = T(4, 2)
    for t, offset in ((lp, 100), (ent, 104), (norm, 108)):
        t.set_grad(at(offset, 4))
    for offset in (5, 37, 57, 61, 99, 103, 105, 111):
        x.set_grad(at(offset, 4, 10))
        if offset != 57:       # over the values of entropy, which are read
            refused("UNSUPPORTED", b, x, tok, stats, lp, ent if offset in (61, 103, 105) else None, norm)
        refused("UNSUPPORTED", b, x, tok, stats, lp, ent, norm)


@pytest.mark.parametrize("rotated,base,factor,slow,fast,context", [(128, 10000.0, 16.0, 1, 32, 4096), (64, 500000.0, 4.0, 1, 32, 8192),
                                                                   (96, 10000.0, 8.0, 2, 20, 2048)])
def test_the_ramp_of_the_parts_table(rotated, base, factor, slow, fast, context):
    """Between the pair that makes `fast` turns over the context and the one that makes `slow`, both rounded outwards to
    whole pairs, the share of the divided frequency grows linearly with the pair's index."""
    i = np.arange(rotated // 2)
    plain = base ** (-2.0 * i / rotated)

    def pair(turns):
        return rotated * np.log(context / (2 * np.pi * turns)) / (2 * np.log(base))

    low, high = np.floor(pair(fast)), np.ceil(pair(slow))
    assert 2 < low and high < rotated // 2 - 2          # the ramp lies inside
    share = np.clip((i - low) / (high - low), 0, 1)
    table, _ = pb.rotary_frequencies(rotated, base, "parts", factor=factor, slow=slow, fast=fast, context=context)
    np.testing.assert_allclose(table, plain / factor * share + plain * (1 - share), rtol=2.0 ** -23)
    assert ((share > 0) & (share < 1)).sum() > 5
