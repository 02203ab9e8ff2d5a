"""What pb.forward and pb.backward hand to the library, seen by a stand-in for the entry point: no GPU needed."""
import numpy as np
import pytest

import plast_b200 as pb


@pytest.fixture
def given(monkeypatch):
    """The (dim, keepdim, fval) that each call hands over."""
    seen = []

    def entry(inputs, output, params):
        seen.append((params.dim, params.keepdim, params.fval))

    for direction in ("forward", "backward"):
        monkeypatch.setitem(pb._ENTRY, (direction, "leaky_relu"), entry)
    return seen


@pytest.mark.parametrize("call", [pb.forward, pb.backward])
@pytest.mark.parametrize("order", [(0.0, -0.0), (-0.0, 0.0)])
def test_both_zeros_arrive(given, call, order):
    x, y = pb.Tensor((3,), device="cpu"), pb.Tensor((3,), device="cpu")
    for fval in order:
        call("leaky_relu", [x], y, fval=fval, check=False)
    assert [np.signbit(g[2]) for g in given] == [np.signbit(v) for v in order]


@pytest.mark.parametrize("call", [pb.forward, pb.backward])
def test_a_scalar_that_changes_is_read_at_every_call(given, call):
    torch = pytest.importorskip("torch")
    x, y = pb.Tensor((3,), device="cpu"), pb.Tensor((3,), device="cpu")
    for slope in (torch.tensor(0.5), np.full((), 0.5, np.float32)):
        del given[:]
        call("leaky_relu", [x], y, fval=slope, check=False)
        slope *= 2
        call("leaky_relu", [x], y, fval=slope, check=False)
        assert [g[2] for g in given] == [0.5, 1.0]
    del given[:]
    call("leaky_relu", [x], y, dim=pb.FULL_REDUCE, keepdim=True, fval=1, check=False)
    assert given == [(pb.FULL_REDUCE, 1, 1.0)]


TENSORS, TENSOR = pb.C.POINTER(pb.C.POINTER(pb.CTensor)), pb.C.POINTER(pb.CTensor)


def takes(name):
    from plast_b200 import graph, optim  # noqa: F401  (they declare entry points of their own)
    return getattr(pb.lib, name).argtypes


@pytest.mark.parametrize("name,wanted", [
    *[(f"{op}_cuda_forward", [TENSORS, TENSOR]) for op in pb.FORWARD_OPS + ["chain", "sum_axis0_noalloc"]],
    *[(f"{op}_cuda_backward", [TENSORS, TENSOR]) for op in pb.BACKWARD_OPS + ["chain"]],
    *[(f"{kind}_step_cuda", [None, TENSORS]) for kind in ("sgd", "adam", "adamw", "muon")],
    ("plast_b200_orthogonalise", [TENSORS, TENSORS]), ("plast_b200_token_logprob", [TENSOR] * 8),
    ("plast_b200_token_logprob_backward", [TENSOR] * 6), ("plast_b200_qk_norm_rotary", [TENSOR] * 8),
    ("plast_b200_qk_norm_rotary_backward", [TENSOR] * 8)])
def test_entry_points_refuse_what_is_no_tensor_pointer(name, wanted):
    """By their declared types (a call with a wrong one must not be made): a number, bytes, an untyped address, one
    level of pointers too few or too many."""
    t = pb.Tensor((2,), device="cpu")
    one, many = pb.C.byref(t.c), pb._ptr_array([t, t])
    for declared, kind in zip(takes(name), wanted):
        if kind is None:
            continue
        declared.from_param(many if kind is TENSORS else one)
        for wrong in (5, b"bytes", pb.C.c_void_p(8), one if kind is TENSORS else many, t):
            with pytest.raises(TypeError):
                declared.from_param(wrong)


def test_the_layer_takes_tensors_only():
    from plast_b200 import optim
    x, row = pb.Tensor((2, 3), device="cpu"), pb.Tensor((2,), device="cpu")
    for wrong in (5, b"bytes", np.zeros(3, np.float32), pb.C.byref(x.c)):
        for call in (lambda: pb.forward("neg", [wrong], x), lambda: pb.forward("neg", [x], wrong),
                     lambda: pb.backward("neg", [wrong], x), lambda: pb.token_logprob(wrong, row, row),
                     lambda: optim.step(optim.SGD(0.1), [wrong]), lambda: optim.orthogonalise([wrong], [x])):
            with pytest.raises((AttributeError, TypeError)):
                call()


def test_a_gradient_that_was_set_stays_its_owners(monkeypatch):
    """Tensors that come and go with one gradient (a step's parameters over the same buffer) do not free it."""
    freed = []

    class Device:
        def __getattr__(self, name):
            return freed.append if name == "arena_free_cuda" else getattr(pb._LazyLib._lib, name)

    grad, other = pb.Tensor((3,), device="cpu"), pb.Tensor((3,), device="cpu")
    monkeypatch.setattr(pb, "lib", Device())
    grad._dptr, other._dptr = 11, 12                     # as if they held device memory
    other.set_grad(grad)
    del other
    assert freed == [12]
    t = pb.Tensor((3,), device="cpu", requires_grad=True)
    t.grad._dptr = 13
    t.free()                                             # its own goes with it
    assert freed == [12, 13]
    t.attach_grad()._dptr = 14
    t.set_grad(grad)                                     # replaced: nobody holds it any more
    assert freed == [12, 13, 14]
    t.free()
    del t
    assert freed == [12, 13, 14] and grad._dptr == 11
    del grad
    assert freed == [12, 13, 14, 11]
    t, other = pb.Tensor((3,), device="cpu"), pb.Tensor((3,), device="cpu")
    other.set_grad(t.attach_grad())
    t.grad._dptr = 15
    del t                                                # the other one holds it
    assert freed[4:] == []
    del other
    assert freed[4:] == [15]


@pytest.mark.parametrize("count", [0, 1, 3, 8, 9, 40])
def test_addresses_are_a_list_of_pointers(count):
    ts = [pb.Tensor((i + 1,), device="cpu") for i in range(count)]
    packed = pb._addresses(ts)
    at = pb.C.cast(pb.C.c_char_p(packed), TENSORS)
    assert len(packed) == 8 * count and [at[i].contents.shape[0] for i in range(count)] == [i + 1 for i in range(count)]


@pytest.mark.parametrize("count", [0, 1])
def test_a_momentum_for_every_parameter(count):
    """The library reads a momentum per parameter from the caller's array."""
    from plast_b200 import optim
    params = [pb.Tensor((4, 4), device="cpu", requires_grad=True) for _ in range(2)]
    opt = optim.Muon.create(moments=[pb.Tensor((4, 4), device="cpu") for _ in range(count)])
    with pytest.raises(ValueError):
        optim.step(opt, params)
