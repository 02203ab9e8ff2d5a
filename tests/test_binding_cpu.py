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
