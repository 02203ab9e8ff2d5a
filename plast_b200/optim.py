"""ctypes mirror of include/plast_b200_optim.h: the optimiser structs of the plast runtime and
the multi-tensor step entry points."""
from __future__ import annotations

import ctypes as C

from . import CTensor, _by_address, check_error, lib


class SGD(C.Structure):
    """include/optimizers/sgd.h:5-7"""
    _fields_ = [("lr", C.c_float)]


class Adam(C.Structure):
    """include/optimizers/adam.h:5-15"""
    _fields_ = [("lr", C.c_float), ("beta1", C.c_float), ("beta2", C.c_float), ("epsilon", C.c_float),
                ("t", C.c_int), ("m", C.POINTER(C.POINTER(CTensor))), ("v", C.POINTER(C.POINTER(CTensor))),
                ("data_arena", C.c_void_p), ("optimizer_arena", C.c_void_p)]


class AdamW(C.Structure):
    """include/optimizers/adamw.h:5-16"""
    _fields_ = [("lr", C.c_float), ("beta1", C.c_float), ("beta2", C.c_float), ("epsilon", C.c_float),
                ("weight_decay", C.c_float), ("t", C.c_int), ("m", C.POINTER(C.POINTER(CTensor))),
                ("v", C.POINTER(C.POINTER(CTensor))), ("data_arena", C.c_void_p), ("optimizer_arena", C.c_void_p)]


MUON_SCALE_ASPECT, MUON_SCALE_RMS, MUON_SCALE_NONE = 0, 1, 2


class Muon(C.Structure):
    """Muon of include/plast_b200_optim.h; `create` fills in the usual settings."""
    _fields_ = [("lr", C.c_float), ("momentum", C.c_float), ("weight_decay", C.c_float), ("epsilon", C.c_float),
                ("nesterov", C.c_int), ("ns_steps", C.c_int), ("scale", C.c_int),
                ("m", C.POINTER(C.POINTER(CTensor)))]

    @classmethod
    def create(cls, lr=0.02, momentum=0.95, weight_decay=0.0, epsilon=1e-7, nesterov=True, ns_steps=5,
               scale=MUON_SCALE_ASPECT, moments=None):
        """`moments`: the caller's momentum Tensors, one per parameter; None: the library creates them."""
        opt = cls(lr, momentum, weight_decay, epsilon, int(bool(nesterov)), ns_steps, scale)
        if moments is not None:
            opt._moments = list(moments)          # keeps the caller's structs alive
            opt._moments_array = param_array(opt._moments)
            opt.m = opt._moments_array
        return opt


assert C.sizeof(Muon) == 40 and Muon.m.offset == 32
assert C.sizeof(SGD) == 4 and C.sizeof(Adam) == 56 and C.sizeof(AdamW) == 56
assert Adam.t.offset == 16 and Adam.m.offset == 24 and AdamW.t.offset == 20 and AdamW.m.offset == 24

for _name, _struct in (("sgd_step_cuda", SGD), ("adam_step_cuda", Adam), ("adamw_step_cuda", AdamW), ("muon_step_cuda", Muon)):
    getattr(lib, _name).argtypes = [C.POINTER(_struct), C.POINTER(C.POINTER(CTensor)), C.c_int]
    getattr(lib, _name).restype = None
lib.plast_b200_adam_state_release.argtypes = [C.POINTER(C.POINTER(CTensor)), C.POINTER(C.POINTER(CTensor))]
lib.plast_b200_adam_state_release.restype = None
lib.plast_b200_muon_state_release.argtypes = [C.POINTER(C.POINTER(CTensor))]
lib.plast_b200_muon_state_release.restype = None
lib.plast_b200_orthogonalise.argtypes = [C.POINTER(C.POINTER(CTensor))] * 2 + [C.c_int, C.c_int, C.c_float]
lib.plast_b200_orthogonalise.restype = None

# by the addresses of _address_array
_STEP = {_struct: _by_address(_name, C.POINTER(_struct), C.c_void_p, C.c_int)
         for _name, _struct in (("sgd_step_cuda", SGD), ("adam_step_cuda", Adam), ("adamw_step_cuda", AdamW), ("muon_step_cuda", Muon))}
_orthogonalise = _by_address("plast_b200_orthogonalise", C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_float)


def param_array(params):
    """Tensor** for a list of plast_b200.Tensor objects; None entries become NULL."""
    arr = (C.POINTER(CTensor) * max(len(params), 1))()
    for i, p in enumerate(params):
        if p is not None:
            arr[i] = C.pointer(p.c)
    return arr


def _address_array(params):
    """param_array() as plain addresses, for the length of one call."""
    return (C.c_void_p * max(len(params), 1))(*[None if p is None else p.address for p in params])


def step(optimizer, params) -> None:
    """One optimiser step on the GPU over a list of parameters (Tensor objects with .grad)."""
    moments = getattr(optimizer, "_moments", None)
    if moments is not None and optimizer.m and len(moments) < len(params):
        raise ValueError(f"{len(params)} parameters, but {len(moments)} momenta were given")
    _STEP[type(optimizer)](C.byref(optimizer), _address_array(params), len(params))
    check_error()


def orthogonalise(inputs, outputs, steps: int = 5, epsilon: float = 1e-7) -> None:
    """outputs[i] = the Newton-Schulz orthogonalisation of inputs[i], all matrices at once."""
    if len(inputs) != len(outputs):
        raise ValueError("as many outputs as inputs")
    _orthogonalise(_address_array(inputs), _address_array(outputs), len(inputs), steps, epsilon)
    check_error()


def muon_status() -> bool:
    """Whether a wait inside a Muon step or an orthogonalisation has run out since the last look: results of such a
    call hold NaN (plast_b200_muon_status). Waits for the library stream."""
    status = lib.plast_b200_muon_status()
    check_error()
    return status != 0


def release_state(optimizer) -> None:
    if isinstance(optimizer, Muon):
        if optimizer.m:
            lib.plast_b200_muon_state_release(optimizer.m)
            optimizer.m = None
    elif not isinstance(optimizer, SGD) and optimizer.m:
        lib.plast_b200_adam_state_release(optimizer.m, optimizer.v)
        optimizer.m = None
        optimizer.v = None
