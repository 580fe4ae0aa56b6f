"""The expert layer's and the adapters' C ABI and argument checks that need no GPU:
the library exports what the header declares, the binding has its arity, and
bad arguments are refused before any device work."""
import os
import re

import pytest
import torch

from camoe_b200 import _lib, adapters, experts

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "camoe_experts.h")
P = 4096  # a 16-byte aligned address that is never used


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return {name: params.count(",") + 1 for name, params in re.findall(r"\b(camoe_(?:ex|ad)_\w+)\s*\(([^)]*)\)\s*;", text)}


def test_exports_and_arity():
    lib, names = _lib.lib(), declared()
    assert sorted(names) == sorted(_lib.EX_EXPORTS)
    for name, n in names.items():
        assert len(getattr(lib, name).argtypes) == n, name


def dispatch(N=4, k=2, E=8, C=16, dtype=0, index=P, index_bytes=8, work=P, nbytes=1 << 20, x=P, offsets=P):
    return _lib.lib().camoe_ex_dispatch(x, dtype, index, index_bytes, P, offsets, P, P, work, nbytes, N, k, E, C, None)


def test_dispatch_statuses():
    assert dispatch(dtype=2) == _lib.ERR_UNSUPPORTED
    assert dispatch(index_bytes=2) == _lib.ERR_UNSUPPORTED
    assert dispatch(E=1025) == _lib.ERR_UNSUPPORTED
    assert dispatch(k=65) == _lib.ERR_UNSUPPORTED
    for bad in (dict(N=-1), dict(k=0), dict(E=0), dict(C=-1), dict(index=None), dict(offsets=None), dict(x=None)):
        assert dispatch(**bad) == _lib.ERR_INVALID_ARG, bad
    assert dispatch(N=1 << 31) == _lib.ERR_SHAPE
    need = _lib.lib().camoe_ex_dispatch_work_bytes(50000, 2, 8)
    assert need > 0 and _lib.lib().camoe_ex_dispatch_work_bytes(4, 2, 8) == 0
    assert dispatch(N=50000, nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert dispatch(N=50000, work=None) == _lib.ERR_INVALID_ARG
    assert _lib.lib().camoe_ex_dispatch_work_bytes(-1, 2, 8) == 0


def test_combine_statuses():
    f, b = _lib.lib().camoe_ex_combine, _lib.lib().camoe_ex_combine_bwd
    assert f(P, 2, P, P, P, 4, 2, 16, None) == _lib.ERR_UNSUPPORTED
    assert f(None, 0, P, P, P, 4, 2, 16, None) == _lib.ERR_INVALID_ARG
    assert f(None, 0, None, None, None, 0, 2, 16, None) == _lib.OK
    assert b(P, 0, P, None, P, P, P, P, 4, 2, 8, 16, None) == _lib.ERR_INVALID_ARG
    assert b(P, 0, P, P, None, P, P, P, 4, 2, 8, 16, None) == _lib.ERR_INVALID_ARG
    assert b(P, 0, P, P, P, P, None, None, 4, 2, 8, 16, None) == _lib.OK


def ffn(R=4, E=2, C=16, F=32, offsets=P, xs=P):
    return _lib.lib().camoe_ex_ffn_fwd(xs, P, P, offsets, P, P, P, R, E, C, F, None)


def test_ffn_statuses():
    for bad in (dict(R=-1), dict(E=0), dict(C=0), dict(F=0), dict(offsets=None), dict(xs=None)):
        assert ffn(**bad) == _lib.ERR_INVALID_ARG, bad
    for bad in (dict(E=1025), dict(C=12), dict(F=20)):
        assert ffn(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert ffn(R=1 << 31) == _lib.ERR_SHAPE
    assert ffn(xs=P + 2) == _lib.ERR_ALIGNMENT
    assert ffn(R=0) == _lib.OK
    b = _lib.lib().camoe_ex_ffn_bwd
    assert b(P + 4, *[P] * 10, 4, 2, 16, 32, None) == _lib.ERR_ALIGNMENT
    assert b(None, *[P] * 10, 4, 2, 16, 32, None) == _lib.ERR_INVALID_ARG


def test_adapter_statuses():
    lib = _lib.lib()
    need = lib.camoe_ad_work_bytes(500, 64, 64, 8, 4)
    assert need > 0 and lib.camoe_ad_work_bytes(500, 60, 64, 8, 4) == 0
    def call(N=500, C=64, M=64, D=8, L=4, x=P, nbytes=need):
        return lib.camoe_ad_linear(x, P, P, P, P, None, P, P, nbytes, N, C, M, D, L, None)
    for bad in (dict(N=-1), dict(C=0), dict(D=0), dict(L=0), dict(x=None)):
        assert call(**bad) == _lib.ERR_INVALID_ARG, bad
    for bad in (dict(C=60), dict(M=4), dict(D=264), dict(D=12), dict(L=1025)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert call(x=P + 8) == _lib.ERR_ALIGNMENT
    assert call(nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert call(N=0) == _lib.OK


def test_python_refuses_cpu_tensors():
    x, index = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int64)
    plan = experts.ExpertPlan(*(torch.zeros(s, dtype=torch.int32) for s in ((4,), (4, 2), (8,))))
    bf = torch.bfloat16
    for call in (lambda: experts.expert_dispatch(x, index, 3),
                 lambda: experts.expert_combine(torch.zeros(8, 16), torch.zeros(4, 2), plan),
                 lambda: experts.expert_ffn(torch.zeros(8, 16, dtype=bf), torch.zeros(3, 32, 16, dtype=bf),
                                            torch.zeros(3, 16, 32, dtype=bf), plan.offsets),
                 lambda: adapters.adapter_linear(torch.zeros(4, 16, dtype=bf), torch.zeros(8, 16, dtype=bf),
                                                 torch.zeros(2, 8, 16, dtype=bf), torch.zeros(2, 8, 8, dtype=bf),
                                                 torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_addresses_off_their_elements_are_refused():
    """Every array of every call, one element's half or less beside its place."""
    lib, want = _lib.lib(), _lib.ERR_ALIGNMENT
    f, b, p = lib.camoe_ex_combine, lib.camoe_ex_combine_bwd, lib.camoe_ex_dispatch
    for dtype, off in ((0, 1), (1, 2)):
        for at, o in ((0, off), (2, off), (3, 2), (4, 2), (5, 2), (6, 2), (7, 2)):
            arrays = [P, P, P, P, P, P, P, P]  # x, index, xs, offsets, position, source, work; the last unused
            if at == 7:
                arrays[1] += 4
            else:
                arrays[at] += o
            x, index, xs, offsets, position, source, work, _ = arrays
            assert p(x, dtype, index, 8, xs, offsets, position, source, work, 1 << 20, 50, 2, 8, 16, None) == want, at
        for at, o in ((0, off), (1, 2), (2, 2), (3, off)):
            rows, weight, position, out = [P + (o if i == at else 0) for i in range(4)]
            assert f(rows, dtype, weight, position, out, 4, 2, 16, None) == want, at
        for at, o in ((0, off), (1, off), (2, 2), (3, 2), (4, 2), (5, off), (6, 2)):
            dout, ys, weight, offsets, position, dys, dweight = [P + (o if i == at else 0) for i in range(7)]
            assert b(dout, dtype, ys, weight, offsets, position, dys, dweight, 4, 2, 8, 16, None) == want, at
    assert p(None, 0, None, 8, None, P + 2, None, None, None, 0, 0, 2, 8, 16, None) == want
    assert ffn(offsets=P + 2) == want
    assert lib.camoe_ex_ffn_bwd(P, P, P, P, P + 1, *[P] * 6, 4, 2, 16, 32, None) == want
    for adapter, scale in ((P + 2, None), (P, P + 1)):
        assert lib.camoe_ad_linear(P, P, P, P, adapter, scale, P, P, 1 << 30, 50, 64, 64, 8, 4, None) == want
