"""Norms around a block without a GPU: refusals of the C entry points and of the
wrappers.  Everything is refused on the host: nothing is launched and the dummy
pointers are never read."""

import ctypes

import pytest
import torch

from pagedmoe_amd import _lib, kernels as K

D = 0x1000


@pytest.mark.parametrize("change,msg", [
    (dict(x=None), b"null"), (dict(weight=None), b"null"), (dict(h=None), b"null"),
    (dict(xd=2), b"fp32 or bf16"), (dict(xd=-1), b"fp32 or bf16"), (dict(wd=2), b"fp32 or bf16"),
    (dict(n=-1), b"hidden"), (dict(d=0), b"hidden"), (dict(d=16385), b"hidden"),
    (dict(n=(1 << 23) + 1), b"2^23"), (dict(eps=-1e-6), b"eps"), (dict(eps=float("nan")), b"eps")])
def test_norm_refusals(change, msg):
    a = dict(x=D, xd=0, weight=D, wd=1, n=3, d=64, eps=1e-6, h=D) | change
    L = _lib.lib()
    assert L.pmoe_block_norm(a["x"], a["xd"], a["weight"], a["wd"], a["n"], a["d"], a["eps"], 0,
                             a["h"], None) == -1
    assert msg in L.pmoe_last_error()


ARRAYS = ("residual", "y", "weights", "shared_y", "shared_logit", "post", "gate", "next")


def join(change):
    a = dict(stream=0, wt=1, kind=0, gt=1, eps=1e-6, n=3, k=1, d=64, out=D, h=None, j=True,
             **dict.fromkeys(ARRAYS)) | dict(residual=D, y=D) | change
    j = _lib.Join()
    j.stream_dtype, j.weight_dtype, j.gate_kind, j.gate_dtype = (a["stream"], a["wt"], a["kind"],
                                                                 a["gt"])
    j.residual_scale = j.branch_scale = 1.0
    j.eps = a["eps"]
    return _lib.lib().pmoe_block_join(ctypes.byref(j) if a["j"] else None, *(a[n] for n in ARRAYS),
                                      a["n"], a["k"], a["d"], a["out"], a["h"], None)


@pytest.mark.parametrize("change,msg", [
    (dict(j=False), b"null"), (dict(residual=None), b"null"), (dict(y=None), b"null"),
    (dict(out=None), b"null"), (dict(stream=2), b"fp32 or bf16"), (dict(wt=2), b"fp32 or bf16"),
    (dict(gt=-1), b"fp32 or bf16"), (dict(n=-1), b"shape"), (dict(k=0), b"shape"),
    (dict(d=0), b"shape"), (dict(d=16392), b"shape"), (dict(n=(1 << 23) + 1), b"2^23"),
    (dict(k=2), b"weights"), (dict(shared_logit=D), b"shared_y"), (dict(gate=D), b"gate"),
    (dict(kind=1), b"gate"), (dict(kind=4, gate=D), b"gate"), (dict(kind=-1, gate=D), b"gate"),
    (dict(next=D), b"together"), (dict(h=D), b"together"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps")])
def test_join_refusals(change, msg):
    assert join(change) == -1
    assert msg in _lib.lib().pmoe_last_error()


def test_no_rows_launch_nothing():
    assert join(dict(n=0)) == 0 and join(dict(n=0, next=D, h=D, kind=3, gate=D, shared_y=D)) == 0
    assert _lib.lib().pmoe_block_norm(D, 0, D, 0, 0, 64, 0.0, 1, D, None) == 0


def test_wrappers_refuse_host_tensors():
    x, w = torch.zeros(2, 64), torch.ones(64)
    with pytest.raises(ValueError):
        K.block_norm(x, w)
    with pytest.raises(TypeError):
        K.block_norm(x.double(), w)
    with pytest.raises(ValueError):
        K.block_join(x, x.to(torch.bfloat16))
    with pytest.raises(TypeError):
        K.block_join(x.half(), x.to(torch.bfloat16))
