"""What kvs_linear, kvs_linear_backward, kvs_distill and kvs_distill_backward refuse, on the host: each
call returns its code before any CUDA call (the pointers here are plain numbers, never followed)."""

import ctypes as C
import math

import pytest

P = 0x10000  # a 256-byte aligned address that nothing reads
E_ARG, E_UNSUPPORTED, E_SCRATCH = -1, -2, -4


@pytest.fixture(scope="module")
def lib():
    from kvstreams import _native as N

    return N.load_library()


def _args(**kw):
    from kvstreams import _native as N

    base = dict(x=P, weight=P, out=P, ld_x=64, ld_w=64, ld_out=32, rows=4, n=32, k=64, dtype=N.KVS_BF16, activation=0,
                pre_dtype=0)
    return N.KvsLinearArgs(**{**base, **kw})


def _grads(**kw):
    from kvstreams import _native as N

    return N.KvsLinearGrads(**{**dict(gy=P, dx=P, dw=P, ld_gy=32, ld_dx=64, ld_dw=64), **kw})


@pytest.mark.parametrize("change,code", [
    (dict(x=None), E_ARG), (dict(weight=None), E_ARG), (dict(out=None), E_ARG),
    (dict(rows=-1), E_ARG), (dict(n=0), E_ARG), (dict(k=0), E_ARG),
    (dict(activation=4), E_ARG), (dict(activation=-1), E_ARG),
    (dict(ld_x=56), E_ARG), (dict(ld_w=56), E_ARG), (dict(ld_out=31), E_ARG),
    (dict(residual=P, ld_res=31), E_ARG), (dict(pre=P, ld_pre=31), E_ARG),
    (dict(weight_up=P, ld_w_up=56), E_ARG), (dict(weight_up=P, ld_w_up=64, bias=P), E_ARG),
    (dict(weight_up=P, ld_w_up=64, residual=P, ld_res=32), E_ARG),
    (dict(weight_up=P, ld_w_up=64, pre=P, ld_pre=63), E_ARG),
    (dict(dtype=0), E_UNSUPPORTED), (dict(dtype=1), E_UNSUPPORTED), (dict(dtype=9), E_UNSUPPORTED),
    (dict(k=60), E_UNSUPPORTED), (dict(rows=(1 << 30) + 1), E_UNSUPPORTED), (dict(ld_x=68), E_UNSUPPORTED), (dict(ld_w=68), E_UNSUPPORTED),
    (dict(x=P + 2), E_UNSUPPORTED), (dict(weight=P + 8), E_UNSUPPORTED),
    (dict(weight_up=P + 8, ld_w_up=64), E_UNSUPPORTED), (dict(pre=P, ld_pre=32, pre_dtype=3), E_UNSUPPORTED),
])
def test_linear(lib, change, code):
    assert lib.kvs_linear(C.byref(_args(**change)), None) == code


def test_linear_without_rows_does_nothing(lib):
    assert lib.kvs_linear(None, None) == E_ARG
    assert lib.kvs_linear(C.byref(_args(rows=0, x=None, out=None)), None) == 0


@pytest.mark.parametrize("args,grads,code", [
    (dict(), dict(gy=None), E_ARG), (dict(), dict(ld_gy=31), E_ARG), (dict(), dict(ld_dx=63), E_ARG),
    (dict(), dict(ld_dw=63), E_ARG), (dict(), dict(dw_up=P), E_ARG), (dict(activation=2), dict(), E_ARG),
    (dict(activation=2, pre=P, ld_pre=31), dict(), E_ARG),
    (dict(weight_up=P, ld_w_up=64, pre=P, ld_pre=64), dict(), E_ARG),                    # dw without dw_up
    (dict(weight_up=P, ld_w_up=64, pre=P, ld_pre=64), dict(dw_up=P, db=P), E_ARG),       # gated has no bias
    (dict(weight_up=P, ld_w_up=64), dict(dw_up=P), E_ARG),                               # gated needs pre
    (dict(k=60), dict(), E_UNSUPPORTED),
    (dict(activation=2, pre=P, ld_pre=32), dict(), E_SCRATCH), (dict(), dict(db=P), E_SCRATCH),
    (dict(), dict(db=P, scratch=P + 8, scratch_bytes=1 << 20), E_SCRATCH),
    (dict(weight_up=P, ld_w_up=64, pre=P, ld_pre=64), dict(dw_up=P, scratch=P, scratch_bytes=100), E_SCRATCH),
])
def test_linear_backward(lib, args, grads, code):
    assert lib.kvs_linear_backward(C.byref(_args(**args)), C.byref(_grads(**grads)), None) == code


def test_backward_scratch(lib):
    """dz of the operands' type in rows padded to 8, bias partials in float32; nothing for a plain
    product whose gradient the tensor maps take as it lies."""
    size = lambda a, g: lib.kvs_linear_backward_scratch_bytes(C.byref(_args(**a)), C.byref(_grads(**g)))  # noqa: E731
    assert size({}, {}) == 0
    assert size({}, dict(ld_gy=33)) >= 4 * 32 * 2
    assert size(dict(n=33), dict(ld_gy=33)) >= 4 * 40 * 2
    assert size(dict(activation=1), {}) >= 4 * 32 * 2
    assert size(dict(weight_up=P, n=33), {}) >= 4 * 80 * 2
    assert size({}, dict(db=P)) >= 32 * 4
    assert size(dict(rows=0), dict(db=P)) == 0


def test_forward_scratch(lib):
    """Only products whose tiles do not come out even have scratch to gain from, and few rows never."""
    size = lambda **kw: lib.kvs_linear_scratch_bytes(C.byref(_args(**kw)))  # noqa: E731
    assert lib.kvs_linear_scratch_bytes(None) == 0
    assert size() == 0 and size(rows=0) == 0
    assert size(rows=128, n=4096, k=14336, ld_x=14336, ld_w=14336, ld_out=4096) == 0
    assert size(rows=1536, n=4096, k=4096, ld_x=4096, ld_w=4096, ld_out=4096) > 0


def test_scratch_of_sizes_past_the_limits(lib):
    """Sizes that the calls refuse have no scratch, also where their block counts would pass 32 bits."""
    for kw in (dict(k=2**31 - 8), dict(n=2**31 - 1), dict(n=(1 << 29) + 8), dict(rows=2**31 - 1)):
        a = _args(**{**dict(rows=300), **kw})
        assert lib.kvs_linear_scratch_bytes(C.byref(a)) == 0
        assert lib.kvs_linear_backward_scratch_bytes(C.byref(a), C.byref(_grads(db=P))) == 0
        assert lib.kvs_linear(C.byref(a), None) == E_UNSUPPORTED


def _distill(lib, **kw):
    a = {**dict(logits=P, ld=100, n_rows=2, vocab=100, ids=P, teacher=P, top=4, temperature=1.0, dtype=0, loss=P,
                lse=P), **kw}
    return lib.kvs_distill(a["logits"], a["ld"], a["n_rows"], a["vocab"], a["ids"], a["teacher"], a["top"],
                           a["temperature"], a["dtype"], a["loss"], a["lse"], None)


def _distill_bwd(lib, **kw):
    a = {**dict(logits=P, ld=100, n_rows=2, vocab=100, ids=P, teacher=P, top=4, lse=P, grad=P, temperature=1.0,
                dtype=0, d=2 * P, ld_out=100, out_dtype=0), **kw}
    return lib.kvs_distill_backward(a["logits"], a["ld"], a["n_rows"], a["vocab"], a["ids"], a["teacher"], a["top"],
                                    a["lse"], a["grad"], a["temperature"], a["dtype"], a["d"], a["ld_out"],
                                    a["out_dtype"], None)


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), E_ARG), (dict(ids=None), E_ARG), (dict(teacher=None), E_ARG), (dict(lse=None), E_ARG),
    (dict(n_rows=-1), E_ARG), (dict(vocab=0), E_ARG), (dict(top=0), E_ARG), (dict(ld=99), E_ARG),
    (dict(temperature=0.0), E_ARG), (dict(temperature=-1.0), E_ARG), (dict(temperature=math.nan), E_ARG),
    (dict(temperature=math.inf), E_ARG), (dict(top=1025), E_UNSUPPORTED), (dict(dtype=4), E_UNSUPPORTED),
    (dict(dtype=-1), E_UNSUPPORTED), (dict(n_rows=0, logits=None), 0),
])
def test_distill(lib, change, code):
    assert _distill(lib, **change) == code
    assert _distill_bwd(lib, **change) == code


def test_distill_backward_types_and_places(lib):
    from kvstreams import _native as N

    assert _distill(lib, loss=None) == E_ARG
    assert _distill_bwd(lib, grad=None) == E_ARG
    assert _distill_bwd(lib, d=None) == E_ARG
    assert _distill_bwd(lib, ld_out=99) == E_ARG
    assert _distill_bwd(lib, d=P, ld_out=101) == E_ARG                 # in place, other rows
    assert _distill_bwd(lib, d=P, out_dtype=N.KVS_BF16) == E_ARG       # in place, other type
    for dtype, out in [(N.KVS_F32, N.KVS_F64), (N.KVS_BF16, N.KVS_F32), (N.KVS_BF16, N.KVS_F16), (N.KVS_F64, N.KVS_F32)]:
        assert _distill_bwd(lib, dtype=dtype, out_dtype=out) == E_UNSUPPORTED


def test_host_tensors_are_refused():
    import torch

    from kvstreams import ops

    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear_backward(torch.zeros(2, 32, dtype=torch.bfloat16), x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.distill(torch.zeros(2, 10), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3))
