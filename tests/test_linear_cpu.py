"""Refusals of the channel-mixing products, checked before any CUDA call, and the clamping of `ends` in the plain form."""
import pytest
import torch

from tests import _linear as ref


def _t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_grouped_linear_refusals():
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    for call, match in (
        (lambda: GroupedLinear(_t(4, 8), _t(2, 6, 8)), 'CUDA'),
        (lambda: GroupedLinear(_t(4, 8), _t(8)), 'weight'),
        (lambda: GroupedLinear(_t(4, 8), _t(2, 8, 6).transpose(1, 2)), None),
        (lambda: GroupedLinear(_t(4, 8, dtype=torch.float32), _t(2, 6, 8, dtype=torch.float32)), 'fp16'),
        (lambda: GroupedLinear(_t(4, 8), _t(2, 6, 8, dtype=torch.bfloat16)), 'fp16'),
        (lambda: GroupedLinear(_t(8, 4).T, _t(2, 6, 8)), 'contiguous'),
        (lambda: GroupedLinear(_t(1, 8).expand(4, 8), _t(2, 6, 8)), 'overlap'),
        (lambda: GroupedLinear(_t(4, 3, 8), _t(2, 6, 8)), 'rows'),
        (lambda: GroupedLinear(_t(1, 8, 2, 3, 4), _t(2, 6, 8)), 'channels_last_3d'),
        (lambda: GroupedLinearDGRAD(_t(4, 8), _t(2, 6)), 'CUDA'),
        (lambda: GroupedLinearWGRAD(_t(4, 8), _t(4, 6, dtype=torch.bfloat16)), 'fp16'),
    ):
        with pytest.raises(AssertionError, match=match):
            call()


def test_int8_linear_refusals():
    from kerops_b200.ops.linear import Int8Linear, QuantRows

    x, w, s = _t(4, 8), _t(2, 6, 8, dtype=torch.int8), _t(2, 6, dtype=torch.float32)
    q = x.to(torch.int8)
    for call, match in (
        (lambda: Int8Linear(x, w, s), 'CUDA'),
        (lambda: Int8Linear(x, w.half(), s), 'int8'),
        (lambda: Int8Linear(x, w, s.half()), 'w_scale'),
        (lambda: Int8Linear(x, w, s[:1]), 'w_scale'),
        (lambda: Int8Linear(x.float(), w, s), 'fp16, bf16 or int8'),
        (lambda: Int8Linear(q, w, s), 'x_scale'),
        (lambda: Int8Linear(q, w, s, x_scale=torch.zeros(4)), 'x_scale and dtype'),
        (lambda: Int8Linear(q, w, s, x_scale=torch.zeros(3), dtype=torch.float16), 'x_scale'),
        (lambda: Int8Linear(q, w, s, x_scale=torch.zeros(4), dtype=torch.float32), 'dtype'),
        (lambda: Int8Linear(x, w, s, x_scale=torch.zeros(4)), 'belongs to int8'),
        (lambda: QuantRows(x), 'CUDA'),
        (lambda: QuantRows(x.float()), 'fp16'),
    ):
        with pytest.raises(AssertionError, match=match):
            call()


def test_ends_refusals():
    from kerops_b200.ops.linear import _launch

    dev = _t(4, 8)
    _launch.check_ends(None, 1, dev)
    _launch.check_ends(torch.zeros(3, dtype=torch.int32), 3, dev)
    for ends, groups in ((None, 2), (torch.zeros(3, dtype=torch.int64), 3), (torch.zeros(2, dtype=torch.int32), 3),
                         (torch.zeros(6, dtype=torch.int32)[::2], 3), (torch.zeros(3, 1, dtype=torch.int32), 3)):
        with pytest.raises(AssertionError, match='ends'):
            _launch.check_ends(ends, groups, dev)


def test_c_entry_points_refuse_bad_arguments(kdw_lib):
    f, i8, q = kdw_lib.kdw_linear_f16, kdw_lib.kdw_linear_i8, kdw_lib.kdw_quant_rows
    P = 4096  # any non-null address: these calls end before it is used
    ok = dict(op=0, a=P, b=P, out=P, ends=P, ws=None, nb=0, T=4, E=2, K=8, N=8, sa=8, sb=8, dt=0)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None)

    assert call(a=None) == call(b=None) == call(out=None) == call(ends=None) == -1
    assert b'null' in kdw_lib.kdw_last_error()
    for kw in (dict(T=0), dict(E=0), dict(K=0), dict(N=-1), dict(T=1 << 31), dict(E=1025), dict(E=1024, N=1 << 22), dict(op=3), dict(op=-1),
               dict(dt=2), dict(sa=7), dict(op=1, N=16), dict(op=2, sb=7)):
        assert call(**kw) == -1, kw
    for kw in (dict(a=P + 1), dict(b=P + 1), dict(out=P + 1), dict(ends=P + 2)):
        assert call(**kw) == -2, kw
    okg = dict(x=P, w=P, g=P, dx=P, dw=P, ends=P, ws=None, nb=0, T=400, E=2, K=9, N=8, sx=9, sg=8, dt=0)

    def callg(**kw):
        return kdw_lib.kdw_linear_grads_f16(*{**okg, **kw}.values(), None)

    for kw in (dict(x=None), dict(w=None), dict(g=None), dict(dx=None), dict(dw=None), dict(ends=None), dict(T=0), dict(sx=8), dict(sg=7),
               dict(dt=2), dict(E=1025)):
        assert callg(**kw) == -1, kw
    for kw in (dict(x=P + 1), dict(w=P + 1), dict(g=P + 1), dict(dx=P + 1), dict(dw=P + 1), dict(ends=P + 1)):
        assert callg(**kw) == -2, kw
    assert callg() == -3 and b'workspace' in kdw_lib.kdw_last_error()  # rows of nine values are copied into it
    ok8 = dict(x=P, xs=P, w=P, ws=P, y=P, ends=P, wsp=None, nb=0, T=4, E=2, K=16, N=8, sx=16, xt=2, dt=0)

    def call8(**kw):
        return i8(*{**ok8, **kw}.values(), None)

    for kw in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(ends=None), dict(K=131072, sx=131072), dict(xt=3),
               dict(dt=2), dict(sx=15), dict(T=0)):
        assert call8(**kw) == -1, kw
    assert call8(xs=P + 2) == call8(ws=P + 1) == call8(y=P + 1) == call8(xt=0, x=P + 1) == -2
    assert call8(xt=0, T=400) == -3 and b'workspace' in kdw_lib.kdw_last_error()
    assert q(None, P, P, 1, 8, 8, 0, None) == q(P, P, P, 0, 8, 8, 0, None) == q(P, P, P, 1, 8, 7, 0, None) == -1
    assert q(P, P, P, 1, 8, 8, 2, None) == -1 and q(P + 1, P, P, 1, 8, 8, 0, None) == -2
    assert kdw_lib.kdw_linear_f16_workspace_bytes(0, P, P, 0, 1, 8, 8, 8, 8, 0) == -1
    assert kdw_lib.kdw_linear_i8_workspace_bytes(P, P, 1, 1, 200000, 8, 200000, 0, 0) == -1


def test_spans_are_clamped():
    assert ref.spans([2, 1, 9, 4], 5) == [(0, 2), (2, 2), (2, 5), (5, 5)]
    assert ref.spans([-3, 2], 5) == [(0, 0), (0, 2)]


def test_the_listed_sizes_get_every_variant(kdw_lib):
    """The sizes that the GPU tests run get the variants they are listed for, and no sizes get a variant that is not listed."""
    auto = kdw_lib.kdw_linear_auto_variant
    for op, variant, T, E, K, N in ref.VARIANTS:
        assert auto(op % 3, 2 if op == 3 else 0, T, E, K, N, 148) == variant, (op, variant)
    listed = {(op, v) for op, v, *_ in ref.VARIANTS}
    g = torch.Generator().manual_seed(0)
    for _ in range(4000):
        T, K, N = (int(2 ** (float(torch.rand((), generator=g)) * b)) for b in (20, 13, 13))
        E, op = int(torch.randint(1, 40, (), generator=g)), int(torch.randint(0, 4, (), generator=g))
        assert (op, auto(op % 3, 2 if op == 3 else 0, T, E, K, N, 148)) in listed
    assert auto(3, 0, 8, 1, 8, 8, 148) == auto(0, 3, 8, 1, 8, 8, 148) == auto(0, 0, 0, 1, 8, 8, 148) == auto(0, 0, 8, 1, 8, 8, 0) == -1
