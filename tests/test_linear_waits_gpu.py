"""Waits of the channel-mixing products between CTAs: of a pair, of a cluster that shares a tile, and behind the row quantiser."""
import pytest
import torch

from tests import _linear as ref

pytestmark = pytest.mark.gpu

# (operation, variant, T, E, K, N) as in _linear.VARIANTS; operation 3: rows of 16 bits, quantised within the call
WAITS = [
    (0, 1256256, 2556, 32, 24, 2592),
    (0, 1256256, 3000, 8, 512, 1536),
    (0, 2256256, 4325, 32, 1416, 168),
    (0, 4256256, 2485, 1, 2064, 144),
    (0, 4128064, 17, 1, 1528, 24),
    (0, 8128064, 17, 2, 5536, 24),
    (1, 1256256, 777, 8, 9536, 24),
    (1, 4256256, 2173, 8, 152, 1960),
    (2, 1256256, 22, 32, 2360, 136),
    (2, 1256256, 3000, 8, 1024, 1024),
    (2, 2256256, 1364, 1, 5232, 136),
    (2, 4256256, 4020, 2, 1160, 144),
    (3, 1128064, 300, 3, 520, 200),
    (3, 1256256, 638, 8, 24, 11160),
    (3, 2256256, 4800, 8, 2760, 160),
    (3, 4256256, 2454, 2, 3936, 136),
    (3, 8128064, 18, 1, 10864, 24),
]


def _call(kdw_lib, op, variant, T, E, K, N):
    """A product of these sizes as a function without arguments, and its exact result."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD, Int8Linear, QuantRows

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms != 148 or kdw_lib.kdw_linear_auto_variant(op % 3, 2 if op == 3 else 0, T, E, K, N, sms) == variant
    ends = ref.uneven_ends(T, E)
    e = ref.tensor_ends(ends)
    if op == 3:
        x = torch.randn(T, K, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').half()
        w, ws = QuantRows(torch.randn(E, N, K, generator=torch.Generator(device='cuda').manual_seed(2), device='cuda').half())
        q, s = QuantRows(x)
        want = ref.fwd(q, w, ends)
        for i, (a, b) in enumerate(ref.spans(ends, T)):
            want[a:b] = want[a:b].float() * s[a:b, None] * ws[i]
        return lambda: Int8Linear(x, w, ws, e), want.half()
    x, g = ref.integers((T, K), torch.float16, 1, top=1), ref.integers((T, N), torch.float16, 2, top=1)
    w = ref.integers((E, N, K), torch.float16, 3, top=1)
    if op == 0:
        return lambda: GroupedLinear(x, w, e), ref.fwd(x, w, ends).half()
    if op == 1:
        return lambda: GroupedLinearDGRAD(g, w, e), ref.dgrad(g, w, ends).half()
    return lambda: GroupedLinearWGRAD(x, g, e), ref.wgrad(x, g, ends).half()


@pytest.mark.parametrize('op,variant,T,E,K,N', WAITS)
def test_calls_close_behind_one_another(kdw_lib, op, variant, T, E, K, N):
    """A CTA leaves its shared memory to a CTA of the next call only when nothing is on its way to it any more."""
    from kerops_b200 import _lib

    call, want = _call(kdw_lib, op, variant, T, E, K, N)
    got = [call() for _ in range(20)]
    assert all(torch.equal(y, want) for y in got)
    assert _lib.device_status() == 0


@pytest.mark.parametrize('op,variant,T,E,K,N', WAITS)
def test_waits_that_run_out_are_reported_and_leave_the_context_usable(kdw_lib, op, variant, T, E, K, N):
    from kerops_b200 import _lib

    call, want = _call(kdw_lib, op, variant, T, E, K, N)
    assert torch.equal(call(), want) and _lib.device_status() == 0
    for stop in (0, 2):  # (of these sizes some CTAs, mostly all of them, load three stages and more)
        try:
            assert kdw_lib.kdw_test_wait_limits(20_000_000, stop) == 0
            call()
            assert _lib.device_status() == 1
        finally:
            kdw_lib.kdw_test_wait_limits(2_000_000_000, -1)
        assert torch.equal(call(), want) and _lib.device_status() == 0


@pytest.mark.parametrize('op,variant,T,E,K,N', [c for c in WAITS if c[0] == 2])
def test_a_pair_keeps_other_groups_rows_out(op, variant, T, E, K, N):
    """The last block of a group's rows reaches into the next group's: both CTAs of a pair clear those before the products
    read them, so that a NaN or an infinity there reaches nothing.  Every second group, and the rows of no group, hold such."""
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import GroupedLinearWGRAD

    ends = [T - 5] if E == 1 else [min(T - 5, (e + 1) * (T // E) + (1, 0, 2)[e % 3]) for e in range(E)]
    x, g = ref.integers((T, K), torch.float16, 1, top=1), ref.integers((T, N), torch.float16, 2, top=1)
    want = ref.wgrad(x, g, ends).half()
    live = torch.zeros(T, dtype=torch.bool, device='cuda')
    for a, b in ref.spans(ends, T)[::2]:
        live[a:b] = True
    x[~live], g[~live] = float('nan'), float('inf')
    e = ref.tensor_ends(ends)
    for _ in range(30):
        got = GroupedLinearWGRAD(x, g, e).view(E, N, K)
        assert torch.equal(got[::2], want[::2])
    assert _lib.device_status() == 0
