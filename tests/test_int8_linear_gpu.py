"""The row quantiser and the 8-bit integer product.  Both are defined to the bit: the quantised values are the exactly
rounded quotients, the integer sums are exact, and the two scales are applied in fp32 one after the other."""
import numpy as np
import pytest
import torch

from tests import _linear as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def _quant(x):
    """64-bit form; a quotient that is no half misses every half by 2^-20 and more, one that is comes out exactly."""
    f = x.double().cpu().numpy()
    top = np.abs(f).max(axis=1, keepdims=True)
    with np.errstate(invalid='ignore', divide='ignore'):
        q = np.where(top > 0, np.rint(f * 127 / top), 0)
    scale = (torch.from_numpy(top[:, 0]).float() / 127).to(x.device)
    return torch.from_numpy(q).to(torch.int8).to(x.device), scale


def _all_values(dtype):
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    return bits[torch.isfinite(bits)].cuda()


@pytest.mark.parametrize('dtype', TYPES)
def test_quant_every_value_against_many_maxima(dtype):
    from kerops_b200.ops.linear import QuantRows

    values = _all_values(dtype)
    g = torch.Generator(device='cuda').manual_seed(0)
    some = values[torch.randint(len(values), (60,), generator=g, device='cuda')].abs()
    edge = torch.tensor([1.0, 127.0, 254.0, 127 * 1.5, 2.0 ** -10, torch.finfo(dtype).max, torch.finfo(dtype).tiny], device='cuda').to(dtype)
    smallest = values[values > 0].min()
    for top in [*some, *edge, smallest]:
        row = torch.where(values.abs() <= top, values, torch.zeros_like(values))
        row = torch.cat([row, top.view(1)])[None]
        q, s = QuantRows(row)
        qr, sr = _quant(row)
        assert torch.equal(q, qr) and torch.equal(s, sr), float(top)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T,K', [(1, 1), (3, 7), (5, 8), (2, 1000), (9, 1024), (7, 1025), (3, 4096), (2, 8200), (1, 40003), (300, 33)])
def test_quant_shapes(T, K, dtype):
    from kerops_b200.ops.linear import QuantRows

    x = torch.randn(T, K, generator=torch.Generator(device='cuda').manual_seed(K), device='cuda').to(dtype)
    x[0] = 0 if T > 1 else x[0]
    q, s = QuantRows(x)
    qr, sr = _quant(x)
    assert q.shape == x.shape and torch.equal(q, qr) and torch.equal(s, sr)
    wide = torch.zeros(T, K + 11, dtype=dtype, device='cuda')
    wide[:, 3:3 + K] = x
    q, s = QuantRows(wide[:, 3:3 + K])
    assert torch.equal(q, qr) and torch.equal(s, sr)


@pytest.mark.parametrize('K', [40, 2000])
def test_quant_rows_that_are_not_finite(K):
    from kerops_b200.ops.linear import QuantRows

    x = torch.randn(6, K, device='cuda').half()
    x[1, K // 2], x[3, 0], x[4, K - 1] = float('nan'), float('inf'), float('-inf')
    q, s = QuantRows(x)
    bad = torch.tensor([False, True, False, True, True, False], device='cuda')
    assert torch.equal(torch.isnan(s), bad) and not q[bad].any()
    qr, sr = _quant(x[~bad])
    assert torch.equal(q[~bad], qr) and torch.equal(s[~bad], sr)


def _int8(T, K, N, E, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randint(-128, 128, (T, K), generator=g, device='cuda', dtype=torch.int8)
    w = torch.randint(-128, 128, (E, N, K), generator=g, device='cuda', dtype=torch.int8)
    return x, torch.rand(T, generator=g, device='cuda') + 0.01, w, (torch.rand(E, N, generator=g, device='cuda') + 0.01) / K


def _product(x, xs, w, ws, ends, dtype):
    sums = ref.fwd(x, w, ends)  # exact in 64 bits
    y = torch.zeros(sums.shape, dtype=dtype, device=x.device)
    for e, (a, b) in enumerate(ref.spans(ends, x.shape[0])):
        y[a:b] = (sums[a:b].float() * xs[a:b, None] * ws[e]).to(dtype)
    return y


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T,K,N,ends', [
    *[(T, K, N, None) for T in (1, 2, 8, 9, 31, 64, 129, 300) for K, N in ((1, 1), (16, 16), (33, 70), (128, 64), (272, 200))],
    (1, 4096, 1000, None), (3, 4100, 264, None), (16, 8192, 512, None), (60, 4096, 384, None), (1000, 512, 640, None),
    (300, 144, 136, [0, 100, 100, 290]), (300, 144, 136, [0, 0, 0]), (300, 70, 33, [200, 100, 400]),
    (12, 2048, 256, [0, 3, 3, 4, 12, 12]), (12, 100, 30, [0, 3, 3, 4, 9, 9]),
])
def test_product_to_the_bit(T, K, N, ends, dtype):
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import Int8Linear

    E = 1 if ends is None else len(ends)
    x, xs, w, ws = _int8(T, K, N, E, T + K + N)
    e = None if ends is None else ref.tensor_ends(ends)
    y = Int8Linear(x, w, ws, e, x_scale=xs, dtype=dtype)
    assert torch.equal(y, _product(x, xs, w, ws, ends or [T], dtype))
    assert _lib.device_status() == 0


@pytest.mark.parametrize('op,variant,T,E,K,N', [c for c in ref.VARIANTS if c[0] == 3])
def test_every_variant(kdw_lib, op, variant, T, E, K, N):
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import Int8Linear

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms != 148 or kdw_lib.kdw_linear_auto_variant(0, 2, T, E, K, N, sms) == variant
    x, xs, w, ws = _int8(T, K, N, E, T)
    ends = ref.uneven_ends(T, E)
    y = Int8Linear(x, w, ws, ref.tensor_ends(ends), x_scale=xs, dtype=torch.bfloat16)
    assert torch.equal(y, _product(x, xs, w, ws, ends, torch.bfloat16))
    assert _lib.device_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T,K,N,ends', [
    (1, 1, 1, None), (1, 4096, 512, None), (1, 1001, 333, None), (5, 2056, 72, None), (8, 64, 64, None), (33, 256, 100, None),
    (200, 1000, 130, None), (64, 4096, 1024, None), (1000, 520, 264, [10, 10, 900]), (7, 640, 128, [1, 1, 4, 6]),
    (16, 9000, 40, None),
])
def test_float_rows_are_quantised_within_the_call(T, K, N, ends, dtype):
    from kerops_b200.ops.linear import Int8Linear

    E = 1 if ends is None else len(ends)
    _, _, w, ws = _int8(T, K, N, E, 1)
    x = torch.randn(T, K, generator=torch.Generator(device='cuda').manual_seed(2), device='cuda').to(dtype)
    if T > 4:
        x[2] = 0
        x[3, 0] = float('inf')
    e = None if ends is None else ref.tensor_ends(ends)
    y = Int8Linear(x, w, ws, e)
    fine = torch.isfinite(x).all(1)
    q, s = _quant(torch.where(fine[:, None], x, torch.zeros_like(x)))
    s = torch.where(fine, s, torch.full_like(s, float('nan')))
    want = _product(q, s, w, ws, ends or [T], dtype)
    assert y.dtype == dtype and torch.equal(y.nan_to_num(7.0), want.nan_to_num(7.0))
    other = torch.bfloat16 if dtype == torch.float16 else torch.float16
    y = Int8Linear(x, w, ws, e, dtype=other)
    assert torch.equal(y.nan_to_num(7.0), _product(q, s, w, ws, ends or [T], other).nan_to_num(7.0))


def test_the_longest_sum_stays_inside_32_bits():
    from kerops_b200.ops.linear import Int8Linear
    from kerops_b200.ops.linear.int8_linear import MAX_K

    for T in (1, 130):
        x = torch.full((T, MAX_K), -128, dtype=torch.int8, device='cuda')
        w = torch.full((1, 24, MAX_K), -128, dtype=torch.int8, device='cuda')
        one = torch.full((T,), 2.0 ** -16, device='cuda')
        y = Int8Linear(x, w, torch.ones(1, 24, device='cuda'), x_scale=one, dtype=torch.float16)
        assert (y == 32768.0).all()  # 2^14 * 131071 / 2^16 = 32767.75, rounded


@pytest.mark.parametrize('T', [3, 200])
def test_small_scales_do_not_underflow_in_a_product_of_their_own(T):
    from kerops_b200.ops.linear import Int8Linear

    x = torch.full((T, 64), 100, dtype=torch.int8, device='cuda')
    w = torch.full((1, 8, 64), 100, dtype=torch.int8, device='cuda')
    y = Int8Linear(x, w, torch.full((1, 8), 1e-22, device='cuda'), x_scale=torch.full((T,), 1e-22, device='cuda'), dtype=torch.bfloat16)
    want = 640000 * 1e-44
    assert torch.all((y.double() - want).abs() <= want * 2 ** -7)


def test_strides_volumes_and_guard_bands():
    from kerops_b200.ops.linear import Int8Linear, QuantRows, _launch

    for T, K, N, pad in ((50, 64, 40, 16), (50, 64, 40, 3), (4, 96, 40, 16), (4, 96, 40, 5), (4, 30, 33, 0)):
        x, xs, w, ws = _int8(T, K + pad, N, 1, 3)
        view, w = x[:, pad // 2:pad // 2 + K], w[:, :, :K].contiguous()
        want = _product(view, xs, w, ws, [T], torch.float16)
        buf = torch.full((T * N + 8192,), 7.0, dtype=torch.float16, device='cuda')
        for shift in (4096, 4097):
            buf.fill_(7.0)
            out = buf[shift:shift + T * N].view(T, N)
            _launch.int8_product(view, xs, w, ws, out, None, T, 1, K, N)
            assert torch.equal(out, want) and (buf[:shift] == 7).all() and (buf[shift + T * N:] == 7).all()
    v = torch.randn(2, 3, 4, 5, 16, device='cuda').half().permute(0, 4, 1, 2, 3)
    wq, ws = QuantRows(torch.randn(2, 24, 16, device='cuda').half())
    e = ref.tensor_ends([60, 120])
    y = Int8Linear(v, wq, ws, e)
    rows = v.permute(0, 2, 3, 4, 1).reshape(120, 16)
    assert y.shape == (2, 24, 3, 4, 5) and y.is_contiguous(memory_format=torch.channels_last_3d)
    assert torch.equal(y.permute(0, 2, 3, 4, 1).reshape(120, 24), Int8Linear(rows, wq, ws, e))
    q, s = QuantRows(v)
    assert torch.equal(Int8Linear(q, wq, ws, e, x_scale=s, dtype=torch.float16), y)
    assert Int8Linear(rows[:0], wq, ws, e).shape == (0, 24)


@pytest.mark.parametrize('T', [2, 300])
def test_streams_and_capture(T):
    from kerops_b200.ops.linear import Int8Linear

    K, N = 1024, 200
    x = torch.randn(T, K, device='cuda').half()
    _, _, w, ws = _int8(1, K, N, 2, 1)
    e = ref.tensor_ends([1, T])
    want = Int8Linear(x, w, ws, e)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got += [Int8Linear(x, w, ws, e) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = Int8Linear(x, w, ws, e)
    x.copy_(torch.randn(T, K, device='cuda').half())
    e.copy_(ref.tensor_ends([0, T - 1]))
    y.fill_(float('nan'))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, Int8Linear(x, w, ws, e)) and not y[T - 1].any()


def test_trained_in_16_bits_then_answering_in_8():
    """The weights that GroupedLinear trains, quantised per output channel and used by Int8Linear: every output is off
    by what the two roundings of its factors allow."""
    from kerops_b200.autograd import ExpertLinear
    from kerops_b200.ops.linear import Int8Linear, QuantRows

    m = ExpertLinear(3, 128, 96, device='cuda', dtype=torch.bfloat16)
    x = torch.randn(100, 128, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').bfloat16()
    ends = [30, 30, 90]
    e = ref.tensor_ends(ends)
    w = m.weight.detach()
    y = Int8Linear(x, *QuantRows(w), e)
    # a value is off by half a step s/2 = max/254: |x w - x' w'| <= |x| dw + |w| dx + dx dw, summed over K; then half
    # a step of bf16 for the result and 2^-22 of it for the fp32 scales
    dx = x.double().abs().amax(1, keepdim=True) / 254
    want = ref.fwd(x, w, ends)
    dw = w.double().abs().amax(2) / 254
    for e_, (a, b) in enumerate(ref.spans(ends, 100)):
        slack = x[a:b].double().abs().sum(1, keepdim=True) * dw[e_] + dx[a:b] * w[e_].double().abs().sum(1) + 128 * dx[a:b] * dw[e_]
        assert ((y[a:b].double() - want[a:b]).abs() <= slack + (2.0 ** -8 + 2.0 ** -22) * (want[a:b].abs() + slack)).all()
    assert not y[90:].any()


@pytest.mark.parametrize('T,K,N,E', [(8, 512, 256, 3), (64, 4096, 2048, 1), (200, 1024, 512, 40), (600, 512, 768, 1),
                                     (777, 1001, 333, 2), (3000, 256, 1024, 5), (9000, 1024, 2048, 3)])
def test_every_operand_made_by_the_call_before(T, K, N, E):
    """Kernels start while the one before them still runs: a chain in which each call reads what the last ones wrote
    (rows, weights, scales and row counts) gives the same bits as with a synchronisation behind every call, and as a
    captured graph."""
    from kerops_b200.ops.linear import GroupedLinear, Int8Linear, QuantRows

    g = torch.Generator(device='cuda').manual_seed(T)
    x0 = torch.randn(T, K, generator=g, device='cuda').bfloat16()
    ws = [(torch.randn(E, N, K, generator=g, device='cuda') / K ** 0.5).bfloat16() for _ in range(3)]
    back = (torch.randn(E, K, N, generator=g, device='cuda') / N ** 0.5).bfloat16()
    counts = [torch.sort(torch.randint(0, T + 1, (E,), generator=g, device='cuda'))[0].int() for _ in range(3)]
    counts = [torch.cat([c[:-1], torch.full_like(c[-1:], T)]) for c in counts]
    e = torch.empty(E, dtype=torch.int32, device='cuda')

    def chain(after):
        x, out = x0, []
        for i in range(6):
            e.copy_(counts[i % 3])
            after()
            q, s = QuantRows(ws[i % 3])
            after()
            y = Int8Linear(x, q, s, e)
            after()
            x = GroupedLinear(y, back, e)
            after()
            out += [y, x]
        return out

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        got = chain(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(3):
        for t in got:
            t.fill_(float('nan'))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T,K', [(2501, k) for k in (1, 7, 8, 9, 16, 24, 31, 32, 40, 63, 64, 100, 128, 129, 136, 200, 256, 257, 300,
                                                     504, 512, 520, 1000, 1024, 1500, 2048, 4096)]
                         + [(700001, 8), (400003, 16), (300007, 33), (330001, 64), (200003, 128)])
def test_quant_many_rows(T, K, dtype):
    """Every split of a row over threads: rows that end inside a CTA's share, rows of zeros, of a NaN, of an infinity among
    others, rows of a wider matrix; and the product that quantises its rows itself."""
    from kerops_b200.ops.linear import Int8Linear, QuantRows

    g = torch.Generator(device='cuda').manual_seed(K)
    x = torch.randn(T, K, generator=g, device='cuda').to(dtype)
    x[::97] = 0
    odd = torch.arange(5, T, 101, device='cuda')
    good = torch.ones(T, dtype=torch.bool, device='cuda')
    good[odd] = False
    xr, sr = _quant(x)
    x[odd, odd % K] = torch.where(odd % 2 == 0, float('nan'), float('-inf')).to(dtype)
    xr[odd] = 0
    for pad, first in ((0, 0), (8, 0), (11, 3)):
        wide = torch.zeros(T, K + pad, dtype=dtype, device='cuda')
        rows = wide[:, first:first + K]
        rows.copy_(x)
        q, s = QuantRows(rows)
        assert torch.equal(q, xr) and torch.equal(s[good], sr[good]) and s[odd].isnan().all()
    w, ws = QuantRows(torch.randn(24, K, generator=g, device='cuda').to(dtype)[None])
    y = Int8Linear(x, w, ws)
    want = Int8Linear(q, w, ws, x_scale=s, dtype=dtype)
    assert torch.equal(y[good], want[good]) and y[odd].isnan().all()


@pytest.mark.parametrize('T,K,N', [(3, 64, 24), (12, 64, 24), (300, 64, 24), (18, 10864, 24), (638, 24, 1116), (300, 512, 400)])
def test_rows_of_large_values_do_not_overflow_on_their_way(T, K, N):
    """bf16 rows reach 3e38: sum times row scale may lie outside fp32 where the result, after the channel's scale, is inside."""
    from kerops_b200.ops.linear import Int8Linear, QuantRows

    g = torch.Generator(device='cuda').manual_seed(K)
    x = (torch.randn(T, K, generator=g, device='cuda') * 2.0 ** 120).bfloat16()
    x[1::3] *= 2.0 ** -100
    w, ws = QuantRows((torch.randn(1, N, K, generator=g, device='cuda') / (4 * K ** 0.5)).bfloat16())
    q, s = QuantRows(x)
    # exact sums; the scales (3 roundings of fp32) and the result (half a step of bf16, 2^-8) are rounded
    want = ref.fwd(q, w, [T]) * s[:, None].double() * ws.double()
    assert (s[0] * ref.fwd(q, w, [T])[0].abs().max().float()).isinf()  # the plain order's first product
    for y in (Int8Linear(x, w, ws), Int8Linear(q, w, ws, x_scale=s, dtype=torch.bfloat16)):
        assert ((y.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs()).all()


@pytest.mark.parametrize('variant,T,E,K,N', [
    (1128064, 17, 3, 32, 24), (1128128, 8484, 32, 32, 24), (1128256, 16926, 32, 32, 24), (1256256, 638, 8, 32, 11160),
    (2128064, 18, 3, 2784, 24), (2128128, 4926, 1, 4240, 24), (2128256, 9872, 2, 4032, 24), (2256256, 4800, 8, 2768, 160),
    (4128064, 17, 2, 2992, 24), (4128128, 1147, 32, 3968, 24), (4128256, 4105, 32, 4000, 24), (4256256, 2454, 2, 3936, 136),
    (8128064, 18, 1, 10864, 24), (8128128, 700, 1, 16000, 136), (8128256, 567, 1, 19200, 504),
])
def test_every_variant_behind_its_own_quantiser(kdw_lib, variant, T, E, K, N):
    """With 16-bit rows and aligned weights every tensor-core variant loads its weights while its rows are being quantised: the
    same bits as from rows quantised before, with other operands' calls close behind."""
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import Int8Linear, QuantRows

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms != 148 or kdw_lib.kdw_linear_auto_variant(0, 2, T, E, K, N, sms) == variant
    ends = ref.uneven_ends(T, E)
    e = ref.tensor_ends(ends)
    cases = []
    for seed in (1, 2):
        _, _, w, ws = _int8(1, K, N, E, seed)
        x = torch.randn(T, K, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda').bfloat16()
        q, s = QuantRows(x)
        y = Int8Linear(q, w, ws, e, x_scale=s, dtype=torch.float16)
        assert torch.equal(y, _product(q, s, w, ws, ends, torch.float16))
        cases.append((x, w, ws, y))
    for _ in range(5):
        got = [Int8Linear(x, w, ws, e, dtype=torch.float16) for x, w, ws, _ in cases]
        assert all(torch.equal(y, c[3]) for y, c in zip(got, cases))
    assert _lib.device_status() == 0


def test_rows_and_weights_beyond_32_bits():
    """More than 2^31 values quantised, multiplied and written; more than 2^31 weights for few rows and for many."""
    from kerops_b200.ops.linear import Int8Linear, QuantRows

    T, K, N, tail = 17_000_100, 136, 136, 2000
    x = torch.zeros(T, K, dtype=torch.float16, device='cuda')
    x[-tail:] = torch.randn(tail, K, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').half()
    w, ws = QuantRows(torch.randn(1, N, K, generator=torch.Generator(device='cuda').manual_seed(2), device='cuda').half())
    qr, sr = _quant(x[-tail:])
    want = _product(qr, sr, w, ws, [tail], torch.float16)
    q, s = QuantRows(x)
    assert torch.equal(q[-tail:], qr) and torch.equal(s[-tail:], sr) and not torch.count_nonzero(q[:-tail]) and not s[:-tail].any()
    for y in (Int8Linear(q, w, ws, x_scale=s, dtype=torch.float16), Int8Linear(x, w, ws)):
        assert torch.equal(y[-tail:], want) and not torch.count_nonzero(y[:-tail])
    del x, q, y
    torch.cuda.empty_cache()
    E, N, K = 40, 8200, 7632
    for T in (3, 12, 40):
        x, xs, wl, ws = _int8(T, K, N, 1, T)
        w = torch.zeros(E, N, K, dtype=torch.int8, device='cuda')
        w[-1] = wl[0]
        wide = torch.ones(E, N, device='cuda')
        wide[-1] = ws[0]
        y = Int8Linear(x, w, wide, ref.tensor_ends([0] * (E - 1) + [T]), x_scale=xs, dtype=torch.bfloat16)
        assert torch.equal(y, _product(x, xs, wl, ws, [T], torch.bfloat16))
        del w
    torch.cuda.empty_cache()
