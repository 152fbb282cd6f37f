"""Products of row groups (forward, input gradient, weight gradient) against a plain 64-bit form.  The inputs are small
whole numbers wherever possible: their sums are exact in fp32 in any order, so the comparison is bit for bit."""
import pytest
import torch

from tests import _linear as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def _check(T, K, N, ends, dtype, seed=0):
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    spec = ends
    ends = [T] if spec is None else spec
    E = len(ends)
    x, g = ref.integers((T, K), dtype, seed), ref.integers((T, N), dtype, seed + 1)
    w = ref.integers((E, N, K), dtype, seed + 2)
    e = None if spec is None else ref.tensor_ends(ends)
    y, dx = GroupedLinear(x, w, e), GroupedLinearDGRAD(g, w, e)
    dw = GroupedLinearWGRAD(x, g, e)
    assert dw.shape == ((N, K) if e is None else (E, N, K))
    assert torch.equal(y, ref.fwd(x, w, ends).to(dtype))
    assert torch.equal(dx, ref.dgrad(g, w, ends).to(dtype))
    assert torch.equal(dw.view(E, N, K), ref.wgrad(x, g, ends).to(dtype))
    assert _lib.device_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T', [1, 2, 9, 17, 33, 64, 127, 128, 129, 300])
@pytest.mark.parametrize('K,N', [(1, 1), (8, 8), (16, 264), (37, 5), (64, 64), (100, 63), (200, 136), (264, 520)])
def test_one_group(T, K, N, dtype):
    _check(T, K, N, None, dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T,ends', [
    (1, [0, 1, 1]),
    (5, [1, 2, 3, 4, 5]),
    (300, [0, 0, 300]),
    (300, [300, 300, 300]),
    (300, [1, 130, 131, 259]),           # rows behind the last group
    (300, [0, 0, 0]),                    # no group has rows
    (300, [200, 100, 250]),              # an end that steps back: an empty group
    (300, [100, 400, 200]),              # ends past the last row
    (300, [-5, 128, 256]),
    (1000, [64, 128, 500, 513, 514, 999]),
])
@pytest.mark.parametrize('K,N', [(64, 72), (33, 130), (320, 64)])
def test_groups(T, ends, K, N, dtype):
    _check(T, K, N, ends, dtype)


@pytest.mark.parametrize('E', [33, 1000, 1024])
def test_many_groups(E):
    g = torch.Generator().manual_seed(E)
    ends = torch.cumsum(torch.randint(0, 4, (E,), generator=g), 0).tolist()
    _check(ends[-1] + 3, 40, 24, ends, torch.bfloat16)


@pytest.mark.parametrize('T,K,N,ends', [
    (4096, 512, 768, None),              # wide tiles
    (3000, 1024, 512, [1000, 1700, 2990]),
    (16, 4096, 512, None),               # a long contraction over few rows: shares that are added afterwards
    (40, 4104, 512, [3, 30]),
    (150, 2048, 130, None),
    (30000, 64, 96, None),               # a long contraction of the weight gradient
    (30011, 40, 72, [29000, 29000, 30000]),
])
def test_larger(T, K, N, ends):
    _check(T, K, N, ends, torch.float16)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('K', [8, 16, 24, 32, 64, 104, 128])
def test_narrow_weights_and_many_rows(K, dtype):
    """Few channels: row products that stream the rows, and weight gradients that fold rows together."""
    for i, N in enumerate((8, 16, 40, 64, 128)):
        _check((8192, 9000, 8200, 8194, 8193)[(i + K // 8) % 5], K, N, None, dtype)
        _check(777, K, N, [771], dtype)


@pytest.mark.parametrize('K,N', [(8, 8), (8, 128), (32, 24), (128, 16), (64, 64)])
@pytest.mark.parametrize('T', [8192, 100000])
def test_one_narrow_group_that_ends_before_the_last_row(T, K, N):
    _check(T, K, N, [T - 70], torch.bfloat16)


def test_one_pass_gradients_keep_rows_apart_and_repeat():
    """NaN and infinities in rows of no group reach nothing, in a row of the group its own dx and dw; same bits every call."""
    from kerops_b200.ops.linear import _launch

    T, K, N = 40000, 32, 64
    x, g, w = ref.integers((T, K), torch.bfloat16, 1), ref.integers((T, N), torch.bfloat16, 2), ref.integers((1, N, K), torch.bfloat16, 3)
    e = ref.tensor_ends([T - 100])
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    want = ref.dgrad(g, w, [T - 100]).bfloat16(), ref.wgrad(x, g, [T - 100]).bfloat16()
    x[T - 100:], g[T - 100:] = float('nan'), float('inf')
    _launch.grads(x, w, g, dx, dw, e, T, 1, K, N)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    g[777, 5] = float('nan')
    _launch.grads(x, w, g, dx, dw, e, T, 1, K, N)
    rows, outs = torch.arange(T, device='cuda') != 777, torch.arange(N, device='cuda') != 5
    assert torch.equal(dx[rows], want[0][rows]) and torch.isnan(dx[777]).all()
    assert torch.equal(dw[:, outs], want[1][:, outs]) and torch.isnan(dw[:, 5]).all()
    x, g = torch.randn(T, K, device='cuda').bfloat16(), torch.randn(T, N, device='cuda').bfloat16()
    first = None
    for _ in range(3):
        _launch.grads(x, w, g, dx, dw, e, T, 1, K, N)
        first = first or (dx.clone(), dw.clone())
        assert torch.equal(dx, first[0]) and torch.equal(dw, first[1])
    # half a step of bf16: values in [2^e, 2^(e+1)) lie 2^(e-7) apart (8 significant bits), so a rounding is off by at most
    # 2^(e-8) <= 2^-8 of the value; and a step of fp32 of the magnitudes for each of the n additions
    for got, f, args, n in ((dx, ref.dgrad, (g, w), N), (dw, ref.wgrad, (x, g), T)):
        full, size = f(*args, [T - 100]), f(*(a.abs() for a in args), [T - 100])
        assert ((got.double() - full).abs() <= 2.0 ** -8 * full.abs() + n * 2.0 ** -23 * size).all()


def test_folded_rows_do_not_mix():
    """A NaN in one voxel stays with its own products: the blocks that pair neighbouring voxels are not summed."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    T, K, N = 16384, 8, 16
    x, g = ref.integers((T, K), torch.float16, 1), ref.integers((T, N), torch.float16, 2)
    w = ref.integers((N, K), torch.float16, 3)
    y, dx = ref.fwd(x, w[None], [T]).half(), ref.dgrad(g, w[None], [T]).half()
    x[1001, 3] = float('nan')
    g[1000] = float('inf')  # the neighbouring voxel
    got = GroupedLinearWGRAD(x, g)
    assert torch.isnan(got[:, 3]).all()
    keep = [0, 1, 2, 4, 5, 6, 7]
    want = ref.wgrad(x[:, keep], g, [T])[0]
    assert torch.equal(got[:, keep].nan_to_num(7.0), want.half().nan_to_num(7.0))
    gy, gdx = GroupedLinear(x, w), GroupedLinearDGRAD(g, w)
    rows = torch.arange(T, device='cuda')
    assert torch.equal(gy[rows != 1001], y[rows != 1001]) and torch.isnan(gy[1001]).all()
    assert torch.equal(gdx[rows != 1000], dx[rows != 1000])


@pytest.mark.parametrize('op,variant,T,E,K,N', [c for c in ref.VARIANTS if c[0] < 3])
def test_every_variant(kdw_lib, op, variant, T, E, K, N):
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms != 148 or kdw_lib.kdw_linear_auto_variant(op, 0, T, E, K, N, sms) == variant
    x, g = ref.integers((T, K), torch.float16, 1, top=1), ref.integers((T, N), torch.float16, 2, top=1)
    w = ref.integers((E, N, K), torch.float16, 3, top=1)
    # the kernels that fold rows take one group of all rows
    ends = [T] if variant // 1000000 == 32 else ref.uneven_ends(T, E)
    e = None if variant // 1000000 == 32 else ref.tensor_ends(ends)
    if op == 0:
        assert torch.equal(GroupedLinear(x, w, e), ref.fwd(x, w, ends).half())
    elif op == 1:
        assert torch.equal(GroupedLinearDGRAD(g, w, e), ref.dgrad(g, w, ends).half())
    else:
        assert torch.equal(GroupedLinearWGRAD(x, g, e).view(E, N, K), ref.wgrad(x, g, ends).half())
    from kerops_b200 import _lib

    assert _lib.device_status() == 0


@pytest.mark.parametrize('dtype', TYPES)
def test_normal_values_within_the_rounding(dtype):
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    T, K, N, ends = 700, 328, 200, [100, 100, 650]
    gen = torch.Generator(device='cuda').manual_seed(4)
    x = torch.randn(T, K, generator=gen, device='cuda').to(dtype)
    g = torch.randn(T, N, generator=gen, device='cuda').to(dtype)
    w = (torch.randn(3, N, K, generator=gen, device='cuda') / K ** 0.5).to(dtype)
    e = ref.tensor_ends(ends)
    # half a step of the result, and for each of the n fp32 additions at most a step of fp32 (2^-23) of the sum of
    # magnitudes; the last term is half the smallest subnormal of fp16
    for got, f, args, n in ((GroupedLinear(x, w, e), ref.fwd, (x, w), K), (GroupedLinearDGRAD(g, w, e), ref.dgrad, (g, w), N),
                            (GroupedLinearWGRAD(x, g, e), ref.wgrad, (x, g), T)):
        want, size = f(*args, ends), f(*(a.abs() for a in args), ends)
        err = (got.double() - want).abs()
        assert (err <= torch.finfo(dtype).eps / 2 * want.abs() + n * 2.0 ** -23 * size + 2.0 ** -25).all()


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_a_group_sees_only_its_rows(bad):
    """NaN and infinities in one group, and in rows of no group, change no other group's results."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    T, K, N, ends = 500, 72, 136, [100, 230, 400]
    x, g = ref.integers((T, K), torch.float16, 1), ref.integers((T, N), torch.float16, 2)
    w = ref.integers((3, N, K), torch.float16, 3)
    e = ref.tensor_ends(ends)
    y, dx, dw = ref.fwd(x, w, ends).half(), ref.dgrad(g, w, ends).half(), ref.wgrad(x, g, ends).half()
    x[100:230], g[100:230], x[400:], g[400:] = bad, bad, bad, bad
    gy, gdx, gdw = GroupedLinear(x, w, e), GroupedLinearDGRAD(g, w, e), GroupedLinearWGRAD(x, g, e)
    keep = [*range(100), *range(230, 500)]
    assert torch.equal(gy[keep], y[keep]) and torch.equal(gdx[keep], dx[keep])
    assert torch.equal(gdw[[0, 2]], dw[[0, 2]])
    assert not torch.isfinite(gdw[1]).any()
    assert torch.isnan(gy[100:230]).all() or torch.isinf(gy[100:230]).any()


@pytest.mark.parametrize('offset,stride', [(0, 80), (8, 88), (1, 80), (0, 73), (3, 91)])
def test_row_strides_and_bases(offset, stride):
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    T, C, N, ends = 333, 72, 72, [10, 300]
    wide_x, wide_g = ref.integers((T, stride + 8), torch.bfloat16, 1), ref.integers((T, stride + 8), torch.bfloat16, 2)
    wide_x, wide_g = wide_x.flatten()[:T * stride + 8], wide_g.flatten()[:T * stride + 8]
    before = wide_x.clone(), wide_g.clone()
    x, g = (torch.as_strided(t, (T, C), (stride, 1), offset) for t in (wide_x, wide_g))
    w = ref.integers((2, N, C), torch.bfloat16, 3)
    e = ref.tensor_ends(ends)
    assert torch.equal(GroupedLinear(x, w, e), ref.fwd(x, w, ends).bfloat16())
    assert torch.equal(GroupedLinearDGRAD(g, w, e), ref.dgrad(g, w, ends).bfloat16())
    assert torch.equal(GroupedLinearWGRAD(x, g, e), ref.wgrad(x, g, ends).bfloat16())
    assert torch.equal(wide_x, before[0]) and torch.equal(wide_g, before[1])


@pytest.mark.parametrize('K', [64, 33])
@pytest.mark.parametrize('rows', [12, 400])
def test_nothing_beyond_the_outputs_is_written(K, rows):
    from kerops_b200.ops.linear import _launch

    N, ends, guard = 72, [rows // 4, rows - 5], 4096
    x, g = ref.integers((rows, K), torch.float16, 1), ref.integers((rows, N), torch.float16, 2)
    w = ref.integers((2, N, K), torch.float16, 3)
    e = ref.tensor_ends(ends)
    for op, a, b, shape, want in ((0, x, w, (rows, N), ref.fwd(x, w, ends)), (1, g, w, (rows, K), ref.dgrad(g, w, ends)),
                                  (2, g, x, (2, N, K), ref.wgrad(x, g, ends))):
        n = torch.Size(shape).numel()
        for shift in (0, 1):  # an aligned output and one that only scalar stores reach
            buf = torch.full((n + 2 * guard,), 7.0, dtype=torch.float16, device='cuda')
            out = buf[guard + shift:guard + shift + n].view(shape)
            _launch.product(op, a, b, out, e, rows, 2, K, N)
            assert torch.equal(out, want.half())
            assert (buf[:guard + shift] == 7).all() and (buf[guard + shift + n:] == 7).all()


def test_volumes_and_empty_inputs():
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    x = ref.integers((2, 3, 5, 7, 16), torch.float16, 1).permute(0, 4, 1, 2, 3)
    g = ref.integers((2, 3, 5, 7, 24), torch.float16, 2).permute(0, 4, 1, 2, 3)
    w = ref.integers((2, 24, 16), torch.float16, 3)
    e = ref.tensor_ends([105, 210])  # a group per sample
    xr, gr = x.permute(0, 2, 3, 4, 1).reshape(210, 16), g.permute(0, 2, 3, 4, 1).reshape(210, 24)
    y, dx = GroupedLinear(x, w, e), GroupedLinearDGRAD(g, w, e)
    assert y.shape == g.shape and y.stride() == g.stride() and dx.shape == x.shape and dx.stride() == x.stride()
    assert torch.equal(y.permute(0, 2, 3, 4, 1).reshape(210, 24), ref.fwd(xr, w, [105, 210]).half())
    assert torch.equal(dx.permute(0, 2, 3, 4, 1).reshape(210, 16), ref.dgrad(gr, w, [105, 210]).half())
    assert torch.equal(GroupedLinearWGRAD(x, g, e), ref.wgrad(xr, gr, [105, 210]).half())
    none = torch.empty(0, 16, dtype=torch.float16, device='cuda')
    assert GroupedLinear(none, w, e).shape == (0, 24)
    assert torch.equal(GroupedLinearWGRAD(none, torch.empty(0, 24, dtype=torch.float16, device='cuda'), e), torch.zeros_like(w))


def test_offsets_beyond_32_bits():
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    T, K, N = 17_000_100, 136, 136  # 2.3e9 values per operand
    ends = [16_999_000, 17_000_050]
    x = torch.zeros(T, K, dtype=torch.float16, device='cuda')
    tail = ref.integers((2000, K), torch.float16, 1)
    x[-2000:] = tail
    w = ref.integers((2, N, K), torch.float16, 2)
    e = ref.tensor_ends(ends)
    local = [t - (T - 2000) for t in ends]
    want = ref.fwd(tail, w, local).half()
    y = GroupedLinear(x, w, e)
    assert torch.equal(y[-2000:], want) and not y[:-2000].any()
    del y
    dx = GroupedLinearDGRAD(x, w, e)
    assert torch.equal(dx[-2000:], ref.dgrad(tail, w, local).half()) and not dx[:-2000].any()
    del dx
    assert torch.equal(GroupedLinearWGRAD(x, x, e), ref.wgrad(tail, tail, local).half())


def test_same_bits_every_call_and_on_any_stream():
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearWGRAD

    T, K, N = 20000, 96, 160
    gen = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randn(T, K, generator=gen, device='cuda', dtype=torch.float16)
    g = torch.randn(T, N, generator=gen, device='cuda', dtype=torch.float16)
    w = torch.randn(3, N, K, generator=gen, device='cuda', dtype=torch.float16)
    e = ref.tensor_ends([3000, 15000, 20000])
    first = GroupedLinear(x, w, e), GroupedLinearWGRAD(x, g, e)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((GroupedLinear(x, w, e), GroupedLinearWGRAD(x, g, e)))
    torch.cuda.synchronize()
    for y, dw in got:
        assert torch.equal(y, first[0]) and torch.equal(dw, first[1])


def test_capture_and_replay():
    """The row counts are read on the device: a captured step replays on other rows, weights and ends."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    T, K, N = 600, 72, 200
    x, g = ref.integers((T, K), torch.float16, 1), ref.integers((T, N), torch.float16, 2)
    w, e = ref.integers((3, N, K), torch.float16, 3), ref.tensor_ends([100, 400, 600])

    def step():
        return GroupedLinear(x, w, e), GroupedLinearDGRAD(g, w, e), GroupedLinearWGRAD(x, g, e)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs do not share a workspace
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for seed, ends in ((10, [1, 1, 590]), (20, [600, 600, 600]), (30, [0, 300, 301])):
        x.copy_(ref.integers((T, K), torch.float16, seed))
        w.copy_(ref.integers((3, N, K), torch.float16, seed + 1))
        e.copy_(ref.tensor_ends(ends))
        for o in outs:
            for t in o:
                t.fill_(float('nan'))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for y, dx, dw in outs:
            assert torch.equal(y, ref.fwd(x, w, ends).half())
            assert torch.equal(dx, ref.dgrad(g, w, ends).half())
            assert torch.equal(dw, ref.wgrad(x, g, ends).half())


@pytest.mark.parametrize('T,K,N,ends', [
    (1, 5, 3, None), (40, 8, 8, None), (300, 37, 64, None), (300, 64, 37, [10, 10, 290]), (9000, 24, 8, None), (9000, 24, 8, [8990]),
    (2000, 512, 264, [700, 1500]), (20000, 72, 130, None), (60, 4096, 520, [0, 60]), (8192, 8, 128, None),
    # one pass over rows and gradients: every width of both
    *[(32768 + 37 * i, K, N, None) for i, (K, N) in enumerate((K, N) for K in (8, 16, 24, 64, 104) for N in (8, 16, 32, 40, 128)
                                                             if K * N <= 2048)],
    (40000, 32, 64, [39987]), (40000, 64, 32, [0]),
])
@pytest.mark.parametrize('offset,extra', [(0, 0), (8, 8), (3, 5)])
def test_both_gradients_of_one_call(T, K, N, ends, offset, extra):
    """One call for both gradients gives what the two operators give, from rows anywhere, and writes nothing else."""
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import _launch

    spec, ends = ends, [T] if ends is None else ends
    E, guard = len(ends), 1024
    e = None if spec is None else ref.tensor_ends(ends)
    x, g = (torch.as_strided(ref.integers((T * (c + extra) + offset,), torch.float16, i, top=1), (T, c), (c + extra, 1), offset)
            for i, c in enumerate((K, N)))
    w = ref.integers((E, N, K), torch.float16, 3, top=1)
    for shift in (0, 1):
        bx, bw = (torch.full((n + 2 * guard,), 7.0, dtype=torch.float16, device='cuda') for n in (T * K, E * N * K))
        dx, dw = bx[guard + shift:guard + shift + T * K].view(T, K), bw[guard + shift:guard + shift + E * N * K].view(E, N, K)
        _launch.grads(x, w, g, dx, dw, e, T, E, K, N)
        assert torch.equal(dx, ref.dgrad(g, w, ends).half()) and torch.equal(dw, ref.wgrad(x, g, ends).half())
        for b, n in ((bx, T * K), (bw, E * N * K)):
            assert (b[:guard + shift] == 7).all() and (b[guard + shift + n:] == 7).all()
    assert _lib.device_status() == 0


def test_a_training_step_is_captured():
    """Forward and backward in a graph, the first calls of this kind in the autograd thread among them."""
    from kerops_b200.autograd import grouped_linear

    T, K, N, ends = 400, 72, 40, [100, 390]
    x, w = ref.integers((T, K), torch.float16, 1), ref.integers((2, N, K), torch.float16, 2)
    g, e = ref.integers((T, N), torch.float16, 3), ref.tensor_ends(ends)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = grouped_linear(xl, wl, e)
        dx, dw = torch.autograd.grad(y, (xl, wl), g)
    for seed in (4, 5):
        x.copy_(ref.integers((T, K), torch.float16, seed))
        g.copy_(ref.integers((T, N), torch.float16, seed + 10))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref.fwd(x, w, ends).half())
        assert torch.equal(dx, ref.dgrad(g, w, ends).half()) and torch.equal(dw, ref.wgrad(x, g, ends).half())


@pytest.mark.parametrize('shape', ['matrix', 'volume'])
def test_autograd_formula_and_differences(shape):
    from kerops_b200.autograd import ExpertLinear, grouped_linear

    T, K, N, ends = 210, 16, 24, [50, 50, 200]
    e = ref.tensor_ends(ends)

    def form(t):
        return t if shape == 'matrix' else t.view(2, 3, 5, 7, -1).permute(0, 4, 1, 2, 3)

    def rows(t):
        return t if shape == 'matrix' else t.permute(0, 2, 3, 4, 1).reshape(T, -1)

    x, w = form(ref.integers((T, K), torch.float16, 1)).requires_grad_(True), ref.integers((3, N, K), torch.float16, 2).requires_grad_(True)
    g = form(ref.integers((T, N), torch.float16, 3))
    y = grouped_linear(x, w, e)
    y.backward(g)
    assert torch.equal(rows(x.grad), ref.dgrad(rows(g), w.detach(), ends).half())
    assert torch.equal(w.grad, ref.wgrad(rows(x.detach()), rows(g), ends).half())
    # the product is linear in each argument: a difference quotient is exact, whatever the step
    dx, dw = form(ref.integers((T, K), torch.float16, 4)), ref.integers((3, N, K), torch.float16, 5)
    with torch.no_grad():
        along_x = grouped_linear(x + dx, w, e).double() - y.double()
        along_w = grouped_linear(x, w + dw, e).double() - y.double()
    assert (along_x * g.double()).sum() == (x.grad.double() * dx.double()).sum()
    assert (along_w * g.double()).sum() == (w.grad.double() * dw.double()).sum()
    # a gradient that is one value expanded, only one of the gradients wanted, and the module
    m = ExpertLinear(3, K, N, device='cuda')
    m(x.detach(), e).sum().backward()
    assert torch.equal(m.weight.grad, ref.wgrad(rows(x.detach()), torch.ones(T, N, device='cuda'), ends).half())
    x.grad = None
    m.weight.requires_grad_(False)
    m(x, e).sum().backward()
    err = (rows(x.grad).double() - ref.dgrad(torch.ones(T, N, device='cuda'), m.weight, ends)).abs()
    assert (err <= 2.0 ** -11 * rows(x.grad).abs() + N * 2.0 ** -23 * N / 4).all()  # |w| <= 1/4


@pytest.mark.parametrize('shape', ['matrix', 'volume'])
@pytest.mark.parametrize('groups', [1, 3])
def test_gradients_of_gradients(shape, groups):
    """s = <u, dx> + <V, dw> of a backward pass, differentiated again: ds/dg = u w + x V, ds/dx = g V, ds/dw = g^T u."""
    from kerops_b200.autograd import grouped_linear

    T, K, N = 210, 16, 24
    ends = [T] if groups == 1 else [50, 50, 200]
    e = None if groups == 1 else ref.tensor_ends(ends)

    def form(t):
        return t if shape == 'matrix' else t.view(2, 3, 5, 7, -1).permute(0, 4, 1, 2, 3)

    def rows(t):
        return t if shape == 'matrix' else t.permute(0, 2, 3, 4, 1).reshape(T, -1)

    x, g, u = (form(ref.integers((T, c), torch.float16, i, top=1)).requires_grad_(True) for i, c in enumerate((K, N, K)))
    w, V = (ref.integers((groups, N, K) if groups > 1 else (N, K), torch.float16, i, top=1).requires_grad_(True) for i in (3, 4))
    dx, dw = torch.autograd.grad(grouped_linear(x, w, e), (x, w), g, create_graph=True)
    s = (dx.float() * u.float()).sum() + (dw.float() * V.float()).sum()
    gg, gx, gw = torch.autograd.grad(s, (g, x, w))
    xr, gr, ur, w3, V3 = rows(x.detach()), rows(g.detach()), rows(u.detach()), w.detach().view(groups, N, K), V.detach().view(groups, N, K)
    assert torch.equal(rows(gg), (ref.fwd(ur, w3, ends) + ref.fwd(xr, V3, ends)).half())
    assert torch.equal(rows(gx), ref.dgrad(gr, V3, ends).half())
    assert torch.equal(gw.view(groups, N, K), ref.wgrad(ur, gr, ends).half())


def test_depthwise_then_pointwise_step():
    """The products behind a depthwise convolution, as a layer uses them: y = experts(dwconv(x)) and all gradients."""
    from kerops_b200.autograd import DepthwiseConv3d, ExpertLinear
    from kerops_b200.ops.conv import DWConv, DWConvWGRAD
    from kerops_b200.autograd import DWConvDGRAD

    C, N = 16, 40
    x = ref.integers((2, 6, 8, 12, C), torch.float16, 1).permute(0, 4, 1, 2, 3).requires_grad_(True)
    conv, mix = DepthwiseConv3d(C, device='cuda'), ExpertLinear(2, C, N, device='cuda')
    conv.weight.data.copy_(ref.integers((3, 3, 3, C), torch.float16, 2, top=1))
    mix.weight.data.copy_(ref.integers((2, N, C), torch.float16, 3, top=1))
    e = ref.tensor_ends([576, 1152])
    g = ref.integers((2, 6, 8, 12, N), torch.float16, 4, top=1).permute(0, 4, 1, 2, 3)
    mix(conv(x), e).backward(g)

    def rows(t):
        return t.permute(0, 2, 3, 4, 1).reshape(1152, -1)

    h = DWConv(x.detach(), conv.weight.detach())
    gh = ref.dgrad(rows(g), mix.weight.detach(), [576, 1152]).half().view(2, 6, 8, 12, C).permute(0, 4, 1, 2, 3)
    assert torch.equal(mix.weight.grad, ref.wgrad(rows(h), rows(g), [576, 1152]).half())
    assert torch.equal(conv.weight.grad, DWConvWGRAD(x.detach(), gh))
    assert torch.equal(x.grad, DWConvDGRAD(gh, conv.weight.detach()))


def test_a_wait_that_runs_out_is_reported_and_leaves_the_context_usable():
    from kerops_b200 import _lib
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearWGRAD

    x, w = ref.integers((600, 512), torch.float16, 1), ref.integers((1, 256, 512), torch.float16, 2)
    g = ref.integers((600, 256), torch.float16, 3)
    lib = _lib.load()
    want = GroupedLinear(x, w), GroupedLinearWGRAD(x, g)
    assert _lib.device_status() == 0
    try:
        for stop in (0, 3):
            assert lib.kdw_test_wait_limits(50_000_000, stop) == 0
            GroupedLinear(x, w)
            assert _lib.device_status() == 1
            GroupedLinearWGRAD(x, g)
            assert _lib.device_status() == 1
    finally:
        lib.kdw_test_wait_limits(2_000_000_000, -1)
    assert torch.equal(GroupedLinear(x, w), want[0]) and torch.equal(GroupedLinearWGRAD(x, g), want[1])
    assert _lib.device_status() == 0


@pytest.mark.parametrize('op', ['forward', 'input gradient', '8-bit'])
def test_more_than_a_billion_channels(op):
    """An output row of more than 2^31 bytes: 54 GB with the weights (8-bit: 54 GB)."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, Int8Linear

    T, few, many, last = 17, 16 if op == '8-bit' else 8, 2 ** 30 + 136, 2 ** 20
    torch.cuda.empty_cache()
    x = ref.integers((T, few), torch.float16, 1)
    if op == 'forward':
        w = torch.zeros(many, few, dtype=torch.float16, device='cuda')
        w[-last:] = ref.integers((last, few), torch.float16, 2)
        y, want = GroupedLinear(x, w), ref.fwd(x, w[None, -last:], [T])
    elif op == 'input gradient':
        w = torch.zeros(few, many, dtype=torch.float16, device='cuda')
        w[:, -last:] = ref.integers((few, last), torch.float16, 2)
        y, want = GroupedLinearDGRAD(x, w), ref.dgrad(x, w[None, :, -last:], [T])
    else:
        w = torch.zeros(many, few, dtype=torch.int8, device='cuda')
        w[-last:] = ref.integers((last, few), torch.int8, 2)
        one = torch.ones(T, device='cuda')
        y = Int8Linear(x.to(torch.int8), w, torch.ones(many, device='cuda'), x_scale=one, dtype=torch.float16)
        want = ref.fwd(x, w[None, -last:], [T])
    assert torch.equal(y[:, -last:], want.half())
    del w
    assert all(not torch.count_nonzero(row[:-last]) for row in y)
    del y
    torch.cuda.empty_cache()


def _behind_zeros(shape, tail, dtype, seed):
    """Zeros but for the last `tail` entries of the first dimension."""
    t = torch.zeros(shape, dtype=dtype, device='cuda')
    t[-tail:] = ref.integers((tail, *shape[1:]), dtype, seed)
    return t


def test_narrow_volumes_beyond_32_bits():
    """More than 2^31 values a row operand, through the kernels of narrow weights and of both gradients in one pass."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD, _launch

    T, K, N, tail = 70_000_011, 32, 32, 3000
    x, w = _behind_zeros((T, K), tail, torch.float16, 1), ref.integers((N, K), torch.float16, 2)
    for f, form in ((GroupedLinear, ref.fwd), (GroupedLinearDGRAD, ref.dgrad)):
        y = f(x, w)
        assert torch.equal(y[-tail:], form(x[-tail:], w[None], [tail]).half()) and not torch.count_nonzero(y[:-tail])
        del y
    want = ref.wgrad(x[-tail:], x[-tail:], [tail]).half()[0]
    assert torch.equal(GroupedLinearWGRAD(x, x), want)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    _launch.grads(x, w, x, dx, dw, None, T, 1, K, N)
    assert torch.equal(dw, want) and torch.equal(dx[-tail:], ref.dgrad(x[-tail:], w[None], [tail]).half())
    assert not torch.count_nonzero(dx[:-tail])
    del x, dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize('T', [6, 40])
def test_weights_beyond_32_bits(T):
    """More than 2^31 weights, the rows in the last group: products of few rows and of tiles, and the weight gradient."""
    from kerops_b200.ops.linear import GroupedLinear, GroupedLinearDGRAD, GroupedLinearWGRAD

    E, N, K = 36, 8200, 7624
    w = _behind_zeros((E, N, K), 1, torch.bfloat16, 1)
    x, g = ref.integers((T, K), torch.bfloat16, 2), ref.integers((T, N), torch.bfloat16, 3)
    ends = [0] * (E - 1) + [T - 1]
    e = ref.tensor_ends(ends)
    last = [T - 1]
    assert torch.equal(GroupedLinear(x, w, e), ref.fwd(x, w[-1:], last).bfloat16())
    assert torch.equal(GroupedLinearDGRAD(g, w, e), ref.dgrad(g, w[-1:], last).bfloat16())
    del w
    dw = GroupedLinearWGRAD(x, g, e)
    assert torch.equal(dw[-1:], ref.wgrad(x, g, last).bfloat16()) and not any(torch.count_nonzero(d) for d in dw[:-1])
    del dw
    torch.cuda.empty_cache()
