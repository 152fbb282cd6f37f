"""Channel-mixing (pointwise) products of row groups: forward, input gradient and weight gradient.  The products along
the channels that follow a depthwise convolution, with one weight matrix per group of rows (an expert each); a single
group is the plain pointwise product.  No counterpart in the reference, whose pointwise operators
(kerops/ops/linear/relu_linear_add.py:20-52) take one square weight matrix and no groups."""
import torch

from . import _launch


def _weight_dims(weight):
    assert weight.ndim in (2, 3), 'weight: [groups, out_channels, in_channels] or [out_channels, in_channels] expected'
    assert weight.is_contiguous()
    return weight.shape if weight.ndim == 3 else (1,) + tuple(weight.shape)


def _check(a, b, groups, ends):
    assert a.dtype == b.dtype and a.dtype in _launch.TYPES, 'both operands fp16 or both bf16 expected'
    assert a.is_cuda and a.get_device() == b.get_device(), 'the operands must be CUDA tensors on one device'
    assert 1 <= groups <= _launch.MAX_GROUPS, f'1 to {_launch.MAX_GROUPS} groups'
    _launch.check_ends(ends, groups, a)


def GroupedLinear(x, weight, ends=None):
    """y[t, :] = weight[e] @ x[t, :] for the rows t of group e; zero for rows of no group.

    x       [T, K] fp16 or bf16 CUDA matrix with contiguous channels (any row stride), or a channels_last_3d
            (N, K, H, W, D) volume, whose voxels in memory order are the rows
    weight  [E, N, K] contiguous, of x's dtype; [N, K] for one group.  At most 1024 groups
    ends    [E] int32 CUDA vector of cumulative row counts: group e is the rows ends[e-1] .. ends[e]-1.  It is read on
            the device; ends that step back or pass T are clamped.  None: one group of all rows
    Returns [T, N] (or a channels_last_3d volume with N channels).  Products are exact and summed in fp32, rounded once.
    """
    E, N, K = _weight_dims(weight)
    rows = _launch.as_rows(x, 'x')
    _check(rows, weight, E, ends)
    T = rows.shape[0]
    assert rows.shape[1] == K and N >= 1 and K >= 1, 'x and weight disagree about the input channels'
    y = x.new_empty((T, N))
    if T:
        _launch.product(_launch.FWD, rows, weight, y, ends, T, E, K, N)
    return _launch.like_rows(y, x)


def GroupedLinearDGRAD(grad, weight, ends=None):
    """Input gradient of GroupedLinear: dx[t, :] = grad[t, :] @ weight[e]; zero for rows of no group.

    grad    [T, N] matrix or channels_last_3d volume with N channels, like x of GroupedLinear
    Returns [T, K] (or a volume with K channels)."""
    E, N, K = _weight_dims(weight)
    rows = _launch.as_rows(grad, 'grad')
    _check(rows, weight, E, ends)
    T = rows.shape[0]
    assert rows.shape[1] == N and N >= 1 and K >= 1, 'grad and weight disagree about the output channels'
    dx = grad.new_empty((T, K))
    if T:
        _launch.product(_launch.DGRAD, rows, weight, dx, ends, T, E, K, N)
    return _launch.like_rows(dx, grad)


def GroupedLinearWGRAD(x, grad, ends=None):
    """Weight gradient of GroupedLinear: dw[e] = sum over the rows t of group e of grad[t, :]^T x[t, :].

    x, grad  [T, K] and [T, N] matrices (or volumes) as for GroupedLinear
    Returns [E, N, K] in their dtype ([N, K] without ends); zero for a group without rows.  Sums are fp32 and added in a
    fixed order, so that a call on the same data returns the same bits."""
    xr, gr = _launch.as_rows(x, 'x'), _launch.as_rows(grad, 'grad')
    E = 1 if ends is None else ends.shape[0]
    _check(gr, xr, E, ends)
    T, K = xr.shape
    N = gr.shape[1]
    assert gr.shape[0] == T and N >= 1 and K >= 1, 'x and grad disagree about the rows'
    if x.ndim == 5 or grad.ndim == 5:
        assert x.ndim == grad.ndim and x.shape[2:] == grad.shape[2:] and x.shape[0] == grad.shape[0], \
            'x and grad disagree about the volume'
    dw = x.new_empty((N, K) if ends is None else (E, N, K))
    if T:
        _launch.product(_launch.WGRAD, gr, xr, dw, ends, T, E, K, N)
    else:
        dw.zero_()
    return dw


def grouped_linear_grads(x, weight, grad, ends, need_x, need_w):
    """(dx, dw) of a GroupedLinear(x, weight, ends) that has been checked when it ran, None for one that is not needed; grad is
    a contiguous gradient of its result, dw has weight's shape."""
    E, N, K = weight.shape if weight.ndim == 3 else (1, *weight.shape)
    xr, gr = _launch.as_rows(x, 'x'), _launch.as_rows(grad, 'grad')
    T = xr.shape[0]
    dx = gr.new_empty((T, K)) if need_x else None
    dw = torch.empty_like(weight) if need_w else None
    if T == 0:
        if need_w:
            dw.zero_()
    elif need_x and need_w:
        _launch.grads(xr, weight, gr, dx, dw, ends, T, E, K, N)
    elif need_x:
        _launch.product(_launch.DGRAD, gr, weight, dx, ends, T, E, K, N)
    elif need_w:
        _launch.product(_launch.WGRAD, gr, xr, dw, ends, T, E, K, N)
    return _launch.like_rows(dx, x) if need_x else None, dw
