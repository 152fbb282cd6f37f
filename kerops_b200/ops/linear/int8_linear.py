"""Channel-mixing product in 8-bit integers with a scale per row (token, voxel) and per output channel, and the row
quantiser for both operands.  No counterpart in the reference (its kerops/ops/quantization.py stores activations in 8
bits with one window for the whole tensor and multiplies nothing)."""
import torch

from . import _launch

MAX_K = 131071  # 128 * 128 * K stays inside a 32-bit sum


def QuantRows(x):
    """8-bit integers and a scale per row: scale = max|x| / 127, q = x * 127 / max|x| rounded to nearest, halves to even.

    x  [T, K] fp16 or bf16 CUDA matrix with contiguous channels (any row stride), a channels_last_3d (N, K, H, W, D)
       volume, whose voxels are the rows, or [E, N, K] contiguous weights, whose output channels are the rows
    Returns (q, scale): q int8 of x's shape (channels_last_3d for a volume), scale fp32 [T] ([E, N] for weights).  A row
    of zeros has q = 0 and scale 0; a row with a NaN or an infinity has q = 0 and scale NaN."""
    assert x.dtype in _launch.TYPES, 'fp16 or bf16 expected'
    assert x.is_cuda, 'CUDA tensor expected'
    assert x.ndim in (2, 3, 5)
    if x.ndim == 3:
        assert x.is_contiguous()
        rows = x.view(-1, x.shape[2])
    else:
        rows = _launch.as_rows(x, 'x')
    q = torch.empty(rows.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows.shape[0], dtype=torch.float32, device=x.device)
    assert rows.shape[1] >= 1, 'a row without values has no scale'
    if rows.shape[0]:
        _launch.quant_rows(rows, q, scale)
    if x.ndim == 3:
        return q.view(x.shape), scale.view(x.shape[:2])
    return _launch.like_rows(q, x), scale


def Int8Linear(x, weight, w_scale, ends=None, *, x_scale=None, dtype=None):
    """y[t, n] = (sum_k x[t, k] * weight[e, n, k]) * x_scale[t] * w_scale[e, n] for the rows t of group e, zero for rows
    of no group; the integer sums are exact.

    x        [T, K] matrix with contiguous channels, or channels_last_3d (N, K, H, W, D) volume, whose voxels are the
             rows: fp16 / bf16, quantised within the call as QuantRows does, or int8 with x_scale [T] fp32
    weight   [E, N, K] (or [N, K]) int8 contiguous and w_scale [E, N] (or [N]) fp32 contiguous: QuantRows(weights)
    ends     [E] int32 cumulative row counts, as for GroupedLinear; None: one group
    dtype    torch.float16 or torch.bfloat16, the result's; x's own by default, needed for int8 x
    Returns [T, N], or a channels_last_3d volume with N channels.  K at most 131071.  Pays with long rows; on volumes of up
    to some 128 channels GroupedLinear on 16-bit weights is faster (8 M voxels, 64 -> 64: 319 and 877 us)."""
    assert weight.ndim in (2, 3) and weight.dtype == torch.int8 and weight.is_contiguous(), \
        'weight: contiguous int8 [groups, out_channels, in_channels] or [out_channels, in_channels] expected'
    E, N, K = weight.shape if weight.ndim == 3 else (1,) + tuple(weight.shape)
    assert w_scale.dtype == torch.float32 and w_scale.shape == weight.shape[:-1] and w_scale.is_contiguous(), \
        'w_scale: contiguous fp32 scale per group and output channel expected'
    rows = _launch.as_rows(x, 'x')
    T = rows.shape[0]
    if x.dtype == torch.int8:
        assert x_scale is not None and dtype is not None, 'int8 x needs x_scale and dtype'
        assert x_scale.dtype == torch.float32 and x_scale.shape == (T,) and x_scale.is_contiguous(), \
            'x_scale: contiguous fp32 scale per row expected'
        assert x_scale.get_device() == x.get_device(), 'x_scale must be on the device of x'
    else:
        assert x.dtype in _launch.TYPES, 'x: fp16, bf16 or int8 expected'
        assert x_scale is None, 'x_scale belongs to int8 x'
        dtype = x.dtype if dtype is None else dtype
    assert dtype in _launch.TYPES, 'dtype: torch.float16 or torch.bfloat16'
    assert x.is_cuda and x.get_device() == weight.get_device() == w_scale.get_device(), 'CUDA tensors on one device expected'
    assert rows.shape[1] == K and N >= 1 and 1 <= K <= MAX_K, 'x and weight disagree about the input channels'
    assert 1 <= E <= _launch.MAX_GROUPS, f'1 to {_launch.MAX_GROUPS} groups'
    _launch.check_ends(ends, E, x)
    y = x.new_empty((T, N), dtype=dtype)
    if T:
        _launch.int8_product(rows, x_scale, weight, w_scale, y, ends, T, E, K, N)
    return _launch.like_rows(y, x)
