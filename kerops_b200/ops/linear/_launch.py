"""Argument marshalling of the channel-mixing products between torch tensors and the C-ABI (include/kdw.h)."""
import functools

import torch

from ... import _lib
from ..conv._launch import _on

# torch dtype -> KDW_F16 / KDW_BF16 (include/kdw.h)
TYPES = {torch.float16: 0, torch.bfloat16: 1}
INT8 = 2  # KDW_I8
FWD, DGRAD, WGRAD = 0, 1, 2
MAX_GROUPS = 1024

# of a device index, and the current one: torch.cuda.current_stream and torch.cuda.device cost 3 us more, beside
# some 10 us that a small call takes
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)  # (absent from builds of torch without CUDA)
_current_device = getattr(torch._C, '_cuda_getDevice', None)


def as_rows(t, name):
    """The [rows, channels] matrix of `t`: `t` itself, or the voxels of a channels_last_3d (N, C, H, W, D) volume."""
    if t.ndim == 2:
        if not t.is_contiguous():
            assert t.stride(1) == 1 or t.shape[1] == 1, f'{name}: the channels of a row must be contiguous'
            assert t.stride(0) >= t.shape[1] or t.shape[0] <= 1, f'{name}: rows must not overlap'
        return t
    assert t.ndim == 5, f'{name}: [rows, channels] matrix or (N, C, H, W, D) volume expected'
    assert t.is_contiguous(memory_format=torch.channels_last_3d), f'{name}: channels_last_3d volume expected'
    return t.permute(0, 2, 3, 4, 1).reshape(-1, t.shape[1])


def like_rows(rows, t):
    """`rows` [T, C'] in the form of `t`: the matrix itself, or a channels_last_3d volume of t's extents."""
    if t.ndim == 2:
        return rows
    n, _, h, w, d = t.shape
    return rows.view(n, h, w, d, rows.shape[1]).permute(0, 4, 1, 2, 3)


def row_stride(t):
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else cols


def check_ends(ends, groups, rows):
    if ends is None:
        assert groups == 1, 'ends is needed with more than one group'
        return
    assert ends.dtype is torch.int32 and ends.ndim == 1 and ends.is_contiguous(), 'ends: contiguous int32 vector expected'
    assert len(ends) == groups, 'ends: one cumulative row count per group expected'
    assert ends.get_device() == rows.get_device(), 'ends must be on the device of the rows'


# The workspace depends on sizes and on the operands' alignment to 16 bytes alone; asking the library costs more than the
# rest of a small call.
@functools.lru_cache(maxsize=4096)
def _product_workspace(device, op, a_align, b_align, T, E, K, N, sa, sb, dtype):
    n = _lib.load().kdw_linear_f16_workspace_bytes(op, 4096 + a_align, 4096 + b_align, T, E, K, N, sa, sb, dtype)
    if n < 0:
        _lib.check(int(n))
    return n


@functools.lru_cache(maxsize=4096)
def _grads_workspace(device, x_align, w_align, g_align, has_ends, T, E, K, N, sx, sg, dtype):
    n = _lib.load().kdw_linear_grads_f16_workspace_bytes(4096 + x_align, 4096 + w_align, 4096 + g_align, has_ends, T, E, K, N, sx, sg, dtype)
    if n < 0:
        _lib.check(int(n))
    return n


@functools.lru_cache(maxsize=4096)
def _int8_workspace(device, x_align, w_align, T, E, K, N, sx, x_type, dtype):
    n = _lib.load().kdw_linear_i8_workspace_bytes(4096 + x_align, 4096 + w_align, T, E, K, N, sx, x_type, dtype)
    if n < 0:
        _lib.check(int(n))
    return n


def product(op, a, b, out, ends, T, E, K, N):
    """Enqueues one product (FWD | DGRAD | WGRAD) of 16-bit operands on a's device / current stream."""
    device = a.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return product(op, a, b, out, ends, T, E, K, N)
    dtype = TYPES[a.dtype]
    sa, sb = row_stride(a), row_stride(b) if op == WGRAD else K
    pa, pb = a.data_ptr(), b.data_ptr()
    nbytes = _product_workspace(device.index, op, pa & 15, pb & 15, T, E, K, N, sa, sb, dtype)
    ws = a.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = _lib.load().kdw_linear_f16(
        op, pa, pb, out.data_ptr(), None if ends is None else ends.data_ptr(), ws.data_ptr() if nbytes else None, nbytes,
        T, E, K, N, sa, sb, dtype, _raw_stream(device.index),
    )
    if rc:
        _lib.check(rc)
    return out


def grads(x, weight, grad, dx, dw, ends, T, E, K, N):
    """Enqueues both gradients of a forward product on x's device / current stream."""
    device = x.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return grads(x, weight, grad, dx, dw, ends, T, E, K, N)
    dtype = TYPES[x.dtype]
    sx, sg = row_stride(x), row_stride(grad)
    px, pw, pg = x.data_ptr(), weight.data_ptr(), grad.data_ptr()
    nbytes = _grads_workspace(device.index, px & 15, pw & 15, pg & 15, ends is not None, T, E, K, N, sx, sg, dtype)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = _lib.load().kdw_linear_grads_f16(
        px, pw, pg, dx.data_ptr(), dw.data_ptr(), None if ends is None else ends.data_ptr(),
        ws.data_ptr() if nbytes else None, nbytes, T, E, K, N, sx, sg, dtype, _raw_stream(device.index),
    )
    if rc:
        _lib.check(rc)


def int8_product(x, x_scale, weight, w_scale, y, ends, T, E, K, N):
    """Enqueues y = Int8Linear(x); x is int8 with x_scale, or 16-bit (x_scale None)."""
    device = x.device
    if device.index != _current_device():
        with torch.cuda.device(device):
            return int8_product(x, x_scale, weight, w_scale, y, ends, T, E, K, N)
    x_type, dtype, sx = TYPES.get(x.dtype, INT8), TYPES[y.dtype], row_stride(x)
    px, pw = x.data_ptr(), weight.data_ptr()
    nbytes = _int8_workspace(device.index, px & 15, pw & 15, T, E, K, N, sx, x_type, dtype)
    ws = y.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = _lib.load().kdw_linear_i8(
        px, None if x_scale is None else x_scale.data_ptr(), pw, w_scale.data_ptr(), y.data_ptr(),
        None if ends is None else ends.data_ptr(), ws.data_ptr() if nbytes else None, nbytes, T, E, K, N, sx, x_type,
        dtype, _raw_stream(device.index),
    )
    if rc:
        _lib.check(rc)
    return y


def quant_rows(x, q, scale):
    """Enqueues q, scale = QuantRows(x) for a [rows, channels] matrix."""
    lib = _lib.load()
    with _on(x.device):
        rc = lib.kdw_quant_rows(x.data_ptr(), q.data_ptr(), scale.data_ptr(), x.shape[0], x.shape[1], row_stride(x),
                                TYPES[x.dtype], _raw_stream(x.device.index))
    _lib.check(rc)
