"""Products in 8 bits: e4m3 values with one scale per block of 128.

The sdfnet's layers multiply bf16 matrices; these operators do the same
contractions on e4m3 operands (four significant bits), at half the bytes and
twice the tensor cores' rate, less the passes that quantize and the scaled sums
between the blocks.  Against a bf16 ``F.linear`` on one B200 (replayed in a
graph, us; rows x outputs x columns) that pays at some sizes only:

    training step     65536 x 256 x 256    91 of 140   16384 x 8192 x 8192  4080 of 4730
                      65536 x 512 x 512   172 of 177   8192 x 4096 x 2048    337 of 317
                      1048576 x 256 x 256 973 of 799   65536 x 1024 x 1024   460 of 366
    forward alone     16384 x 8192 x 8192 1213 of 1512 (1123 with the weight quantized once)
                      8192 x 4096 x 2048   104 of 96   (89)
                      65536 x 256 x 256     28 of 13   (26)

Operands that are in 8 bits already (a checkpoint's weight and scales) need
``block_matmul`` in any case.

``quantize_blocks`` turns a matrix into e4m3 values and power-of-two scales,
``dequantize_blocks`` turns them back, ``block_matmul`` multiplies two such
matrices (with any fp32 scales, as a checkpoint may bring them), and
``block_linear`` is a layer for training: its forward and both of its
gradients are 8-bit products of operands quantized on the way.
"""
from __future__ import annotations

import math
import threading

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.SDFOAM_F32, torch.float16: _lib.SDFOAM_F16, torch.bfloat16: _lib.SDFOAM_BF16}
_E4M3 = torch.float8_e4m3fn
_BLOCK = 128


def _blocks(n: int) -> int:
    return (n + _BLOCK - 1) // _BLOCK


def _cuda(what: str, x: torch.Tensor, device=None):
    if x.device.type != "cuda":
        raise RuntimeError(f"{what} must be on CUDA device")
    if device is not None and x.device != device:
        raise RuntimeError(f"{what} must be on the device of the other arguments")


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x itself when its rows are contiguous (any distance apart), else a copy.
    A view that negates as it is read (the imaginary part of a conjugate) is
    written out: the kernels read memory."""
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.contiguous()


# One word per device in pinned host memory, which a kernel that gives up
# waiting writes and the host reads without a copy: (tensor, its numpy view,
# its address).  Made once, under the lock: kernels hold the address.
_flags: dict = {}
_flags_lock = threading.Lock()


def _flag(device: torch.device) -> int:
    f = _flags.get(device.index)
    if f is None:
        with _flags_lock:
            f = _flags.get(device.index)
            if f is None:
                t = torch.zeros(1, dtype=torch.int32, pin_memory=True)
                f = _flags[device.index] = (t, t.numpy(), t.data_ptr())
    if f[1][0]:
        _raise(f)
    return f[2]


def _raise(f):
    f[1][0] = 0
    raise RuntimeError("an 8-bit product gave up waiting on the tensor-core pipeline and wrote NaN")


def check_block_flags():
    """Waits for the devices that have run 8-bit products and raises
    RuntimeError if one of them gave up waiting on the tensor-core pipeline
    (the next product on the device raises it too)."""
    for index, f in list(_flags.items()):
        torch.cuda.synchronize(index)
        if f[1][0]:
            _raise(f)


def _values(rows: int, columns: int, device) -> torch.Tensor:
    """An e4m3 matrix whose rows start on 16 bytes."""
    ld = (columns + 15) // 16 * 16
    v = torch.empty((rows, ld), dtype=_E4M3, device=device)
    return v if ld == columns else v[:, :columns]


def _quantize(x, block_rows, turned):
    """(values, scales) of x, or of x turned."""
    x = _matrix(x)
    m, k = x.shape
    dev = x.device
    rows, columns = (k, m) if turned else (m, k)
    v = _values(rows, columns, dev)
    s = torch.empty((_blocks(columns), rows if block_rows == 1 else _blocks(rows)), dtype=torch.float32, device=dev)
    at = (v.data_ptr(), max(v.stride(0), columns), s.data_ptr())
    lib = _lib.load()
    with _lib.on(dev):
        _lib.check(lib.sdfoam_block_quantize(x.data_ptr(), max(x.stride(0), k), _DTYPES[x.dtype], m, k, block_rows,
                                             *((None, 0, None, *at) if turned else (*at, None, 0, None)), None, 0,
                                             None, _lib.stream(dev)))
    return v, s.t()


def quantize_blocks(x: torch.Tensor, block_rows: int = 1, transpose: bool = False):
    """(values, scales) of a matrix in blocks of ``block_rows`` x 128 (1:
    activations, 128: weights), of ``x.t()`` with ``transpose``.

    values: float8_e4m3fn, rows 16 bytes aligned; scales: float32
    [ceil(rows / block_rows), ceil(columns / 128)] with the rows' scales of one
    block of columns next to each other in memory, per block the smallest
    power of two s >= 2^-126 with ``448 s`` at least the block's largest
    magnitude (1 for a block of zeros).  values = x / s to the nearest, ties to
    even.  Infinities and NaN become NaN and do not count in the block's
    largest magnitude.  Not differentiable; see :func:`block_linear`."""
    if x.dim() != 2:
        raise RuntimeError("x must have 2 dimensions")
    if x.dtype not in _DTYPES:
        raise RuntimeError("x must have float32, float16 or bfloat16 dtype")
    if block_rows not in (1, _BLOCK):
        raise RuntimeError("block_rows must be 1 or 128")
    _cuda("x", x)
    return _quantize(x, block_rows, bool(transpose))


def _block_rows(what: str, values: torch.Tensor, scales: torch.Tensor) -> int:
    if values.dim() != 2 or scales.dim() != 2:
        raise RuntimeError(f"{what} and its scales must have 2 dimensions")
    if values.dtype != _E4M3:
        raise RuntimeError(f"{what} must have float8_e4m3fn dtype")
    if scales.dtype != torch.float32:
        raise RuntimeError(f"the scales of {what} must have float32 dtype")
    m, k = values.shape
    rows, columns = scales.shape
    if columns == _blocks(k):
        if rows == m:
            return 1
        if rows == _blocks(m):
            return _BLOCK
    raise RuntimeError(f"the scales of {what} must have shape [{m} or {_blocks(m)}, {_blocks(k)}]")


def dequantize_blocks(values: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """values * scales as a contiguous matrix of ``dtype``; the blocks follow
    from the shape of the scales.  Not differentiable."""
    block_rows = _block_rows("values", values, scales)
    if dtype not in _DTYPES:
        raise RuntimeError("dtype must be float32, float16 or bfloat16")
    _cuda("values", values)
    _cuda("scales", scales, values.device)
    v, s = _matrix(values), scales
    m, k = v.shape
    out = torch.empty((m, k), dtype=dtype, device=v.device)
    lib = _lib.load()
    with _lib.on(v.device):
        _lib.check(lib.sdfoam_block_dequantize(v.data_ptr(), max(v.stride(0), k), s.data_ptr(), s.stride(0), s.stride(1),
                                               block_rows, m, k, _DTYPES[dtype], out.data_ptr(),
                                               _lib.stream(v.device)))
    return out


def _operand(v: torch.Tensor):
    """(v, bytes between its rows): rows 16 bytes aligned, as the copies into
    shared memory need them."""
    rows, step = v.stride()
    k = v.shape[1]
    if step == 1 and rows >= k and rows % 16 == 0 and v.data_ptr() % 16 == 0:
        return v, rows
    out = _values(v.shape[0], k, v.device)
    out.copy_(v)
    return out, max(out.stride(0), k)


def _check_bias(bias, n, device):
    if bias.dtype not in _DTYPES or bias.dim() != 1 or bias.shape[0] != n:
        raise RuntimeError(f"bias must be a float32, float16 or bfloat16 vector of {n}")
    _cuda("bias", bias, device)


def block_matmul(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor,
                 bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(a * a_scales) @ (b * b_scales).t() + bias`` of e4m3 matrices a [M, K]
    and b [N, K] with a scale per 1 x 128 or 128 x 128 block (any fp32 values;
    the shape of the scales says which; the product of two may leave fp32 where
    the sum times both does not).  fp32 sums in a fixed order, rounded once to ``out_dtype`` (float32, float16 or bfloat16).  Not differentiable;
    see :func:`block_linear`."""
    a_rows = _block_rows("a", a, a_scales)
    b_rows = _block_rows("b", b, b_scales)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise RuntimeError(f"a and b must have the same number of columns, got {k} and {b.shape[1]}")
    if out_dtype not in _DTYPES:
        raise RuntimeError("out_dtype must be float32, float16 or bfloat16")
    dev = a.device
    if dev.type != "cuda" or a_scales.device != dev or b.device != dev or b_scales.device != dev:
        _cuda("a", a)
        for what, t in (("a_scales", a_scales), ("b", b), ("b_scales", b_scales)):
            _cuda(what, t, dev)
    if bias is not None:
        _check_bias(bias, n, dev)
        bias = bias.resolve_neg().contiguous()
    lib = _lib.load()
    nbytes = lib.sdfoam_block_matmul_workspace_bytes(m, n, k)
    with _lib.on(dev):
        a, lda = _operand(a)
        b, ldb = _operand(b)
        out = torch.empty((m, n), dtype=out_dtype, device=dev)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None
        _lib.check(lib.sdfoam_block_matmul(
            a.data_ptr(), lda, a_scales.data_ptr(), *a_scales.stride(), a_rows, m,
            b.data_ptr(), ldb, b_scales.data_ptr(), *b_scales.stride(), b_rows, n, k,
            None if bias is None else bias.data_ptr(), 0 if bias is None else _DTYPES[bias.dtype],
            out.data_ptr(), max(n, 1), _DTYPES[out_dtype], None if ws is None else ws.data_ptr(), nbytes, _flag(dev),
            _lib.stream(dev)))
    return out


class _BlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_mode):
        # x is kept (turned, in 8 bits) for the weight's gradient and the
        # weight for x's (needs_input_grad does not know the grad mode, which
        # is off in here)
        keep_w, keep_x = (grad_mode and need for need in ctx.needs_input_grad[:2])
        x, weight = _matrix(x), _matrix(weight)
        m, k = x.shape
        n = weight.shape[0]
        dev = x.device
        lib = _lib.load()
        y = torch.empty((m, n), dtype=x.dtype, device=dev)
        saved_bytes = lib.sdfoam_block_linear_saved_bytes(m, n, k, keep_x, keep_w)
        saved = torch.empty((saved_bytes,), dtype=torch.uint8, device=dev)
        nbytes = lib.sdfoam_block_linear_workspace_bytes(m, n, k)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        if bias is not None:
            bias = bias.resolve_neg().contiguous()
        with _lib.on(dev):
            _lib.check(lib.sdfoam_block_linear_forward(
                x.data_ptr(), max(x.stride(0), k), _DTYPES[x.dtype], m, weight.data_ptr(), max(weight.stride(0), k),
                _DTYPES[weight.dtype], n, k, None if bias is None else bias.data_ptr(),
                0 if bias is None else _DTYPES[bias.dtype], y.data_ptr(), saved.data_ptr(), saved_bytes, keep_x, keep_w,
                ws.data_ptr(), nbytes, _flag(dev), _lib.stream(dev)))
        ctx.save_for_backward(saved)
        ctx.kept = keep_x, keep_w
        ctx.sizes = m, n, k
        ctx.dtypes = x.dtype, weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (saved,) = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        m, n, k = ctx.sizes
        grad = _matrix(grad)
        dev = grad.device
        lib = _lib.load()
        dx = torch.empty((m, k), dtype=ctx.dtypes[0], device=dev) if need_x else None
        dw = torch.empty((n, k), dtype=ctx.dtypes[1], device=dev) if need_w else None
        db = torch.empty((n,), dtype=ctx.dtypes[2], device=dev) if need_b else None
        nbytes = lib.sdfoam_block_linear_workspace_bytes(m, n, k)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        with _lib.on(dev):
            _lib.check(lib.sdfoam_block_linear_backward(
                grad.data_ptr(), max(grad.stride(0), n), _DTYPES[grad.dtype], m, n, k, saved.data_ptr(),
                saved.numel(), *ctx.kept, None if dx is None else dx.data_ptr(), _DTYPES[ctx.dtypes[0]],
                None if dw is None else dw.data_ptr(), _DTYPES[ctx.dtypes[1]], None if db is None else db.data_ptr(),
                0 if db is None else _DTYPES[db.dtype], ws.data_ptr(), nbytes, _flag(dev), _lib.stream(dev)))
        return dx, dw, db, None


def block_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.t() + bias`` with 8-bit products: x [..., K], weight [N, K]
    (float32, float16 or bfloat16), output of x's type.

    With Q the values that :func:`quantize_blocks` keeps, in blocks of 1 x 128
    of x and 128 x 128 of the weight:

        y = Q(x) Q(weight)^T + bias
        dx = Q(dy) Q(weight),  dweight = Q(dy^T) Q(x^T)^T,  dbias = sum dy

    the blocks of dy along the reduction of each product (its columns for dx,
    its rows for dweight).  For a weight that stays as it is, quantize it once
    and call :func:`block_matmul`."""
    if weight.dim() != 2 or x.dim() < 1:
        raise RuntimeError("weight must have 2 dimensions and x at least 1")
    if x.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"x must have {weight.shape[1]} columns, got {x.shape[-1]}")
    for what, t in (("x", x), ("weight", weight)):
        if t.dtype not in _DTYPES:
            raise RuntimeError(f"{what} must have float32, float16 or bfloat16 dtype")
    _cuda("x", x)
    _cuda("weight", weight, x.device)
    if bias is not None:
        _check_bias(bias, weight.shape[0], x.device)
    if x.dim() == 2:
        return _BlockLinear.apply(x, weight, bias, torch.is_grad_enabled())
    y = _BlockLinear.apply(x.reshape(math.prod(x.shape[:-1]), x.shape[-1]), weight, bias, torch.is_grad_enabled())
    return y.reshape(*x.shape[:-1], weight.shape[0])
