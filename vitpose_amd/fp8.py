"""Linears on 8-bit floating-point operands: e4m3 numbers with one f32 scale per block of 128 (vit.py:66-74,93,96 in
evaluation).

    wq, ws = quantize_weight(weight)                       # once: [N, K] -> e4m3 [N, Kp], scales of its 128 x 128 squares
    y = linear(x, wq, ws, bias, act='gelu')                # x f32 or bf16 [M, K] -> bf16 [M, N]

or, where several products read the same rows,

    xq, xs = quantize_rows(x)                              # e4m3 [M, Kp], scales [Kp / 128, M]
    y = product(xq, xs, wq, ws, bias)

`layernorm_rows` gives the rows behind a LayerNorm in that form, and a product with out_dtype = torch.float8_e4m3fn its
result: what lies between two products then never exists in 16 bits.

Kp is K rounded up to 128.  Sums are f32 but for the matrix instruction's eights: it adds eight products at a time, each of which may
lose 2^-13 of the largest of the eight (5e-5 of a result's norm, against 3e-2 for the rounding of the operands).  Nothing here synchronises or records gradients (rows that require one are refused outside no_grad).
"""
import ctypes

import torch

from . import _lib
from ._lib import VP_BF16, VP_E4M3, VP_F32, Fp8Args

BLOCK = 128
_F8, _BF16, _F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32
_NOT_PLAIN = (AttributeError, TypeError, ValueError, RuntimeError)
_ACTS = {None: 0, 'gelu': 1}
_INSTEAD = 'detach it, or call under torch.no_grad()'


def _on_device(t, what, dev=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{what}: expected a tensor, got {type(t).__name__}')
    if t.device.type != 'cuda':
        raise RuntimeError(f'{what} is on {t.device}: the 8-bit products run on a HIP device only')
    if dev is not None and t.device != dev:
        raise ValueError(f'{what}: on {t.device}, other operands on {dev}')


def _real_matrix(t, what, dev=None):
    """(dtype tag, leading dimension) of an f32 or bf16 [rows][K] matrix that the quantizers read."""
    _on_device(t, what, dev)
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f'{what}: expected float32 or bfloat16, got {t.dtype}')
    if t.dim() != 2 or t.shape[1] < 8 or t.shape[1] % 8:
        raise ValueError(f'{what}: shape {tuple(t.shape)}, expected [rows, K] with K a multiple of 8')
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if t.numel() and (t.stride(1) != 1 or ld < t.shape[1] or ld % 8 or t.data_ptr() % 16):
        raise ValueError(f'{what}: rows must be contiguous, a multiple of 8 elements apart and on 16-byte boundaries')
    return (VP_F32 if t.dtype == torch.float32 else VP_BF16), ld


def _codes(t, what, dev):
    """Leading dimension of an e4m3 [rows][Kp] matrix."""
    _on_device(t, what, dev)
    if t.dtype != _F8:
        raise TypeError(f'{what}: expected {_F8}, got {t.dtype}')
    if t.dim() != 2 or t.shape[1] < BLOCK or t.shape[1] % BLOCK:
        raise ValueError(f'{what}: shape {tuple(t.shape)}, expected [rows, Kp] with Kp a multiple of {BLOCK}')
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if t.numel() and (t.stride(1) != 1 or ld < t.shape[1] or ld % 16 or t.data_ptr() % 16):
        raise ValueError(f'{what}: rows must be contiguous, a multiple of 16 elements apart and on 16-byte boundaries')
    return ld


def _vector(t, what, shape, dev):
    _on_device(t, what, dev)
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f'{what}: expected contiguous float32 {list(shape)}, got {t.dtype} {list(t.shape)}')


def _rows(x):
    """(device number, pointer, dtype tag, leading dimension) of the rows that a call rounds."""
    try:
        d, p = x.get_device(), x.data_ptr()
        _, K = x.shape
        if (d >= 0 and (x.dtype is _BF16 or x.dtype is _F32) and K >= 8 and not (K & 7 or p & 15) and x.is_contiguous() and
                not x.requires_grad):
            return d, p, VP_BF16 if x.dtype is _BF16 else VP_F32, K
    except _NOT_PLAIN:
        pass
    tag, ld = _real_matrix(x, 'x')
    _lib.records_none(x, 'x', _INSTEAD)
    return x.get_device(), x.data_ptr(), tag, ld


def quantize_rows(x):
    """x f32 or bf16 [M, K] -> (e4m3 [M, Kp], f32 scales [Kp / 128, M])."""
    d, p, tag, ld = _rows(x)
    M, K = x.shape
    if (M | K) >> 31:
        _lib.too_large(M, K)
    kb = (K + 127) // BLOCK
    q = x.new_empty((M, kb * BLOCK), dtype=_F8)
    scale = x.new_empty((kb, M), dtype=_F32)
    if M:
        _lib.launch(d, _lib.lib().vp_quantize_fp8_rows, p, tag, ld, M, K, q.data_ptr(), scale.data_ptr())
    return q, scale


def quantize_weight(w):
    """w f32 or bf16 [N, K] -> (e4m3 [N, Kp], f32 scales [ceil(N / 128), Kp / 128])."""
    tag, ld = _real_matrix(w, 'w')
    N, K = w.shape
    if N < 1:
        raise ValueError('w: no rows')
    if (N | K) >> 31:
        _lib.too_large(N, K)
    kb = (K + BLOCK - 1) // BLOCK
    q = torch.empty(N, kb * BLOCK, dtype=_F8, device=w.device)
    scale = torch.empty((N + BLOCK - 1) // BLOCK, kb, dtype=torch.float32, device=w.device)
    _lib.launch(w.get_device(), 'vp_quantize_fp8_weight', w.data_ptr(), tag, ld, N, K, q.data_ptr(), scale.data_ptr())
    return q, scale


def layernorm_rows(x, weight, bias, eps=1e-6):
    """quantize_rows of the LayerNorm of x f32 [M, E] over its rows (E a multiple of 8, at most 2048)."""
    tag, ld = _real_matrix(x, 'x')
    _lib.records_none(x, 'x', _INSTEAD)
    M, E = x.shape
    if tag != VP_F32:
        raise TypeError('x: expected float32 (the residual stream)')
    if ld != E or E > 2048:
        raise ValueError(f'x: shape {tuple(x.shape)}, strides {x.stride()}: contiguous rows of at most 2048 values')
    for t, what in ((weight, 'weight'), (bias, 'bias')):
        _vector(t, what, (E,), x.device)
        if t.data_ptr() % 16:
            raise ValueError(f'{what}: must start on a 16-byte boundary')
    if M >> 31:
        _lib.too_large(M, E)
    kb = (E + BLOCK - 1) // BLOCK
    q = x.new_empty((M, kb * BLOCK), dtype=_F8)
    scale = x.new_empty((kb, M))
    if M:
        _lib.launch(x.get_device(), 'vp_layernorm_fp8', x.data_ptr(), weight.data_ptr(), bias.data_ptr(), eps, M, E, q.data_ptr(), scale.data_ptr())
    return q, scale


def _result(M, N, out, out_dtype, like):
    """(result, its leading dimension, dtype tag)."""
    if out is None:
        if out_dtype is not _BF16 and out_dtype is not _F32:
            raise TypeError(f'out_dtype: bfloat16 or float32, got {out_dtype}')
        return like.new_empty((M, N), dtype=out_dtype), N, VP_BF16 if out_dtype is _BF16 else VP_F32
    _on_device(out, 'out', like.device)
    if out.dtype not in (_BF16, _F32):
        raise TypeError(f'out: expected bfloat16 or float32, got {out.dtype}')
    if tuple(out.shape) != (M, N):
        raise ValueError(f'out: shape {tuple(out.shape)}, expected ({M}, {N})')
    ldo = out.stride(0) if M > 1 else N
    if out.numel() and ((out.stride(1) != 1 and N > 1) or ldo < N or out.data_ptr() % 16):
        raise ValueError('out: rows must be contiguous and start on a 16-byte boundary')
    _lib.records_none(out, 'out', _INSTEAD)
    return out, ldo, VP_F32 if out.dtype is _F32 else VP_BF16


def _apart(out, resid, *operands):
    """Refuses a given result that a workgroup could write while another still reads an operand there (the residual is read by the lane
    that writes, so it may be the result itself)."""
    for name, t in operands:
        if t is not None and _lib.shares_memory(out, t):
            raise ValueError(f'out shares memory with {name}, which is read while it is written')
    if resid is not None and _lib.shares_memory(out, resid) and (
            resid.data_ptr() != out.data_ptr() or (resid.stride(0) != out.stride(0) and out.shape[0] > 1)):
        raise ValueError('out shares memory with resid, but is not the same matrix')


def _weights(wq, ws, bias, act, d, dev):
    """(leading dimension of wq, N, Kp, pointer of bias); d and dev name the rows' device."""
    try:
        N, Kp = wq.shape
        plain = (wq.dtype is _F8 and Kp >= BLOCK and not (Kp & 127 or wq.data_ptr() & 15) and wq.is_contiguous() and
                 wq.get_device() == d and ws.dtype is _F32 and ws.shape == ((N + 127) // BLOCK, Kp // BLOCK) and
                 ws.is_contiguous() and ws.get_device() == d and
                 (bias is None or (bias.dtype is _F32 and bias.shape == (N,) and bias.is_contiguous() and bias.get_device() == d)))
    except _NOT_PLAIN:
        plain = False
    ldw = Kp if plain else _codes(wq, 'wq', dev)
    if not plain:
        N, Kp = wq.shape
        _vector(ws, 'ws', ((N + BLOCK - 1) // BLOCK, Kp // BLOCK), dev)
        if bias is not None:
            _vector(bias, 'bias', (N,), dev)
    if act not in _ACTS:
        raise ValueError(f'act {act!r}: one of {list(_ACTS)}')
    return ldw, N, Kp, bias.data_ptr() if bias is not None else None


def _residual(resid, M, N, tag, dev):
    """(pointer, leading dimension) of the f32 [M, N] matrix that is added to an f32 result."""
    _on_device(resid, 'resid', dev)
    _lib.records_none(resid, 'resid', _INSTEAD)
    if tag != VP_F32:
        raise TypeError('resid: the result has to be float32 too')
    if resid.dtype is not _F32 or tuple(resid.shape) != (M, N):
        raise ValueError(f'resid: expected float32 {[M, N]}, got {resid.dtype} {list(resid.shape)}')
    ldr = resid.stride(0) if M > 1 else N
    if resid.numel() and ((resid.stride(1) != 1 and N > 1) or ldr < N or resid.data_ptr() % 16):
        raise ValueError('resid: rows must be contiguous and start on a 16-byte boundary')
    return resid.data_ptr(), ldr


def product(xq, xs, wq, ws, bias=None, act=None, out_dtype=torch.bfloat16, out=None, resid=None):
    """act(xq wq^T with the blocks' scales + bias) (+ resid), bf16 or f32 [M, N]; operands as the quantizers return them.
    resid (f32 results only) may be `out` itself; nothing else may lie in its memory.  out_dtype = torch.float8_e4m3fn: (codes, scales) of the result, as
    quantize_rows would return them, but from the sums before they are rounded to 16 bits (no out, no resid)."""
    try:
        d, p = xq.get_device(), xq.data_ptr()
        M, Kx = xq.shape
        plain = (d >= 0 and xq.dtype is _F8 and Kx >= BLOCK and not (Kx & 127 or p & 15) and xq.is_contiguous() and
                 xs.dtype is _F32 and xs.shape == (Kx // BLOCK, M) and xs.is_contiguous() and xs.get_device() == d)
    except _NOT_PLAIN:
        plain = False
    if not plain:
        _on_device(xq, 'xq')
        ldx = _codes(xq, 'xq', xq.device)
        M, Kx = xq.shape
        _vector(xs, 'xs', (Kx // BLOCK, M), xq.device)
        d, p = xq.get_device(), xq.data_ptr()
    else:
        ldx = Kx
    ldw, N, Kp, pb = _weights(wq, ws, bias, act, d, xq.device)
    if Kx != Kp:
        raise ValueError(f'xq {tuple(xq.shape)} against wq {tuple(wq.shape)}: Kp differs')
    if (M | N | Kp) >> 31:
        _lib.too_large(M, N, Kp)
    if out_dtype is _F8:
        if out is not None or resid is not None:
            raise ValueError('out_dtype float8_e4m3fn takes neither out nor resid')
        nb = (N + 127) // BLOCK
        q, s = xs.new_empty((M, nb * BLOCK), dtype=_F8), xs.new_empty((nb, M))
        if M:
            args = Fp8Args(M, N, Kp, p, ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), pb, _ACTS[act], q.data_ptr(), nb * BLOCK,
                           VP_E4M3, None, 0, s.data_ptr())
            _lib.launch(d, _lib.lib().vp_gemm_fp8, ctypes.byref(args))
        return q, s
    given = out is not None
    out, ldo, tag = _result(M, N, out, out_dtype, xs)
    pr, ldr = _residual(resid, M, N, tag, xq.device) if resid is not None else (None, 0)
    if given:
        _apart(out, resid, ('xq', xq), ('xs', xs), ('wq', wq), ('ws', ws), ('bias', bias))
    if M and N:
        args = Fp8Args(M, N, Kp, p, ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), pb, _ACTS[act], out.data_ptr(), ldo, tag,
                       pr, ldr)
        _lib.launch(d, _lib.lib().vp_gemm_fp8, ctypes.byref(args))
    return out


def linear(x, wq, ws, bias=None, act=None, out_dtype=torch.bfloat16, out=None, resid=None):
    """act(x w^T + bias) (+ resid) with x rounded to e4m3 on the way: `quantize_rows` and `product` in one call (one launch where the
    rows are few; the blocks of K may then be added up in another order)."""
    if out_dtype is _F8:
        return product(*quantize_rows(x), wq, ws, bias, act, out_dtype, out, resid)
    d, p, tag, ldx = _rows(x)
    M, K = x.shape
    ldw, N, Kp, pb = _weights(wq, ws, bias, act, d, x.device)
    if (K + 127) // BLOCK * BLOCK != Kp:
        raise ValueError(f'x {tuple(x.shape)} against wq {tuple(wq.shape)}')
    if (M | N | Kp) >> 31:
        _lib.too_large(M, N, Kp)
    given = out is not None
    out, ldo, otag = _result(M, N, out, out_dtype, x)
    pr, ldr = _residual(resid, M, N, otag, x.device) if resid is not None else (None, 0)
    if given:
        _apart(out, resid, ('x', x), ('wq', wq), ('ws', ws), ('bias', bias))
    if M and N:
        L = _lib.lib()
        q = s = None
        if not L.vp_linear_fp8_fused(M, N, K, tag):
            scratch = x.new_empty(M * (Kp + Kp // BLOCK * 4), dtype=torch.uint8)       # codes, then scales
            q = scratch.data_ptr()
            s = q + M * Kp
        args = Fp8Args(M, N, Kp, None, 0, None, wq.data_ptr(), ldw, ws.data_ptr(), pb, _ACTS[act], out.data_ptr(), ldo, otag, pr, ldr)
        _lib.launch(d, L.vp_linear_fp8, ctypes.byref(args), p, tag, ldx, K, q, s)
    return out
