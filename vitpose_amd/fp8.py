"""Linears on 8-bit floating-point operands: e4m3 numbers with one f32 scale per block of 128 (vit.py:66-74,93,96 in
evaluation).

    wq, ws = quantize_weight(weight)                       # once: [N, K] -> e4m3 [N, Kp], scales of its 128 x 128 squares
    y = linear(x, wq, ws, bias, act='gelu')                # x f32 or bf16 [M, K] -> bf16 [M, N]

or, where several products read the same rows,

    xq, xs = quantize_rows(x)                              # e4m3 [M, Kp], scales [Kp / 128, M]
    y = product(xq, xs, wq, ws, bias)

Kp is K rounded up to 128.  Nothing here synchronises.
"""
import ctypes

import torch

from . import _lib
from ._lib import VP_BF16, VP_F32, Fp8Args

BLOCK = 128
_F8 = torch.float8_e4m3fn
_ACTS = {None: 0, 'gelu': 1}


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


def quantize_rows(x):
    """x f32 or bf16 [M, K] -> (e4m3 [M, Kp], f32 scales [Kp / 128, M])."""
    tag, ld = _real_matrix(x, 'x')
    M, K = x.shape
    kb = (K + BLOCK - 1) // BLOCK
    q = torch.empty(M, kb * BLOCK, dtype=_F8, device=x.device)
    scale = torch.empty(kb, M, dtype=torch.float32, device=x.device)
    if M:
        _lib.launch(x.device, 'vp_quantize_fp8_rows', x.data_ptr(), tag, ld, M, K, q.data_ptr(), scale.data_ptr())
    return q, scale


def quantize_weight(w):
    """w f32 or bf16 [N, K] -> (e4m3 [N, Kp], f32 scales [ceil(N / 128), Kp / 128])."""
    tag, ld = _real_matrix(w, 'w')
    N, K = w.shape
    if N < 1:
        raise ValueError('w: no rows')
    kb = (K + BLOCK - 1) // BLOCK
    q = torch.empty(N, kb * BLOCK, dtype=_F8, device=w.device)
    scale = torch.empty((N + BLOCK - 1) // BLOCK, kb, dtype=torch.float32, device=w.device)
    _lib.launch(w.device, 'vp_quantize_fp8_weight', w.data_ptr(), tag, ld, N, K, q.data_ptr(), scale.data_ptr())
    return q, scale


def _result(M, N, out, out_dtype, dev):
    if out is None:
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f'out_dtype: bfloat16 or float32, got {out_dtype}')
        out = torch.empty(M, N, dtype=out_dtype, device=dev)
        return out, N
    _on_device(out, 'out', dev)
    if out.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f'out: expected bfloat16 or float32, got {out.dtype}')
    if tuple(out.shape) != (M, N):
        raise ValueError(f'out: shape {tuple(out.shape)}, expected ({M}, {N})')
    ldo = out.stride(0) if M > 1 else N
    if out.numel() and ((out.stride(1) != 1 and N > 1) or ldo < N or out.data_ptr() % 16):
        raise ValueError('out: rows must be contiguous and start on a 16-byte boundary')
    return out, ldo


def _operand_checks(wq, ws, bias, act, dev):
    ldw = _codes(wq, 'wq', dev)
    N, Kp = wq.shape
    _vector(ws, 'ws', ((N + BLOCK - 1) // BLOCK, Kp // BLOCK), dev)
    if bias is not None:
        _vector(bias, 'bias', (N,), dev)
    if act not in _ACTS:
        raise ValueError(f'act {act!r}: one of {list(_ACTS)}')
    return ldw, N, Kp


def product(xq, xs, wq, ws, bias=None, act=None, out_dtype=torch.bfloat16, out=None):
    """act(xq wq^T with the blocks' scales + bias), bf16 or f32 [M, N]; operands as the quantizers return them."""
    _on_device(xq, 'xq')
    dev = xq.device
    ldx = _codes(xq, 'xq', dev)
    ldw, N, Kp = _operand_checks(wq, ws, bias, act, dev)
    M = xq.shape[0]
    if xq.shape[1] != Kp:
        raise ValueError(f'xq {tuple(xq.shape)} against wq {tuple(wq.shape)}: Kp differs')
    _vector(xs, 'xs', (Kp // BLOCK, M), dev)
    out, ldo = _result(M, N, out, out_dtype, dev)
    if M and N:
        args = Fp8Args(M, N, Kp, xq.data_ptr(), ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(),
                       bias.data_ptr() if bias is not None else None, _ACTS[act], out.data_ptr(), ldo,
                       VP_F32 if out.dtype == torch.float32 else VP_BF16)
        _lib.launch(dev, 'vp_gemm_fp8', ctypes.byref(args))
    return out


def linear(x, wq, ws, bias=None, act=None, out_dtype=torch.bfloat16, out=None):
    """act(x w^T + bias) with x rounded to e4m3 on the way: `quantize_rows` and `product` in one call (one launch where the
    rows are few; the blocks of K may then be added up in another order)."""
    tag, ldx = _real_matrix(x, 'x')
    dev, (M, K) = x.device, x.shape
    ldw, N, Kp = _operand_checks(wq, ws, bias, act, dev)
    if (K + BLOCK - 1) // BLOCK * BLOCK != Kp:
        raise ValueError(f'x {tuple(x.shape)} against wq {tuple(wq.shape)}')
    out, ldo = _result(M, N, out, out_dtype, dev)
    if M and N:
        L = _lib.lib()
        q = s = None
        if not L.vp_linear_fp8_fused(M, N, K, tag):
            q = torch.empty(M * Kp, dtype=torch.uint8, device=dev)
            s = torch.empty(Kp // BLOCK * M, dtype=torch.float32, device=dev)
        args = Fp8Args(M, N, Kp, None, 0, None, wq.data_ptr(), ldw, ws.data_ptr(), bias.data_ptr() if bias is not None else None,
                       _ACTS[act], out.data_ptr(), ldo, VP_F32 if out.dtype == torch.float32 else VP_BF16)
        _lib.launch(dev, 'vp_linear_fp8', ctypes.byref(args), x.data_ptr(), tag, ldx, K, q.data_ptr() if q is not None else None,
                    s.data_ptr() if s is not None else None)
    return out
