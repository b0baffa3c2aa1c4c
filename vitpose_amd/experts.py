"""Linears whose weight is chosen row by row: the expert layers of a mixture-of-experts model with any number of rows per
expert (MoEMlp.experts, mmpose/models/backbones/vit_moe.py:92-111, chooses per image and evaluates every expert on every
row).

    rows, offsets = expert_rows(expert, num_expert)                 # int32 [T] -> row list, int32 [num_expert + 1]
    y = grouped_linear(x, weight, bias, offsets, rows)              # bf16 [T, N]
    dx = grouped_linear_dgrad(dy, weight, offsets, rows)            # bf16 [T, K]
    dweight, dbias = grouped_linear_wgrad(dy, x, offsets, rows)     # f32 [E, N, K], [E, N]

`ExpertLinear` is the module with f32 master parameters and autograd on top of them.  Operands are bf16, sums f32.  The
routing stays on the device; nothing here synchronises.
"""
import ctypes

import torch
from torch import nn

from . import _lib
from ._lib import GroupedArgs

MAX_EXPERTS = 512


def _on_device(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{what}: expected a tensor, got {type(t).__name__}')
    if t.device.type != 'cuda':
        raise RuntimeError(f'{what} is on {t.device}: the expert products run on a HIP device only')


def _matrix(t, what, cols, dev, rows=None):
    """A bf16 [rows][cols] operand whose rows lie one after another at a multiple of 8 elements."""
    _on_device(t, what)
    if t.dtype != torch.bfloat16:
        raise TypeError(f'{what}: expected torch.bfloat16, got {t.dtype}')
    if t.dim() != 2 or (cols is not None and t.shape[1] != cols) or (rows is not None and t.shape[0] != rows):
        raise ValueError(f'{what}: shape {tuple(t.shape)}, expected [{rows if rows is not None else "T"}, {cols}]')
    if t.device != dev:
        raise ValueError(f'{what}: on {t.device}, other operands on {dev}')
    if t.shape[1] % 8 or t.shape[1] < 8:
        raise ValueError(f'{what}: {t.shape[1]} columns, a multiple of 8 is needed')
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if (t.stride(1) != 1 or ld % 8 or ld < t.shape[1] or t.data_ptr() % 16) and t.numel():
        raise ValueError(f'{what}: rows must be contiguous, a multiple of 8 elements apart and on 16-byte boundaries')
    return ld


def _weight(w, dev):
    _on_device(w, 'weight')
    if w.dtype != torch.bfloat16:
        raise TypeError(f'weight: expected torch.bfloat16, got {w.dtype}')
    if w.dim() != 3 or w.shape[0] < 1 or w.shape[1] < 8 or w.shape[2] < 8 or w.shape[1] % 8 or w.shape[2] % 8:
        raise ValueError(f'weight: shape {tuple(w.shape)}, expected [experts, N, K] with N and K multiples of 8')
    if w.device != dev:
        raise ValueError(f'weight: on {w.device}, other operands on {dev}')
    se, sn, sk = w.stride()
    if sk != 1 or sn % 8 or sn < w.shape[2] or se % 8 or w.data_ptr() % 16:
        raise ValueError('weight: K must be contiguous, rows and experts multiples of 8 elements apart, on 16-byte boundaries')
    return se, sn


def _routing(offsets, rows, E, T, dev):
    _on_device(offsets, 'offsets')
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() != E + 1 or not offsets.is_contiguous():
        raise ValueError(f'offsets: expected a contiguous int32 tensor of {E + 1} values, got {offsets.dtype} {tuple(offsets.shape)}')
    if offsets.device != dev or (rows is not None and rows.device != dev):
        raise ValueError(f'offsets and rows must be on {dev}')
    if rows is not None and (rows.dtype != torch.int32 or rows.dim() != 1 or rows.numel() != T or not rows.is_contiguous()):
        raise ValueError(f'rows: expected a contiguous int32 tensor of {T} values, got {rows.dtype} {tuple(rows.shape)}')


def expert_rows(expert, num_expert):
    """expert: int32 [T] -> (rows int32 [T], offsets int32 [num_expert + 1]): the row numbers in the order of their
    experts, rows of one expert ascending, then the rows whose entry is not in [0, num_expert); rows offsets[e] up to
    offsets[e + 1] of the list are expert e's."""
    _on_device(expert, 'expert')
    if expert.dtype != torch.int32 or expert.dim() != 1 or not expert.is_contiguous():
        raise ValueError(f'expert: expected a contiguous one-dimensional int32 tensor, got {expert.dtype} {tuple(expert.shape)}')
    if not 1 <= num_expert <= MAX_EXPERTS:
        raise ValueError(f'num_expert {num_expert}: 1 to {MAX_EXPERTS} are supported')
    rows = torch.empty_like(expert)
    offsets = torch.empty(num_expert + 1, dtype=torch.int32, device=expert.device)
    _lib.launch(expert.device, 'vp_expert_rows', expert.data_ptr(), expert.numel(), num_expert, rows.data_ptr(),
                offsets.data_ptr())
    return rows, offsets


def _product(name, src, src_cols, weight, bias, offsets, rows, out, out_cols):
    dev, T = src.device, src.shape[0]
    se, sn = _weight(weight, dev)
    E, N, K = weight.shape
    if src.shape[1] != src_cols:
        raise ValueError(f'{tuple(src.shape)} rows against a weight of {tuple(weight.shape)}')
    _routing(offsets, rows, E, T, dev)
    sb = 0
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E, N) or bias.device != dev:
            raise ValueError(f'bias: expected float32 [{E}, {N}] on {dev}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}')
        sb = bias.stride(0) if E > 1 else N
        if bias.stride(1) != 1 or sb % 4 or bias.data_ptr() % 16:
            raise ValueError('bias: contiguous rows a multiple of 4 elements apart, on 16-byte boundaries')
    fresh = out is None
    if fresh:
        out = torch.empty(T, out_cols, dtype=torch.bfloat16, device=dev)
    ldo = out_cols if fresh else _matrix(out, 'out', out_cols, dev, T)
    if T == 0:
        return out
    ld = src.stride(0) if T > 1 else src_cols
    fwd = name == 'vp_grouped_fwd'
    p = src.data_ptr()
    args = GroupedArgs(T, E, N, K, offsets.data_ptr(), rows.data_ptr() if rows is not None else None,
                       p if fwd else None, ld, weight.data_ptr(), sn, se, bias.data_ptr() if bias is not None else None, sb,
                       None if fwd else p, ld, out.data_ptr(), ldo, fresh)
    _lib.launch(dev, name, ctypes.byref(args))
    return out


def grouped_linear(x, weight, bias, offsets, rows=None, out=None):
    """out[t] = x[t] @ weight[e].T + bias[e] for every row t of expert e.  x bf16 [T, K], weight bf16 [E, N, K], bias f32
    [E, N] or None; offsets / rows as `expert_rows` returns them (rows None: the rows lie in the order of their experts).
    A new result has zeros in the rows that no expert takes; a given `out` keeps them as they are."""
    _on_device(x, 'x')
    _matrix(x, 'x', None, x.device)
    return _product('vp_grouped_fwd', x, weight.shape[-1], weight, bias, offsets, rows, out, weight.shape[1])


def grouped_linear_dgrad(dy, weight, offsets, rows=None, out=None):
    """The gradient of x: out[t] = dy[t] @ weight[e] for every row t of expert e, bf16 [T, K] (other rows as above)."""
    _on_device(dy, 'dy')
    _matrix(dy, 'dy', None, dy.device)
    return _product('vp_grouped_dgrad', dy, weight.shape[1], weight, None, offsets, rows, out, weight.shape[-1])


def grouped_linear_wgrad(dy, x, offsets, rows=None, want_bias=True):
    """(dweight f32 [E, N, K], dbias f32 [E, N] or None): sums of dy[t]^T x[t] and dy[t] over every expert's rows."""
    _on_device(x, 'x')
    dev, T = x.device, x.shape[0]
    ldx = _matrix(x, 'x', None, dev)
    ldy = _matrix(dy, 'dy', None, dev, T)
    _on_device(offsets, 'offsets')
    E, N, K = offsets.numel() - 1, dy.shape[1], x.shape[1]
    if E < 1:
        raise ValueError('offsets: at least two values are needed')
    _routing(offsets, rows, E, T, dev)
    dw = torch.empty(E, N, K, dtype=torch.float32, device=dev)
    db = torch.empty(E, N, dtype=torch.float32, device=dev) if want_bias else None
    slices = _lib.lib().vp_grouped_wgrad_slices(T, E, N, K)
    need = slices * E * N * (K + (1 if want_bias else 0)) if slices > 1 else 0
    ws = torch.empty(need, dtype=torch.float32, device=dev) if need else None
    args = GroupedArgs(T, E, N, K, offsets.data_ptr(), rows.data_ptr() if rows is not None else None, x.data_ptr(), ldx,
                       None, 0, 0, None, 0, dy.data_ptr(), ldy, None, 0, 0)
    _lib.launch(dev, 'vp_grouped_wgrad', ctypes.byref(args), dw.data_ptr(), db.data_ptr() if want_bias else None,
                ws.data_ptr() if need else None, need * 4)
    return dw, db


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, rows, weight_bf16):
        ctx.save_for_backward(x, weight_bf16, offsets, rows)
        ctx.has_bias = bias is not None
        return grouped_linear(x, weight_bf16, bias, offsets, rows)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, offsets, rows = ctx.saved_tensors
        dy = dy.contiguous()
        dx = grouped_linear_dgrad(dy, w, offsets, rows) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw, db = grouped_linear_wgrad(dy, x, offsets, rows, want_bias=ctx.has_bias)
        return dx, dw, db, None, None, None


class ExpertLinear(nn.Module):
    """num_expert Linears of one shape, one per row: y[t] = x[t] @ weight[expert[t]].T + bias[expert[t]], zeros where
    expert[t] is not in [0, num_expert).  f32 master parameters (torch optimizers apply); every call rounds them to bf16
    once.  x bf16 [T, in_features], expert int32 [T]."""

    def __init__(self, num_expert, in_features, out_features, bias=True, device=None):
        super().__init__()
        if not 1 <= num_expert <= MAX_EXPERTS:
            raise ValueError(f'num_expert {num_expert}: 1 to {MAX_EXPERTS} are supported')
        if in_features < 8 or out_features < 8 or in_features % 8 or out_features % 8:
            raise ValueError(f'{in_features} -> {out_features}: multiples of 8 are needed')
        self.num_expert, self.in_features, self.out_features = num_expert, in_features, out_features
        self.weight = nn.Parameter(torch.empty(num_expert, out_features, in_features, device=device))
        self.bias = nn.Parameter(torch.empty(num_expert, out_features, device=device)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        """nn.Linear's: uniform in +- in_features^-1/2."""
        r = self.in_features ** -0.5
        nn.init.uniform_(self.weight, -r, r)
        if self.bias is not None:
            nn.init.uniform_(self.bias, -r, r)

    def forward(self, x, expert):
        rows, offsets = expert_rows(expert, self.num_expert)
        return _GroupedLinear.apply(x, self.weight, self.bias, offsets, rows, self.weight.detach().bfloat16())

    def extra_repr(self):
        return f'num_expert={self.num_expert}, in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}'
