"""Linears whose weight is chosen row by row: the expert layers of a mixture-of-experts model with any number of rows per
expert (MoEMlp.experts, mmpose/models/backbones/vit_moe.py:92-111, chooses per image and evaluates every expert on every
row).

    rows, offsets = expert_rows(expert, num_expert)                 # int32 [T] -> row list, int32 [num_expert + 1]
    y = grouped_linear(x, weight, bias, offsets, rows)              # bf16 [T, N]
    dx = grouped_linear_dgrad(dy, weight, offsets, rows)            # bf16 [T, K]
    dweight, dbias = grouped_linear_wgrad(dy, x, offsets, rows)     # f32 [E, N, K], [E, N]

`ExpertLinear` is the module with f32 master parameters and autograd on top of them.  Operands are bf16, sums f32.  The
routing stays on the device; nothing here synchronises.  The module records gradients, the functions do not (outside no_grad they
refuse rows and weights that require one).
"""
import ctypes

import torch
from torch import nn

from . import _lib
from ._lib import GroupedArgs

MAX_EXPERTS = 512
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_INSTEAD = 'use ExpertLinear, detach it, or call under torch.no_grad()'
_NOT_PLAIN = (AttributeError, TypeError, ValueError, RuntimeError)


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
    if expert.dtype is not _I32 or expert.dim() != 1 or not expert.is_contiguous():
        raise ValueError(f'expert: expected a contiguous one-dimensional int32 tensor, got {expert.dtype} {tuple(expert.shape)}')
    if not 1 <= num_expert <= MAX_EXPERTS:
        raise ValueError(f'num_expert {num_expert}: 1 to {MAX_EXPERTS} are supported')
    T = expert.shape[0]
    if T >> 31:
        _lib.too_large(T)
    rows, offsets = expert.new_empty(T), expert.new_empty(num_expert + 1)
    _lib.launch(expert.get_device(), _lib.lib().vp_expert_rows, expert.data_ptr(), T, num_expert, rows.data_ptr(), offsets.data_ptr())
    return rows, offsets


def _plain_routing(offsets, rows, E, T, d):
    """Whether offsets and rows are what the kernels take as they are (cheap: `_routing` finds the words for what is not)."""
    return (offsets.dtype is _I32 and offsets.shape == (E + 1,) and offsets.is_contiguous() and offsets.get_device() == d and
            (rows is None or (rows.dtype is _I32 and rows.shape == (T,) and rows.is_contiguous() and rows.get_device() == d)))


def _product(fwd, src, what, weight, bias, offsets, rows, out):
    try:
        T, C = src.shape
        E, N, K = weight.shape
        d, p, pw = src.get_device(), src.data_ptr(), weight.data_ptr()
        plain = (d >= 0 and src.dtype is _BF16 and weight.dtype is _BF16 and C == (K if fwd else N) and E and N and K and
                 not ((N | K) & 7 or (p | pw) & 15) and src.is_contiguous() and weight.is_contiguous() and
                 weight.get_device() == d and not (src.requires_grad or weight.requires_grad) and _plain_routing(offsets, rows, E, T, d) and
                 (bias is None or (bias.dtype is _F32 and bias.shape == (E, N) and bias.is_contiguous() and
                                   bias.get_device() == d and not bias.data_ptr() & 15)))
    except _NOT_PLAIN:
        plain = False
    if plain:
        se, sn, sb, ld = N * K, K, N, C
    else:
        _on_device(src, what)
        dev = src.device
        ld = _matrix(src, what, None, dev)
        se, sn = _weight(weight, dev)
        _lib.records_none(src, what, _INSTEAD)
        _lib.records_none(weight, 'weight', _INSTEAD)
        E, N, K = weight.shape
        T, C = src.shape
        if C != (K if fwd else N):
            raise ValueError(f'{what} {tuple(src.shape)} against a weight of {tuple(weight.shape)}')
        _routing(offsets, rows, E, T, dev)
        sb = 0
        if bias is not None:
            if bias.dtype != _F32 or tuple(bias.shape) != (E, N) or bias.device != dev:
                raise ValueError(f'bias: expected float32 [{E}, {N}] on {dev}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}')
            sb = bias.stride(0) if E > 1 else N
            if bias.stride(1) != 1 or sb % 4 or bias.data_ptr() % 16:
                raise ValueError('bias: contiguous rows a multiple of 4 elements apart, on 16-byte boundaries')
        d, p, pw = src.get_device(), src.data_ptr(), weight.data_ptr()
    if (T | E | N | K) >> 31:
        _lib.too_large(T, E, N, K)
    cols = N if fwd else K
    fresh = out is None
    if fresh:
        out = src.new_empty((T, cols))
    ldo = cols if fresh else _matrix(out, 'out', cols, src.device, T)
    if not fresh:
        _lib.records_none(out, 'out', _INSTEAD)
        for t, name in ((src, what), (weight, 'weight'), (bias, 'bias'), (offsets, 'offsets'), (rows, 'rows')):
            if t is not None and _lib.shares_memory(out, t):
                raise ValueError(f'out shares memory with {name}, which is read while it is written')
    if T:
        args = GroupedArgs(T, E, N, K, offsets.data_ptr(), rows.data_ptr() if rows is not None else None,
                           p if fwd else None, ld, pw, sn, se, bias.data_ptr() if bias is not None else None, sb,
                           None if fwd else p, ld, out.data_ptr(), ldo, fresh)
        L = _lib.lib()
        _lib.launch(d, L.vp_grouped_fwd if fwd else L.vp_grouped_dgrad, ctypes.byref(args))
    return out


def grouped_linear(x, weight, bias, offsets, rows=None, out=None):
    """out[t] = x[t] @ weight[e].T + bias[e] for every row t of expert e.  x bf16 [T, K], weight bf16 [E, N, K], bias f32
    [E, N] or None; offsets / rows as `expert_rows` returns them (rows None: the rows lie in the order of their experts), or
    E + 1 neighbours of its offsets for a run of the experts.  A new result has zeros in the rows that no expert takes; a given
    `out` keeps them as they are.  (A list that does not name every row needs an `out`: rows that it leaves out are not
    written.  `out` may not lie in an operand's memory.)"""
    return _product(True, x, 'x', weight, bias, offsets, rows, out)


def grouped_linear_dgrad(dy, weight, offsets, rows=None, out=None):
    """The gradient of x: out[t] = dy[t] @ weight[e] for every row t of expert e, bf16 [T, K] (other rows as above)."""
    return _product(False, dy, 'dy', weight, None, offsets, rows, out)


def grouped_linear_wgrad(dy, x, offsets, rows=None, want_bias=True):
    """(dweight f32 [E, N, K], dbias f32 [E, N] or None): sums of dy[t]^T x[t] and dy[t] over every expert's rows."""
    try:
        (T, K), (T2, N) = x.shape, dy.shape
        E = offsets.shape[0] - 1
        d, px, py = x.get_device(), x.data_ptr(), dy.data_ptr()
        plain = (d >= 0 and T == T2 and x.dtype is _BF16 and dy.dtype is _BF16 and N and K and E >= 1 and
                 not ((N | K) & 7 or (px | py) & 15) and x.is_contiguous() and dy.is_contiguous() and dy.get_device() == d and
                 not (x.requires_grad or dy.requires_grad) and
                 _plain_routing(offsets, rows, E, T, d))
    except _NOT_PLAIN:
        plain = False
    if plain:
        ldx, ldy = K, N
    else:
        _on_device(x, 'x')
        dev, T = x.device, x.shape[0]
        ldx = _matrix(x, 'x', None, dev)
        ldy = _matrix(dy, 'dy', None, dev, T)
        _lib.records_none(x, 'x', _INSTEAD)
        _lib.records_none(dy, 'dy', _INSTEAD)
        _on_device(offsets, 'offsets')
        E, N, K = offsets.numel() - 1, dy.shape[1], x.shape[1]
        if E < 1:
            raise ValueError('offsets: at least two values are needed')
        _routing(offsets, rows, E, T, dev)
        d, px, py = x.get_device(), x.data_ptr(), dy.data_ptr()
    if (T | E | N | K) >> 31:
        _lib.too_large(T, E, N, K)
    dw = x.new_empty((E, N, K), dtype=_F32)
    db = x.new_empty((E, N), dtype=_F32) if want_bias else None
    L = _lib.lib()
    slices = L.vp_grouped_wgrad_slices(T, E, N, K)
    need = slices * E * N * (K + (1 if want_bias else 0)) if slices > 1 else 0
    ws = x.new_empty(need, dtype=_F32) if need else None
    args = GroupedArgs(T, E, N, K, offsets.data_ptr(), rows.data_ptr() if rows is not None else None, px, ldx,
                       None, 0, 0, None, 0, py, ldy, None, 0, 0)
    _lib.launch(d, L.vp_grouped_wgrad, ctypes.byref(args), dw.data_ptr(), db.data_ptr() if want_bias else None,
                ws.data_ptr() if need else None, need * 4)
    return dw, db


def _bf16(w):
    """bf16 copy of f32 master weights."""
    _on_device(w, 'weight')
    if w.dtype is not _F32 or not w.is_contiguous() or w.data_ptr() % 16:
        raise ValueError(f'weight: expected contiguous float32 on a 16-byte boundary, got {w.dtype}, strides {w.stride()}')
    out = torch.empty(w.shape, dtype=_BF16, device=w.device)
    _lib.launch(w.get_device(), 'vp_cast_f32_bf16', w.data_ptr(), out.data_ptr(), w.numel())
    return out


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
        if dy.data_ptr() % 16:
            dy = dy.clone()
        dx = grouped_linear_dgrad(dy, w, offsets, rows) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw, db = grouped_linear_wgrad(dy, x, offsets, rows, want_bias=ctx.has_bias)
        return dx, dw, db, None, None, None


class ExpertLinear(nn.Module):
    """num_expert Linears of one shape, one per row: y[t] = x[t] @ weight[expert[t]].T + bias[expert[t]], zeros where
    expert[t] is not in [0, num_expert).  f32 master parameters (torch optimizers apply); every call rounds them to bf16
    once.  x bf16 [T, in_features], expert int32 [T].  A backward pass may be captured into a graph while no graph of an eager
    pass over the same parameters is alive (torch ends the process otherwise)."""

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
        return _GroupedLinear.apply(x, self.weight, self.bias, offsets, rows, _bf16(self.weight))

    def extra_repr(self):
        return f'num_expert={self.num_expert}, in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}'
