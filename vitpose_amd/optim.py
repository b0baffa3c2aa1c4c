"""Optimizer-side host logic: the layer-wise lr-decay parameter groups of the
reference's LayerDecayOptimizerConstructor
(mmcv_custom/layer_decay_optimizer_constructor.py:6-78), the step / warm-up lr
schedule of the ViTPose configs, and the chunk table that drives the fused AdamW
kernel over the flat parameter buffer.
"""
from ctypes import c_void_p
from typing import Dict, List, Sequence, Tuple

import torch

from . import _lib

CHUNK = 1 << 11  # elements per AdamW workgroup: two float4 per lane; measured 596 us per step for 90 M
# parameters (norm + update) against 637 us at 1 << 16, whose 1472 workgroups leave an uneven last round


def get_num_layer_for_vit(var_name: str, num_max_layer: int) -> int:
    """Layer id of a TopDown parameter name (layer_decay_optimizer_constructor.py:6-15)."""
    if var_name in ('backbone.cls_token', 'backbone.mask_token', 'backbone.pos_embed'):
        return 0
    if var_name.startswith('backbone.patch_embed'):
        return 0
    if var_name.startswith('backbone.blocks'):
        return int(var_name.split('.')[2]) + 1
    return num_max_layer - 1


def layer_decay_param_groups(named_shapes: Sequence[Tuple[str, Tuple[int, ...]]], num_layers: int,
                             layer_decay_rate: float, base_lr: float, base_wd: float) -> Dict[str, dict]:
    """Per-parameter {lr_scale, lr, weight_decay, group_name}: the groups `add_params` builds
    (same file, :32-65).  `num_layers` is the config value (depth); the constructor adds 2."""
    n = num_layers + 2
    out = {}
    for name, shape in named_shapes:
        if len(shape) == 1 or name.endswith('.bias') or 'pos_embed' in name:
            gname, wd = 'no_decay', 0.
        else:
            gname, wd = 'decay', base_wd
        lid = get_num_layer_for_vit(name, n)
        scale = layer_decay_rate ** (n - lid - 1)
        out[name] = dict(group_name=f'layer_{lid}_{gname}', lr_scale=scale, lr=scale * base_lr, weight_decay=wd)
    return out


def step_lr(base_lr: float, it: int, epoch: int, steps=(170, 200), gamma=0.1, warmup_iters=500,
            warmup_ratio=0.001) -> float:
    """mmcv StepLrUpdaterHook with linear warm-up, as configured at
    configs/.../ViTPose_base_coco_256x192.py:32-38."""
    lr = base_lr * gamma ** sum(epoch >= s for s in steps)
    if it < warmup_iters:
        k = (1 - it / warmup_iters) * (1 - warmup_ratio)
        lr = lr * (1 - k)
    return lr


# ---------------------------------------------------------------------------------------------------------------
# moments in 8 bits
# ---------------------------------------------------------------------------------------------------------------
STATE_BLOCK = 128      # state values that share one scale
_F8, _F32, _I64 = torch.float8_e4m3fn, torch.float32, torch.int64


def new_state8(numel: int, device):
    """Zero moments for `numel` state values (a multiple of 128): (exp_avg e4m3 [numel], its scales f32 [numel / 128],
    sqrt(exp_avg_sq) e4m3 [numel], its scales f32 [numel / 128])."""
    if numel % STATE_BLOCK:
        raise ValueError(f'state values come in blocks of {STATE_BLOCK}, got {numel}')

    def codes():
        return torch.zeros(numel, dtype=torch.uint8, device=device).view(_F8)

    def scales():
        return torch.zeros(numel // STATE_BLOCK, dtype=torch.float32, device=device)
    return codes(), scales(), codes(), scales()


def noise_key(seed: int, step: int) -> int:
    """The `noise` argument of step number `step` of a run with `seed`: 31 bits, the same on every rank."""
    def mix(h):
        h ^= h >> 16
        h = h * 0x85EBCA6B & 0xFFFFFFFF
        h ^= h >> 13
        h = h * 0xC2B2AE35 & 0xFFFFFFFF
        return h ^ (h >> 16)
    return mix((seed & 0xFFFFFFFF) ^ mix(step & 0xFFFFFFFF)) & 0x7FFFFFFF


def _flat_arg(t, dtype, name, device, numel=None):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f'{name}: expected a {dtype} tensor, got {getattr(t, "dtype", type(t).__name__)}')
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f'{name}: must be one-dimensional and contiguous')
    if t.device != device:
        raise ValueError(f'{name}: on {t.device}, the parameters on {device}')
    if numel is not None and t.numel() != numel:
        raise ValueError(f'{name}: {t.numel()} values, expected {numel}')


def adamw8_step(param, grad, state, chunks, *, lr, betas=(0.9, 0.999), eps=1e-8, step, noise, half=None,
                max_grad_norm=0.0, grad_scale=1.0):
    """One AdamW step over flat f32 buffers whose moments are held in 8 bits (torch.optim.AdamW's update).

    param, grad: f32 [numel], numel a multiple of 4;  half: bf16 [numel] copy of the new weights, or None;  state: as `new_state8` makes it;
    chunks: device tensors (start int64, length int32, lr_scale f32, weight_decay f32, state_start int64), one entry per
    run of at most 2048 consecutive elements of one tensor (starts and lengths multiples of 4, state starts multiples
    of 128, no overlaps; an entry that leaves the buffers is skipped);  step: number of this step, from 1;  noise: key
    of this step's random numbers (`noise_key`).  max_grad_norm > 0 clips the gradients of the table's elements by their
    norm first.  Everything is updated in place on the current stream; nothing synchronises.  lr, step and noise are arguments
    of the launch: a captured graph repeats the ones that it was captured with."""
    m8, ms, r8, rs = state
    start, length, lr_scale, decay, state_start = chunks or (None,) * 5
    b1, b2 = betas
    try:
        d, n, ns, nc = param.get_device(), param.shape, m8.shape, start.shape
        (nb,) = ns
        plain = (d >= 0 and len(n) == 1 and len(nc) == 1 and not nb & 127 and
                 all(t.shape == sh and t.dtype is dt and t.is_contiguous() and t.get_device() == d for t, sh, dt in (
                     (param, n, _F32), (grad, n, _F32), (m8, ns, _F8), (r8, ns, _F8), (ms, (nb >> 7,), _F32), (rs, (nb >> 7,), _F32),
                     (start, nc, _I64), (length, nc, torch.int32), (lr_scale, nc, _F32), (decay, nc, _F32),
                     (state_start, nc, _I64))) and
                 (half is None or (half.shape == n and half.dtype is torch.bfloat16 and half.is_contiguous() and half.get_device() == d)))
    except (AttributeError, TypeError, ValueError, RuntimeError):
        plain = False
    if not plain:
        _check_adamw8(param, grad, state, chunks, half)
    if step < 1 or not (0 <= b1 < 1 and 0 <= b2 < 1) or not (eps == 0 or eps >= 1.2e-38):
        raise ValueError(f'step {step}, betas {betas}, eps {eps}: step >= 1, betas in [0, 1) and eps 0 or a normal f32 number needed')
    if not 0 <= noise < 1 << 32:
        raise ValueError('noise is a 32-bit key')
    d, n, ns, nc = param.get_device(), param.numel(), m8.numel(), start.numel()
    if n & 3:
        raise ValueError(f'param: {n} values; a run is a multiple of 4 long, so one that reaches the end would leave the buffer: pad it')
    if nc >> 31:
        _lib.too_large(nc)
    if nc == 0:
        return
    L = _lib.lib()
    partials, npart = None, 0
    if max_grad_norm > 0:
        npart = min(256, (nc + 3) // 4)
        partials = param.new_empty(npart, dtype=torch.float64)
        _lib.launch(d, L.vp_sumsq_chunks_f64, grad.data_ptr(), start.data_ptr(), length.data_ptr(), nc, n, partials.data_ptr(), npart)
    _lib.launch(d, L.vp_adamw8_step, param.data_ptr(), grad.data_ptr(), m8.data_ptr(), ms.data_ptr(), r8.data_ptr(),
                rs.data_ptr(), half.data_ptr() if half is not None else None, start.data_ptr(), length.data_ptr(),
                lr_scale.data_ptr(), decay.data_ptr(), state_start.data_ptr(), nc, n, ns, lr, b1, b2, eps, step,
                partials.data_ptr() if npart else None, npart, max_grad_norm, grad_scale, noise)


def _check_adamw8(param, grad, state, chunks, half):
    """The words for what `adamw8_step` cannot take."""
    dev = param.device
    if dev.type != 'cuda':
        raise RuntimeError('adamw8_step runs on a HIP device only')
    n = param.numel()
    _flat_arg(param, torch.float32, 'param', dev)
    _flat_arg(grad, torch.float32, 'grad', dev, n)
    if half is not None:
        _flat_arg(half, torch.bfloat16, 'half', dev, n)
    m8, ms, r8, rs = state
    ns = m8.numel()
    if ns % STATE_BLOCK:
        raise ValueError(f'state values come in blocks of {STATE_BLOCK}, got {ns}')
    _flat_arg(m8, _F8, 'exp_avg', dev)
    _flat_arg(r8, _F8, 'exp_avg_sq', dev, ns)
    _flat_arg(ms, torch.float32, 'exp_avg scale', dev, ns // STATE_BLOCK)
    _flat_arg(rs, torch.float32, 'exp_avg_sq scale', dev, ns // STATE_BLOCK)
    start, length, lr_scale, decay, state_start = chunks
    nc = start.numel()
    _flat_arg(start, torch.int64, 'chunk start', dev)
    _flat_arg(length, torch.int32, 'chunk length', dev, nc)
    _flat_arg(lr_scale, torch.float32, 'chunk lr scale', dev, nc)
    _flat_arg(decay, torch.float32, 'chunk weight decay', dev, nc)
    _flat_arg(state_start, torch.int64, 'chunk state start', dev, nc)


class FlatAdamW:
    """torch.optim.AdamW semantics over a ParamStore, one fused kernel per step.

    state_bits = 8 holds both moments in 8 bits (`adamw8_step`; 2.06 bytes of state a parameter instead of 8): its
    random numbers follow from `noise_seed` and the step count, so ranks that hold the same gradients stay identical."""

    def __init__(self, store, groups: Dict[str, dict], lr: float, betas=(0.9, 0.999), eps=1e-8,
                 max_grad_norm: float = 0.0, frozen: Sequence[str] = (), state_bits: int = 32, noise_seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits is 8 or 32, got {state_bits}')
        self.state_bits, self.noise_seed = state_bits, noise_seed
        self.store, self.lr, self.betas, self.eps = store, lr, betas, eps
        self.max_grad_norm = max_grad_norm
        self.step_count = 0
        self.frozen = tuple(frozen)
        dev = store.device
        starts, lens, scales, wds, sstarts, soff = [], [], [], [], [], 0
        self.state_offsets = {}
        for name in store.names:
            if name in frozen:
                continue
            grp = groups[name]
            n = store.view(name).numel()
            n_pad = (n + 3) // 4 * 4  # padding inside the 64-element alignment gap: zeros stay zeros
            off = store.offsets[name]
            self.state_offsets[name] = soff
            for c0 in range(0, n_pad, CHUNK):
                starts.append(off + c0)
                lens.append(min(CHUNK, n_pad - c0))
                scales.append(grp['lr_scale'])
                wds.append(grp['weight_decay'])
                sstarts.append(soff + c0)
            soff += (n_pad + STATE_BLOCK - 1) // STATE_BLOCK * STATE_BLOCK
        self.nchunks = len(starts)
        self.chunk_start = torch.tensor(starts, dtype=torch.int64, device=dev)
        self.chunk_len = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.chunk_lr_scale = torch.tensor(scales, dtype=torch.float32, device=dev)
        self.chunk_wd = torch.tensor(wds, dtype=torch.float32, device=dev)
        if state_bits == 8:
            self.chunk_state = torch.tensor(sstarts, dtype=torch.int64, device=dev)
            self.state8 = new_state8(soff, dev)
            return
        self.exp_avg = torch.zeros_like(store.data)
        self.exp_avg_sq = torch.zeros_like(store.data)
        self.gnorm_sq = torch.zeros(1, dtype=torch.float32, device=dev)
        # per-workgroup partial sums of the gradient norm: summed in a fixed order, so that every data-parallel
        # replica derives the same clip factor, bit for bit, from the same all-reduced gradients
        self.gnorm_partials = torch.zeros(2048, dtype=torch.float32, device=dev)

    def step(self, lr: float = None, grad_scale: float = 1.0):
        if self.state_bits == 8:
            st = self.store
            self.step_count += 1
            adamw8_step(st.data, st.grad, self.state8, (self.chunk_start, self.chunk_len, self.chunk_lr_scale,
                                                        self.chunk_wd, self.chunk_state),
                        lr=self.lr if lr is None else lr, betas=self.betas, eps=self.eps, step=self.step_count,
                        noise=noise_key(self.noise_seed, self.step_count), half=st.half,
                        max_grad_norm=self.max_grad_norm, grad_scale=grad_scale)
            return
        L = _lib.lib()
        s = c_void_p(torch.cuda.current_stream().cuda_stream)
        st = self.store
        self.step_count += 1
        gn = None
        if self.max_grad_norm > 0:
            # the norm runs over the optimizer's own chunks: parameters it does not update (frozen ones) stay out of
            # the clip factor, as torch's clip_grad_norm_ over the parameters with requires_grad leaves them out
            rc = L.vp_sumsq_chunks_det(c_void_p(st.grad.data_ptr()), c_void_p(self.chunk_start.data_ptr()),
                                       c_void_p(self.chunk_len.data_ptr()), self.nchunks,
                                       c_void_p(self.gnorm_sq.data_ptr()), c_void_p(self.gnorm_partials.data_ptr()),
                                       self.gnorm_partials.numel(), s)
            if rc:
                raise RuntimeError(f'vp_sumsq_chunks_det failed: {rc}')
            gn = c_void_p(self.gnorm_sq.data_ptr())
        rc = L.vp_adamw_step(
            c_void_p(st.data.data_ptr()), c_void_p(st.grad.data_ptr()), c_void_p(self.exp_avg.data_ptr()),
            c_void_p(self.exp_avg_sq.data_ptr()), c_void_p(st.half.data_ptr()),
            c_void_p(self.chunk_start.data_ptr()), c_void_p(self.chunk_len.data_ptr()),
            c_void_p(self.chunk_lr_scale.data_ptr()), c_void_p(self.chunk_wd.data_ptr()), self.nchunks,
            self.lr if lr is None else lr, self.betas[0], self.betas[1], self.eps, self.step_count, gn,
            self.max_grad_norm, grad_scale, s)
        if rc:
            raise RuntimeError(f'vp_adamw_step failed: {rc}')

    # -- checkpointing (the reference saves optimizer.state_dict() next to the weights,
    #    mmcv_custom/checkpoint.py:490-552; runner.resume restores it) --
    def state_dict(self):
        """Adam moments per parameter NAME (CPU tensors) + the step count and hyper-parameters.  8-bit moments are
        saved as they are held (e4m3 codes as bytes + block scales), so that a resumed run continues bit for bit."""
        st = self.store
        names = [n for n in st.names if n not in self.frozen]
        if self.state_bits == 8:
            return {'format': 'vitpose_amd.FlatAdamW8/1', 'step': self.step_count, 'noise_seed': self.noise_seed,
                    'hyper': dict(lr=self.lr, betas=tuple(self.betas), eps=self.eps, max_grad_norm=self.max_grad_norm),
                    'state': {n: {k: v.detach().cpu().clone() for k, v in self._state8_views(n).items()} for n in names}}
        return {'format': 'vitpose_amd.FlatAdamW/1', 'step': self.step_count,
                'hyper': dict(lr=self.lr, betas=tuple(self.betas), eps=self.eps, max_grad_norm=self.max_grad_norm),
                'state': {n: {'exp_avg': st._v(self.exp_avg, n).detach().cpu().clone(),
                              'exp_avg_sq': st._v(self.exp_avg_sq, n).detach().cpu().clone()} for n in names}}

    def _state8_views(self, name):
        """The blocks of one parameter in the 8-bit state, codes as bytes."""
        n = self.store.view(name).numel()
        b0 = self.state_offsets[name] // STATE_BLOCK
        b1 = b0 + (n + STATE_BLOCK - 1) // STATE_BLOCK
        m8, ms, r8, rs = self.state8
        return {'exp_avg': m8.view(torch.uint8)[b0 * STATE_BLOCK:b1 * STATE_BLOCK], 'exp_avg_scale': ms[b0:b1],
                'exp_avg_sq_root': r8.view(torch.uint8)[b0 * STATE_BLOCK:b1 * STATE_BLOCK], 'exp_avg_sq_scale': rs[b0:b1]}

    def load_state_dict(self, sd):
        want = 'vitpose_amd.FlatAdamW8/1' if self.state_bits == 8 else 'vitpose_amd.FlatAdamW/1'
        if sd.get('format') != want:
            raise ValueError(f'not a FlatAdamW state dict of {self.state_bits}-bit moments (expected format "{want}")')
        st = self.store
        names = [n for n in st.names if n not in self.frozen]
        missing = [n for n in names if n not in sd['state']]
        unexpected = [n for n in sd['state'] if n not in names]
        if missing or unexpected:
            raise KeyError(f'optimizer state does not match the model: missing {missing[:3]}, unexpected {unexpected[:3]}')
        if self.state_bits == 8:
            for n in names:
                for key, view in self._state8_views(n).items():
                    v = sd['state'][n][key]
                    if v.shape != view.shape or v.dtype != view.dtype:
                        raise ValueError(f'{n}.{key}: {v.dtype} {tuple(v.shape)} != {view.dtype} {tuple(view.shape)}')
            for n in names:
                for key, view in self._state8_views(n).items():
                    view.copy_(sd['state'][n][key])
            self.noise_seed = int(sd['noise_seed'])
        for n in names if self.state_bits == 32 else ():
            for key, buf in (('exp_avg', self.exp_avg), ('exp_avg_sq', self.exp_avg_sq)):
                v = sd['state'][n][key]
                if tuple(v.shape) != tuple(st.shapes[n]):
                    raise ValueError(f'{n}.{key}: shape {tuple(v.shape)} != {tuple(st.shapes[n])}')
                st._v(buf, n).copy_(v.to(st.device, torch.float32))
        self.step_count = int(sd['step'])
        h = sd.get('hyper', {})
        self.lr = h.get('lr', self.lr)
        self.betas = tuple(h.get('betas', self.betas))
        self.eps = h.get('eps', self.eps)
        self.max_grad_norm = h.get('max_grad_norm', self.max_grad_norm)
