"""Refusals that the host sides of the C entry points make before anything reaches a device, and host arithmetic of the
operators for expert layers and 8-bit formats."""
import pytest
import torch

from vitpose_amd import _lib, optim

ERR_ARG = -1


def adamw8(**over):
    a = dict(p=64, g=64, m=64, ms=64, r=64, rs=64, half=None, start=64, length=64, scale=64, wd=64, state=64, nchunks=1, numel=128,
             state_numel=128, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, step=1, partials=None, npartials=0, max_norm=0.0,
             grad_scale=1.0, noise=0)
    a.update(over)
    return _lib.lib().vp_adamw8_step(*a.values(), None)


@pytest.mark.parametrize('over', [dict(p=None), dict(g=None), dict(m=None), dict(rs=None), dict(start=None), dict(state=None),
                                  dict(step=0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(nchunks=-1), dict(numel=-1),
                                  dict(state_numel=100), dict(p=72), dict(g=68), dict(m=65), dict(half=66), dict(npartials=257),
                                  dict(npartials=3), dict(npartials=3, partials=64, max_norm=0.0)])
def test_adamw8_refuses_on_the_host(over):
    assert adamw8(**over) == ERR_ARG


def test_adamw8_with_an_empty_table_does_nothing():
    assert adamw8(nchunks=0, p=None, g=None) == 0


@pytest.mark.parametrize('over', [dict(partials=None), dict(n=0), dict(n=257), dict(x=None), dict(x=72), dict(nchunks=-1)])
def test_sumsq_chunks_f64_refuses_on_the_host(over):
    a = dict(x=64, start=64, length=64, nchunks=1, numel=4, partials=64, n=1)
    a.update(over)
    assert _lib.lib().vp_sumsq_chunks_f64(*a.values(), None) == ERR_ARG


def test_adamw8_needs_a_device():
    st = optim.new_state8(128, 'cpu')
    with pytest.raises(RuntimeError):
        optim.adamw8_step(torch.zeros(4), torch.zeros(4), st, (), lr=1e-3, step=1, noise=0)
    with pytest.raises(ValueError):
        optim.new_state8(100, 'cpu')


def test_noise_keys_differ_by_step_and_seed():
    keys = {optim.noise_key(s, t) for s in range(8) for t in range(1, 129)}
    assert len(keys) == 8 * 128 and all(0 <= k < 1 << 31 for k in keys)


def grouped(entry, *more, **over):
    from vitpose_amd._lib import GroupedArgs
    import ctypes
    a = dict(T=16, E=2, N=16, K=32, offsets=64, rows=64, x=64, ldx=32, w=64, ldw=32, stride_w=512, bias=64, stride_b=16, dy=64,
             ldy=16, out=64, ldo=32, zero_rest=0)
    a.update(over)
    return getattr(_lib.lib(), entry)(ctypes.byref(GroupedArgs(*a.values())), *more, None)


COMMON = [dict(T=-1), dict(E=0), dict(N=12), dict(N=0), dict(K=20), dict(offsets=None)]


@pytest.mark.parametrize('over', COMMON + [dict(x=None), dict(x=72), dict(w=None), dict(w=66), dict(out=None), dict(out=8), dict(ldx=24),
                                           dict(ldx=36), dict(ldw=24), dict(ldo=8), dict(ldo=20), dict(stride_w=100), dict(bias=68),
                                           dict(stride_b=18)])
def test_grouped_fwd_refuses_on_the_host(over):
    assert grouped('vp_grouped_fwd', **over) == ERR_ARG


@pytest.mark.parametrize('over', COMMON + [dict(dy=None), dict(dy=72), dict(w=None), dict(out=8), dict(ldy=8), dict(ldy=20), dict(ldo=24)])
def test_grouped_dgrad_refuses_on_the_host(over):
    assert grouped('vp_grouped_dgrad', **over) == ERR_ARG


@pytest.mark.parametrize('over', COMMON + [dict(dy=None), dict(x=None), dict(x=72), dict(ldx=24), dict(ldy=12)])
def test_grouped_wgrad_refuses_on_the_host(over):
    assert grouped('vp_grouped_wgrad', 64, 64, None, 0, **over) == ERR_ARG


def test_grouped_wgrad_refuses_missing_results_and_workspace():
    assert grouped('vp_grouped_wgrad', None, 64, None, 0) == ERR_ARG
    assert grouped('vp_grouped_wgrad', 72, 64, None, 0) == ERR_ARG
    assert _lib.lib().vp_grouped_wgrad_slices(100000, 1, 16, 32) > 1
    assert grouped('vp_grouped_wgrad', 64, 64, None, 0, T=100000, E=1) == ERR_ARG
    assert grouped('vp_grouped_wgrad', 64, 64, 64, 1024, T=100000, E=1) == ERR_ARG


def test_grouped_products_of_no_rows_touch_nothing():
    assert grouped('vp_grouped_fwd', T=0, x=None, out=None) == 0
    assert grouped('vp_grouped_dgrad', T=0, dy=None, out=None) == 0


def test_expert_rows_refuses_on_the_host():
    L = _lib.lib()
    for a in ((64, -1, 2, 64, 64), (64, 8, 0, 64, 64), (None, 8, 2, 64, 64), (64, 8, 2, None, 64), (64, 8, 2, 64, None)):
        assert L.vp_expert_rows(*a, None) == ERR_ARG
    assert L.vp_expert_rows(64, 8, 513, 64, 64, None) == -2


def test_expert_operators_need_a_device():
    from vitpose_amd import experts
    x, w = torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    offsets = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        experts.expert_rows(offsets, 2)
    with pytest.raises(RuntimeError):
        experts.grouped_linear(x, w, None, offsets)
    with pytest.raises(RuntimeError):
        experts.grouped_linear_dgrad(x[:, :8], w, offsets)
    with pytest.raises(RuntimeError):
        experts.grouped_linear_wgrad(x, x, offsets)
    with pytest.raises(ValueError):
        experts.ExpertLinear(2, 12, 16)
    with pytest.raises(ValueError):
        experts.ExpertLinear(513, 16, 16)
    assert set(experts.ExpertLinear(2, 16, 8).state_dict()) == {'weight', 'bias'}


def fp8_gemm(**over):
    import ctypes
    from vitpose_amd._lib import Fp8Args
    a = dict(M=4, N=8, K=128, xq=64, ldx=128, xs=64, wq=64, ldw=128, ws=64, bias=None, act=0, out=64, ldo=8, out_dtype=1)
    a.update(over)
    return _lib.lib().vp_gemm_fp8(ctypes.byref(Fp8Args(*a.values())), None)


@pytest.mark.parametrize('over', [dict(M=-1), dict(N=0), dict(K=0), dict(K=100), dict(K=192), dict(act=2), dict(out_dtype=2), dict(xq=None),
                                  dict(xq=68), dict(xs=None), dict(wq=None), dict(wq=65), dict(ws=None), dict(out=None), dict(out=8),
                                  dict(ldx=112), dict(ldx=136), dict(ldw=0), dict(ldo=7)])
def test_gemm_fp8_refuses_on_the_host(over):
    assert fp8_gemm(**over) == ERR_ARG


@pytest.mark.parametrize('entry', ['vp_quantize_fp8_rows', 'vp_quantize_fp8_weight'])
def test_fp8_quantizers_refuse_on_the_host(entry):
    f = getattr(_lib.lib(), entry)
    ok = dict(x=64, dtype=0, ld=16, rows=2, K=16, q=64, scale=64)
    for over in (dict(x=None), dict(x=72), dict(dtype=2), dict(ld=8), dict(ld=20), dict(rows=-1), dict(K=0), dict(K=12), dict(q=None),
                 dict(q=72), dict(scale=None)):
        assert f(*{**ok, **over}.values(), None) == ERR_ARG, over


def test_fp8_of_no_rows_touches_nothing_and_needs_a_device():
    from vitpose_amd import fp8
    assert fp8_gemm(M=0, xq=None, out=None) == 0
    assert _lib.lib().vp_quantize_fp8_rows(None, 0, 16, 0, 16, None, None, None) == 0
    x = torch.zeros(4, 16)
    with pytest.raises(RuntimeError):
        fp8.quantize_rows(x)
    with pytest.raises(RuntimeError):
        fp8.quantize_weight(x)
    with pytest.raises(RuntimeError):
        fp8.linear(x, x, x)


def linear_fp8(**over):
    import ctypes
    from vitpose_amd._lib import Fp8Args
    a = dict(M=4, N=8, K=128, xq=None, ldx=0, xs=None, wq=64, ldw=128, ws=64, bias=None, act=0, out=64, ldo=8, out_dtype=1)
    more = dict(x=64, dtype=1, rows=16, k=16, q=64, s=64)
    for k, v in over.items():
        (more if k in more else a)[k] = v
    return _lib.lib().vp_linear_fp8(ctypes.byref(Fp8Args(*a.values())), *more.values(), None)


@pytest.mark.parametrize('over', [dict(M=-1), dict(N=0), dict(K=100), dict(wq=None), dict(wq=72), dict(ws=None), dict(out=None), dict(ldw=64),
                                  dict(ldo=4), dict(act=5), dict(out_dtype=7), dict(x=None), dict(x=72), dict(dtype=2), dict(rows=8),
                                  dict(rows=20), dict(k=12), dict(k=0), dict(k=136, rows=136), dict(M=100000, N=5120, q=None),
                                  dict(M=100000, N=5120, s=None)])
def test_linear_fp8_refuses_on_the_host(over):
    over = dict(over)
    if over.get('N') == 5120:
        over['ldo'] = 5120
    assert linear_fp8(**over) == ERR_ARG


def test_linear_fp8_of_no_rows_touches_nothing():
    assert linear_fp8(M=0, x=None, q=None, s=None, out=None) == 0
    L = _lib.lib()
    assert L.vp_linear_fp8_fused(1, 5120, 1280, 1) == 1 and L.vp_linear_fp8_fused(24576, 1280, 5120, 1) == 0
    assert L.vp_linear_fp8_fused(0, 8, 8, 1) == 0


@pytest.mark.parametrize('over', [dict(resid=64, ldr=8), dict(resid=64, ldr=7, out_dtype=0), dict(resid=68, ldr=8, out_dtype=0), dict(M=(1 << 29) + 1)])
def test_fp8_residuals_and_row_counts_refused_on_the_host(over):
    assert fp8_gemm(**over) == ERR_ARG and (over.get('M') or linear_fp8(**over) == ERR_ARG)


@pytest.mark.parametrize('over', [dict(oscale=None), dict(ldo=120), dict(ldo=136), dict(N=136), dict(resid=64)])
def test_fp8_results_as_codes_refused_on_the_host(over):
    a = dict(out_dtype=2, ldo=128, resid=None, ldr=8, oscale=64)
    a.update(over)
    assert fp8_gemm(**a) == ERR_ARG
    assert linear_fp8(**dict(a, ldo=128, N=8, resid=None, oscale=64)) == ERR_ARG


@pytest.mark.parametrize('over', [dict(x=None), dict(x=4), dict(gamma=None), dict(gamma=8), dict(beta=None), dict(beta=4), dict(M=-1), dict(M=1 << 30), dict(E=0),
                                  dict(E=12), dict(E=2056), dict(q=None), dict(q=8), dict(s=None)])
def test_layernorm_fp8_refuses_on_the_host(over):
    a = dict(x=64, gamma=64, beta=64, eps=1e-6, M=4, E=64, q=64, s=64)
    a.update(over)
    assert _lib.lib().vp_layernorm_fp8(*a.values(), None) == ERR_ARG


def test_layernorm_fp8_of_no_rows_touches_nothing():
    assert _lib.lib().vp_layernorm_fp8(None, None, None, 1e-6, 0, 64, None, None, None) == 0


def test_every_entry_is_called_with_the_header_s_arguments():
    """Number and kind of the arguments in the ctypes table against the prototypes: a missing one would hand the callee a truncated
    pointer."""
    import ctypes
    import os
    import re
    with open(os.path.join(os.path.dirname(__file__), '..', 'include', 'vitpose_hip.h')) as f:
        text = re.sub(r'/\*.*?\*/', '', f.read(), flags=re.S)
    kinds = {'int': ctypes.c_int, 'long': ctypes.c_long, 'size_t': ctypes.c_size_t, 'float': ctypes.c_float, 'double': ctypes.c_double}
    checked = 0
    for name, params in re.findall(r'\bint (vp_\w+)\(([^;{]*)\);', text):
        types = _lib.SIGNATURES.get(name)
        if types is None:
            continue
        params = [p.strip() for p in params.split(',') if p.strip() not in ('', 'void')]
        assert len(types) == len(params), f'{name}: {len(types)} arguments, {len(params)} in the header'
        for t, p in zip(types, params):
            plain = '*' not in p and '[' not in p and not p.startswith('vp_stream_t')
            words = [w for w in p.split()[:-1] if w not in ('const', 'unsigned')]
            if plain and words and words[0] in kinds and 'unsigned' not in p:
                assert t is kinds[words[0]], f'{name}: {p} is called with {t.__name__}'
            elif not plain:
                assert ctypes.sizeof(t) == ctypes.sizeof(ctypes.c_void_p), f'{name}: {p}'
        checked += 1
    assert checked > 40


@pytest.mark.parametrize('eps,rc', [(0.0, 0), (1e-8, 0), (1.2e-38, 0), (1e-40, ERR_ARG), (float('nan'), ERR_ARG)])
def test_adamw8_takes_no_eps_that_the_division_flushes(eps, rc):
    # (an empty table: nothing is launched, only the arguments are looked at)
    assert adamw8(eps=eps, nchunks=0) == rc


def test_row_counts_beyond_32_bit_arithmetic_are_refused():
    import ctypes
    from vitpose_amd._lib import GroupedArgs
    L, T = _lib.lib(), (1 << 30) + 1
    assert L.vp_expert_rows(64, T, 4, 64, 64, None) == ERR_ARG
    a = GroupedArgs(T, 4, 64, 64, 64, 64, 64, 64, 64, 64, 64 * 64, None, 0, 64, 64, 64, 64, 0)
    assert L.vp_grouped_fwd(ctypes.byref(a), None) == ERR_ARG
    assert L.vp_grouped_dgrad(ctypes.byref(a), None) == ERR_ARG
    assert L.vp_grouped_wgrad(ctypes.byref(a), 64, None, None, 0, None) == ERR_ARG


def test_which_tensors_share_memory():
    share = _lib.shares_memory
    flat = torch.zeros(4096)
    a = flat[:1024].view(16, 64)
    assert share(a, a) and share(a, a[3:5]) and share(a[:, :8], a[:, 4:12]) and share(flat, a) and share(a.view(16, 8, 8), a)
    assert not share(a, flat[1024:2048].view(16, 64)) and not share(a[:8], a[8:]) and not share(flat[1024:], a)
    # beside each other in the rows of one array, whichever begins first, also with single rows and other types
    assert not share(a[:, :32], a[:, 32:]) and not share(a[:, 32:], a[:, :32]) and not share(a[:9, 40:], a[2:, 8:40])
    assert share(a[:, :33], a[:, 32:]) and share(a[:, 32:], a[1:, :33])
    assert not share(a[3:4, :32], a[:, 32:]) and share(a[3:4, :33], a[:, 32:]) and share(a[3:4], a[3:4]) and not share(a[3:4], a[4:5])
    half = flat.view(torch.bfloat16)[:2048].view(16, 128)
    assert not share(half[:, :64], a[:, 32:]) and share(half[:, :66], a[:, 32:]) and not share(half[:, 64:], a[:, :32])
    # rows of another distance: the whole ranges count
    assert share(a[:, :8], flat[8:2056].view(16, 128)[:, :8])
    assert not share(a, a[:0]) and not share(a[:, :0], a)


def test_no_kernel_is_chosen_that_needs_more_threads_than_a_launch_takes():
    """2^32 threads: 2^23 workgroups of 512."""
    L, unsupported = _lib.lib(), -2
    assert L.vp_linear_fp8_fused(16, 8, 128, 1) == 1
    for M in (1 << 28, 1 << 29):             # 16 rows a workgroup: 2^24 and more of them
        assert L.vp_linear_fp8_fused(M, 8, 128, 1) == 0
    big = 1 << 29
    assert fp8_gemm(M=big, N=1024, ldo=1024) == unsupported
    assert fp8_gemm(M=big, N=1024, ldo=1024, act=1) == unsupported
    assert grouped('vp_grouped_fwd', T=1 << 30, N=136, ldo=136, E=2) == unsupported
    assert grouped('vp_grouped_dgrad', T=1 << 30, K=136, ldw=136, ldo=136, E=2) == unsupported
    assert grouped('vp_grouped_dgrad', T=1 << 30, K=136, ldw=136, N=520, ldy=520, ldo=136, E=2) == unsupported
    assert grouped('vp_grouped_wgrad', 64, 64, None, 0, T=8, E=1 << 24) == unsupported


def test_the_package_imports_on_a_torch_built_without_a_gpu():
    import os
    import subprocess
    import sys
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "from vitpose_amd import _lib, experts, fp8, optim\n"
            "optim.new_state8(128, 'cpu')\n"
            "experts.ExpertLinear(2, 16, 8)\n")
    run = subprocess.run([sys.executable, '-c', code], cwd=os.path.join(os.path.dirname(__file__), '..'), capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


def test_rows_that_require_a_gradient_are_refused_where_none_is_recorded():
    """(the tensors pass as far as the check: they say that they lie on a device)"""
    from vitpose_amd import experts, fp8

    class OnDevice(torch.Tensor):
        device = torch.device('cuda', 0)
        is_cuda = True

        def get_device(self):
            return 0

    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice).requires_grad_()
    x, w = t(8, 16), t(2, 8, 16)
    offsets, f = torch.zeros(3, dtype=torch.int32), t(16, dtype=torch.float32)
    for call in (lambda: fp8.quantize_rows(x), lambda: fp8.linear(x, x, x), lambda: fp8.layernorm_rows(t(8, 16, dtype=torch.float32), f, f),
                 lambda: experts.grouped_linear(x, w.detach(), None, offsets), lambda: experts.grouped_linear(x.detach(), w, None, offsets),
                 lambda: experts.grouped_linear_dgrad(t(8, 8), w.detach(), offsets), lambda: experts.grouped_linear_wgrad(t(8, 8), x.detach(), offsets)):
        with pytest.raises(RuntimeError, match='requires a gradient'):
            call()
    _lib.records_none(x.detach(), 'x', '')
    with torch.no_grad():
        _lib.records_none(x, 'x', '')


def record_fp8(monkeypatch, E, heads, B, **cfg):
    """Entry points and workspace of an evaluation plan on 8-bit products, recorded over host buffers (nothing runs)."""
    from vitpose_amd import engine, plan
    monkeypatch.setattr(plan, '_p', lambda t: None if t is None else t.data_ptr())
    cfg = dict(img_size=(256, 192), patch_size=16, in_chans=3, embed_dim=E, depth=1, num_heads=heads, mlp_ratio=4, qkv_bias=True, ratio=1, **cfg)
    vit, ws, recorded = engine.VitRunner(cfg, engine.ParamStore(engine.vit_param_shapes(cfg), 'cpu')), engine.Workspace('cpu'), plan.Plan()
    vit.record_forward(recorded, ws, torch.zeros(B, 3, 256, 192), B, training=False, fp8=True)
    return [c[0] for c in recorded.calls], ws.bufs


def test_channels_that_the_8_bit_layernorm_cannot_take_are_refused_when_the_plan_is_recorded(monkeypatch):
    with pytest.raises(ValueError, match='embed_dim 2112'):
        record_fp8(monkeypatch, 2112, 33, 1)
    assert 'vp_layernorm_fp8' in record_fp8(monkeypatch, 64, 2, 1)[0]


@pytest.mark.parametrize('B,few', [(2, True), (64, False)])
@pytest.mark.parametrize('routed', [False, True])
def test_an_8_bit_evaluation_holds_no_buffer_that_no_launch_touches(monkeypatch, B, few, routed):
    E, Hd, M = 128, 512, 192 * B
    calls, bufs = record_fp8(monkeypatch, E, 4, B, **(dict(num_expert=3, part_features=32) if routed else {}))
    assert (_lib.lib().vp_linear_fp8_fused(M, E, Hd, _lib.VP_BF16) == 1) == few
    assert calls.count('vp_gemm_fp8') == (2 if few or routed else 3)
    codes = not few and not routed
    assert ('h' in bufs) == (not codes) and ('fp8_hq' in bufs) == ('fp8_hs' in bufs) == codes
    width = Hd if few and not routed else E
    assert bufs['fp8_q'].numel() == M * width and bufs['fp8_s'].numel() == M * width // 128
    assert not codes or (bufs['fp8_hq'].numel() == M * Hd and bufs['fp8_hs'].numel() == M * Hd // 128)


def test_adamw8_takes_buffers_of_whole_fours():
    """Runs are multiples of 4 long: the last one of such a buffer, rounded up, would be skipped in silence."""
    assert adamw8(numel=126) == ERR_ARG and adamw8(numel=129, nchunks=0) == ERR_ARG and adamw8(numel=124, nchunks=0) == 0


def test_sizes_beyond_32_bits_are_refused_and_not_cut():
    """(tensors without memory that say they lie on a device: nothing is allocated, and nothing must be launched)"""
    from vitpose_amd import experts, fp8

    class OnDevice(torch.Tensor):
        device = torch.device('cuda', 0)
        is_cuda = True

        def get_device(self):
            return 0

    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device='meta').as_subclass(OnDevice)
    far, f8, f32, i32 = 2 ** 32 + 8, torch.float8_e4m3fn, torch.float32, torch.int32
    wq, ws = t(8, 128, dtype=f8), t(1, 1, dtype=f32)
    for call in (lambda: fp8.quantize_rows(t(far, 8)), lambda: fp8.quantize_rows(t(1, far)), lambda: fp8.quantize_weight(t(far, 8)),
                 lambda: fp8.linear(t(far, 8), wq, ws), lambda: fp8.product(t(far, 128, dtype=f8), t(1, far, dtype=f32), wq, ws),
                 lambda: fp8.product(t(4, 128, dtype=f8), t(1, 4, dtype=f32), t(far, 128, dtype=f8), t((far + 127) // 128, 1, dtype=f32)),
                 lambda: fp8.layernorm_rows(t(far, 8, dtype=f32), t(8, dtype=f32), t(8, dtype=f32)),
                 lambda: experts.expert_rows(t(far, dtype=i32), 4),
                 lambda: experts.grouped_linear(t(far, 8), t(2, 16, 8), None, t(3, dtype=i32)),
                 lambda: experts.grouped_linear(t(4, 8), t(2, far, 8), None, t(3, dtype=i32)),
                 lambda: experts.grouped_linear_dgrad(t(far, 16), t(2, 16, 8), t(3, dtype=i32)),
                 lambda: experts.grouped_linear_wgrad(t(far, 16), t(far, 8), t(3, dtype=i32)),
                 lambda: optim.adamw8_step(t(8, dtype=f32), t(8, dtype=f32), (t(128, dtype=f8), ws[0], t(128, dtype=f8), ws[0]),
                                           (t(far, dtype=torch.int64), t(far, dtype=i32), t(far, dtype=f32), t(far, dtype=f32), t(far, dtype=torch.int64)),
                                           lr=1e-3, step=1, noise=0)):
        with pytest.raises(ValueError, match='below 2'):
            call()


def test_rows_longer_than_32_bit_column_numbers_are_refused():
    """A tile's or a block's last column passes 2^31 where K nearly does."""
    far = (1 << 31) - 8
    for entry, more in (('vp_grouped_fwd', ()), ('vp_grouped_dgrad', ()), ('vp_grouped_wgrad', (64, 64, None, 0))):
        for over in (dict(K=far, ldx=far, ldw=far, ldo=far), dict(N=far, ldy=far, ldo=far)):
            assert grouped(entry, *more, T=1, E=1, **over) == ERR_ARG
    L = _lib.lib()
    assert L.vp_quantize_fp8_rows(64, 1, far, 1, far, 64, 64, None) == ERR_ARG
    assert L.vp_quantize_fp8_weight(64, 1, far, 1, far, 64, 64, None) == ERR_ARG
    wide = (1 << 30) + 128
    assert linear_fp8(K=wide, ldw=wide, k=wide, rows=wide) == ERR_ARG
    assert linear_fp8(K=128, ldw=(1 << 22) + 128) == ERR_ARG
