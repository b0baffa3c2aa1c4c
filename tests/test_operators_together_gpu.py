"""The 8-bit optimizer, the expert products and the 8-bit products in one program, as a user runs them: train an expert layer
one step and evaluate it on 8-bit operands; train a ViTPose one step with 8-bit moments and evaluate it with `fp8`.  Every
stage is compared in 64 bits on the inputs that the stage before it left.

Tolerances (U = 2^-24): a sum of n products is off by at most (n + 2) U of the sum of the magnitudes, a bf16 result by half a
step (2^-8) more; the first AdamW step moves a parameter by lr g / (|g| + eps) up to some twenty roundings, and the weight
decay adds four of the parameter's; what the 8-bit products lose between their codes and their result is derived in
test_fp8_gpu."""
import pytest
import torch

from test_fp8_gpu import check_layernorm, check_rounded, close, oracle as fp8_oracle
from test_model_gpu import TOY, make_engine, relerr

from oracle import vitpose_oracle as O
from vitpose_amd import fp8
from vitpose_amd.experts import ExpertLinear

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def within(got, want, tol, what):
    off = (got.detach().cpu().double() - want).abs()
    assert (off <= tol).all(), f'{what}: {(off / tol.clamp(min=1e-300)).max().item():.3g} of the bound'


def bound(n, mag, got, want):
    tol = (n + 4) * U * mag
    return tol + (2.0 ** -8 * (want.abs() + tol) if got.dtype == torch.bfloat16 else 0) + 1e-30


@pytest.mark.parametrize('T,E,K,Hd,N', [(1, 4, 64, 136, 64), (333, 6, 128, 264, 72)])
def test_an_expert_ffn_trains_a_step_and_answers_in_8_bits(T, E, K, Hd, N):
    from vitpose_amd.engine import ParamStore
    from vitpose_amd.optim import FlatAdamW
    g = torch.Generator().manual_seed(T + N)
    layers = [ExpertLinear(E, K, Hd), ExpertLinear(E, Hd, N)]
    shapes = [(f'fc{i + 1}.{n}', tuple(p.shape)) for i, m in enumerate(layers) for n, p in m.named_parameters()]
    store = ParamStore(shapes, 'cuda')
    for i, m in enumerate(layers):
        for n, p in list(m.named_parameters()):
            v = store.view(f'fc{i + 1}.{n}')
            v.copy_(torch.randn(p.shape, generator=g) * (0.05 if n == 'weight' else 0.5))
            setattr(m, n, torch.nn.Parameter(v))                # the layers' parameters are the flat buffer's
            getattr(m, n).grad = store.gview(f'fc{i + 1}.{n}')  # autograd adds to the flat gradients
    groups = {n: dict(lr_scale=1.0 if n.startswith('fc1') else 0.5, weight_decay=0.1 if n.endswith('weight') else 0.0) for n, _ in shapes}
    lr = 1e-2
    opt = FlatAdamW(store, groups, lr, max_grad_norm=1.0, state_bits=8, noise_seed=5)
    x = torch.randn(T, K, generator=g).bfloat16().cuda()
    expert = torch.randint(-1, E - 1, (T,), generator=g).int()  # some rows of no expert, one expert of no rows
    c = torch.randn(T, N, generator=g).bfloat16().cuda()
    ed = expert.cuda()

    h = layers[0](x, ed)
    h.retain_grad()
    a = torch.nn.functional.gelu(h)
    a.retain_grad()
    y = layers[1](a, ed)
    y.backward(c)

    on = expert >= 0
    pick = expert.clamp(min=0).long()
    onehot = torch.nn.functional.one_hot(pick, E).double() * on[:, None]
    for m, xin, out, dout, dx in ((layers[0], x, h, h.grad, None), (layers[1], a, y, c, a.grad)):
        W, b = m.weight.detach().bfloat16().cpu().double(), m.bias.detach().cpu().double()
        xd, dd = xin.detach().cpu().double(), dout.cpu().double()
        n = xd.shape[1]
        want = (torch.einsum('tk,tnk->tn', xd, W[pick]) + b[pick]) * on[:, None]
        mag = (torch.einsum('tk,tnk->tn', xd.abs(), W[pick].abs()) + b[pick].abs()) * on[:, None]
        within(out, want, bound(n, mag, out, want), 'forward')
        if dx is not None:
            want = torch.einsum('tn,tnk->tk', dd, W[pick]) * on[:, None]
            mag = torch.einsum('tn,tnk->tk', dd.abs(), W[pick].abs()) * on[:, None]
            within(dx, want, bound(dd.shape[1], mag, dx, want), 'gradient of the rows')
        want, mag = (torch.einsum('te,tn,tk->enk', onehot, p, q) for p, q in ((dd, xd), (dd.abs(), xd.abs())))
        within(m.weight.grad, want, bound(T, mag, m.weight.grad, want), 'gradient of the weights')
        want, mag = (torch.einsum('te,tn->en', onehot, p) for p in (dd, dd.abs()))
        within(m.bias.grad, want, bound(T, mag, m.bias.grad, want), 'gradient of the biases')
        assert not m.weight.grad[E - 1].any() and not m.bias.grad[E - 1].any()
    assert not y[~on.cuda()].any()

    before, grads = store.data.clone(), store.grad.clone()
    norm = min(1.0, 1.0 / (grads.double().norm().item() + 1e-6))
    opt.step()
    for name, _ in shapes:
        p, q, gr = (store._v(t, name).cpu().double() for t in (before, store.data, grads))
        step = lr * groups[name]['lr_scale']
        upd = step * gr * norm / ((gr * norm).abs() + 1e-8)
        want = p * (1 - step * groups[name]['weight_decay']) - upd
        within(q, want, 4 * U * p.abs() + 40 * U * upd.abs() + 1e-30, f'step of {name}')
        assert torch.equal(store.hview(name), store.view(name).bfloat16())
    for _ in range(2):                                          # gradients stay: later steps read the 8-bit moments
        opt.step()
    assert torch.isfinite(store.data).all()

    # the trained layer on 8-bit operands: one Linear per expert over its rows
    for e in range(E):
        rows = (expert == e).nonzero()[:, 0]
        wq, ws = fp8.quantize_weight(layers[0].weight.detach()[e])
        xe = x[rows.cuda()]
        got = fp8.linear(xe, wq, ws, layers[0].bias.detach()[e], act='gelu')
        assert got.shape == (len(rows), Hd)
        if len(rows):
            xq, xs = fp8.quantize_rows(xe)
            close(got, *fp8_oracle(xq, xs, wq, ws, layers[0].bias.detach()[e].cpu()), wq.shape[1], 'gelu')


@pytest.mark.parametrize('B', [2, 24])
def test_a_vit_trained_with_8_bit_moments_evaluates_on_8_bit_products(B):
    hc = O.classic_head_cfg(64)
    eng = make_engine(TOY, hc, O.synth_vit_weights(TOY, seed=1), O.synth_head_weights(hc, seed=2), 'cuda:0')
    img, target, tw = O.synth_batch(B, seed=3)
    img = img.cuda()
    old = eng.infer(img, fp8=True)
    eng.setup_optimizer(lr=1e-3, state_bits=8, noise_seed=1)
    eng.forward_backward(img[:2], target[:2].cuda(), tw[:2].cuda())
    eng.optimizer_step()
    heat = eng.infer(img, fp8=True)
    assert not torch.equal(heat, old) and eng.optimizer.step_count == 1

    # the step's weights are the ones that were rounded
    weights = eng.vit._fp8[0]
    assert len(weights) == 4 * TOY['depth']
    for name, (wq, ws) in weights.items():
        q, s = fp8.quantize_weight(eng.store.view('backbone.' + name + '.weight'))
        assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, ws)

    # call by call: what the LayerNorms and the 8-bit products got and gave
    plan, _, out = eng.plans[('infer', B, 'fp8')]
    buf, vit = eng.ws_infer.bufs, eng.vit
    E, M, Hd = TOY['embed_dim'], B * 192, 4 * TOY['embed_dim']
    rows = lambda q, s, K: (buf[q][:M * -(-K // 128) * 128].view(M, -1).view(torch.float8_e4m3fn).clone(),  # noqa: E731
                            buf[s][:M * -(-K // 128)].view(-1, M).clone())
    few = bool(plan.L.vp_linear_fp8_fused(M, E, Hd, 1))
    stages = [('norm1', 'x_a'), ('attn.qkv', 'qkv', None), ('attn.proj', 'x_b', 'x_a'), ('norm2', 'x_b'),
              ('mlp.fc1', 'h' if few else None, None), ('mlp.fc2', 'x_a', 'x_b')]
    seen, codes = 0, None
    for i, (entry, _, _) in enumerate(plan.calls):
        if not entry.endswith('_fp8'):
            plan.run(i, i + 1)
            continue
        block, stage = divmod(seen, 6)
        name, dst = f'blocks.{block}.' + stages[stage][0], stages[stage][1]
        if 'norm' in name:
            x = buf[dst].cpu().double()
            plan.run(i, i + 1)
            codes = rows('fp8_q', 'fp8_s', E)
            check_layernorm(x, vit.w(name + '.weight').cpu(), vit.w(name + '.bias').cpu(), *codes)
        else:
            r = buf[stages[stage][2]].cpu().double() if stages[stage][2] else 0.0
            if entry == 'vp_linear_fp8':
                codes = fp8.quantize_rows(buf['ao' if 'proj' in name else 'h'])
            plan.run(i, i + 1)
            wq, ws = weights[name]
            want, mag = fp8_oracle(*codes, wq, ws, vit.w(name + '.bias').cpu())
            want, mag = want + r, mag + (r.abs() if stages[stage][2] else 0.0)
            if dst is None:
                codes = rows('fp8_hq', 'fp8_hs', Hd)
                check_rounded(want, mag, wq.shape[1], *codes, act='gelu')
            else:
                assert buf[dst].dtype == (torch.float32 if stages[stage][2] else torch.bfloat16)
                close(buf[dst], want, mag, wq.shape[1], 'gelu' if 'fc1' in name else None)
        seen += 1
    assert seen == 6 * TOY['depth'] and torch.equal(out, heat)
    # the same network: every operand is off by 3 % in the mean, which is some 5 % of a Linear's result; a wrong scale, a lost
    # residual or a skipped Linear is of the size of the maps themselves
    rel = relerr(heat, eng.infer(img))[0]
    print(f'heat maps on 8-bit products against bf16: {rel:.3f}')
    assert rel < 0.25
    with pytest.raises(ValueError):
        eng.infer(img, fp8=True, exact=True)
    with pytest.raises(ValueError):
        eng.infer(img, fp8=True, fold_ln=True)
    assert eng.infer(img[:1], fp8=True).shape[0] == 1
    # an engine set to 8 bits still takes another path where a call names it
    eng.fp8 = True
    want = [eng.infer(img, fp8=False, fold_ln=True), eng.infer(img, fp8=False), eng.infer(img, fp8=False, exact=True)]
    assert torch.equal(eng.infer(img, fold_ln=True), want[0]) and torch.equal(eng.infer(img, exact=True), want[2])
    assert torch.equal(eng.infer(img), heat) and not torch.equal(heat, want[1])


def test_test_cfg_chooses_8_bit_products_and_refuses_two_paths_at_once():
    import vitpose_amd.models  # noqa: F401
    from vitpose_amd.builder import build_posenet
    hc = O.classic_head_cfg(64)

    def model(**cfg):
        torch.manual_seed(0)
        return build_posenet(dict(type='TopDown', backbone=dict(TOY, type='ViT'),
                                  keypoint_head=dict(hc, type='TopdownHeatmapSimpleHead', loss_keypoint=dict(type='JointsMSELoss', use_target_weight=True)),
                                  train_cfg=dict(), test_cfg=dict(flip_test=False, post_process='default', shift_heatmap=False,
                                                                  use_udp=False, **cfg))).to('cuda').eval()
    img = O.synth_batch(2, seed=3)[0].cuda()
    with torch.no_grad():
        m = model(fp8=True)
        heat = m.forward_dummy(img)
        assert ('infer', 2, 'fp8') in m._engine.plans and ('infer', 2) not in m._engine.plans
        assert torch.equal(heat, m._engine.infer(img, fp8=True))
        assert not torch.equal(heat, m._engine.infer(img, fp8=False)) and ('infer', 2) in m._engine.plans
        for other in ('fp32_exact', 'fold_layernorm'):
            with pytest.raises(ValueError):
                model(fp8=True, **{other: True}).forward_dummy(img)


def test_a_routed_vit_evaluates_on_8_bit_products():
    """ViTMoE: the routed fc2 keeps its bf16 product, the other three Linears of a Block are 8-bit ones."""
    cfg = dict(TOY, num_expert=3, part_features=16)
    hc = O.classic_head_cfg(64)
    from vitpose_amd.pose_engine import PoseEngine
    eng = PoseEngine(cfg, hc, 'cuda:0')
    g = torch.Generator().manual_seed(7)
    eng.load_state_dict({n: (0.1 * torch.randn(s, generator=g) + (1.0 if 'norm' in n and n.endswith('weight') else 0.0))
                         for n, s in eng.named_shapes()}, strict=False)
    img = O.synth_batch(3, seed=3)[0].cuda()
    heat = eng.infer(img, fp8=True, dataset_source=[0, 2, 1])
    names = [c[0] for c in eng.plans[('infer', 3, 'fp8')][0].calls]
    assert sum(n in ('vp_linear_fp8', 'vp_gemm_fp8') for n in names) == 3 * TOY['depth']
    assert relerr(heat, eng.infer(img, dataset_source=[0, 2, 1]))[0] < 0.25
    assert not torch.equal(heat, eng.infer(img, fp8=True, dataset_source=[0, 1, 1]))
