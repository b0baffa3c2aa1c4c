"""AdamW with 8-bit moments (vp_adamw8_step, optim.adamw8_step, FlatAdamW(state_bits=8)) against the update in 64 bits.

Tolerances, from the arithmetic (eps = 2^-24, half a step of f32):
* exp_avg' = m + (1 - b1)(g - m) may cancel, so its error goes by what is added: m is one rounding of a product (eps |m|), the
  difference and its product with 1 - b1 (itself rounded) are three of (1 - b1)(|g| + |m|) on top of what they inherit, the
  clipped g two, the sum one of |m'| <= |m| + |g|: together less than 4 eps (|m| + |g|) for b1 >= 0.5;
* weights: p (1 - lr wd) - rate m / (sqrt(v) / bc2 + eps): the decay is 3 roundings of values near p, the quotient that error of
  m and at most 16 roundings of values near the update (v 8 halved by the root, division and products 5), one for the
  difference;
* a code: exp_avg is off by half a spacing of e4m3 plus the f32 error of the value in front of it (8 roundings);
  sqrt(exp_avg_sq) is one of the two neighbours of its value, and the one its random number names unless that number is
  within 2^-17 of the border (32 roundings of numbers near x^2, a spacing of x^2 being at least x^2 / 8)."""
import ctypes
import math

import pytest
import torch

from vitpose_amd import _lib, optim

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
SIZES = [1, 3, 17, 64, 127, 128, 129, 1000, 2047, 2048, 2049, 5000]


def layout(sizes, lr_scales, decays):
    """(table, floats, state values): tensors at multiples of 64 as in ParamStore, their state at multiples of 128."""
    rows, at, sat = [], 0, 0
    for n, s, d in zip(sizes, lr_scales, decays):
        n4 = (n + 3) // 4 * 4
        for c in range(0, n4, 2048):
            rows.append((at + c, min(2048, n4 - c), s, d, sat + c))
        at += (n + 63) // 64 * 64
        sat += (n4 + 127) // 128 * 128
    cols = list(zip(*rows))
    kinds = (torch.int64, torch.int32, torch.float32, torch.float32, torch.int64)
    return tuple(torch.tensor(c, dtype=k) for c, k in zip(cols, kinds)), at, sat


def mix32(h):
    low = 0xFFFFFFFF
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & low
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & low
    return h ^ (h >> 16)


def exact_step(p, g, m, r, chunks, hyper, clip=1.0):
    """Per chunk, in 64 bits: (new p, m, v, the update, the error of m and what of it reaches the update)."""
    lr, (b1, b2), eps, t = hyper
    out = []
    for s, n, scale, wd, q in zip(*[c.tolist() for c in chunks]):
        gd, pd = g[s:s + n].double() * clip, p[s:s + n].double()
        mm = b1 * m[q:q + n] + (1 - b1) * gd
        v = b2 * r[q:q + n] ** 2 + (1 - b2) * gd * gd
        rate = lr * scale
        upd = rate / (1 - b1 ** t) * mm / ((v / (1 - b2 ** t)).sqrt() + eps)
        merr = 4 * EPS * (m[q:q + n].abs() + gd.abs())
        out.append((pd - rate * wd * pd - upd, mm, v, upd, merr, merr * rate / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + eps)))
    return out


def decode(state):
    m8, ms, r8, rs = [x.cpu() for x in state]
    return (m8.double().view(-1, 128) * ms.double()[:, None]).view(-1), (r8.double().view(-1, 128) * rs.double()[:, None]).view(-1)


def spacing(x):
    """Distance of e4m3 neighbours at |x|."""
    return torch.exp2((torch.frexp(x.abs())[1] - 1).clamp(min=-6).double() - 3)


def check(p0, g, st0, chunks, hyper, noise, clip, p1, half, st1):
    m0, r0 = decode(st0)
    m8, ms, r8, rs = [x.cpu() for x in st1]
    for (s, n, q), (pe, me, ve, upd, merr, uerr) in zip(zip(chunks[0].tolist(), chunks[1].tolist(), chunks[4].tolist()),
                                            exact_step(p0, g, m0, r0, chunks, hyper, clip)):
        tol = 4 * EPS * p0[s:s + n].abs().double() + 20 * EPS * upd.abs() + uerr + 1e-45
        assert ((p1[s:s + n].double() - pe).abs() <= tol).all()
        if half is not None:
            assert torch.equal(half[s:s + n], p1[s:s + n].bfloat16())
        for b in range(0, n, 128):
            i, j, blk = b, min(n, b + 128), (q + b) // 128
            amax, rmax = me[i:j].abs().max(), ve[i:j].max().sqrt()
            assert abs(ms[blk].double() - amax / 448) <= 4 * EPS * amax / 448 + merr[i:j].max() / 448 if amax >= 2.0 ** -99 else ms[blk] == 0
            assert abs(rs[blk].double() - rmax / 448) <= 12 * EPS * rmax / 448 if rmax >= 2.0 ** -99 else rs[blk] == 0
            if ms[blk] > 0:
                x = me[i:j] / ms[blk].double()
                err = (m8[q + i:q + j].double() - x).abs()
                assert (err <= spacing(x) / 2 + 8 * EPS * x.abs() + merr[i:j] / ms[blk].double()).all()
            if rs[blk] > 0:
                x = (ve[i:j].sqrt() / rs[blk].double()).clamp(max=448)
                lo = torch.floor(x / spacing(x)) * spacing(x)
                hi = lo + spacing(x)
                prob = (x * x - lo * lo) / (hi * hi - lo * lo)
                u = (mix32((torch.arange(q + i, q + j) & 0xFFFFFFFF) ^ noise) >> 8).double() * 2.0 ** -24
                want = torch.where(x > 0, torch.where(u < prob, hi, lo).clamp(2.0 ** -9, 448), torch.zeros_like(x))
                got = r8[q + i:q + j].double()
                sure = ((u - prob).abs() > 2.0 ** -17) & (prob > 2.0 ** -17) & (prob < 1 - 2.0 ** -17)
                assert torch.equal(got[sure], want[sure])
                near = (got - x).abs() <= spacing(x) * (1 + 2.0 ** -12)
                assert (near | ((x < 2.0 ** -9) & (got == 2.0 ** -9) & (x > 0)) | ((x == 0) & (got == 0))).all()


def make(sizes, seed, scales=None, state=True):
    gen = torch.Generator().manual_seed(seed)
    k = len(sizes)
    chunks, n, ns = layout(sizes, [0.75 ** (i % 5) for i in range(k)], [0.1 if i % 2 else 0.0 for i in range(k)])
    p, g = torch.zeros(n), torch.zeros(n)
    m, r = torch.zeros(ns), torch.zeros(ns)
    for s, ln, q in zip(chunks[0].tolist(), chunks[1].tolist(), chunks[4].tolist()):
        loud = 10 ** (torch.rand(1, generator=gen) * 6 - 7)
        p[s:s + ln] = torch.randn(ln, generator=gen) * 0.02
        g[s:s + ln] = torch.randn(ln, generator=gen) * loud
        m[q:q + ln] = torch.randn(ln, generator=gen) * loud
        r[q:q + ln] = torch.rand(ln, generator=gen) * loud
    st = optim.new_state8(ns, 'cpu')
    if state and ns:
        mb, rb = m.view(-1, 128), r.view(-1, 128)
        st[1].copy_(mb.abs().amax(1) / 448)
        st[3].copy_(rb.amax(1) / 448)
        st[0].copy_((mb / st[1].clamp(min=1e-30)[:, None]).view(-1))
        st[2].copy_((rb / st[3].clamp(min=1e-30)[:, None]).view(-1))
    return p, g, st, chunks


def on_gpu(*xs):
    return tuple(x.cuda() for x in xs)


def step(p, g, st, chunks, hyper, noise, half=True, **kw):
    lr, betas, eps, t = hyper
    pd, gd, std, chd = p.cuda(), g.cuda(), on_gpu(*st), on_gpu(*chunks)
    h = torch.zeros(p.numel(), dtype=torch.bfloat16, device='cuda') if half else None
    optim.adamw8_step(pd, gd, std, chd, lr=lr, betas=betas, eps=eps, step=t, noise=noise, half=h, **kw)
    return pd.cpu(), h.cpu() if half else None, std


HYPER = (3e-3, (0.9, 0.999), 1e-8, 7)


@pytest.mark.parametrize('sizes', [SIZES, [1], [2048], [2049], [100_003, 5, 40_000]])
@pytest.mark.parametrize('t', [1, 7, 100_000])
def test_step_matches_the_update_in_64_bits(sizes, t):
    hyper = (3e-3, (0.9, 0.999), 1e-8, t)
    p, g, st, chunks = make(sizes, 3, state=t > 1)
    noise = optim.noise_key(5, t)
    p1, half, st1 = step(p, g, st, chunks, hyper, noise)
    check(p, g, st, chunks, hyper, noise, 1.0, p1, half, st1)


@pytest.mark.parametrize('max_norm,scale', [(1e-3, 1.0), (1e6, 1.0), (0.5, 0.25)])
def test_step_clips_by_the_norm_of_the_table(max_norm, scale):
    p, g, st, chunks = make(SIZES, 4)
    # elements that no chunk covers (frozen tensors) stay out of the norm and keep what they hold
    keep = [i for i in range(chunks[0].numel()) if i not in (2, 6)]
    gone = [i for i in (2, 6)]
    table = tuple(c[keep].contiguous() for c in chunks)
    p1, half, st1 = step(p, g, st, table, HYPER, 9, max_grad_norm=max_norm, grad_scale=scale)
    norm = math.sqrt(sum(float(g[s:s + n].double().square().sum()) for s, n in zip(table[0].tolist(), table[1].tolist())))
    clip = scale * min(1.0, max_norm / (norm * scale + 1e-6))
    check(p, g, st, table, HYPER, 9, clip, p1, half, st1)
    for i in gone:
        s, n, q = int(chunks[0][i]), int(chunks[1][i]), int(chunks[4][i])
        assert torch.equal(p1[s:s + n], p[s:s + n]) and not half[s:s + n].any()
        assert torch.equal(st1[0].cpu().view(torch.uint8)[q:q + n], st[0].view(torch.uint8)[q:q + n])


def test_zero_gradients_and_empty_state_only_decay():
    p, g, st, chunks = make([300, 2048], 5, state=False)
    g.zero_()
    p1, half, st1 = step(p, g, st, chunks, HYPER, 1)
    check(p, g, st, chunks, HYPER, 1, 1.0, p1, half, st1)
    assert not any(x.cpu().view(torch.uint8).any() for x in st1)


def test_blocks_below_the_smallest_scale_are_stored_as_zeros():
    p, g, st, chunks = make([256], 6, state=False)
    g.fill_(1e-37)
    p1, half, st1 = step(p, g, st, chunks, HYPER, 1)
    m8, ms, r8, rs = st1
    assert not ms.any() and not m8.cpu().view(torch.uint8).any() and not rs.any() and torch.isfinite(p1).all()


def test_small_elements_of_a_block_keep_a_divisor():
    """A non-zero second moment never becomes zero, whatever its neighbours: no later step divides by eps alone."""
    p, g, st, chunks = make([128], 7, state=False)
    g.fill_(1e-9)
    g[0] = 10.0
    for noise in range(8):
        _, _, st1 = step(p, g, st, chunks, HYPER, noise)
        assert (st1[2].cpu().view(torch.uint8)[1:] == 1).all()


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_what_is_not_finite_marks_its_own_block(bad):
    p, g, st, chunks = make([640], 8)
    g[200] = bad
    p1, half, st1 = step(p, g, st, chunks, HYPER, 3)
    q, ok = 200 // 128, [0, 2, 3, 4]
    assert torch.isnan(st1[1][q]) and torch.isnan(st1[3][q])
    assert torch.isfinite(st1[1][ok]).all() and torch.isfinite(st1[3][ok]).all()
    assert not torch.isfinite(p1[200]) and torch.isfinite(p1[:200]).all() and torch.isfinite(p1[201:]).all()
    p2, _, _ = step(p, g, st, chunks, HYPER, 3, max_grad_norm=1.0)       # the norm carries it to every element
    assert not torch.isfinite(p2).any() if math.isnan(bad) else not torch.isfinite(p2[200])


def test_rounding_keeps_the_expected_second_moment():
    """Mean over keys of the decoded second moment = its exact value: 4096 independent draws of each element, five
    standard errors (a draw's deviation is at most half the distance of the neighbours' squares)."""
    p, g, st, chunks = make([256], 9)
    m0, r0 = decode(st)
    _, _, ve, *_ = exact_step(p, g, m0, r0, chunks, HYPER)[0]
    total, gd, chd = torch.zeros(256, dtype=torch.float64, device='cuda'), g.cuda(), on_gpu(*chunks)
    for k in range(4096):
        std = on_gpu(*st)
        optim.adamw8_step(p.cuda(), gd, std, chd, lr=1e-3, step=7, noise=optim.noise_key(1, k))
        total += ((std[2].double().view(-1, 128) * std[3].double()[:, None]) ** 2).view(-1)
    scale = std[3].cpu().double().repeat_interleave(128)
    x = ve.sqrt() / scale
    lo = torch.floor(x / spacing(x)) * spacing(x)
    width = ((lo + spacing(x)) ** 2 - lo ** 2) * scale ** 2
    fine = x >= 2.0 ** -9
    assert (((total.cpu() / 4096 - ve).abs() <= 5 * width / 2 / 64 + 1e-4 * width)[fine]).all()


def test_rows_of_the_table_that_leave_the_buffers_are_skipped():
    p, g, st, chunks = make([2048, 500], 10)
    table = [c.clone() for c in chunks]
    extra = [(p.numel() - 4, 8, 1.0, 0.0, 0), (-4, 4, 1.0, 0.0, 0), (0, 4, 1.0, 0.0, st[0].numel()), (2, 4, 1.0, 0.0, 0),
             (0, 4, 1.0, 0.0, 64), (0, 6, 1.0, 0.0, 0), (0, 4096, 1.0, 0.0, 0), (0, 0, 1.0, 0.0, 0)]
    wide = tuple(torch.cat([c, torch.tensor([e[i] for e in extra], dtype=c.dtype)]) for i, c in enumerate(table))
    a = step(p, g, st, chunks, HYPER, 2, max_grad_norm=1.0)
    b = step(p, g, st, wide, HYPER, 2, max_grad_norm=1.0)
    # (the norm of the longer table is added up by more workgroups: compare without the clip's last bit)
    torch.testing.assert_close(a[0], b[0], rtol=1e-6, atol=0)
    a, b = step(p, g, st, chunks, HYPER, 2), step(p, g, st, wide, HYPER, 2)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a[2], b[2]))


def test_same_inputs_same_bits_on_another_stream_and_in_a_replayed_graph():
    p, g, st, chunks = make(SIZES, 11)
    want = step(p, g, st, chunks, HYPER, 2, max_grad_norm=1e-2)
    gd, chd = g.cuda(), on_gpu(*chunks)
    pd, std = p.cuda(), on_gpu(*st)
    h = torch.zeros(p.numel(), dtype=torch.bfloat16, device='cuda')
    side = torch.cuda.Stream()
    lr, betas, eps, t = HYPER

    def call():
        optim.adamw8_step(pd, gd, std, chd, lr=lr, betas=betas, eps=eps, step=t, noise=2, half=h, max_grad_norm=1e-2)

    def same():
        assert torch.equal(pd.cpu(), want[0]) and torch.equal(h.cpu(), want[1])
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(std, want[2]))

    def reset():
        pd.copy_(p)
        for a, b in zip(std, st):
            a.copy_(b)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    same()
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        same()
        (gd * 2).sum().item()


def test_refusals():
    p, g, st, chunks = make([300], 12)
    pd, gd, std, chd = p.cuda(), g.cuda(), on_gpu(*st), on_gpu(*chunks)

    def call(param=pd, grad=gd, state=std, table=chd, **kw):
        optim.adamw8_step(param, grad, state, table, **{**dict(lr=1e-3, step=1, noise=0), **kw})
    with pytest.raises(RuntimeError):
        call(param=p)
    with pytest.raises(TypeError):
        call(param=pd.half())
    with pytest.raises(ValueError):
        call(grad=gd[:-1])
    with pytest.raises(ValueError):
        call(grad=g)
    with pytest.raises(ValueError):
        call(param=pd.view(-1, 2))
    with pytest.raises(ValueError):
        call(param=torch.zeros(640, device='cuda')[::2])
    with pytest.raises(ValueError):
        call(state=(std[0], std[1][:-1], std[2], std[3]))
    with pytest.raises(TypeError):
        call(state=(std[0].view(torch.uint8), std[1], std[2], std[3]))
    with pytest.raises(ValueError):
        call(state=(std[0][:-4], std[1], std[2][:-4], std[3]))
    with pytest.raises(TypeError):
        call(table=(chd[0].int(),) + chd[1:])
    with pytest.raises(ValueError):
        call(step=0)
    with pytest.raises(ValueError):
        call(betas=(1.0, 0.9))
    with pytest.raises(ValueError):
        call(noise=-1)
    with pytest.raises(TypeError):
        call(half=torch.zeros(pd.numel(), device='cuda'))
    with pytest.raises(RuntimeError):      # a buffer off its 16-byte boundary
        call(param=torch.zeros(pd.numel() + 1, device='cuda')[1:])


def _store(seed):
    from vitpose_amd.engine import ParamStore
    store = ParamStore([('backbone.blocks.0.w', (40, 33)), ('backbone.blocks.0.bias', (17,)), ('head.w', (130, 70)),
                        ('head.frozen', (50,))], 'cuda')
    gen = torch.Generator().manual_seed(seed)
    for n in store.names:
        store.view(n).copy_(torch.randn(store.shapes[n], generator=gen) * 0.1)
    store.half.copy_(store.data)
    return store


def _optimizer(store, **kw):
    groups = {n: dict(lr_scale=0.5 if 'backbone' in n else 1.0, weight_decay=0.0 if 'bias' in n else 0.1) for n in store.names}
    return optim.FlatAdamW(store, groups, lr=1e-2, max_grad_norm=1.0, frozen=['head.frozen'], **kw)


def test_flat_optimizer_follows_the_32_bit_one_and_resumes_bit_for_bit():
    stores = [_store(1) for _ in range(3)]
    opts = [_optimizer(stores[0]), _optimizer(stores[1], state_bits=8, noise_seed=4), _optimizer(stores[2], state_bits=8, noise_seed=4)]
    start = stores[0].data.clone()
    gen = torch.Generator().manual_seed(2)
    grads = [torch.randn(stores[0].numel, generator=gen) * 0.1 for _ in range(12)]

    def run(k, a, b):
        for i in range(a, b):
            stores[k].grad.copy_(grads[i])
            opts[k].step()
    run(0, 0, 12)
    run(1, 0, 12)
    run(2, 0, 5)
    saved = opts[2].state_dict()
    again = _optimizer(stores[2], state_bits=8)
    again.load_state_dict(saved)
    opts[2] = again
    run(2, 5, 12)
    assert torch.equal(stores[1].data, stores[2].data) and torch.equal(stores[1].half, stores[1].data.bfloat16())
    assert torch.equal(stores[1].view('head.frozen').cpu(), start[stores[1].offsets['head.frozen']:][:50].cpu())
    # the first step starts from exact (zero) moments: the same weights up to the clip factor's rounding; after that a
    # moment is off by at most half (exp_avg) and a whole (root of exp_avg_sq) spacing of an eighth, so an update is off by
    # less than 1 / 16 + 1 / 8 + their product of itself, for elements above a 2^-6 of their block's largest
    moved = (stores[0].data - start).double()
    off = (stores[1].data - stores[0].data).double()
    assert off.norm() < 0.2 * moved.norm()
    with pytest.raises(ValueError):
        opts[0].load_state_dict(saved)
    with pytest.raises(ValueError):
        opts[1].load_state_dict(opts[0].state_dict())
    saved['state']['head.w']['exp_avg'] = saved['state']['head.w']['exp_avg'][:-1]
    with pytest.raises(ValueError):
        opts[1].load_state_dict(saved)
    with pytest.raises(ValueError):
        _optimizer(stores[0], state_bits=16)


def test_flat_optimizer_first_step_equals_the_32_bit_one():
    a, b = _store(3), _store(3)
    x, y = _optimizer(a), _optimizer(b, state_bits=8)
    for s in (a, b):
        s.grad.copy_(torch.randn(s.numel, generator=torch.Generator().manual_seed(5)) * 1e-3)
    before = a.data.clone()
    x.step()
    y.step()
    # both compute the update in f32, 20 roundings each, from the same numbers
    tol = 4 * EPS * before.abs() + 40 * EPS * (a.data - before).abs() + 1e-12
    assert ((a.data - b.data).abs() <= tol).all()


def test_rows_whose_end_passes_64_bits_are_skipped():
    """A start next to 2^63: start + length is negative there, so the buffer's end has to be compared by differences."""
    p, g, st, chunks = make([2048, 500], 10)
    far = 2 ** 63
    extra = [(far - 4, 8, 1.0, 0.0, 0), (far - 2048, 2048, 1.0, 0.0, 0), (0, 4, 1.0, 0.0, far - 128), (0, 2048, 1.0, 0.0, far - 2048)]
    wide = tuple(torch.cat([c, torch.tensor([e[i] for e in extra], dtype=c.dtype)]) for i, c in enumerate(chunks))
    a, b = step(p, g, st, chunks, HYPER, 2), step(p, g, st, wide, HYPER, 2)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a[2], b[2]))
    only = tuple(c[-4:-2].contiguous() for c in wide)            # (those that the norm reads too)
    c = step(p, g, st, only, HYPER, 2, max_grad_norm=1.0)
    assert torch.equal(c[0], p)


@pytest.mark.parametrize('size', [1e-28, 1e-25, 1e-18, 1e-12, 1e19, 1e25, 1e36])
@pytest.mark.parametrize('eps', [1e-8, 0.0])
def test_gradients_of_any_size(size, eps):
    """What is kept is the ROOT of the second moment, so neither a gradient whose square leaves 32 bits nor eps = 0 makes a difference."""
    p, g, st, chunks = make([300, 2048, 5], 13, state=False)
    gen = torch.Generator().manual_seed(14)
    for t in (1, 2, 3):
        g = torch.zeros(g.numel())
        for s, n in zip(chunks[0].tolist(), chunks[1].tolist()):
            g[s:s + n] = (0.1 + torch.rand(n, generator=gen)) * (1 - 2 * torch.randint(0, 2, (n,), generator=gen)) * size
        hyper = (3e-3, (0.9, 0.999), eps, t)
        p1, half, st1 = step(p, g, st, chunks, hyper, t)
        check(p, g, st, chunks, hyper, t, 1.0, p1, half, st1)
        p, st = p1, tuple(x.cpu() for x in st1)


def test_without_eps_what_has_no_gradient_only_decays():
    hyper = (3e-3, (0.9, 0.999), 0.0, 1)
    p, g, st, chunks = make([300, 2048], 15, state=False)
    g.zero_()
    g[7] = 2.0
    p1, half, st1 = step(p, g, st, chunks, hyper, 1)
    assert torch.isfinite(p1).all()
    still = p.clone()
    still[320:] *= 1 - 0.75 * 3e-3 * 0.1            # (the second tensor's rate and decay)
    assert ((p1 - still).abs() <= 4 * EPS * p.abs())[torch.arange(p.numel()) != 7].all()
    # a gradient whose root of the second moment is below the smallest scale while its first moment is not: no trace of either is kept
    g.fill_(1e-29)
    p2, _, st2 = step(p1, g, optim.new_state8(st[0].numel(), 'cpu'), chunks, hyper, 2)
    p3, _, _ = step(p2, torch.zeros_like(g), tuple(x.cpu() for x in st2), chunks, (3e-3, (0.9, 0.999), 0.0, 2), 3)
    assert torch.isfinite(p3).all() and ((p3 - p2).abs() <= 10 * 3e-3 + p2.abs() * 1e-2).all()


def test_a_root_far_below_its_block_keeps_a_divisor_too():
    p, g, st, chunks = make([128], 16, state=False)
    g.fill_(1e-35)
    g[0] = 1e14
    _, _, st1 = step(p, g, st, chunks, HYPER, 1)
    assert (st1[2].cpu().view(torch.uint8)[1:] == 1).all()


def test_a_buffer_whose_last_run_would_leave_it_is_refused():
    p, g, st, chunks = make([2046], 17)
    cut = [x[:2046].cuda() for x in (p, g)]
    assert chunks[1].tolist() == [2048]
    with pytest.raises(ValueError, match='multiple of 4'):
        optim.adamw8_step(*cut, on_gpu(*st), on_gpu(*chunks), lr=1e-3, step=1, noise=0)
    cut = [x[:2048].cuda() for x in (p, g)]
    optim.adamw8_step(*cut, on_gpu(*st), on_gpu(*chunks), lr=1e-3, step=1, noise=0)
    assert not torch.equal(cut[0].cpu(), p[:2048])
