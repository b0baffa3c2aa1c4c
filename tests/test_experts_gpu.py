"""Expert products (vp_expert_rows, vp_grouped_*, vitpose_amd.experts) against sums in 64 bits.

Tolerances: a sum of n products in f32 is off by at most (n + 2) 2^-24 of the sum of their magnitudes, in any order; a bf16
result by half a step more, 2^-8 of itself.  Products of small whole numbers whose sums stay below 2^8 are exact in both."""
import pytest
import torch

from vitpose_amd import experts

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def routing(T, E, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == 'even':
        ids = torch.arange(T) % E
    elif kind == 'one':
        ids = torch.full((T,), E - 1)
    elif kind == 'gaps':              # every other expert without a row, some rows without an expert
        ids = torch.randint(0, E, (T,), generator=g) // 2 * 2
        ids[torch.rand(T, generator=g) < 0.1] = -1
        ids[torch.rand(T, generator=g) < 0.05] = E + 3
    else:                             # most rows at the first experts
        ids = (torch.rand(T, generator=g) ** 4 * E).long().clamp(max=E - 1)
    return ids[torch.randperm(T, generator=g)].int()


def lists(ids, E):
    key = torch.where((ids >= 0) & (ids < E), ids, torch.full_like(ids, E))
    order = torch.sort(key, stable=True).indices.int()
    count = torch.bincount(key.long(), minlength=E + 1)[:E]
    return order, torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]).int()


def oracle(x, w, b, dy, ids):
    """(y, dx, dw, db) in 64 bits and the sums of magnitudes behind them."""
    x, w, dy = x.double(), w.double(), dy.double()
    E = w.shape[0]
    y, ya = torch.zeros(2, x.shape[0], w.shape[1], dtype=torch.float64)
    dx, dxa = torch.zeros(2, *x.shape, dtype=torch.float64)
    dw, dwa = torch.zeros(2, *w.shape, dtype=torch.float64)
    db, dba = torch.zeros(2, E, w.shape[1], dtype=torch.float64)
    for e in range(E):
        m = (ids == e).nonzero().flatten()
        if m.numel():
            y[m], ya[m] = x[m] @ w[e].t(), x[m].abs() @ w[e].abs().t()
            if b is not None:
                y[m] += b[e].double()
                ya[m] += b[e].double().abs()
            dx[m], dxa[m] = dy[m] @ w[e], dy[m].abs() @ w[e].abs()
            dw[e], dwa[e] = dy[m].t() @ x[m], dy[m].abs().t() @ x[m].abs()
            db[e], dba[e] = dy[m].sum(0), dy[m].abs().sum(0)
    return (y, dx, dw, db), (ya, dxa, dwa, dba)


def close(got, want, mags, n, what):
    tol = (n + 2) * U * mags + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0)
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= tol).all(), f'{what}: worst {((off - tol) / (tol + 1e-300)).max().item():.3g} over the bound at {(off - tol).argmax().item()}'


CASES = [
    # T, E, K, N, routing
    (1, 1, 8, 8, 'even'), (1, 6, 1536, 96, 'one'), (2, 5, 64, 16, 'even'), (7, 3, 72, 24, 'gaps'), (64, 4, 128, 64, 'even'),
    (65, 2, 136, 72, 'one'), (128, 1, 64, 128, 'even'), (129, 8, 200, 136, 'skewed'), (192, 6, 1024, 256, 'gaps'),
    (300, 64, 96, 40, 'even'), (333, 100, 64, 64, 'skewed'), (600, 512, 40, 24, 'even'), (1000, 6, 1280, 320, 'skewed'),
    (1537, 3, 264, 200, 'gaps'), (2048, 1, 72, 8, 'even'), (5003, 24, 88, 104, 'gaps'), (9000, 2, 64, 64, 'skewed'),
    (40000, 7, 16, 8, 'gaps'),
]


def data(T, E, K, N, seed, whole=False):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s):
        if whole:
            return torch.randint(-1, 2, s, generator=g).bfloat16()
        return (torch.randn(*s, generator=g) * torch.exp(torch.randn(s[-1], generator=g))).bfloat16()
    return rnd(T, K), rnd(E, N, K), torch.randn(E, N, generator=g), rnd(T, N)


@pytest.mark.parametrize('T,E,K,N,kind', CASES)
def test_rows_are_ordered_by_expert(T, E, K, N, kind):
    ids = routing(T, E, kind, T)
    rows, offsets = experts.expert_rows(ids.cuda(), E)
    order, offs = lists(ids, E)
    assert torch.equal(offsets.cpu(), offs) and torch.equal(rows.cpu(), order)


def test_rows_of_none_and_of_one():
    rows, offsets = experts.expert_rows(torch.empty(0, dtype=torch.int32, device='cuda'), 3)
    assert rows.numel() == 0 and offsets.tolist() == [0, 0, 0, 0]
    rows, offsets = experts.expert_rows(torch.tensor([-7], dtype=torch.int32, device='cuda'), 2)
    assert rows.tolist() == [0] and offsets.tolist() == [0, 0, 0]


@pytest.mark.parametrize('T,E,K,N,kind', CASES)
@pytest.mark.parametrize('listed', [True, False])
def test_products_match_sums_in_64_bits(T, E, K, N, kind, listed):
    ids = routing(T, E, kind, T + 1)
    x, w, b, dy = data(T, E, K, N, T + 2)
    order, offsets = lists(ids, E)
    if not listed:                    # the arrays lie in the order of the experts; rows of no expert last
        ids = ids[order.long()]
        rows = None
    else:
        rows = order.cuda()
    offsets = offsets.cuda()
    (y, dx, dw, db), (ya, dxa, dwa, dba) = oracle(x, w, b, dy, ids)
    xd, wd, bd, dyd = x.cuda(), w.cuda(), b.cuda(), dy.cuda()
    got_dw, got_db = experts.grouped_linear_wgrad(dyd, xd, offsets, rows)
    n = int(torch.bincount(ids[(ids >= 0) & (ids < E)].long(), minlength=E).max())
    close(experts.grouped_linear(xd, wd, bd, offsets, rows), y, ya, K + 1, 'y')
    close(experts.grouped_linear(xd, wd, None, offsets, rows), oracle(x, w, None, dy, ids)[0][0], ya, K, 'y without bias')
    close(experts.grouped_linear_dgrad(dyd, wd, offsets, rows), dx, dxa, N, 'dx')
    close(got_dw, dw, dwa, n, 'dw')
    close(got_db, db, dba, n, 'db')
    again = experts.grouped_linear_wgrad(dyd, xd, offsets, rows)
    assert torch.equal(again[0], got_dw) and torch.equal(again[1], got_db)


@pytest.mark.parametrize('T,E,K,N,kind', [c for c in CASES if c[2] <= 256 and c[3] <= 256])
def test_whole_numbers_come_out_exactly(T, E, K, N, kind):
    """Also the test against differences: y is linear in x, so <dy, y(x + d) - y(x)> = <dx, d>, to the last bit here."""
    ids = routing(T, E, kind, T + 3)
    x, w, _, dy = data(T, E, K, N, T + 4, whole=True)
    d = data(T, E, K, N, T + 5, whole=True)[0]
    x = torch.where(d == 1, x.clamp(max=0), torch.where(d == -1, x.clamp(min=0), x))     # x + d stays in -1, 0, 1
    rows, offsets = experts.expert_rows(ids.cuda(), E)
    (y, dx, dw, db), _ = oracle(x, w, None, dy, ids)
    xd, wd, dyd = x.cuda(), w.cuda(), dy.cuda()
    got = experts.grouped_linear(xd, wd, None, offsets, rows)
    gx = experts.grouped_linear_dgrad(dyd, wd, offsets, rows)
    gw, gb = experts.grouped_linear_wgrad(dyd, xd, offsets, rows)
    assert torch.equal(got.cpu().double(), y) and torch.equal(gx.cpu().double(), dx)
    assert torch.equal(gw.cpu().double(), dw) and torch.equal(gb.cpu().double(), db)
    moved = experts.grouped_linear((x + d).cuda(), wd, None, offsets, rows)
    assert ((moved.double() - got.double()) * dyd.double()).sum() == (gx.double() * d.cuda().double()).sum()


def test_what_lies_beside_the_operands_does_not_enter():
    """Padding behind a row, rows without an expert and experts without a row hold NaN; given results keep the rows that
    nobody computes."""
    T, E, K, N = 203, 5, 72, 40
    ids = routing(T, E, 'gaps', 1)
    x, w, b, dy = data(T, E, K, N, 2)
    (y, dx, dw, db), (ya, dxa, dwa, dba) = oracle(x, w, b, dy, ids)
    nan = float('nan')

    def wide(t, pad):
        buf = torch.full((*t.shape[:-1], t.shape[-1] + pad), nan, dtype=t.dtype, device='cuda')
        buf[..., :t.shape[-1]] = t.cuda()
        return buf[..., :t.shape[-1]]
    gone = (ids < 0) | (ids >= E)
    x[gone], dy[gone] = nan, nan
    for e in range(E):
        if not (ids == e).any():
            w[e], b[e] = nan, nan
    xd, wd, bd, dyd = wide(x, 8), wide(w, 24), wide(b, 4), wide(dy, 16)
    rows, offsets = experts.expert_rows(ids.cuda(), E)
    close(experts.grouped_linear(xd, wd, bd, offsets, rows), y, ya, K + 1, 'y')
    close(experts.grouped_linear_dgrad(dyd, wd, offsets, rows), dx, dxa, N, 'dx')
    gw, gb = experts.grouped_linear_wgrad(dyd, xd, offsets, rows)
    close(gw, dw, dwa, T, 'dw')
    close(gb, db, dba, T, 'db')
    assert experts.grouped_linear_wgrad(dyd, xd, offsets, rows, want_bias=False)[1] is None
    for call, src, want, cols in ((experts.grouped_linear, xd, y, N), (experts.grouped_linear_dgrad, dyd, dx, K)):
        buf = torch.full((T, cols + 8), 7.0, dtype=torch.bfloat16, device='cuda')
        args = (src, wd, bd, offsets, rows) if call is experts.grouped_linear else (src, wd, offsets, rows)
        assert call(*args, out=buf[:, :cols]).data_ptr() == buf.data_ptr()
        kept = buf.cpu()
        assert (kept[:, cols:] == 7).all() and (kept[gone] == 7).all()
        assert not (kept[~gone][:, :cols] == 7).all()


def test_lists_and_offsets_that_leave_the_arrays_are_cut():
    T, E, K, N = 100, 3, 64, 16
    x, w, b, dy = data(T, E, K, N, 3, whole=True)
    xd, wd, dyd = x.cuda(), w.cuda(), dy.cuda()
    rows = torch.arange(T, dtype=torch.int32)
    rows[5], rows[70] = -4, T + 9
    offsets = torch.tensor([-3, 40, 20, 400], dtype=torch.int32)       # expert 1 has no rows, expert 2 has 20..99
    ids = torch.full((T,), -1)
    ids[0:40] = 0
    ids[20:100] = 2                                                    # rows 20..39 belong to experts 0 and 2: not compared
    ids[5], ids[70] = -1, -1
    clean = torch.ones(T, dtype=torch.bool)
    clean[20:40] = False
    (y, dx, dw, db), _ = oracle(x, w, None, dy, ids)
    got = experts.grouped_linear(xd, wd, None, offsets.cuda(), rows.cuda(), out=torch.zeros(T, N, dtype=torch.bfloat16, device='cuda'))
    gx = experts.grouped_linear_dgrad(dyd, wd, offsets.cuda(), rows.cuda(), out=torch.zeros(T, K, dtype=torch.bfloat16, device='cuda'))
    gw, gb = experts.grouped_linear_wgrad(dyd, xd, offsets.cuda(), rows.cuda())
    assert torch.equal(got.cpu().double()[clean], y[clean]) and torch.equal(gx.cpu().double()[clean], dx[clean])
    assert torch.equal(gw[2].cpu().double(), dw[2]) and torch.equal(gb[2].cpu().double(), db[2]) and not gw[1].any()


def test_no_rows_at_all():
    w = torch.ones(3, 16, 24, dtype=torch.bfloat16, device='cuda')
    offsets = torch.zeros(4, dtype=torch.int32, device='cuda')
    x, dy = torch.empty(0, 24, dtype=torch.bfloat16, device='cuda'), torch.empty(0, 16, dtype=torch.bfloat16, device='cuda')
    assert experts.grouped_linear(x, w, None, offsets).shape == (0, 16)
    assert experts.grouped_linear_dgrad(dy, w, offsets).shape == (0, 24)
    dw, db = experts.grouped_linear_wgrad(dy, x, offsets)
    assert dw.shape == (3, 16, 24) and not dw.any() and not db.any()
    # rows, but none with an expert
    x = torch.full((9, 24), float('nan'), dtype=torch.bfloat16, device='cuda')
    assert not experts.grouped_linear(x, w, None, offsets).any()


def test_weights_inside_a_flat_buffer():
    """Experts of one layer as ParamStore keeps them: weight and bias of an expert in turn, every tensor at a multiple of
    64 elements."""
    T, E, K, N = 150, 4, 72, 24
    ids = routing(T, E, 'skewed', 5)
    x, w, b, dy = data(T, E, K, N, 6)
    step = (N * K + 63) // 64 * 64 + 64
    flat = torch.full((E * step,), float('nan'), device='cuda')
    for e in range(E):
        flat[e * step:e * step + N * K] = w[e].float().flatten().cuda()
        flat[e * step + step - 64:e * step + step - 64 + N] = b[e].cuda()
    half = flat.bfloat16()
    wv = half.as_strided((E, N, K), (step, K, 1))
    bv = flat.as_strided((E, N), (step, 1), step - 64)
    rows, offsets = experts.expert_rows(ids.cuda(), E)
    (y, dx, _, _), (ya, dxa, _, _) = oracle(x, w, b, dy, ids)
    close(experts.grouped_linear(x.cuda(), wv, bv, offsets, rows), y, ya, K + 1, 'y')
    close(experts.grouped_linear_dgrad(dy.cuda(), wv, offsets, rows), dx, dxa, N, 'dx')


def test_another_stream_and_replayed_graphs_with_new_routing():
    T, E, K, N = 500, 6, 128, 64
    x, w, b, dy = [t.cuda() for t in data(T, E, K, N, 7, whole=True)]
    ids = [routing(T, E, k, 8).cuda() for k in ('even', 'gaps', 'one')]
    static = ids[0].clone()

    def call():
        rows, offsets = experts.expert_rows(static, E)
        return (experts.grouped_linear(x, w, None, offsets, rows), experts.grouped_linear_dgrad(dy, w, offsets, rows),
                *experts.grouped_linear_wgrad(dy, x, offsets, rows))
    want = []
    for i in ids:
        static.copy_(i)
        want.append([t.clone() for t in call()])
    side = torch.cuda.Stream()
    static.copy_(ids[1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want[1]))
    graphs = []
    for _ in range(2):                 # two graphs of the same calls: nothing of theirs is shared
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for k in (2, 0, 1):
        static.copy_(ids[k])
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = call()
        for _, out in graphs:
            assert all(torch.equal(a, c) and torch.equal(a, d) for a, c, d in zip(out, want[k], eager))


def test_expert_linear_and_its_gradients():
    T, E, K, N = 257, 5, 64, 48
    torch.manual_seed(3)
    layer = experts.ExpertLinear(E, K, N, device='cuda')
    ids = routing(T, E, 'gaps', 9)
    x, _, _, dy = data(T, E, K, N, 10)
    xd = x.cuda().requires_grad_()
    y = layer(xd, ids.cuda())
    y.backward(dy.cuda())
    w, b = layer.weight.detach().bfloat16().cpu(), layer.bias.detach().cpu()
    (ye, dx, dw, db), (ya, dxa, dwa, dba) = oracle(x, w, b, dy, ids)
    close(y.detach(), ye, ya, K + 1, 'y')
    close(xd.grad, dx, dxa, N, 'dx')
    close(layer.weight.grad, dw, dwa, T, 'dw')
    close(layer.bias.grad, db, dba, T, 'db')
    # the gradient of a sum reaches the kernel as one expanded value; weights that changed are seen at once
    layer.zero_grad()
    with torch.no_grad():
        layer.weight.mul_(2.0)
    y2 = layer(xd, ids.cuda())
    y2.sum().backward()
    (ye, _, dw, _), (ya, _, dwa, _) = oracle(x, layer.weight.detach().bfloat16().cpu(), b, torch.ones(T, N), ids)
    close(y2.detach(), ye, ya, K + 1, 'y')
    close(layer.weight.grad, dw, dwa, T, 'dw')
    frozen = experts.ExpertLinear(E, K, N, bias=False, device='cuda').requires_grad_(False)
    x3 = x.cuda().requires_grad_()
    frozen(x3, ids.cuda()).backward(dy.cuda())
    assert x3.grad is not None and frozen.weight.grad is None


def test_refusals():
    T, E, K, N = 32, 3, 64, 16
    x, w, b, dy = [t.cuda() for t in data(T, E, K, N, 11)]
    rows, offsets = experts.expert_rows(routing(T, E, 'even', 1).cuda(), E)
    ok = (x, w, b, offsets, rows)

    def swap(i, v):
        return tuple(v if k == i else t for k, t in enumerate(ok))
    for bad in (swap(0, x.float()), swap(1, w.float())):
        with pytest.raises(TypeError):
            experts.grouped_linear(*bad)
    for bad in (swap(0, x[:, :-8]), swap(0, x[0]), swap(0, x[:, 1:57]), swap(1, w[0]), swap(1, w[:, :12]), swap(2, b.bfloat16()),
                swap(2, b[:2]), swap(3, offsets[:-1]), swap(3, offsets.long()), swap(4, rows[:-1]), swap(4, rows.long()),
                swap(0, x.t().contiguous().t())):
        with pytest.raises(ValueError):
            experts.grouped_linear(*bad)
    for bad in (swap(0, x.cpu()), swap(1, w.cpu())):
        with pytest.raises(RuntimeError):
            experts.grouped_linear(*bad)
    with pytest.raises(ValueError):
        experts.grouped_linear(*ok, out=torch.empty(T, N + 8, dtype=torch.bfloat16, device='cuda'))
    with pytest.raises(ValueError):
        experts.grouped_linear_dgrad(x, w, offsets, rows)
    with pytest.raises(ValueError):
        experts.grouped_linear_wgrad(dy[:-1], x, offsets, rows)
    with pytest.raises(ValueError):
        experts.expert_rows(rows.long(), 3)
    for n in (0, 513):
        with pytest.raises(ValueError):
            experts.expert_rows(rows, n)


def test_a_gradient_off_its_sixteen_bytes_and_a_layer_without_bias():
    """autograd may hand over any contiguous view; a layer whose input needs no gradient still gets its weights'."""
    g = torch.Generator().manual_seed(3)
    layer = experts.ExpertLinear(3, 16, 8, bias=False, device='cuda')
    x = torch.randn(5, 16, generator=g).bfloat16().cuda()
    e = torch.tensor([2, 0, 2, 1, -1], dtype=torch.int32).cuda()
    flat = torch.randn(5 * 8 + 1, generator=g).bfloat16().cuda()
    dy = flat[1:].view(5, 8)
    assert dy.data_ptr() % 16
    y = layer(x, e)
    y.backward(dy)
    want = torch.zeros(3, 8, 16, dtype=torch.float64)
    for t, k in enumerate(e.tolist()):
        if k >= 0:
            want[k] += dy[t].cpu().double()[:, None] * x[t].cpu().double()
    # two products of bf16 numbers at most are added in f32
    assert (layer.weight.grad.cpu().double() - want).abs().max() <= 4 * 2.0 ** -24 * 16


@pytest.mark.parametrize('T,E,K,N,listed', [(5003, 8, 72, 1024, True), (12300, 6, 40, 320, False), (16384, 3, 136, 256, True), (9001, 1, 64, 520, True),
                                            (6144, 6, 72, 320, True), (6100, 5, 200, 312, False), (9000, 6, 40, 192, True),
                                            (2500, 6, 136, 256, True), (12288, 6, 40, 256, False)])
def test_forward_products_of_many_rows(T, E, K, N, listed):
    """Row counts at which the 64-, 128- and 192-row tiles take turns."""
    g = torch.Generator().manual_seed(T)
    x, w, b = torch.randn(T, K, generator=g).bfloat16(), torch.randn(E, N, K, generator=g).bfloat16(), torch.randn(E, N, generator=g)
    ids = torch.randint(-1, E, (T,), generator=g).int()
    ids[torch.rand(T, generator=g) < 0.4] = 0
    if not listed:
        ids = ids.clamp(min=0).sort()[0].int()
    rows, offsets = experts.expert_rows(ids.cuda(), E)
    got = experts.grouped_linear(x.cuda(), w.cuda(), b.cuda(), offsets, rows if listed else None).cpu().double()
    want, mag = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    for e in range(E):
        s = ids == e
        want[s] = x[s].double() @ w[e].double().t() + b[e].double()
        mag[s] = x[s].double().abs() @ w[e].double().abs().t() + b[e].double().abs()
    tol = (K + 4) * 2.0 ** -24 * mag
    assert ((got - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()


@pytest.mark.parametrize('T', [1, 63, 1910, 1911, 2021, 5210, 5211, 16383, 16384, 16385, 40001])
@pytest.mark.parametrize('E', [1, 2, 15, 16, 31, 32, 300])
def test_rows_are_ordered_whichever_kernel_does_it(T, E):
    g = torch.Generator().manual_seed(T + E)
    ids = torch.randint(-2, E + 2, (T + 1,), generator=g).int()
    if E > 2:
        ids[torch.rand(T + 1, generator=g) < 0.3] = 1
    for first in (0, 1):                    # on sixteen bytes and off them
        some = ids[first:first + T]
        rows, offsets = experts.expert_rows(ids.cuda()[first:first + T], E)
        key = torch.where((some >= 0) & (some < E), some, torch.full_like(some, E)).long()
        assert torch.equal(rows.cpu().long(), torch.argsort(key, stable=True))
        assert torch.equal(offsets.cpu().long(), torch.bincount(key, minlength=E + 1).cumsum(0)[:E + 1] - torch.bincount(key, minlength=E + 1)[:E + 1])


@pytest.mark.parametrize('T,E,K,N', [(5003, 3, 264, 776), (9000, 2, 136, 520), (2600, 24, 200, 400), (700, 40, 72, 408), (6000, 1, 1024, 392)])
def test_gradients_of_long_reductions(T, E, K, N):
    """dx at sizes of every tile, dW and db in one and in several slices."""
    g = torch.Generator().manual_seed(T)
    x, dy, w = torch.randn(T, K, generator=g).bfloat16(), torch.randn(T, N, generator=g).bfloat16(), torch.randn(E, N, K, generator=g).bfloat16()
    ids = torch.randint(-1, E, (T,), generator=g).int()
    ids[torch.rand(T, generator=g) < 0.3] = 0
    rows, offsets = experts.expert_rows(ids.cuda(), E)
    dx = experts.grouped_linear_dgrad(dy.cuda(), w.cuda(), offsets, rows).cpu().double()
    dw, db = [t.cpu().double() for t in experts.grouped_linear_wgrad(dy.cuda(), x.cuda(), offsets, rows)]
    alone, none = experts.grouped_linear_wgrad(dy.cuda(), x.cuda(), offsets, rows, want_bias=False)
    assert none is None and torch.equal(alone.cpu().double(), dw)
    u = 2.0 ** -24
    for e in range(-1, E):
        s = ids == e
        d, xe = dy[s].double(), x[s].double()
        if e < 0:
            assert not dx[s].any()
            continue
        want, mag = d @ w[e].double(), d.abs() @ w[e].double().abs()
        tol = (N + 4) * u * mag
        assert ((dx[s] - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()
        n = int(s.sum()) + 4
        assert ((dw[e] - d.t() @ xe).abs() <= n * u * (d.abs().t() @ xe.abs())).all()
        assert ((db[e] - d.sum(0)).abs() <= n * u * d.abs().sum(0)).all()


@pytest.mark.parametrize('T,E,K,N', [(1, 2, 16, 8), (5, 2, 64, 16), (203, 3, 72, 40), (700, 40, 72, 408), (2500, 6, 136, 256), (5003, 3, 264, 776),
                                     (6144, 6, 72, 320), (12300, 6, 40, 320), (9000, 100, 136, 520)])
@pytest.mark.parametrize('listed', [True, False])
@pytest.mark.parametrize('kind', ['some', 'all before', 'all behind'])
def test_a_run_of_the_experts_leaves_zeros_in_every_other_row(T, E, K, N, listed, kind):
    """Offsets of experts 2 .. E + 1 of E + 4: a new result has zeros in the rows of those before and behind, whatever its memory held."""
    g = torch.Generator().manual_seed(T + N)
    x, w, b, dy = [t.cuda() for t in data(T, E, K, N, T)]
    ids = torch.randint(-1, E + 4, (T,), generator=g).int()
    if kind != 'some':
        ids.fill_(1 if kind == 'all before' else E + 2)
    if not listed:
        ids = torch.where(ids < 0, torch.full_like(ids, E + 9), ids).sort()[0].int()
    rows, offsets = experts.expert_rows(ids.cuda(), E + 4)
    rows, offsets = rows if listed else None, offsets[2:E + 3]
    mine = ((ids >= 2) & (ids < E + 2)).cuda()

    def poison(cols):
        held = [torch.full((T, cols), float('nan'), dtype=torch.bfloat16, device='cuda') for _ in range(3)]
        del held

    for call, cols in ((lambda **k: experts.grouped_linear(x, w, b, offsets, rows, **k), N),
                       (lambda **k: experts.grouped_linear_dgrad(dy, w, offsets, rows, **k), K)):
        want = call(out=torch.zeros(T, cols, dtype=torch.bfloat16, device='cuda'))
        assert not want[~mine].any() and (kind != 'some' or T < 100 or want[mine].any())
        for _ in range(2):
            poison(cols)
            assert torch.equal(call(), want)


def test_a_result_in_an_operand_s_memory_is_refused():
    T, E, N = 40, 3, 64
    x, w, b, _ = [t.cuda() for t in data(T, E, N, N, 12)]
    rows, offsets = experts.expert_rows(routing(T, E, 'even', 1).cuda(), E)
    for call in (lambda out: experts.grouped_linear(x, w, b, offsets, rows, out=out), lambda out: experts.grouped_linear_dgrad(x, w, offsets, rows, out=out)):
        for out in (x, w.view(-1, N)[:T], w.view(-1)[64:64 + T * N].view(T, N)):
            with pytest.raises(ValueError):
                call(out)
    both = torch.zeros(T, 2 * N, dtype=torch.bfloat16, device='cuda')       # beside each other in one array
    both[:, :N] = x
    y = experts.grouped_linear(both[:, :N], w, b, offsets, rows, out=both[:, N:])
    assert torch.equal(y, experts.grouped_linear(x, w, b, offsets, rows)) and torch.equal(both[:, :N], x)


def test_rows_and_weights_that_require_a_gradient():
    x, w, b, dy = [t.cuda() for t in data(16, 2, 64, 32, 13)]
    rows, offsets = experts.expert_rows(routing(16, 2, 'even', 1).cuda(), 2)
    want = experts.grouped_linear(x, w, b, offsets, rows)
    for call in (lambda: experts.grouped_linear(x.clone().requires_grad_(), w, b, offsets, rows),
                 lambda: experts.grouped_linear(x, w.clone().requires_grad_(), b, offsets, rows),
                 lambda: experts.grouped_linear_dgrad(dy.clone().requires_grad_(), w, offsets, rows),
                 lambda: experts.grouped_linear_wgrad(dy, x.clone().requires_grad_(), offsets, rows)):
        with pytest.raises(RuntimeError, match='requires a gradient'):
            call()
    with torch.no_grad():
        assert torch.equal(experts.grouped_linear(x.clone().requires_grad_(), w.clone().requires_grad_(), b, offsets, rows), want)
    layer = experts.ExpertLinear(2, 64, 32, device='cuda')
    assert layer(x, routing(16, 2, 'even', 1).cuda()).requires_grad
