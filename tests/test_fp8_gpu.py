"""Block-scaled e4m3 products (vp_quantize_fp8_*, vp_gemm_fp8, vitpose_amd.fp8) against the definition in 64 bits.

Tolerances (U = 2^-24, half a step of f32): a scale is one product of amax and the rounded constant 1 / 448 (2 U); the value in
front of the rounding to e4m3 passes a reciprocal and two products (4 U), so a code is the nearest one up to that, which is half a
spacing plus 4 U of the value; a sum over Kp products in blocks, each block's sum times the product of two scales, is off by at
most (Kp + blocks + 4) U of the sum of the magnitudes; a bf16 result by half a step more (2^-8), the GELU's polynomial by 2.5e-5
and its slope is at most 1.13."""
import pytest
import torch

from vitpose_amd import fp8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def spacing(x):
    return torch.exp2((torch.frexp(x.abs())[1] - 1).clamp(min=-6).double() - 3)


def padded(x):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 128))


def check_codes(x, q, scale):
    """x f64 [..., 128] of one block each, q its codes' values, scale f32."""
    amax = x.abs().amax(-1)
    live = amax >= 2.0 ** -100
    assert ((scale.double() - amax / 448).abs() <= 2.1 * U * amax / 448)[live].all() and not scale[~live].any() and not q[~live].any()
    v = x[live] * 448 / amax[live][..., None]
    assert ((q[live] - v).abs() <= spacing(v) / 2 + 6 * U * v.abs()).all()
    # the largest magnitude is the largest code
    assert (q[live].abs().amax(-1) == 448).all()


SHAPES = [(1, 8), (1, 128), (3, 136), (17, 1000), (64, 384), (200, 72), (129, 1280)]


@pytest.mark.parametrize('M,K', SHAPES + [(5000, 264)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rows_are_rounded_block_by_block(M, K, dtype):
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(4 * torch.randn(M, K, generator=g))).to(dtype)
    x[0, :8] = 0
    if M > 2:
        x[1] = 0
        x[2] *= 2.0 ** -60
        x[2] *= 2.0 ** -60          # some blocks below 2^-100
    q, s = fp8.quantize_rows(x.cuda())
    kb = (K + 127) // 128
    assert q.shape == (M, kb * 128) and s.shape == (kb, M) and q.dtype == torch.float8_e4m3fn
    check_codes(padded(x.double()).view(M, kb, 128), q.cpu().double().view(M, kb, 128), s.cpu().t())
    wide = torch.full((M, K + 16), float('nan'), dtype=dtype, device='cuda')
    wide[:, :K] = x.cuda()
    q2, s2 = fp8.quantize_rows(wide[:, :K])
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


@pytest.mark.parametrize('N,K', SHAPES + [(300, 600)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_weights_are_rounded_square_by_square(N, K, dtype):
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn(N, K, generator=g) * torch.exp(2 * torch.randn(N, K, generator=g))).to(dtype)
    q, s = fp8.quantize_weight(w.cuda())
    nb, kb = (N + 127) // 128, (K + 127) // 128
    assert q.shape == (N, kb * 128) and s.shape == (nb, kb)

    def squares(t):
        t = torch.nn.functional.pad(t, (0, kb * 128 - t.shape[1], 0, nb * 128 - N))
        return t.view(nb, 128, kb, 128).permute(0, 2, 1, 3).reshape(nb, kb, 128 * 128)
    check_codes(squares(w.double()), squares(q.cpu().double()), s.cpu())


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_what_is_not_finite_marks_its_block(bad):
    x = torch.ones(4, 384, device='cuda')
    x[1, 200] = bad
    q, s = fp8.quantize_rows(x)
    assert torch.isnan(s[1, 1]) and int(torch.isnan(s).sum()) == 1
    w = torch.ones(200, 384, device='cuda')
    wq, ws = fp8.quantize_weight(w)
    y = fp8.product(q, s, wq, ws)
    assert torch.isnan(y[1]).all() and (y[[0, 2, 3]] == 384).all()
    w[150, 300] = bad
    wq, ws = fp8.quantize_weight(w)
    assert torch.isnan(ws[1, 2]) and int(torch.isnan(ws).sum()) == 1
    q, s = fp8.quantize_rows(torch.ones(4, 384, device='cuda'))
    y = fp8.product(q, s, wq, ws)
    assert torch.isnan(y[:, 128:]).all() and (y[:, :128] == 384).all()


GEMMS = [(1, 1, 128), (1, 17, 256), (2, 5120, 1280), (3, 64, 136), (16, 96, 1536), (17, 130, 384), (33, 1000, 200), (64, 128, 128),
         (65, 777, 1000), (127, 129, 640), (128, 256, 2048), (192, 1024, 1024), (257, 320, 5120), (513, 72, 264), (1001, 777, 1000),
         (2000, 33, 8)]


def operands(M, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g))
    w = torch.randn(N, K, generator=g) * 0.05
    return x.bfloat16(), w, torch.randn(N, generator=g)


def oracle(xq, xs, wq, ws, bias):
    """(y, magnitudes) in 64 bits from the quantized operands."""
    x = xq.cpu().double() * xs.cpu().t().double().repeat_interleave(128, 1)
    w = wq.cpu().double() * ws.cpu().double().repeat_interleave(128, 0)[:wq.shape[0]].repeat_interleave(128, 1)
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    eights = [t.abs().view(t.shape[0], -1, 8).amax(2) for t in (x, w)]
    mag += 7 * 2.0 ** -13 / ((x.shape[1] + x.shape[1] // 128 + 4) * U) * (eights[0] @ eights[1].t())     # in units of close()'s
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def close(got, want, mag, Kp, act=None):
    tol = (Kp + Kp // 128 + 4) * U * mag
    if act:
        want, tol = torch.nn.functional.gelu(want), 1.13 * tol + (2.6e-5 if got.dtype == torch.bfloat16 else 4 * U * want.abs())
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all() and (off <= tol).all(), f'{(off / tol).max().item():.3g} of the bound'


@pytest.mark.parametrize('M,N,K', GEMMS)
@pytest.mark.parametrize('out_dtype', [torch.bfloat16, torch.float32])
def test_products_match_sums_in_64_bits(M, N, K, out_dtype):
    x, w, b = operands(M, N, K, M + N + K)
    xq, xs = fp8.quantize_rows(x.cuda())
    wq, ws = fp8.quantize_weight(w.cuda())
    Kp = wq.shape[1]
    for bias, act in ((None, None), (b, None), (b, 'gelu')):
        want, mag = oracle(xq, xs, wq, ws, bias)
        bd = bias.cuda() if bias is not None else None
        got = fp8.product(xq, xs, wq, ws, bd, act=act, out_dtype=out_dtype)
        close(got, want, mag, Kp, act)
        # (the call that rounds x itself may add up the blocks in another order)
        close(fp8.linear(x.cuda(), wq, ws, bd, act=act, out_dtype=out_dtype), want, mag, Kp, act)
    x32 = x.float().cuda()
    close(fp8.linear(x32, wq, ws, out_dtype=out_dtype), *oracle(xq, xs, wq, ws, None), Kp)


@pytest.mark.parametrize('M,N,K', GEMMS)
def test_whole_numbers_come_out_exactly(M, N, K):
    """Codes of small whole numbers with scales of whole powers of two: every product and sum is exact."""
    g = torch.Generator().manual_seed(M * N + K)
    Kp = (K + 127) // 128 * 128
    xq = torch.randint(-8, 9, (M, Kp), generator=g).float().to(torch.float8_e4m3fn)
    wq = torch.randint(-8, 9, (N, Kp), generator=g).float().to(torch.float8_e4m3fn)
    xs = torch.exp2(torch.randint(-3, 3, (Kp // 128, M), generator=g).float())
    ws = torch.exp2(torch.randint(-3, 3, ((N + 127) // 128, Kp // 128), generator=g).float())
    want, _ = oracle(xq, xs, wq, ws, None)
    got = fp8.product(xq.cuda(), xs.cuda(), wq.cuda(), ws.cuda(), out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize('M,N', [(3, 50), (40, 130), (300, 264)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_operands_and_results_inside_larger_arrays(M, N, dtype):
    K = 200
    x, w, b = operands(M, N, K, 3)
    xq, xs = fp8.quantize_rows(x.cuda())
    wq, ws = fp8.quantize_weight(w.cuda())
    want = fp8.product(xq, xs, wq, ws, b.cuda(), out_dtype=dtype)
    nan = torch.full((M + N, 256 + 48), 0x7F, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
    nan.view(torch.uint8)[:M, :256] = xq.view(torch.uint8)
    nan.view(torch.uint8)[M:, :256] = wq.view(torch.uint8)
    for pad in (8, 5):                     # rows of the result on and off 8-byte boundaries
        out = torch.full((M, N + pad), 7.0, dtype=dtype, device='cuda')
        got = fp8.product(nan[:M, :256], xs, nan[M:, :256], ws, b.cuda(), out=out[:, :N])
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and (out[:, N:] == 7).all()
        out.fill_(7.0)
        lin = fp8.linear(x.cuda(), wq, ws, b.cuda(), out=out[:, :N])
        assert (out[:, N:] == 7).all()
        torch.testing.assert_close(lin, want, rtol=2.0 ** -7 if dtype == torch.bfloat16 else 1e-4, atol=1e-4)


def test_no_rows():
    wq, ws = fp8.quantize_weight(torch.ones(24, 64, device='cuda'))
    assert fp8.linear(torch.empty(0, 64, device='cuda'), wq, ws).shape == (0, 24)
    q, s = fp8.quantize_rows(torch.empty(0, 64, device='cuda', dtype=torch.bfloat16))
    assert q.shape == (0, 128) and s.shape == (1, 0)


@pytest.mark.parametrize('M', [4, 500])
def test_another_stream_and_replayed_graphs(M):
    x, w, b = operands(M, 200, 264, 5)
    wq, ws = fp8.quantize_weight(w.cuda())
    xs = [(x * k).cuda() for k in (1.0, -2.0, 0.5)]
    bd, static = b.cuda(), xs[0].clone()
    want = [fp8.linear(v, wq, ws, bd, act='gelu') for v in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp8.linear(static, wq, ws, bd, act='gelu')
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8.linear(static, wq, ws, bd, act='gelu')
        graphs.append((graph, out))
    for k in (1, 2, 0, 1):
        static.copy_(xs[k])
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[k]) for _, out in graphs)
        assert torch.equal(fp8.linear(xs[k], wq, ws, bd, act='gelu'), want[k])


def test_refusals():
    x, w, b = [t.cuda() for t in operands(32, 48, 136, 6)]
    wq, ws = fp8.quantize_weight(w)
    xq, xs = fp8.quantize_rows(x)
    for bad in (x.half(), x.int()):
        with pytest.raises(TypeError):
            fp8.quantize_rows(bad)
    for bad in (x[0], x[:, :100], x[:, 1:129], x.t(), torch.zeros(4, 0, device='cuda')):
        with pytest.raises(ValueError):
            fp8.quantize_rows(bad)
    with pytest.raises(RuntimeError):
        fp8.quantize_rows(x.cpu())
    with pytest.raises(ValueError):
        fp8.quantize_weight(w[:0])

    def call(**kw):
        a = dict(xq=xq, xs=xs, wq=wq, ws=ws, bias=b)
        a.update(kw)
        return fp8.product(a.pop('xq'), a.pop('xs'), a.pop('wq'), a.pop('ws'), a.pop('bias'), **a)
    for kw in (dict(xq=xq.view(torch.uint8)), dict(out_dtype=torch.float16), dict(out=torch.empty(32, 48, device='cuda').half())):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(xq=xq[:, :128]), dict(xq=xq[:, 16:144]), dict(xs=xs.t()), dict(xs=xs[:1]), dict(ws=ws.t()), dict(ws=ws.double()),
               dict(bias=b[:-1]), dict(bias=b.bfloat16()), dict(act='relu'), dict(out=torch.empty(32, 49, device='cuda')),
               dict(out=torch.empty(48, 32, device='cuda').t())):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(wq=wq.cpu())
    with pytest.raises(ValueError):
        fp8.linear(x[:, :128], wq, ws)


@pytest.mark.parametrize('M,N,K', [(1, 5, 128), (3, 136, 64), (17, 130, 384), (40, 264, 1000), (300, 1000, 264), (2100, 1280, 256), (2100, 1281, 256)])
@pytest.mark.parametrize('act', [None, 'gelu'])
def test_a_residual_is_added_behind_the_activation(M, N, K, act):
    x, w, b = operands(M, N, K, M + N + K)
    g = torch.Generator().manual_seed(9)
    r = torch.randn(M, N, generator=g).cuda()
    xq, xs = fp8.quantize_rows(x.cuda())
    wq, ws = fp8.quantize_weight(w.cuda())
    bd = b.cuda()
    for call in (lambda **k: fp8.product(xq, xs, wq, ws, bd, act=act, **k), lambda **k: fp8.linear(x.cuda(), wq, ws, bd, act=act, **k)):
        plain = call(out_dtype=torch.float32)
        want = plain + r                                      # one f32 sum of the same two numbers
        assert torch.equal(call(out_dtype=torch.float32, resid=r), want)
        wide = torch.full((M, N + 7), float('nan'), device='cuda')
        wide[:, :N] = r
        assert torch.equal(call(out_dtype=torch.float32, resid=wide[:, :N]), want)
        got = call(out=wide[:, :N], resid=wide[:, :N])        # in place
        assert torch.equal(got, want) and torch.isnan(wide[:, N:]).all()
        with pytest.raises(TypeError):
            call(resid=r)
        for bad in (r.double(), r[:, :N - 1], r.t() if M != N else r[:1]):
            with pytest.raises(ValueError):
                call(out_dtype=torch.float32, resid=bad)
        with pytest.raises(RuntimeError):
            call(out_dtype=torch.float32, resid=r.cpu())


def check_rounded(want, mag, Kp, q, scale, act=None):
    """Codes and scales of a product's result against the exact result: the result itself is off by close()'s bound (before its
    rounding to 16 bits), a scale by its block's largest such error and 2 U, a code by half a spacing and that error in its units."""
    tol = (Kp + Kp // 128 + 4) * U * mag
    if act:
        want, tol = torch.nn.functional.gelu(want), 1.13 * tol + 2.6e-5
    M, N = want.shape
    x, t = [padded(v).view(M, -1, 128) for v in (want, tol)]
    check_codes_within(x, t, q, scale)
    assert not q.cpu().double()[:, N:].any()


def check_codes_within(x, t, q, scale):
    """x f64 [M, blocks, 128], known to t."""
    M, kb, _ = x.shape
    assert q.shape == (M, kb * 128) and scale.shape == (kb, M) and torch.isfinite(scale).all()
    got, s = q.cpu().double().view(M, kb, 128), scale.cpu().t().double()
    amax, tmax = x.abs().amax(-1), t.amax(-1)
    assert ((s - amax / 448).abs() <= (tmax + 2.1 * U * amax) / 448).all()
    safe = s.clamp(min=1e-30)[..., None]
    v, e = x / safe, t / safe
    assert ((got - v).abs() <= spacing(v.abs() + e) / 2 + e + 6 * U * v.abs()).all()
    assert (got.abs().amax(-1)[s > 0] == 448).all()


def check_layernorm(x, gamma, beta, q, scale, eps=1e-6):
    """x f64.  A mean of E values in f32 is off by (E + 2) U of their mean magnitude A, so a difference from it by that and U of
    itself; the standard deviation s, from a sum of squares, by (E / 2 + 4) U of itself and the mean's error; then come four products
    and a sum.  Together under (E + 10) U (2 A / s + |z|) |gamma| + 2 U |result| in the result."""
    E = x.shape[1]
    mean, var = x.mean(1, keepdim=True), x.var(1, unbiased=False, keepdim=True)
    sd = (var + eps).sqrt()
    z = (x - mean) / sd
    want = z * gamma.double() + beta.double()
    tol = (E + 10) * U * (2 * x.abs().mean(1, keepdim=True) / sd + z.abs()) * gamma.double().abs() + 2 * U * (want.abs() + beta.double().abs())
    check_codes_within(*[padded(v).view(len(x), -1, 128) for v in (want, tol)], q, scale)
    assert not q.cpu().double()[:, E:].any()


@pytest.mark.parametrize('M,E', [(1, 8), (3, 64), (5, 384), (17, 520), (64, 768), (9, 1024), (130, 1280), (7, 1536), (33, 2048), (9000, 72)])
def test_layernorm_in_front_of_the_rounding(M, E):
    g = torch.Generator().manual_seed(M + E)
    x = torch.randn(M, E, generator=g) * torch.exp(torch.randn(M, 1, generator=g)) + 3 * torch.randn(M, 1, generator=g)
    gamma, beta = 1 + 0.5 * torch.randn(E, generator=g), 0.3 * torch.randn(E, generator=g)
    if M > 2:
        x[2] = 1.5                          # no variance: the bias is left
    q, s = fp8.layernorm_rows(x.cuda(), gamma.cuda(), beta.cuda())
    check_layernorm(x.double(), gamma, beta, q, s)
    if M > 1:
        x[1, E // 2] = float('nan')
        q2, s2 = fp8.layernorm_rows(x.cuda(), gamma.cuda(), beta.cuda())
        assert torch.isnan(s2[:, 1]).all() and torch.equal(s2[:, 0], s[:, 0]) and torch.equal(s2[:, 2:], s[:, 2:])


@pytest.mark.parametrize('M,N,K', [(1, 8, 128), (17, 130, 384), (130, 128, 64), (257, 777, 264), (300, 1000, 1000), (600, 72, 256), (4100, 1281, 136)])
@pytest.mark.parametrize('act', [None, 'gelu'])
def test_a_result_as_codes_for_the_next_product(M, N, K, act):
    x, w, b = operands(M, N, K, M + N + K)
    xq, xs = fp8.quantize_rows(x.cuda())
    wq, ws = fp8.quantize_weight(w.cuda())
    bd = b.cuda()
    if N > 200:
        bd[128:256] = 0
        wq.view(torch.uint8)[128:256] = 0   # a block of zeros
    q, s = fp8.product(xq, xs, wq, ws, bd, act=act, out_dtype=torch.float8_e4m3fn)
    want, mag = oracle(xq, xs, wq, ws, bd.cpu())
    check_rounded(want, mag, wq.shape[1], q, s, act)
    if N > 200:
        # the GELU's polynomial may give up to 2.5e-5 at zero, so its scale up to that over 448 (and two roundings)
        assert (s[1] <= 2.6e-5 / 448).all() if act else not s[1].any()
    q2, s2 = fp8.linear(x.cuda(), wq, ws, bd, act=act, out_dtype=torch.float8_e4m3fn)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    # and the next product takes it
    w2q, w2s = fp8.quantize_weight(torch.randn(40, N + -N % 8, generator=torch.Generator().manual_seed(1)).cuda())
    close(fp8.product(q, s, w2q, w2s), *oracle(q, s, w2q, w2s, None), w2q.shape[1])
    xs[0, 0] = float('nan')
    q, s = fp8.product(xq, xs, wq, ws, bd, act=act, out_dtype=torch.float8_e4m3fn)
    assert torch.isnan(s[:, 0]).all() and torch.isfinite(s[:, 1:]).all()
    with pytest.raises(ValueError):
        fp8.product(xq, xs, wq, ws, out_dtype=torch.float8_e4m3fn, resid=torch.zeros(M, N, device='cuda'))
    with pytest.raises(ValueError):
        fp8.linear(x.cuda(), wq, ws, out_dtype=torch.float8_e4m3fn, out=torch.zeros(M, N, device='cuda'))


def test_layernorm_refusals():
    x, w = torch.zeros(4, 64, device='cuda'), torch.ones(64, device='cuda')
    assert fp8.layernorm_rows(x[:0], w, w)[0].shape == (0, 128)
    with pytest.raises(TypeError):
        fp8.layernorm_rows(x.bfloat16(), w, w)
    wide = torch.ones(2056, device='cuda')
    for bad in ((x[:, :32], w[:32], w[:32]), (x, w[:32], w), (x, w, w.bfloat16()), (torch.zeros(2, 2056, device='cuda'), wide, wide),
                (x, torch.ones(65, device='cuda')[1:], w)):
        with pytest.raises(ValueError):
            fp8.layernorm_rows(*bad)
    with pytest.raises(RuntimeError):
        fp8.layernorm_rows(x, w.cpu(), w)


def test_codes_from_layernorm_to_product_on_another_stream_and_in_replayed_graphs():
    g = torch.Generator().manual_seed(4)
    M, E, N = 300, 264, 520
    xs = [torch.randn(M, E, generator=g).cuda() * k for k in (1.0, 3.0, 0.2)]
    gamma, beta = torch.randn(E, generator=g).cuda(), torch.randn(E, generator=g).cuda()
    w1, w2 = fp8.quantize_weight(torch.randn(N, E, generator=g).cuda()), fp8.quantize_weight(torch.randn(E, N, generator=g).cuda())

    def run(x):
        h = fp8.product(*fp8.layernorm_rows(x, gamma, beta), *w1, act='gelu', out_dtype=torch.float8_e4m3fn)
        return fp8.product(*h, *w2, out_dtype=torch.float32, resid=x)
    want = [run(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = xs[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = run(static)
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static)
        graphs.append((graph, out))
    for k in (1, 2, 0, 1):
        static.copy_(xs[k])
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[k]) for _, out in graphs) and torch.equal(run(xs[k]), want[k])


@pytest.mark.parametrize('N', [257, 258, 260, 263, 383])
@pytest.mark.parametrize('M', [40, 700, 2600])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rows_that_begin_anywhere(M, N, dtype):
    """Results of odd lengths and odd strides, every element in its place and nothing beside them."""
    x, w, b = operands(M, N, 136, M + N)
    xq, xs = fp8.quantize_rows(x.cuda())
    wq, ws = fp8.quantize_weight(w.cuda())
    want, mag = oracle(xq, xs, wq, ws, b)
    for pad in (0, 1, 3, 5):
        out = torch.full((M, N + pad), 7.0, dtype=dtype, device='cuda')
        got = fp8.product(xq, xs, wq, ws, b.cuda(), out=out[:, :N])
        close(got, want, mag, wq.shape[1])
        assert (out[:, N:] == 7).all()


@pytest.mark.parametrize('M', [1, 3, 300, 4100])
@pytest.mark.parametrize('out_dtype', [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
def test_the_gelu_of_small_values_and_of_its_tail(M, out_dtype):
    """The sums are zeros here, so a column's GELU is that of its bias: blocks of 128 of every size, zeros, and the tail below zero, each
    within a few roundings of ITSELF.  With t = |x|, in U: t / (t + c) is off by 4, the fit by 2, its eight-term polynomial by what its
    partial sums come to, at most 2 + 2.8 t, the exponential by 2 and by the three roundings of its argument, 1.5 t^2; two products and
    the difference add 3: below 14 + 3 t + 1.5 t^2 (the first 4 count in full only near zero)."""
    sizes = [0.0, 1e-25, 1e-12, 1e-5, 1e-4, 1e-3, 0.1, 1.0]
    g = torch.Generator().manual_seed(M)
    b = torch.cat([torch.randn(128, generator=g) * s for s in sizes] + [-torch.linspace(2, 5, 128), -torch.linspace(5, 11, 128)])
    N, K = b.numel(), 256
    x = torch.randn(M, K, generator=g).cuda()
    wq, ws = fp8.quantize_weight(torch.zeros(N, K, device='cuda'))
    want = (b.double() * torch.special.erfc(-b.double() * 0.5 ** 0.5) / 2).expand(M, N)
    tol = (14 + 3 * b.double().abs() + 1.5 * b.double() ** 2) * U * want.abs()
    for call in (lambda: fp8.product(*fp8.quantize_rows(x), wq, ws, b.cuda(), act='gelu', out_dtype=out_dtype),
                 lambda: fp8.linear(x, wq, ws, b.cuda(), act='gelu', out_dtype=out_dtype)):
        got = call()
        if out_dtype == torch.float8_e4m3fn:
            q, s = got
            assert not s[0].any() and not q[:, :128].view(torch.uint8).any()
            check_codes_within(want.reshape(M, -1, 128), tol.reshape(M, -1, 128), q, s)
        else:
            off = (got.cpu().double() - want).abs()
            bound = tol + (2.0 ** -8 * (want.abs() + tol) if out_dtype == torch.bfloat16 else 0)
            assert (off <= bound).all(), [f'{v:.3g}' for v in (off / bound.clamp(min=1e-300)).view(M, -1, 128).amax((0, 2)).tolist()]


def test_a_result_in_an_operand_s_memory_is_refused():
    M, N, K = 64, 64, 64
    x, w, b = [t.cuda() for t in operands(M, N, K, 7)]
    wq, ws = fp8.quantize_weight(w)
    xq, xs = fp8.quantize_rows(x)
    for out in (x, wq.view(torch.bfloat16), xq.view(torch.bfloat16)):
        with pytest.raises(ValueError):
            (fp8.linear if out is x else fp8.product)(*((x,) if out is x else (xq, xs)), wq, ws, out=out)
    flat = torch.zeros(M * N + 256, device='cuda')
    out = flat[:M * N].view(M, N)
    for resid in (flat[4:M * N + 4].view(M, N), flat[N:M * N + N].view(M, N), flat.as_strided((M, N), (N + 4, 1))):
        for call in (lambda **k: fp8.product(xq, xs, wq, ws, **k), lambda **k: fp8.linear(x, wq, ws, **k)):
            with pytest.raises(ValueError):
                call(out=out, resid=resid)
    both = torch.zeros(M, 2 * N, device='cuda')
    both[:, N:] = 1.0
    y = fp8.product(xq, xs, wq, ws, out=both[:, :N], resid=both[:, N:])
    assert torch.equal(y, fp8.product(xq, xs, wq, ws, out_dtype=torch.float32) + 1) and (both[:, N:] == 1).all()


def test_rows_that_require_a_gradient():
    x, w, _ = [t.cuda() for t in operands(8, 24, 64, 8)]
    wq, ws = fp8.quantize_weight(torch.nn.Parameter(w))
    want = fp8.linear(x, wq, ws)
    x.requires_grad_()
    for call in (fp8.quantize_rows, lambda x: fp8.linear(x, wq, ws), lambda x: fp8.linear(x.detach(), wq, ws, out_dtype=torch.float32,
                                                                                          resid=torch.zeros(8, 24, device='cuda').requires_grad_())):
        with pytest.raises(RuntimeError, match='requires a gradient'):
            call(x)
    with torch.no_grad():
        assert torch.equal(fp8.linear(x, wq, ws), want)
    assert torch.equal(fp8.linear(x.detach(), wq, ws), want)


@pytest.mark.parametrize('large,small,exact', [(256.0, 2.0 ** -9, False), (16.0, 2.0 ** -5, True)])
def test_what_the_matrix_instruction_s_eights_may_lose(large, small, exact):
    """A large product in each eight and seven small ones, every number exact in e4m3: the sum is within 7 x 2^-13 of the large products,
    and exact where the small ones lie within the 13 bits below."""
    M, N, K = 300, 40, 128
    x, w = torch.full((M, K), small), torch.ones(N, K)
    x[:, ::8], w[:, ::8] = large, large
    xq, wq = x.to(torch.float8_e4m3fn).cuda(), w.to(torch.float8_e4m3fn).cuda()
    want = 16 * (large * large + 7 * small)
    for rows in (3, M):
        y = fp8.product(xq[:rows], torch.ones(1, rows, device='cuda'), wq, torch.ones(1, 1, device='cuda'), out_dtype=torch.float32).cpu().double()
        assert ((y - want).abs() <= (0 if exact else 16 * 7 * 2.0 ** -13 * large * large)).all()
