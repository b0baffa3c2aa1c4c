"""Expert layers, 8-bit products and the 8-bit optimizer on arrays of more than 2^31 elements: what lies at their ends is computed as
in a small call.  Tolerances as in test_experts_gpu and test_fp8_gpu."""
import pytest
import torch

from test_fp8_gpu import check_layernorm, check_rounded, close, oracle

from vitpose_amd import experts, fp8, optim

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def release():
    yield
    torch.cuda.empty_cache()


def zeros_but_the_end(rows, cols, last, seed, dtype=torch.bfloat16):
    t = torch.zeros(rows, cols, dtype=dtype, device='cuda')
    t[-last:] = torch.randn(last, cols, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    assert t.numel() > 2 ** 31 or cols < 100
    return t


def near(got, want, mag, n):
    tol = (n + 4) * U * mag + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0) + 1e-30
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize('listed', [False, True])
def test_expert_products_of_300000_long_rows(listed):
    T, K, N, last = 300001, 7168, 8, 70
    x, dy = zeros_but_the_end(T, K, last, 1), zeros_but_the_end(T, N, last, 2)
    w = torch.randn(2, N, K, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    b = torch.randn(2, N, generator=torch.Generator().manual_seed(4)).cuda()
    if listed:                              # expert 0 takes the last rows
        rows, mine = torch.arange(T - 1, -1, -1, dtype=torch.int32, device='cuda'), 0
        offsets = torch.tensor([0, last, T], dtype=torch.int32, device='cuda')
    else:
        rows, mine = None, 1
        offsets = torch.tensor([0, T - last, T], dtype=torch.int32, device='cuda')
    y = experts.grouped_linear(x, w, b, offsets, rows)
    xd, wd, dd = x[-last:].cpu().double(), w[mine].cpu().double(), dy[-last:].cpu().double()
    near(y[-last:], xd @ wd.t() + b[mine].cpu().double(), xd.abs() @ wd.abs().t() + b[mine].cpu().double().abs(), K)
    assert torch.equal(y[:T - last], b[1 - mine].bfloat16().expand(T - last, N))
    dx = experts.grouped_linear_dgrad(dy, w, offsets, rows)
    near(dx[-last:], dd @ wd, dd.abs() @ wd.abs(), N)
    assert not dx[:1000].any() and not dx[T // 2:T // 2 + 1000].any() and not dx[T - last - 1000:T - last].any()
    del dx
    dw, db = experts.grouped_linear_wgrad(dy, x, offsets, rows)
    near(dw[mine], dd.t() @ xd, dd.abs().t() @ xd.abs(), T)
    near(db[mine], dd.sum(0), dd.abs().sum(0), T)
    assert not dw[1 - mine].any() and not db[1 - mine].any()


def test_8_bit_products_of_two_million_rows():
    M, K, N, last = 2 ** 21 + 77, 1032, 1040, 50
    x = zeros_but_the_end(M, K, last, 1)
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(2)).cuda()
    b = torch.randn(N, generator=torch.Generator().manual_seed(3)).cuda()
    wq, ws = fp8.quantize_weight(w)
    xq, xs = fp8.quantize_rows(x)
    q, s = fp8.quantize_rows(x[-last:].clone())
    assert torch.equal(xq[-last:].view(torch.uint8), q.view(torch.uint8)) and torch.equal(xs[:, -last:], s)
    want, mag = oracle(q, s.contiguous(), wq, ws, b.cpu())
    y = fp8.product(xq, xs, wq, ws, b)
    close(y[-last:], want, mag, wq.shape[1])
    assert torch.equal(y[M // 2:M // 2 + 1000], b.bfloat16().expand(1000, N))
    del y
    yq, ys = fp8.product(xq, xs, wq, ws, b, out_dtype=torch.float8_e4m3fn)
    check_rounded(want, mag, wq.shape[1], yq[-last:], ys[:, -last:])
    del yq, ys, xq, xs
    r = torch.zeros(M, N, device='cuda')
    r[-last:] = 1.0
    got = fp8.linear(x, wq, ws, b, out=r, resid=r)
    assert got is r
    close(r[-last:], want + 1, mag + 1, wq.shape[1])
    assert torch.equal(r[:1000], b.expand(1000, N))


def test_layernorm_of_two_million_rows():
    M, E, last = 2 ** 21 + 77, 1032, 50
    x = zeros_but_the_end(M, E, last, 1, torch.float32)
    g = torch.Generator().manual_seed(2)
    gamma, beta = torch.randn(E, generator=g), torch.randn(E, generator=g)
    q, s = fp8.layernorm_rows(x, gamma.cuda(), beta.cuda())
    check_layernorm(x[-last:].cpu().double(), gamma, beta, q[-last:], s[:, -last:])
    check_layernorm(torch.zeros(5, E, dtype=torch.float64), gamma, beta, q[:5], s[:, :5])


def test_adamw8_at_the_end_of_two_billion_parameters():
    n, last = 2 ** 31 + 8192, 4096
    g = torch.Generator().manual_seed(1)
    p0, g0 = torch.randn(last, generator=g).cuda(), torch.randn(last, generator=g).cuda()

    def run(numel, offset):
        param, grad = torch.zeros(numel, device='cuda'), torch.zeros(numel, device='cuda')
        param[offset:], grad[offset:] = p0, g0
        state = optim.new_state8(numel, 'cuda')
        start = torch.tensor([offset, offset + 2048], device='cuda')
        table = (start, torch.full((2,), 2048, dtype=torch.int32, device='cuda'), torch.ones(2, device='cuda'),
                 torch.full((2,), 0.1, device='cuda'), start.clone())
        for step in (1, 2):
            optim.adamw8_step(param, grad, state, table, lr=1e-2, step=step, noise=0, max_grad_norm=1.0)
            if step == 1:                   # (later steps read sqrt(v), whose rounding is keyed by the position)
                one = param[offset:].clone()
        m8, ms, r8, rs = state
        assert not param[:offset].any() and not m8.view(torch.uint8)[:offset].any() and torch.isfinite(param[offset:]).all()
        return one, m8.view(torch.uint8)[offset:].clone(), ms[offset // 128:].clone(), rs[offset // 128:].clone()
    for a, b in zip(run(n, n - last), run(last, 0)):
        assert a.shape == b.shape
        if a.dtype == torch.float32 and a.numel() == last or a.dtype == torch.uint8:
            assert torch.equal(a, b)


def test_8_bit_products_of_more_rows_than_small_workgroups_can_be_started_for():
    M, N, K, last = 2 ** 27 + 77, 8, 128, 50
    g = torch.Generator().manual_seed(1)
    w = torch.randn(N, K, generator=g).cuda()
    wq, ws = fp8.quantize_weight(w)
    q, s = fp8.quantize_rows(torch.randn(last, K, generator=g).cuda())
    xq, xs = torch.zeros(M, K, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn), torch.zeros(1, M, device='cuda')
    xq.view(torch.uint8)[-last:], xs[:, -last:] = q.view(torch.uint8), s
    y = fp8.product(xq, xs, wq, ws)
    close(y[-last:], *oracle(q, s, wq, ws, None), K)
    assert not y[:1000].any() and not y[M // 2:M - last].any()
    del xq, xs
    x = torch.zeros(M, K, dtype=torch.bfloat16, device='cuda')
    x[-last:] = 1.0
    y = fp8.linear(x, wq, ws)
    assert torch.equal(y[-last:], y[-1:].expand(last, N)) and not y[:M - last].any()
    close(y[-1:], *oracle(*fp8.quantize_rows(x[-1:].clone()), wq, ws, None), K)


def test_expert_products_of_a_billion_rows():
    T, N, last = 2 ** 30, 8, 70
    x = zeros_but_the_end(T, N, last, 1)
    w = torch.randn(2, N, N, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    offsets = torch.tensor([0, T - last, T], dtype=torch.int32, device='cuda')
    xd, wd = x[-last:].cpu().double(), w[1].cpu().double()
    y = experts.grouped_linear(x, w, None, offsets)
    near(y[-last:], xd @ wd.t(), xd.abs() @ wd.abs().t(), N)
    assert not y[:1000].any() and not y[T // 2:T // 2 + 1000].any()
    del y
    dx = experts.grouped_linear_dgrad(x, w, offsets)
    near(dx[-last:], xd @ wd, xd.abs() @ wd.abs(), N)
    assert not dx[:1000].any() and not dx[T // 2:T // 2 + 1000].any()
