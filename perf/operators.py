"""Measured cases of the framework's operators for expert layers and 8-bit formats.

Three families, each as a user's program calls it:

* ``experts``: products of rows with the weight of the expert each row belongs to (``vitpose_amd.experts``): the forward
  product, the gradients of its input, weight and bias, and the ordering of rows by expert in front of them;
* ``fp8``: a Linear whose operands are e4m3 numbers with one f32 scale per block of 128 (``vitpose_amd.fp8``);
* ``adamw8``: one AdamW step over a model's tensors with both moments held in 8 bits (``vitpose_amd.optim``).

``own`` false computes the same by elementary torch operations in 32 bits; ``exact`` in 64 bits from the definitions.
"""
import math

import torch

own = False

BLOCK = 128          # values that share one scale
E4M3_MAX = 448.0
TINY = 2.0 ** -100   # a block whose largest magnitude is below this is stored as zeros


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one row of a ViTPose+-S expert layer (hidden 1536, 96 expert channels): the latency of a single token
        dict(name='experts_one_row', kind='experts', rows=1, experts=6, k=1536, n=96, skew='even', order='sorted', train=False),
        # one 256 x 192 crop (192 tokens) of ViTPose+-L, tokens routed one by one, two experts without a row
        dict(name='experts_one_image', kind='experts', rows=192, experts=6, k=4096, n=256, skew='gaps', order='ids', train=False),
        # an evaluation batch of 64 crops of ViTPose+-L whose datasets come in uneven shares
        dict(name='experts_batch_L', kind='experts', rows=12288, experts=6, k=4096, n=256, skew='skewed', order='ids', train=False),
        # a training step of ViTPose+-H's expert layer on 32 crops: product and all gradients
        dict(name='experts_train_H', kind='experts', rows=6144, experts=6, k=5120, n=320, skew='skewed', order='sorted', train=True),
        # many experts, odd extents, rows that no expert takes: token routing in a layer of its own
        dict(name='experts_train_odd', kind='experts', rows=5003, experts=24, k=1000, n=328, skew='gaps', order='ids', train=True),
        # one row through ViTPose-H's fc1: reading the weights is all there is
        dict(name='fp8_one_row', kind='fp8', rows=1, k=1280, n=5120, bias=True, act='', keep=False),
        # one crop through ViTPose-L's fc1 with its GELU
        dict(name='fp8_one_image', kind='fp8', rows=192, k=1024, n=4096, bias=True, act='gelu', keep=False),
        # extents that are multiples of nothing: a regression layer behind flattened features
        dict(name='fp8_odd', kind='fp8', rows=1001, k=1000, n=777, bias=False, act='', keep=True),
        # an evaluation batch of 128 crops through ViTPose-H's fc2
        dict(name='fp8_batch_H', kind='fp8', rows=24576, k=5120, n=1280, bias=True, act='', keep=True),
        # fine-tuning a head alone: a few tensors, the launch counts; gradients clipped by their norm
        dict(name='adamw8_head', kind='adamw8', tensors=14, largest=1 << 20, total=2_200_000, clip=True),
        # ViTPose-B with its head: 90 M parameters in 160 tensors, clipped
        dict(name='adamw8_B', kind='adamw8', tensors=160, largest=2_359_296, total=90_000_000, clip=True),
        # ViTPose-L: 304 M parameters
        dict(name='adamw8_L', kind='adamw8', tensors=300, largest=4_194_304, total=304_000_000, clip=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['experts', 'experts', 'fp8', 'fp8', 'adamw8'])
    if kind == 'experts':
        train = rng.random() < 0.5
        rows = _log(rng, 1, 16384)
        k, n = 8 * _log(rng, 8, 640), 8 * _log(rng, 2, 128)
        while rows * k * n > 2 ** 33:
            rows = max(1, rows // 2)
        return dict(kind='experts', rows=rows, experts=_log(rng, 1, 48), k=k, n=n, skew=rng.choice(['even', 'skewed', 'gaps']),
                    order=rng.choice(['sorted', 'ids']), train=train)
    if kind == 'fp8':
        rows, k, n = _log(rng, 1, 24576), 8 * _log(rng, 8, 640), _log(rng, 17, 5120)
        while rows * k * n > 2 ** 37:
            rows = max(1, rows // 2)
        return dict(kind='fp8', rows=rows, k=k, n=n, bias=rng.random() < 0.7, act=rng.choice(['', '', 'gelu']),
                    keep=rng.random() < 0.5)
    total = _log(rng, 100_000, 150_000_000)
    tensors = _log(rng, 4, 300)
    return dict(kind='adamw8', tensors=tensors, largest=max(1024, int(total * rng.uniform(0.03, 0.4))), total=total,
                clip=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _shares(case):
    """Rows per expert, and rows that no expert takes: from the case alone."""
    rows, e, skew = case['rows'], case['experts'], case['skew']
    if skew == 'even':
        weights = [1.0] * e
    elif skew == 'skewed':
        weights = [1.0 / (1 + i) for i in range(e)]
    else:                                   # every third expert has no row at all
        weights = [0.0 if i % 3 == 1 else 1.0 + (i * 7 % 5) for i in range(e)]
    none = rows // 20 if skew == 'gaps' else 0
    left = rows - none
    whole = [int(left * w / sum(weights)) for w in weights]
    whole[max(range(e), key=lambda i: weights[i])] += left - sum(whole)
    return whole, none


def _tensor_sizes(case):
    """Element counts of the model's tensors: weights that share the total, small vectors (biases, norms) between them."""
    out, left = [], case['total']
    for i in range(case['tensors']):
        if i % 2:
            n = min(left, 17 + (i * 193) % 5120)
        else:
            n = min(left, case['largest'], max(1, left // max(1, (case['tensors'] - i + 1) // 2)))
        if n > 0:
            out.append(n)
            left -= n
    return out


def _experts_state(case, gen, dev):
    rows, e, k, n = case['rows'], case['experts'], case['k'], case['n']
    counts, none = _shares(case)
    ids = torch.repeat_interleave(torch.arange(e + 1, device=dev, dtype=torch.int32),
                                  torch.tensor(counts + [none], device=dev))
    s = dict(case=case, most=max(counts))
    if case['order'] == 'ids':
        ids = torch.where(ids == e, torch.full_like(ids, -1), ids)
        s['ids'] = ids[torch.randperm(rows, generator=gen, device=dev)].contiguous()
    else:
        offs = [0]
        for c in counts:
            offs.append(offs[-1] + c)
        s['offsets'] = torch.tensor(offs, dtype=torch.int32, device=dev)
    s['x'] = torch.randn(rows, k, generator=gen, device=dev).bfloat16()
    s['w'] = (torch.randn(e, n, k, generator=gen, device=dev) * k ** -0.5).bfloat16()
    s['b'] = torch.randn(e, n, generator=gen, device=dev) * 0.02
    if case['train']:
        s['dy'] = (torch.randn(rows, n, generator=gen, device=dev) * 1e-2).bfloat16()
    return s


def _blocks(x):
    """[rows][k] as [rows][blocks][BLOCK], the last block filled with zeros."""
    rows, k = x.shape
    pad = -k % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).view(rows, (k + pad) // BLOCK, BLOCK)


def _scale_of(amax):
    """The scale of a block, amax / 448, and what its values are multiplied by; zero for a block below TINY."""
    live = amax >= TINY
    safe = torch.where(live, amax, torch.ones_like(amax))
    zero = torch.zeros_like(amax)
    return torch.where(live, safe * (1 / E4M3_MAX), zero), torch.where(live, safe.reciprocal() * E4M3_MAX, zero)


def _quantize_weight(w):
    """w [n][k] f32 -> e4m3 [n][kp] and scales [ceil(n / 128)][kp / 128]: a block is 128 x 128."""
    n, k = w.shape
    padded = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    tiles = padded.view(padded.shape[0] // BLOCK, BLOCK, padded.shape[1] // BLOCK, BLOCK)
    scale, inv = _scale_of(tiles.abs().amax((1, 3)))
    q = (tiles * inv[:, None, :, None]).reshape(padded.shape)[:n].to(torch.float8_e4m3fn)
    return q.contiguous(), scale.contiguous()


def _fp8_state(case, gen, dev):
    rows, k, n = case['rows'], case['k'], case['n']
    x = torch.randn(rows, k, generator=gen, device=dev)
    # a few channels of a transformer's activations are many times the others
    loud = torch.rand(k, generator=gen, device=dev) < 0.02
    x = (x * torch.where(loud, 12.0, 1.0)).bfloat16()
    wq, ws = _quantize_weight(torch.randn(n, k, generator=gen, device=dev) * 0.02)
    b = torch.randn(n, generator=gen, device=dev) * 0.02 if case['bias'] else None
    return dict(case=case, x=x, wq=wq, ws=ws, b=b)


def _adamw_state(case, gen, dev):
    """Flat buffers with every tensor at a multiple of 128 elements, the tables that drive a step over them, and moments
    as a hundred steps leave them."""
    sizes = _tensor_sizes(case)
    start, length, scale, decay, at = [], [], [], [], 0
    per_block_scale, per_block_decay = [], []
    for i, n in enumerate(sizes):
        blocks = -(-n // BLOCK)
        lr_scale, wd = 0.75 ** (i % 13), 0.0 if i % 2 else 0.1
        n4 = -(-n // 4) * 4
        for c in range(0, n4, 2048):
            start.append(at + c)
            length.append(min(2048, n4 - c))
            scale.append(lr_scale)
            decay.append(wd)
        per_block_scale.append((lr_scale, blocks))
        per_block_decay.append((wd, blocks))
        at += blocks * BLOCK
    total = at

    def per_block(pairs):
        return torch.repeat_interleave(torch.tensor([v for v, _ in pairs], device=dev),
                                       torch.tensor([c for _, c in pairs], device=dev))
    sizes_dev = torch.tensor(sizes, device=dev)
    begins = torch.cumsum((sizes_dev + BLOCK - 1) // BLOCK * BLOCK, 0) - (sizes_dev + BLOCK - 1) // BLOCK * BLOCK
    owner = torch.repeat_interleave(torch.arange(len(sizes), device=dev), (sizes_dev + BLOCK - 1) // BLOCK)
    within = (torch.arange(total // BLOCK, device=dev) * BLOCK - begins[owner])[:, None] + torch.arange(BLOCK, device=dev)
    inside = within < sizes_dev[owner][:, None]
    loud = torch.exp(1.5 * torch.randn(total // BLOCK, 1, generator=gen, device=dev)) * 1e-4

    def noise():
        return torch.randn(total // BLOCK, BLOCK, generator=gen, device=dev) * inside

    m, r = noise() * loud * 0.3, noise().abs() * loud + inside * loud * 0.1
    (ms, mi), (rs, ri) = _scale_of(m.abs().amax(1)), _scale_of(r.amax(1))
    state = (((m * mi[:, None]).to(torch.float8_e4m3fn)).view(-1), ms,
             torch.where(inside, (r * ri[:, None]).clamp_min(2.0 ** -9), torch.zeros_like(r)).to(torch.float8_e4m3fn).view(-1), rs)
    p = (noise() * 0.02).view(-1)
    grad = (noise() * loud).view(-1)
    start = torch.tensor(start, dtype=torch.int64, device=dev)
    chunks = (start, torch.tensor(length, dtype=torch.int32, device=dev), torch.tensor(scale, device=dev),
              torch.tensor(decay, device=dev), start)
    return dict(case=case, p=p, grad=grad, half=p.bfloat16(), state=state, chunks=chunks, scale=per_block(per_block_scale),
                decay=per_block(per_block_decay), noise=int(torch.randint(1 << 31, (1,), generator=gen, device=dev)))


# the schedule of the last epochs: base rate 5e-4 after its steps, layer decay in the tables
ADAM = dict(lr=1e-5, betas=(0.9, 0.999), eps=1e-8, step=100)
MAX_NORM = 1.0


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    return {'experts': _experts_state, 'fp8': _fp8_state, 'adamw8': _adamw_state}[case['kind']](case, gen, dev)


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_experts(s):
    case, x, w, out = s['case'], s['x'].float(), s['w'].float(), {}
    e, rows = case['experts'], case['rows']
    if case['order'] == 'ids':
        key = torch.where((s['ids'] >= 0) & (s['ids'] < e), s['ids'], torch.full_like(s['ids'], e))
        order = torch.argsort(key, stable=True)
        count = (key[:, None] == torch.arange(e, device=key.device)).sum(0)
        offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
        out['rows'], out['offsets'] = order.int(), offsets.int()
    else:
        order, offsets = torch.arange(rows, device=x.device), s['offsets'].long()
    # every expert's rows in a slab of the longest one's length
    place = offsets[:-1, None] + torch.arange(max(1, s['most']), device=x.device)
    valid = (place < offsets[1:, None])[..., None]
    take = order[place.clamp(max=rows - 1)]
    xs = x[take] * valid
    y = torch.bmm(xs, w.transpose(1, 2).contiguous()) + s['b'][:, None]
    # rows that no expert takes come out as zeros; slots behind an expert's rows go to a row of their own
    spot = torch.where(valid[..., 0], take, torch.full_like(take, rows)).view(-1)
    out['y'] = x.new_zeros(rows + 1, case['n']).index_copy_(0, spot, y.view(-1, case['n']))[:rows].bfloat16()
    if case['train']:
        dy = s['dy'].float()[take] * valid
        dx = torch.bmm(dy, w)
        out['dx'] = x.new_zeros(rows + 1, case['k']).index_copy_(0, spot, dx.view(-1, case['k']))[:rows].bfloat16()
        out['dw'] = torch.bmm(dy.transpose(1, 2).contiguous(), xs)
        out['db'] = dy.sum(1)
    return out


def _plain_fp8(s):
    case = s['case']
    blocks = _blocks(s['x'].float())
    scale, inv = _scale_of(blocks.abs().amax(2))
    q = (blocks * inv[..., None]).to(torch.float8_e4m3fn)
    x = (q.float() * scale[..., None]).view(case['rows'], -1)
    wide = s['ws'].repeat_interleave(BLOCK, 0)[:case['n']].repeat_interleave(BLOCK, 1)
    y = x @ (s['wq'].float() * wide).t()
    if s['b'] is not None:
        y = y + s['b']
    if case['act'] == 'gelu':
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    out = {'y': y.bfloat16()}
    if case['keep']:
        out.update(q=q.view(case['rows'], -1), scale=scale.t().contiguous())
    return out


def _mix32(h):
    """The 32-bit finalizer of MurmurHash3 on int64 tensors that hold 32-bit values."""
    low = 0xFFFFFFFF
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & low
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & low
    return h ^ (h >> 16)


def _uniform(total, noise, dev):
    """One number in [0, 1) for each element: 24 bits of a hash of its position and the step's key."""
    at = torch.arange(total, device=dev)
    return (_mix32((at & 0xFFFFFFFF) ^ noise) >> 8).float() * 2.0 ** -24


def _plain_adamw(s):
    lr, (b1, b2), eps, step = ADAM['lr'], ADAM['betas'], ADAM['eps'], ADAM['step']
    m8, ms, r8, rs = s['state']
    p, g = s['p'].view(-1, BLOCK), s['grad'].view(-1, BLOCK)
    if s['case']['clip']:
        norm = g.square().sum(dtype=torch.float64).sqrt().float()
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    lr_c = lr * s['scale'][:, None]
    m, r = m8.view(-1, BLOCK).float() * ms[:, None], r8.view(-1, BLOCK).float() * rs[:, None]
    m = m + (1 - b1) * (g - m)
    v = b2 * (r * r) + ((1 - b2) * g) * g
    r = v.sqrt()
    new = p * (1 - lr_c * s['decay'][:, None]) - ((lr_c / (1 - b1 ** step)) * m) / (r / math.sqrt(1 - b2 ** step) + eps)
    ms_new, mi = _scale_of(m.abs().amax(1))
    rs_new, ri = _scale_of(r.amax(1))
    # the root of the second moment goes to one of its two neighbours, up with the probability that keeps its square
    x = torch.clamp(r * ri[:, None], max=E4M3_MAX)
    low = torch.where(x >= 2.0 ** -6, (x.view(torch.int32) & -0x100000).view(torch.float32), torch.floor(x * 512) / 512)
    high = torch.where(x >= 2.0 ** -6, ((x.view(torch.int32) & -0x100000) + 0x100000).view(torch.float32), low + 1 / 512)
    up = _uniform(p.numel(), s['noise'], p.device).view(-1, BLOCK) * (high * high - low * low) < x * x - low * low
    q = torch.where(up, high, low)
    q = torch.where(x > 0, q.clamp(2.0 ** -9, E4M3_MAX), torch.zeros_like(q))
    s['p'].copy_(new.view(-1))
    s['half'].copy_(new.view(-1))
    m8.copy_((m * mi[:, None]).view(-1))
    ms.copy_(ms_new)
    r8.copy_(q.view(-1))
    rs.copy_(rs_new)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return dict(p=s['p'], half=s['half'], exp_avg=s['state'][0], exp_avg_scale=s['state'][1], exp_avg_sq_root=s['state'][2],
                exp_avg_sq_scale=s['state'][3])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_experts(s):
    from vitpose_amd import experts
    out, rows = {}, None
    if s['case']['order'] == 'ids':
        rows, offsets = experts.expert_rows(s['ids'], s['case']['experts'])
        out['rows'], out['offsets'] = rows, offsets
    else:
        offsets = s['offsets']
    out['y'] = experts.grouped_linear(s['x'], s['w'], s['b'], offsets, rows)
    if s['case']['train']:
        out['dx'] = experts.grouped_linear_dgrad(s['dy'], s['w'], offsets, rows)
        out['dw'], out['db'] = experts.grouped_linear_wgrad(s['dy'], s['x'], offsets, rows)
    return out


def _own_fp8(s):
    from vitpose_amd import fp8
    act = s['case']['act'] or None
    if s['case']['keep']:
        q, scale = fp8.quantize_rows(s['x'])
        return {'y': fp8.product(q, scale, s['wq'], s['ws'], s['b'], act=act), 'q': q, 'scale': scale}
    return {'y': fp8.linear(s['x'], s['wq'], s['ws'], s['b'], act=act)}


def _own_adamw(s):
    from vitpose_amd import optim
    optim.adamw8_step(s['p'], s['grad'], s['state'], s['chunks'], half=s['half'], noise=s['noise'],
                      max_grad_norm=MAX_NORM if s['case']['clip'] else 0.0, **ADAM)
    return _adamw_outputs(s)


def run(state):
    kind = state['case']['kind']
    if own:
        return {'experts': _own_experts, 'fp8': _own_fp8, 'adamw8': _own_adamw}[kind](state)
    return {'experts': _plain_experts, 'fp8': _plain_fp8, 'adamw8': _plain_adamw}[kind](state)


# ------------------------------------------------------------------------------------------------ work and exact values
def work(case):
    if case['kind'] == 'experts':
        counts, none = _shares(case)
        live, hit = sum(counts), sum(c > 0 for c in counts)
        k, n, e, rows = case['k'], case['n'], case['experts'], case['rows']
        moved = 2 * live * k + 2 * hit * k * n + 4 * hit * n + 2 * rows * n + (4 * rows if case['order'] == 'ids' else 0)
        flops = 2 * live * k * n
        if case['train']:
            moved += 2 * live * n + 2 * rows * k + 4 * e * n * (k + 1)
            flops *= 3
        return {'bytes': moved, 'flops': flops}
    if case['kind'] == 'fp8':
        m, k, n = case['rows'], case['k'], case['n']
        kp = -(-k // BLOCK) * BLOCK
        moved = 2 * m * k + n * kp + 4 * -(-n // BLOCK) * (kp // BLOCK) + 2 * m * n + (4 * n if case['bias'] else 0)
        if case['keep']:
            moved += m * kp + 4 * m * (kp // BLOCK)
        return {'bytes': moved, 'flops': 2 * m * k * n}
    n = sum(_tensor_sizes(case))
    return {'bytes': 18 * n + 16 * (n // BLOCK), 'flops': 20 * n}


def _e4m3_64(x):
    """The e4m3 number nearest to each value of |x| <= 448, ties to the even one, in 64 bits."""
    _, power = torch.frexp(x)
    step = torch.exp2((power - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def _scale_64(amax):
    ones = torch.where(amax < TINY, torch.ones_like(amax), amax)
    return torch.where(amax < TINY, torch.zeros_like(amax), ones / E4M3_MAX), ones / E4M3_MAX


def _exact_experts(case, s):
    x, w, b = s['x'].double(), s['w'].double(), s['b'].double()
    rows, e = case['rows'], case['experts']
    y = x.new_zeros(rows, case['n'])
    out = {'y': y}
    if case['train']:
        dy = s['dy'].double()
        out.update(dx=torch.zeros_like(x), dw=torch.zeros_like(w), db=torch.zeros_like(b))
    if case['order'] == 'ids':
        member = [torch.nonzero(s['ids'] == i).flatten() for i in range(e)]
        rest = torch.nonzero((s['ids'] < 0) | (s['ids'] >= e)).flatten()
        out['rows'] = torch.cat(member + [rest]).int()
        out['offsets'] = torch.tensor([sum(m.numel() for m in member[:i]) for i in range(e + 1)], dtype=torch.int32)
    else:
        at = s['offsets'].tolist()
        member = [torch.arange(at[i], at[i + 1], device=x.device) for i in range(e)]
    for i, mine in enumerate(member):
        if mine.numel():
            y[mine] = x[mine] @ w[i].t() + b[i]
            if case['train']:
                out['dx'][mine] = dy[mine] @ w[i]
                out['dw'][i] = dy[mine].t() @ x[mine]
                out['db'][i] = dy[mine].sum(0)
    return out


def _exact_fp8(case, s):
    x = s['x'].double()
    k, kp = case['k'], s['wq'].shape[1]
    full = x.new_zeros(case['rows'], kp)
    full[:, :k] = x
    parts = full.split(BLOCK, 1)
    scales = [_scale_64(c.abs().max(1).values) for c in parts]
    qs = [_e4m3_64(c / d[:, None]) for c, (_, d) in zip(parts, scales)]
    y = x.new_zeros(case['rows'], case['n'])
    for i, (q, (sc, _)) in enumerate(zip(qs, scales)):
        wb = s['wq'][:, i * BLOCK:(i + 1) * BLOCK].double()
        for j in range(s['ws'].shape[0]):
            cols = slice(j * BLOCK, min((j + 1) * BLOCK, case['n']))
            y[:, cols] += (q @ wb[cols].t()) * sc[:, None] * s['ws'][j, i].double()
    if s['b'] is not None:
        y += s['b'].double()
    if case['act'] == 'gelu':
        y = y * torch.special.ndtr(y)
    out = {'y': y}
    if case['keep']:
        out.update(q=torch.cat(qs, 1), scale=torch.stack([sc for sc, _ in scales]))
    return out


def _exact_adamw(case, s):
    lr, (b1, b2), eps, t = ADAM['lr'], ADAM['betas'], ADAM['eps'], ADAM['step']
    m8, ms, r8, rs = s['state']
    shape = (-1, BLOCK)
    g = s['grad'].double().view(shape)
    if case['clip']:
        g = g * min(1.0, MAX_NORM / (float(torch.linalg.vector_norm(g)) + 1e-6))
    rate = (lr * s['scale'].double())[:, None]
    m = b1 * (m8.view(shape).double() * ms.double()[:, None]) + (1 - b1) * g
    v = b2 * (r8.view(shape).double() * rs.double()[:, None]) ** 2 + (1 - b2) * g ** 2
    p = s['p'].double().view(shape)
    p = p - rate * s['decay'].double()[:, None] * p - rate * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    m_scale, m_div = _scale_64(m.abs().max(1).values)
    r_scale, r_div = _scale_64(v.max(1).values.sqrt())
    x = v.sqrt() / r_div[:, None]
    step = torch.exp2((torch.frexp(x)[1] - 1).clamp(min=-6).double() - 3)
    low = torch.floor(x / step) * step
    u = (_mix32(torch.arange(p.numel(), device=p.device) ^ s['noise']) >> 8).double().view(shape) * 2.0 ** -24
    q = torch.where(u < (x ** 2 - low ** 2) / ((low + step) ** 2 - low ** 2), low + step, low).clamp(2.0 ** -9, E4M3_MAX)
    q = torch.where(x > 0, q, torch.zeros_like(q))
    flat = p.reshape(-1)
    return dict(p=flat, half=flat, exp_avg=_e4m3_64(m / m_div[:, None]).reshape(-1), exp_avg_scale=m_scale,
                exp_avg_sq_root=q.reshape(-1), exp_avg_sq_scale=r_scale)


def exact(case, seed):
    s = prepare(case, seed)
    return {'experts': _exact_experts, 'fp8': _exact_fp8, 'adamw8': _exact_adamw}[case['kind']](case, s)
