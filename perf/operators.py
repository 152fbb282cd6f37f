"""Cases, plain forms and 64-bit values of the channel-mixing products: the products grouped by expert with their
gradients, and the 8-bit integer product with a scale per row and per channel.

A case's `op` is 'fwd' (the grouped product), 'train' (the product and both of its gradients) or 'int8' (rows
quantised to 8 bits, multiplied with 8-bit weights, scaled back).  `rows` rows of `k` values meet `experts` weight
matrices of `n` x `k`; the rows are sorted by expert, `ends` holds the cumulative row counts, and the last `behind`
rows belong to no expert (their results are zero).
"""
import math

import torch

own = False

DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def listed():
    return [
        # one token sent to 8 of 64 experts while it is being generated: latency and the weights' bytes
        dict(name='fwd token', op='fwd', dtype='bf16', rows=8, experts=64, k=2048, n=1024, behind=0),
        # a batch of 64 tokens sent to 8 experts each: every expert's weights are read for a handful of rows
        dict(name='fwd batch', op='fwd', dtype='bf16', rows=512, experts=64, k=2048, n=1024, behind=0),
        # the experts of a long prompt: bound by the tensor cores
        dict(name='fwd prompt', op='fwd', dtype='bf16', rows=32768, experts=16, k=2048, n=4096, behind=0),
        # the pointwise product behind a depthwise convolution of the benchmark's (1, 64, 350, 350, 128) volume
        dict(name='fwd volume', op='fwd', dtype='fp16', rows=350 * 350 * 128, experts=1, k=64, n=64, behind=0),
        # a training step of small odd sizes, with rows that no expert takes
        dict(name='train odd', op='train', dtype='fp16', rows=1003, experts=5, k=203, n=77, behind=9),
        # a training step of a mixture-of-experts layer
        dict(name='train experts', op='train', dtype='bf16', rows=16384, experts=32, k=1024, n=2048, behind=0),
        # a training step of the pointwise product on 100 planes of 350 x 128 voxels
        dict(name='train volume', op='train', dtype='fp16', rows=100 * 350 * 128, experts=1, k=32, n=64, behind=0),
        # one token while it is being generated, weights held in 8 bits
        dict(name='int8 token', op='int8', dtype='bf16', rows=1, experts=1, k=4096, n=4096, behind=0),
        # 64 sequences, a token each
        dict(name='int8 batch', op='int8', dtype='bf16', rows=64, experts=1, k=4096, n=8192, behind=0),
        # a long prompt: bound by the tensor cores
        dict(name='int8 prompt', op='int8', dtype='bf16', rows=8192, experts=1, k=4096, n=8192, behind=0),
        # experts whose weights are held in 8 bits
        dict(name='int8 experts', op='int8', dtype='fp16', rows=4096, experts=32, k=1024, n=2048, behind=5),
        # sizes that are multiples of nothing
        dict(name='int8 odd', op='int8', dtype='fp16', rows=777, experts=1, k=1001, n=333, behind=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['fwd', 'train', 'int8'])
    dtype = rng.choice(['fp16', 'bf16'])
    while True:
        if op != 'int8' and rng.random() < 0.3:  # a volume's voxels as rows, few channels
            rows, experts, behind = _log(rng, 20000, 15000000), 1, 0
            k, n = rng.choice([8, 16, 32, 64, 128]), rng.choice([8, 16, 32, 64, 128])
        else:
            rows, experts = _log(rng, 1, 32768), rng.choice([1, 1, 2, 5, 8, 16, 32, 64])
            k, n = _log(rng, 16, 4096), _log(rng, 16, 8192)
            step = rng.choice([1, 8, 64])  # odd, aligned and round sizes
            k, n = max(step, k // step * step), max(step, n // step * step)
            behind = rng.choice([0, 0, rng.randint(0, rows // 8)]) if experts > 1 else 0
        case = dict(op=op, dtype=dtype, rows=rows, experts=experts, k=k, n=n, behind=behind)
        w = work(case)
        if w['flops'] <= 5e11 and w['bytes'] <= 4e9 and experts * k * n <= 3e8:
            return case


def _ends(case, seed):
    """Cumulative row ends: few rows go to experts of their own, as a token's do; more rows in unequal shares."""
    g = torch.Generator().manual_seed(seed)
    rows, experts = case['rows'] - case['behind'], case['experts']
    if experts == 1:
        return [rows]
    if rows <= experts:
        counts = torch.zeros(experts, dtype=torch.int64)
        counts[torch.randperm(experts, generator=g)[:rows]] = 1
    else:
        share = torch.rand(experts, generator=g) + 0.2
        counts = torch.floor(share / share.sum() * rows).to(torch.int64)
        counts[int(torch.randint(experts, (1,), generator=g))] += rows - int(counts.sum())
    return torch.cumsum(counts, 0).tolist()


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    rows, experts, k, n = case['rows'], case['experts'], case['k'], case['n']

    def normal(*shape, type=dtype):
        return torch.randn(*shape, generator=g, device='cuda', dtype=type)

    s = dict(op=case['op'], dtype=dtype, x=normal(rows, k), host_ends=_ends(case, seed))
    s['ends'] = torch.tensor(s['host_ends'], dtype=torch.int32, device='cuda') if experts > 1 else None
    if case['op'] == 'int8':
        w = normal(experts, n, k, type=torch.float32)
        top = w.abs().amax(2, keepdim=True)
        s['w'] = torch.round(w * 127 / top).to(torch.int8)
        s['w_scale'] = (top / 127 / math.sqrt(k)).squeeze(2).contiguous()
    else:
        s['w'] = (normal(experts, n, k) / math.sqrt(k)).to(dtype)
    if case['op'] == 'train':
        s['grad'] = normal(rows, n)
        s['x'].requires_grad_(True)
        s['w'].requires_grad_(True)
    return s


def _groups(ends):
    """(expert, first row, end row) of the experts that have rows."""
    return [(e, a, b) for e, (a, b) in enumerate(zip([0] + ends, ends)) if b > a]


def _fwd(x, w, ends):
    y = x.new_zeros(x.shape[0], w.shape[1])
    for e, a, b in _groups(ends):
        y[a:b] = (x[a:b].float() @ w[e].float().T).to(x.dtype)
    return y


def _train(x, w, grad, ends):
    x, w = x.detach(), w.detach()
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for e, a, b in _groups(ends):
        g = grad[a:b].float()
        dx[a:b] = (g @ w[e].float()).to(x.dtype)
        dw[e] = (g.T @ x[a:b].float()).to(w.dtype)
    return _fwd(x, w, ends), dx, dw


def _int8(x, w, w_scale, ends):
    # 127 x is exact in 32 bits and the rounded quotient never crosses a half, so q is the exact one; the integer
    # sums pass 2^24 and are taken in 64 bits
    f = x.float()
    top = f.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(f * 127 / top), 0.0)
    scale = top / 127
    y = x.new_zeros(x.shape[0], w.shape[1])
    for e, a, b in _groups(ends):
        sums = (q[a:b].double() @ w[e].double().T).float()
        y[a:b] = (sums * scale[a:b] * w_scale[e]).to(x.dtype)
    return y


def run(state):
    s = state
    if own:
        if s['op'] == 'int8':
            from kerops_b200.ops.linear import Int8Linear

            return Int8Linear(s['x'], s['w'], s['w_scale'], s['ends'])
        if s['op'] == 'fwd':
            from kerops_b200.ops.linear import GroupedLinear

            return GroupedLinear(s['x'], s['w'], s['ends'])
        from kerops_b200.autograd import grouped_linear

        y = grouped_linear(s['x'], s['w'], s['ends'])
        dx, dw = torch.autograd.grad(y, (s['x'], s['w']), s['grad'])
        return y.detach(), dx, dw
    if s['op'] == 'int8':
        return _int8(s['x'], s['w'], s['w_scale'], s['host_ends'])
    if s['op'] == 'fwd':
        return _fwd(s['x'], s['w'], s['host_ends'])
    return _train(s['x'], s['w'], s['grad'], s['host_ends'])


def work(case):
    t, e, k, n = case['rows'], case['experts'], case['k'], case['n']
    live = t - case['behind']
    used = min(e, live)  # experts that can have rows
    if case['op'] == 'int8':
        return dict(bytes=2 * live * k + 2 * t * n + used * n * k + 4 * used * n, flops=2 * live * n * k)
    if case['op'] == 'fwd':
        return dict(bytes=2 * (live * k + t * n + used * n * k), flops=2 * live * n * k)
    # y, dx and dw are written whole; x, the weights and the gradient are read once
    return dict(bytes=2 * (live * k + live * n + used * n * k + t * n + t * k + e * n * k), flops=6 * live * n * k)


def exact(case, seed):
    s = prepare(case, seed)
    x, w = s['x'].detach().double(), s['w'].detach()
    t, n, k = case['rows'], case['n'], case['k']
    y = torch.zeros(t, n, dtype=torch.float64, device='cuda')
    if case['op'] == 'int8':
        top = x.abs().max(dim=1).values
        q = torch.round(x * (127 / torch.where(top == 0, 1.0, top))[:, None])
        # the quotient in 64 bits is within 2^-45 of the true one; a half is hit exactly or missed by 2^-20 or more
        near = x * 127 / torch.where(top == 0, 1.0, top)[:, None]
        q = torch.where((near - torch.floor(near) - 0.5).abs() < 2.0 ** -30, 2 * torch.round(near / 2), q)
    start = 0
    out = [y]
    if case['op'] == 'train':
        g = s['grad'].double()
        dx = torch.zeros(t, k, dtype=torch.float64, device='cuda')
        dw = torch.zeros(case['experts'], n, k, dtype=torch.float64, device='cuda')
        out = [y, dx, dw]
    for e, end in enumerate(s['host_ends']):
        r = slice(start, end)
        start = end
        if case['op'] == 'int8':
            y[r] = torch.einsum('tk,nk->tn', q[r], w[e].double()) * (top[r] / 127)[:, None] * s['w_scale'][e].double()
            continue
        we = w[e].double()
        y[r] = torch.einsum('tk,nk->tn', x[r], we)
        if case['op'] == 'train':
            dx[r] = torch.einsum('tn,nk->tk', g[r], we)
            dw[e] = torch.einsum('tn,tk->nk', g[r], x[r])
    return y if len(out) == 1 else tuple(out)
