"""Plain 64-bit forms of the channel-mixing products, and inputs on which every order of summation is exact."""
import torch


def integers(shape, dtype, seed, top=2, device='cuda'):
    """Small whole numbers: products and sums of up to 2^24 / top^2 of them are exact in fp32 in any order, so a result
    equals the plain form's rounded once, bit for bit."""
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g, device=device).to(dtype)


def spans(ends, T):
    """Row ranges of the groups; ends that step back or pass T are clamped."""
    out, begin = [], 0
    for e in ends:
        end = min(max(begin, e), T)
        out.append((begin, end))
        begin = end
    return out


def fwd(x, w, ends):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    for e, (a, b) in enumerate(spans(ends, x.shape[0])):
        y[a:b] = x[a:b].double() @ w[e].double().T
    return y


def dgrad(g, w, ends):
    dx = torch.zeros(g.shape[0], w.shape[2], dtype=torch.float64, device=g.device)
    for e, (a, b) in enumerate(spans(ends, g.shape[0])):
        dx[a:b] = g[a:b].double() @ w[e].double()
    return dx


def wgrad(x, g, ends):
    dw = torch.zeros(len(ends), g.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    for e, (a, b) in enumerate(spans(ends, x.shape[0])):
        dw[e] = g[a:b].double().T @ x[a:b].double()
    return dw


def tensor_ends(ends):
    return torch.tensor(ends, dtype=torch.int32, device='cuda')


# (operation, variant, T, E, K, N): for every kernel variant of kdw_linear_auto_variant, sizes that get it on 148 SMs.
# Operation 0 to 2: KDW_LINEAR_FWD, DGRAD, WGRAD; 3: the 8-bit product.
VARIANTS = [
    (0, 1, 9, 3, 72, 40),
    (3, 1, 9, 3, 80, 40),
    (0, 2, 17, 1, 24, 24),
    (0, 1128064, 17, 2, 24, 24),
    (0, 1128128, 8548, 32, 24, 24),
    (0, 1128256, 16961, 32, 24, 24),
    (0, 1256256, 2556, 32, 24, 2592),
    (0, 2128064, 17, 3, 1368, 24),
    (0, 2128128, 4970, 1, 2128, 24),
    (0, 2128256, 9614, 3, 2040, 24),
    (0, 2256256, 4325, 32, 1416, 168),
    (0, 4128064, 17, 1, 1528, 24),
    (0, 4128128, 1100, 32, 2504, 24),
    (0, 4128256, 4839, 1, 2032, 24),
    (0, 4256256, 2485, 1, 2064, 144),
    (0, 8128064, 17, 2, 5536, 24),
    (0, 8128128, 768, 8, 8016, 24),
    (0, 8128256, 2105, 3, 8728, 24),
    (1, 2, 17, 1, 24, 24),
    (1, 1128064, 17, 3, 24, 24),
    (1, 1128128, 8585, 32, 24, 24),
    (1, 1128256, 17155, 32, 24, 24),
    (1, 1256256, 777, 8, 9536, 24),
    (1, 2128064, 18, 1, 24, 1408),
    (1, 2128128, 4520, 8, 24, 2152),
    (1, 2128256, 8546, 32, 24, 2048),
    (1, 2256256, 4771, 2, 136, 1416),
    (1, 4128064, 17, 1, 24, 1416),
    (1, 4128128, 1114, 32, 24, 2048),
    (1, 4128256, 3761, 32, 24, 2384),
    (1, 4256256, 2173, 8, 152, 1960),
    (1, 8128064, 17, 1, 24, 5928),
    (1, 8128128, 838, 8, 24, 7944),
    (1, 8128256, 1935, 8, 24, 8912),
    (2, 1128064, 17, 8, 24, 24),
    (2, 1128128, 23, 32, 264, 24),
    (2, 1128256, 18, 32, 576, 24),
    (2, 1256256, 22, 32, 2360, 136),
    (2, 2128064, 10873, 8, 24, 24),
    (2, 2128128, 2119, 1, 5456, 24),
    (2, 2128256, 2042, 1, 9744, 24),
    (2, 2256256, 1364, 1, 5232, 136),
    (2, 4128064, 11311, 8, 24, 24),
    (2, 4128128, 1957, 1, 2136, 24),
    (2, 4128256, 73470, 32, 136, 24),
    (2, 4256256, 4020, 2, 1160, 144),
    (2, 8128128, 8138, 1, 1544, 24),
    (2, 8128256, 7955, 1, 3008, 24),
    (2, 16128064, 1223, 1, 24, 24),
    (2, 16128128, 115491, 1, 72, 24),
    (2, 16128256, 231060, 3, 136, 24),
    (2, 16256256, 71659, 1, 160, 144),
    (2, 32128064, 8362, 1, 24, 24),
    (2, 32128128, 237740, 1, 40, 24),
    (2, 32128256, 9732, 1, 3552, 24),
    (3, 1128064, 17, 3, 24, 24),
    (3, 1128128, 8484, 32, 24, 24),
    (3, 1128256, 16926, 32, 24, 24),
    (3, 1256256, 638, 8, 24, 11160),
    (3, 2128064, 18, 3, 2776, 24),
    (3, 2128128, 4926, 1, 4232, 24),
    (3, 2128256, 9872, 2, 4024, 24),
    (3, 2256256, 4800, 8, 2760, 160),
    (3, 4128064, 17, 2, 2992, 24),
    (3, 4128128, 1147, 32, 3960, 24),
    (3, 4128256, 4105, 32, 4000, 24),
    (3, 4256256, 2454, 2, 3936, 136),
    (3, 8128064, 18, 1, 10864, 24),
]


def uneven_ends(T, E):
    """Groups of different sizes, some without rows, the last rows in no group."""
    if E == 1:
        return [T - min(T - 1, 3)]
    g = torch.Generator().manual_seed(T + E)
    share = torch.rand(E, generator=g) ** 2
    share[E // 2] = 0
    ends = torch.cumsum(share / share.sum() * (T - min(T - 1, 3)), 0).to(torch.int64).tolist()
    return ends
