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
