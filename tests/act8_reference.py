"""Plain 64-bit statements of the 8-bit checkpoint format and of the residual norms, for the tests."""
import torch

GROUP = 32


def quantise(x):
    """float64 [rows, d] -> (values float64 [rows, d], scale bytes uint8 [rows, ceil(d / 32)])."""
    x = x.double()
    rows, d = x.shape
    g = torch.nn.functional.pad(x, (0, -d % GROUP)).reshape(rows, -1, GROUP)
    fin = torch.isfinite(g)
    amax = torch.where(fin, g.abs(), torch.zeros_like(g)).amax(-1)
    m, e = torch.frexp(amax / 448.0)                       # amax / 448 = m 2^e, 1/2 <= m < 1; smallest 2^k >= it
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(amax == 0, torch.full_like(e, -117), e).clamp(-117, 119)
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double()).unsqueeze(-1)
    v = (g / s).clamp(-448.0, 448.0)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    q = torch.round(v / step) * step                       # torch.round: ties to even
    q = torch.where(fin, q, torch.full_like(q, float("nan")))
    return (q * s).reshape(rows, -1)[:, :d], (e + 127).to(torch.uint8)


def values(act):
    """float64 values of an Act8, decoded on the CPU."""
    q = act.q.detach().cpu().float().double()
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), act.scale.detach().cpu().view(torch.uint8).double() - 127.0)
    return (q * s.repeat_interleave(GROUP, 1))[:, :act.d]


def norm_fwd(x, res, gamma, beta, kind, eps):
    """-> dict of float64 s, mu, rstd, n, y."""
    s = x.double() if res is None else x.double() + res.double()
    mu = s.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(s[:, :1])
    rstd = 1.0 / torch.sqrt(((s - mu) ** 2).mean(1, keepdim=True) + eps)
    n = (s - mu) * rstd
    y = n if gamma is None else n * gamma.double()
    if beta is not None:
        y = y + beta.double()
    return dict(s=s, mu=mu[:, 0], rstd=rstd[:, 0], n=n, y=y)


def norm_bwd(dy, n, rstd, gamma, kind, dx_in):
    """-> dict of float64 dx, dgamma, dbeta and the sizes of the terms that dx is made of."""
    dy, n, rstd = dy.double(), n.double(), rstd.double()[:, None]
    h = dy if gamma is None else dy * gamma.double()
    c1 = h.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(rstd)
    c2 = (h * n).mean(1, keepdim=True)
    dx = rstd * (h - c1 - n * c2)
    size = rstd * (h.abs() + h.abs().mean(1, keepdim=True) + n.abs() * (h * n).abs().mean(1, keepdim=True))
    if dx_in is not None:
        dx = dx + dx_in.double()
        size = size + dx_in.double().abs()
    return dict(dx=dx, size=size, dgamma=(dy * n).sum(0), dgamma_size=(dy * n).abs().sum(0), dbeta=dy.sum(0), dbeta_size=dy.abs().sum(0))


def gelu(z):
    z = z.double()
    cdf = 0.5 * torch.erfc(-z / 2 ** 0.5)
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
