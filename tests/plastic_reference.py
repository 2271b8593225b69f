"""The gated delta rule token by token in 64 bits, on the CPU, with gradients by autograd."""
import torch


def delta_rule(q, k, v, g, beta, scale, initial=None, lengths=None):
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    S = torch.zeros(B, Hv, dk, dv, dtype=torch.float64) if initial is None else initial
    head = torch.arange(Hv) // (Hv // Hk)
    live = torch.ones(B, T, dtype=torch.bool) if lengths is None else torch.arange(T) < lengths.view(-1, 1)
    out = []
    for t in range(T):
        m = live[:, t].view(B, 1, 1)
        kt = torch.where(m, k[:, t, head], 0.)
        qt = torch.where(m, q[:, t, head], 0.)
        vt = torch.where(m, v[:, t], 0.)
        a = torch.where(m[..., 0], torch.exp(g[:, t]), 1.).view(B, Hv, 1, 1)
        b = torch.where(m[..., 0], beta[:, t], 0.).unsqueeze(-1)
        S = a * S
        u = b * (vt - (kt.unsqueeze(-2) @ S).squeeze(-2))
        S = S + kt.unsqueeze(-1) * u.unsqueeze(-2)
        out.append(scale * (qt.unsqueeze(-2) @ S).squeeze(-2))
    o = torch.stack(out, 1) if T else torch.zeros(B, 0, Hv, dv, dtype=torch.float64)
    return o, S


def inputs(B, T, Hk, Hv, dk, dv, dtype, seed=0, state=True, alike=0.0):
    """Unit keys (``alike`` > 0: with a common part), decays of several strengths, learning rates in (0, 1)."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    q, k = unit(n(B, T, Hk, dk)), unit(n(B, T, Hk, dk) + alike * n(Hk, dk))
    g = -torch.exp(n(Hv) - 3) * torch.nn.functional.softplus(n(B, T, Hv))
    args = {'q': q.to(dtype), 'k': k.to(dtype), 'v': n(B, T, Hv, dv).to(dtype), 'g': g.float(),
            'beta': torch.sigmoid(n(B, T, Hv)).float()}
    if state:
        args['initial'] = (0.3 * n(B, Hv, dk, dv)).float()
    return args


def error(x, y):
    """2-norm of the difference over that of the reference ``y``."""
    x, y = x.detach().cpu().double(), y.detach().double()
    if not torch.equal(torch.isfinite(x), torch.isfinite(y)):
        return float('inf')
    return float((x - y).norm() / y.norm().clamp_min(1e-30)) if y.numel() else 0.0
