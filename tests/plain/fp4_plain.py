"""Weights in 4 bits by their definition, in float64 on the CPU: what packing gives, and a bound on the rounding of a product's sums."""
import torch

MAGNITUDES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def values(w: torch.Tensor, group: int) -> torch.Tensor:
    """The values that a packed w [..., K] stands for, float64."""
    w = w.detach().cpu().double()
    out = torch.empty_like(w)
    for k0 in range(0, w.shape[-1], group):
        part = w[..., k0:k0 + group]
        most = part.abs().amax(-1, keepdim=True)
        most = torch.where(part.isnan().any(-1, keepdim=True), torch.full_like(most, float("nan")), most)
        m, e = torch.frexp(most / 6)
        scale = torch.ldexp(torch.round(m * 64) / 64, e)                 # six significant bits, ties to even
        scale = torch.where(most.isfinite(), scale, torch.full_like(scale, float("nan")))
        far = (part.abs().unsqueeze(-1) - scale.unsqueeze(-1) * MAGNITUDES).abs()
        # the nearest magnitude; of two equally near the one with the even code
        near = far.amin(-1, keepdim=True)
        ties = far == near
        code = torch.where(ties & (torch.arange(8) % 2 == 0), torch.arange(8) + 100, torch.where(ties, torch.arange(8), torch.tensor(-1))).argmax(-1)
        value = MAGNITUDES[code] * scale * torch.sign(part)
        out[..., k0:k0 + group] = torch.where(scale > 0, value, torch.where(scale == 0, torch.zeros_like(value), torch.full_like(value, float("nan"))))
    return out


def sum_bound(x: torch.Tensor, w: torch.Tensor, group: int) -> torch.Tensor:
    """How far a 32-bit sum of x w^T may be off, [rows, N]: the products are exact, a group's are added one by one, then the groups; an
    addition of the matrix cores is taken to be off by a whole last place (2^-23 of the sum so far, which the sum of magnitudes bounds)."""
    depth = group + -(-w.shape[-1] // group) + 16
    return depth * 2.0 ** -23 * (x.double().cpu().abs() @ w.double().cpu().abs().T)


def act(z: torch.Tensor, alpha=1.0, limit=0.0, shift=0.0) -> torch.Tensor:
    g, u = z[..., 0::2], z[..., 1::2]
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g / (1 + torch.exp(-alpha * g)) * (u + shift)
