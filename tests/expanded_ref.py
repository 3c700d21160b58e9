"""The expanded form of latent attention in 64 bits, and bounds of what 16-bit kernels may differ by.

attention() gives, for the keys and values rounded to the type (as the operator's definition has
them), the outputs and three sums of each that the bounds below are made of.

Bounds, with u = eps / 2 of the type, for weights p (sum 1), values v and outputs o = sum p v:
  a key's component rounded to a neighbour of its own nearest (the float32 sum in front of that
  rounding is not the 64-bit one) is off by at most 2 u relative, so a score by at most
  e = 2 u sum |q k| / scale, the weight by a factor within exp(+-e); a value likewise by 2 u; the
  rounding of the weights gives u; sums in float32 are below u / 16 for up to 2^12 terms.  So
    |o' - o| <= sum p |v| (2 (exp(e) - 1) + 4 u) + 2 u |o|     for each output (`worst`), and
  as those roundings are rare and zero in the mean, while the weights' and the output's, each at
  most u, are everywhere and independent, in the 2-norm over many outputs
    |o' - o|_2 <= | sqrt(sum (p v)^2) u |_2 + u |o|_2          (`usual`; the factor sqrt(3) between
  a rounding's largest and its root mean square is the room for the rare ones).
fp16 weights below 2^-22 of the row's largest are rounded to multiples of 2^-33 of it, at most.
"""

from __future__ import annotations

import math

import torch


def attention(q_nope, q_rope, lat, rot, W_uk, W_uv, scale, lims, dtype):
    """One sequence: q_* [n, H, .], lat [keys, 512], rot [keys, 64], query i sees keys <= lims[i].
    Returns out, worst, usual [n, H, 128] in float64."""
    u = torch.finfo(dtype).eps / 2
    dev = q_nope.device
    n, H, _ = q_nope.shape
    keys = lat.size(0)
    out = torch.zeros(n, H, 128, dtype=torch.float64, device=dev)
    worst, usual = torch.zeros_like(out), torch.zeros_like(out)
    if keys == 0:
        return out, worst, usual
    hide = torch.arange(keys, device=dev)[None] > torch.as_tensor(lims, device=dev)[:, None]
    r = rot.double()
    for h in range(H):
        k = (lat.double() @ W_uk[h].double().t()).to(dtype).double()
        v = (lat.double() @ W_uv[h].double().t()).to(dtype).double()
        q, qr = q_nope[:, h].double(), q_rope[:, h].double()
        t = ((q @ k.t() + qr @ r.t()) / scale).masked_fill(hide, -math.inf)
        p = torch.softmax(t, -1).nan_to_num()
        e = 2 * u * (q.abs() @ k.abs().t()) / scale
        o = p @ v
        out[:, h] = o
        g = p * (2 * torch.expm1(e) + 4 * u)
        worst[:, h] = g @ v.abs() + 2 * u * o.abs() + keys * 2.0 ** -33 * v.abs().amax()
        usual[:, h] = u * ((p * p) @ (v * v)).sqrt() + u * o.abs()
    return out, worst, usual


def check(got, out, worst, usual, name=""):
    d = (got.double() - out).abs()
    assert torch.isfinite(got).all(), name
    assert (d <= worst).all(), f"{name}: {(d - worst).max().item():.3e} past the bound"
    total, most = d.norm().item(), usual.norm().item()
    assert total <= most, f"{name}: distance {total:.3e}, at most {most:.3e}"


def limits(Sq, length, new, causal):
    """What each of the last `new` rows sees (largest key index)."""
    return [min(length - Sq + i, length - 1) if causal else length - 1 for i in range(Sq - new, Sq)]
