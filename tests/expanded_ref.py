"""The expanded form of latent attention in 64 bits, and bounds of what the kernels may differ by.

attention() gives the exact outputs for 16-bit inputs and two bounds of each output.  What is rounded on
the way: keys, values and weights p (sum 1, values v, outputs o = sum p v) to 11 bits, each by at most
h = 2^-11 relative, and the output to its type, by u = eps / 2.  So a score is off by at most
e = h sum |q k| / scale and the weight by a factor within exp(+-e), and
    |o' - o| <= sum p |v| (2 (exp(e) - 1) + 2 h) (1 + h) + u |o|         for each output (`worst`).
The roundings are independent and zero in the mean, so over many outputs, in the 2-norm, a score's
error counts as r = h sqrt(sum (q k)^2) / scale and moves o by p (v - o) r, and
    |o' - o|_2 <= | sqrt(sum (p (v - o) r)^2) + sqrt(2) h sqrt(sum (p v)^2) + u |o| |_2   (`usual`),
where a rounding's root mean square, 1 / sqrt(3) of its largest, leaves room for what is small: float32
sums of up to 2^12 terms (below h / 64), and what fp16's subnormals cost under the kernel's powers of
two, which `worst` counts: 2^-24 of the largest cache value in a component of a key or value, 2^-33 of
the row's largest weight in a weight, 2^k times that where 64-key units differ by 2^k in size.
"""

from __future__ import annotations

import math

import torch

H = 2.0 ** -11


def attention(q_nope, q_rope, lat, rot, W_uk, W_uv, scale, lims, dtype):
    """One sequence: q_* [n, H, .], lat [keys, 512], rot [keys, 64], query i sees keys <= lims[i].
    Returns out, worst, usual [n, H, 128] in float64."""
    u = torch.finfo(dtype).eps / 2
    dev = q_nope.device
    n, heads, _ = q_nope.shape
    keys = lat.size(0)
    out = torch.zeros(n, heads, 128, dtype=torch.float64, device=dev)
    worst, usual = torch.zeros_like(out), torch.zeros_like(out)
    if keys == 0:
        return out, worst, usual
    hide = torch.arange(keys, device=dev)[None] > torch.as_tensor(lims, device=dev)[:, None]
    lat, r = lat.double(), rot.double()
    size = torch.maximum(lat.abs().amax(1), r.abs().amax(1))
    units = [size[i:i + 64].max().item() for i in range(0, keys, 64)]
    apart = 4 * max(units) / max(min(units), 2.0 ** -100)
    tiny = 2.0 ** -24 * max(units)
    for h in range(heads):
        k, v = lat @ W_uk[h].double().t(), lat @ W_uv[h].double().t()
        q, qr = q_nope[:, h].double(), q_rope[:, h].double()
        t = ((q @ k.t() + qr @ r.t()) / scale).masked_fill(hide, -math.inf)
        p = torch.softmax(t, -1).nan_to_num()
        top = p.amax(-1, keepdim=True)
        o = p @ v
        out[:, h] = o
        e = (H * (q.abs() @ k.abs().t()) + tiny * (q.abs().sum(1) + qr.abs().sum(1))[:, None]) / scale
        g = p * (2 * torch.expm1(e) + 2 * H) * (1 + H) + top * min(1.0, 2.0 ** -33 * apart)
        worst[:, h] = g @ (v.abs() + tiny) + u * o.abs() + tiny
        s = p * H * ((q * q) @ (k * k).t()).sqrt() / scale
        s = s * s
        moved = (s @ (v * v) - 2 * o * (s @ v) + o * o * s.sum(1, keepdim=True)).clamp(min=0).sqrt()
        usual[:, h] = moved + math.sqrt(2) * H * ((p * p) @ (v * v)).sqrt() + u * o.abs()
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
