"""The decoding-step operators from their definitions in 64 bits, one sequence at a time (no code of the package)."""

import math

import torch

BLOCK = 64


def rotate(x, cos, sin, dtype):
    """``[H, n, D]`` by ``[n, D]`` tables; a cached value has the activation type."""

    half = x.shape[-1] // 2
    a, b = x[..., :half].double(), x[..., half:].double()
    c, s = cos[:, :half].double(), sin[:, :half].double()
    return torch.cat((a * c - b * s, b * c + a * s), -1).to(dtype).double()


def held(x):
    """What a cache holds of ``[H, n, D]`` tokens from position 0 on: finished blocks in steps of 1/127 of their largest value."""

    out = x.double().clone()
    for lo in range(0, x.shape[1] - BLOCK + 1, BLOCK):
        blk = out[:, lo:lo + BLOCK]
        amax = blk.abs().amax((1, 2), keepdim=True)
        codes = torch.where(amax > 0, torch.round(blk * 127 / amax.clamp_min(1e-300)), torch.zeros_like(blk))
        out[:, lo:lo + BLOCK] = torch.where(torch.isfinite(amax), codes * (amax / 127), torch.full_like(blk, math.nan))
    return out


def attend(q, keys, values, start):
    """``q`` [Hq, n, D] at positions start ..., cached ``[Hkv, start + n, D]``: output and, for error bounds, sum p |v|."""

    group = q.shape[0] // keys.shape[0]
    k, v = keys.repeat_interleave(group, 0), values.repeat_interleave(group, 0)
    s = q.double() @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
    n = q.shape[1]
    seen = torch.arange(k.shape[1], device=q.device) <= start + torch.arange(n, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    return p @ v, p @ v.abs()


def moe(x, router, gate_up, down, top_k, normalize):
    xd = x.double()
    logits = xd @ router.double().t()
    probs = torch.softmax(logits, -1)
    out = torch.zeros_like(xd)
    inter = down.shape[2]
    for t in range(x.shape[0]):
        row = logits[t].tolist()
        chosen = sorted(range(len(row)), key=lambda e: (-row[e], e))[:top_k]
        w = probs[t, chosen]
        w = w / w.sum() if normalize else w
        for e, we in zip(chosen, w):
            gu = gate_up[e].double() @ xd[t]
            g, u = gu[:inter], gu[inter:]
            out[t] += we * (down[e].double() @ (g * torch.sigmoid(g) * u))
    return out
