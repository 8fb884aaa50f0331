"""Library-op backend (cuBLAS GEMMs, SDPA attention): the measured baseline.

Numerical contract as in minitrain/kernels/torch_ops.py:13-150: reductions in fp32,
activations returned in the input dtype, dropless MoE that keeps zero-weight routes.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from mini_train_sys_b200.models.ops import RouterPostprocessOutput
from mini_train_sys_b200.ops import kv_cache


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    lo, hi = x.chunk(2, dim=-1)
    return torch.cat((-hi, lo), dim=-1)


def check_router_args(logits: torch.Tensor, top_k: int) -> None:
    if logits.ndim != 2 or logits.dtype != torch.float32:
        raise ValueError("router logits must be a 2D fp32 tensor")
    if logits.shape[0] == 0:
        raise ValueError("router logits must contain at least one token")
    if not 1 <= top_k <= logits.shape[1]:
        raise ValueError(f"top_k must be in [1, {logits.shape[1]}], got {top_k}")


def check_moe_tokens(x: torch.Tensor, router_weight: torch.Tensor, gate_up_proj: torch.Tensor, down_proj: torch.Tensor, top_k: int) -> None:
    if x.ndim != 2 or router_weight.ndim != 2 or gate_up_proj.ndim != 3 or down_proj.ndim != 3:
        raise ValueError("moe_tokens expects x [T, H], router [E, H], gate_up [E, 2 I, H] and down [E, H, I]")
    n_exp, hidden = router_weight.shape
    if x.shape[1] != hidden or gate_up_proj.shape != (n_exp, 2 * down_proj.shape[2], hidden) or down_proj.shape[:2] != (n_exp, hidden):
        raise ValueError(f"moe_tokens shapes do not fit: x {tuple(x.shape)}, router {tuple(router_weight.shape)}, "
                         f"gate_up {tuple(gate_up_proj.shape)}, down {tuple(down_proj.shape)}")
    if not 1 <= top_k <= n_exp:
        raise ValueError(f"top_k must be in [1, {n_exp}], got {top_k}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, router_weight, gate_up_proj, down_proj)):
        raise RuntimeError("moe_tokens is for inference (use torch.no_grad()); fused_moe has a gradient")


class TorchOpsBackend:
    name = "torch"

    def rmsnorm(self, x, weight, eps):
        xf = x.float()
        inv = torch.rsqrt(xf.square().mean(dim=-1, keepdim=True) + eps)
        return (xf * inv * weight.float()).to(x.dtype)

    def rope(self, q, k, cos, sin):
        c = cos[None, None].to(q.dtype)
        s = sin[None, None].to(q.dtype)
        return q * c + rotate_half(q) * s, k * c + rotate_half(k) * s

    def swiglu(self, gate, up):
        return F.silu(gate) * up

    def attention(self, q, k, v, *, is_causal, dropout_p):
        return F.scaled_dot_product_attention(q, k, v, is_causal=is_causal, dropout_p=dropout_p)

    def cross_entropy(self, logits, targets):
        return F.cross_entropy(logits.float(), targets)

    def fused_linear_cross_entropy(self, x, weight, targets):
        return F.cross_entropy(F.linear(x, weight).float(), targets)

    def router_postprocess(self, logits, top_k, *, normalize):
        check_router_args(logits, top_k)
        lse = torch.logsumexp(logits, dim=-1, keepdim=True)
        probs = (logits - lse).exp()
        w, idx = probs.topk(top_k, dim=-1)
        if normalize:
            w = w / w.sum(-1, keepdim=True).clamp_min(torch.finfo(w.dtype).eps)
        ent = -(probs * probs.clamp_min(1e-9).log()).sum(-1).mean().detach()
        return RouterPostprocessOutput(w, idx.to(torch.int32), probs.mean(0), lse.square().mean(), ent)

    def fused_moe(self, x, gate_up_proj, down_proj, top_k_index, top_k_weights):
        out = torch.zeros_like(x)
        for e in torch.unique(top_k_index).tolist():
            tok, slot = torch.where(top_k_index == e)  # zero-weight routes stay in the graph
            if tok.numel() == 0:
                continue
            g, u = F.linear(x[tok], gate_up_proj[e]).chunk(2, dim=-1)
            y = F.linear(F.silu(g) * u, down_proj[e]) * top_k_weights[tok, slot, None]
            out.index_add_(0, tok, y.to(out.dtype))
        return out

    # -- decoding step (hooks outside the 8-op protocol) -----------------------------------------
    def kv_append(self, cache, layer, k, v, *, q=None, cos=None, sin=None):
        """Append a step's keys and values (``[B, kv heads, T, D]``) to ``cache``; with rotary tables, rotate k and q first.

        Token t of sequence b goes to position ``cache.lengths[b] + t`` while ``t < cache.counts[b]``; padding is not looked
        at.  Returns the (rotated) ``q`` with zeroed padding rows, or None without one."""

        kv_cache.check_append(cache, k, v, q, cos, sin)
        return kv_cache.append_plain(cache, layer, k, v, q, cos, sin)

    def kv_read(self, cache, layer, first, n):
        """What the cache holds at positions ``first[b] ... first[b] + n - 1``: fp32 ``(k, v)`` ``[B, kv heads, n, D]``; zeros
        at positions that hold no token."""

        kv_cache.check_read(cache, first, n)
        return kv_cache.read_plain(cache, layer, first, n)

    def cached_attention(self, q, cache, layer):
        """Attention of a step's queries ``[B, heads, T, D]`` over the cached tokens and, causally, the step's own (which
        ``kv_append`` has put there).  Heads that share a K/V head are adjacent.  Padding rows are zero."""

        kv_cache.check_attention(cache, q)
        return kv_cache.attention_plain(q, cache, layer)

    def moe_tokens(self, x, router_weight, gate_up_proj, down_proj, top_k, *, normalize):
        """A whole routed SwiGLU layer for the few tokens ``[T, H]`` of a decoding step (no gradient, no balance statistics)."""

        check_moe_tokens(x, router_weight, gate_up_proj, down_proj, top_k)
        if x.shape[0] == 0:
            return torch.empty_like(x)
        with torch.autocast(device_type=x.device.type, enabled=False):
            logits = F.linear(x.float(), router_weight.float())
            # ties go to the lower expert, as in the kernels
            order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top_k]
            weights = torch.softmax(logits, -1).gather(1, order)
            if normalize:
                weights = weights / weights.sum(-1, keepdim=True).clamp_min(torch.finfo(weights.dtype).eps)
            out = torch.zeros_like(x, dtype=torch.float32)
            for e in torch.unique(order).tolist():
                tok, slot = torch.where(order == e)
                g, u = F.linear(x[tok].float(), gate_up_proj[e].float()).chunk(2, dim=-1)
                out.index_add_(0, tok, F.linear(F.silu(g) * u, down_proj[e].float()) * weights[tok, slot, None])
        return out.to(x.dtype)
