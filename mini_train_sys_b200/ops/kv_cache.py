"""Key / value cache in 8 bits for decoding, and the plain forms of the operators on it.

Tokens of a (sequence, K/V head) are grouped in blocks of 64.  A finished block is held as 8-bit codes with one fp32 scale
for its keys and one for its values; the unfinished block stays in the activation type.  A value is therefore rounded to 8
bits once, and what the cache holds does not depend on how many calls brought the tokens:

    a = max |x| over the block's 64 x D values        scale = a / 127        code = rint(127 x / a), half to even

A block that holds a NaN or an infinity gets a NaN scale: everything that attends to it reads NaN.

A step brings up to ``padded`` new tokens for every sequence (``begin``), each layer appends and attends, ``commit`` moves the
lengths on.  Until then a step may be repeated: appending again at the same lengths writes the same blocks (the tail has
room for two unfinished blocks, so a finished one can be rebuilt; steps of more than 64 tokens that start inside a block
are the exception, they may overwrite the older tokens they were built from).
"""

from __future__ import annotations

import torch

BLOCK = 64
HEAD = 16                      # bytes of a record before its codes
# where a row of values keeps a token: finished blocks, and each half of the unfinished one
_HALF_SLOT = [((t & 7) >> 1) * 8 + (t >> 4) * 4 + ((t >> 3) & 1) * 2 + (t & 1) for t in range(BLOCK // 2)]
_SLOT = [((t & 7) >> 1) * 16 + (t >> 4) * 4 + ((t >> 3) & 1) * 2 + (t & 1) for t in range(BLOCK)]


class QuantizedKVCache:
    """Cache of all layers of a model; the operators take it with a layer index.

    The buffers are made once and written in place (captured graphs and the native layers hold their addresses); a copy of the
    object (``copy.deepcopy``) has its own."""

    def __init__(self, *, layers: int, batch: int, kv_heads: int, head_dim: int, capacity: int, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> None:
        for name, value in (("layers", layers), ("batch", batch), ("kv_heads", kv_heads), ("head_dim", head_dim), ("capacity", capacity)):
            if value <= 0:
                raise ValueError(f"all cache dimensions must be positive (got {name}={value})")
        if dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"Unsupported cache activation dtype: {dtype}")
        self.layers, self.batch, self.kv_heads, self.head_dim = layers, batch, kv_heads, head_dim
        self.blocks = -(-capacity // BLOCK)
        self.capacity = self.blocks * BLOCK
        self.dtype = dtype
        lead = (layers, batch, kv_heads)
        # a finished block: the fp32 scales of its keys and values, 8 bytes of padding, the codes of its keys and of its values
        self.records = torch.full((*lead, self.blocks, HEAD + 2 * BLOCK * head_dim), 128, dtype=torch.uint8, device=device)
        self.records[..., :HEAD] = 0
        self.tail = torch.zeros(*lead, 2, 2, BLOCK * head_dim, dtype=dtype, device=device)
        self.device = self.records.device
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)     # tokens before the step
        self.counts = torch.zeros(batch, dtype=torch.int32, device=device)      # new tokens of the step
        self.held = 0                   # upper bound of the lengths, known without asking the device
        self.padded: int | None = None  # padded number of new tokens of the open step

        self.native: dict[int, object] = {}     # layers as the native backend holds them

    def __getstate__(self) -> dict:
        return {**self.__dict__, "native": {}}      # a copy (of a beam, of a shared prompt) has buffers of its own

    @property
    def codes(self) -> torch.Tensor:
        """``[layers, B, heads, blocks, 2, 64 * D]`` view of the codes (128 stands for zero)."""

        return self.records[..., HEAD:].unflatten(-1, (2, BLOCK * self.head_dim))

    @property
    def scale(self) -> torch.Tensor:
        """``[layers, B, heads, blocks, 2]`` view of the scales of keys and values."""

        return self.records[..., :8].view(torch.float32)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.records, self.tail, self.lengths, self.counts))

    def begin(self, count: torch.Tensor | None = None, *, padded: int = 1) -> None:
        """Open a step of up to ``padded`` new tokens per sequence: ``count[b]`` of them, or all of them where it is None."""

        if padded <= 0:
            raise ValueError("a step needs at least one token")
        if self.held + padded > self.capacity:
            raise ValueError(f"{self.held} cached + {padded} new tokens exceed the cache's capacity of {self.capacity}")
        if count is None:
            self.counts.fill_(padded)
        else:
            if count.shape != (self.batch,) or count.dtype not in (torch.int32, torch.int64):
                raise ValueError("count must hold one integer per sequence")
            self.counts.copy_(count.clamp(0, padded))
        self.padded = padded

    def commit(self) -> None:
        """Close the step: its tokens count as cached."""

        if self.padded is None:
            raise RuntimeError("no step is open")
        self.lengths += self.counts
        self.counts.zero_()
        self.held += self.padded
        self.padded = None

    def replayed(self, padded: int) -> None:
        """Account for a step whose ``begin`` and ``commit`` ran inside a replayed CUDA graph.  Call it before the replay: it
        refuses a step that the cache has no room for."""

        if self.held + padded > self.capacity:
            raise ValueError(f"{self.held} cached + {padded} new tokens exceed the cache's capacity of {self.capacity}")
        self.held += padded

    def reset(self) -> None:
        """Forget all tokens."""

        self.lengths.zero_()
        self.counts.zero_()
        self.held, self.padded = 0, None

    def check_layer(self, index: int) -> int:
        if not 0 <= index < self.layers:
            raise IndexError(f"cache layer {index} of {self.layers}")
        return index


def check_rows(cache: QuantizedKVCache, name: str, x: torch.Tensor, heads: int | None = None, tokens: int | None = None) -> None:
    if x.dim() != 4 or x.shape[0] != cache.batch or x.shape[3] != cache.head_dim:
        raise ValueError(f"{name} must be [{cache.batch}, heads, T, {cache.head_dim}], got {tuple(x.shape)}")
    if heads is not None and x.shape[1] != heads:
        raise ValueError(f"{name} must have {heads} heads, got {x.shape[1]}")
    if x.shape[1] == 0 or x.shape[1] % cache.kv_heads:
        raise ValueError(f"{name} must have a multiple of {cache.kv_heads} heads, got {x.shape[1]}")
    if x.dtype != cache.dtype:
        raise ValueError(f"{name} must have the cache's activation type {cache.dtype}, got {x.dtype}")
    if x.device != cache.device:
        raise ValueError(f"{name} must be on {cache.device}, got {x.device}")
    if tokens is not None and x.shape[2] != tokens:
        raise ValueError(f"{name} must hold the {tokens} padded tokens of the open step, got {x.shape[2]}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError(f"{name} requires a gradient: the cache operators are for inference (use torch.no_grad())")


def check_append(cache, k, v, q, cos, sin) -> None:
    if cache.padded is None:
        raise RuntimeError("open a step with begin() first")
    check_rows(cache, "k", k, cache.kv_heads, cache.padded)
    check_rows(cache, "v", v, cache.kv_heads, cache.padded)
    if q is not None:
        check_rows(cache, "q", q, None, cache.padded)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != cache.head_dim:
            raise ValueError(f"rotary tables must be [positions, {cache.head_dim}]")
        if cos.dtype != cache.dtype or sin.dtype != cache.dtype or cos.device != k.device or sin.device != k.device:
            raise ValueError("rotary tables must match the cache's activation type and device")
        if cos.shape[0] < cache.held + cache.padded:
            raise ValueError(f"rotary tables hold {cos.shape[0]} positions, the step reaches {cache.held + cache.padded}")


def check_attention(cache, q) -> None:
    if cache.padded is None:
        raise RuntimeError("open a step with begin() first")
    check_rows(cache, "q", q, None, cache.padded)


def check_read(cache, first, n) -> None:
    if first.shape != (cache.batch,) or first.dtype != torch.int32 or first.device != cache.device:
        raise ValueError("first must hold one int32 position per sequence, on the cache's device")
    if n < 0:
        raise ValueError("the number of positions must not be negative")


# ---------------------------------------------------------------------------------------------
# plain forms (any device): what the native kernels are tested against in structure, and the path of CPU runs
# ---------------------------------------------------------------------------------------------
def rotate_rows(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Half-split rotation of ``[..., T, D]`` in fp32, rounded to the type of ``x``."""

    half = x.shape[-1] // 2
    xf, c, s = x.float(), cos.float()[..., :half], sin.float()[..., :half]
    lo, hi = xf[..., :half], xf[..., half:]
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1).to(x.dtype)


def quantize_block(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``[..., 64, D]`` -> excess-128 codes (uint8) and the fp32 scale of each block."""

    xd = x.double()
    amax = xd.abs().amax((-1, -2), keepdim=True)
    finite = torch.isfinite(amax)
    usable = finite & (amax > 0)
    codes = torch.where(usable, torch.round(xd * 127.0 / amax), torch.zeros_like(xd))
    scale = torch.where(finite, amax.float() / 127.0, torch.full_like(amax, float("nan")).float())
    return (codes + 128).to(torch.uint8), scale[..., 0, 0]


def _pack_values(rows: torch.Tensor, *, tail: bool) -> torch.Tensor:
    """``[heads, 64, D]`` -> the order in which a record or the tail holds values."""

    heads, _, dim = rows.shape
    slots = torch.tensor(_HALF_SLOT if tail else _SLOT, device=rows.device)
    parts = rows.view(heads, -1, len(slots), dim).transpose(2, 3)        # [heads, 1 or 2 halves, D, tokens]
    out = torch.empty_like(parts, memory_format=torch.contiguous_format)
    out[..., slots] = parts
    return out.view(heads, -1)


def _unpack_values(flat: torch.Tensor, dim: int, *, tail: bool) -> torch.Tensor:
    """Inverse of ``_pack_values`` over the last dimension: ``[..., 64 D]`` -> ``[..., 64, D]``."""

    slots = torch.tensor(_HALF_SLOT if tail else _SLOT, device=flat.device)
    return flat.unflatten(-1, (-1, dim, len(slots)))[..., slots].transpose(-1, -2).flatten(-3, -2)


def append_plain(cache: QuantizedKVCache, layer: int, k, v, q=None, cos=None, sin=None):
    cache.check_layer(layer)
    codes, scale, tail, lengths, counts = cache.codes[layer], cache.scale[layer], cache.tail[layer], cache.lengths, cache.counts
    new, dim, heads = k.shape[2], cache.head_dim, cache.kv_heads
    start = lengths.long().clamp(0, cache.capacity)
    t = torch.arange(new, device=k.device)
    pos = start[:, None] + t
    live = (t < counts[:, None]) & (pos < cache.capacity)
    q_out = None
    if cos is not None:
        at = pos.clamp_max(cos.shape[0] - 1)
        c, s = cos[at][:, None], sin[at][:, None]
        k = rotate_rows(k, c, s)
        q_out = rotate_rows(q, c, s) if q is not None else None
    elif q is not None:
        q_out = q
    if q_out is not None:
        q_out = torch.where(live[:, None, :, None], q_out, torch.zeros_like(q_out))
    for b in range(cache.batch):
        lo, hi = int(start[b]), int(start[b]) + int(live[b].sum())
        for blk in range(lo // BLOCK, -(-hi // BLOCK) if hi > lo else lo // BLOCK):
            base = blk * BLOCK
            first, last = max(lo, base), min(hi, base + BLOCK)
            held = tail[b, :, blk & 1]
            blocks = torch.stack((held[:, 0].view(heads, BLOCK, dim), _unpack_values(held[:, 1], dim, tail=True)), 1)
            blocks[:, 0, first - base:last - base] = k[b, :, first - lo:last - lo]
            blocks[:, 1, first - base:last - base] = v[b, :, first - lo:last - lo]
            open_ = last < base + BLOCK
            if open_:
                dest, rows = held, blocks
            else:
                rows, scales = quantize_block(blocks)
                dest = codes[b, :, blk]
                scale[b, :, blk] = scales
            dest[:, 0] = rows[:, 0].reshape(heads, -1)
            dest[:, 1] = _pack_values(rows[:, 1], tail=open_)
    return q_out


def read_plain(cache: QuantizedKVCache, layer: int, first: torch.Tensor, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    cache.check_layer(layer)
    dim, dev = cache.head_dim, cache.device
    total = (cache.lengths.long().clamp(0, cache.capacity) + cache.counts).clamp_max(cache.capacity)
    pos = first.long()[:, None] + torch.arange(n, device=dev)
    live = (pos >= 0) & (pos < total[:, None])
    pos = torch.where(live, pos, torch.zeros_like(pos))
    last = total // BLOCK
    which = torch.arange(cache.batch, device=dev)
    tail = cache.tail[layer][which, :, last & 1]                          # [B, heads, 2, 64 D]
    out = []
    for side in range(2):
        codes, scale = cache.codes[layer][:, :, :, side], cache.scale[layer][:, :, :, side]
        done = codes.unflatten(-1, (BLOCK, dim)) if side == 0 else _unpack_values(codes, dim, tail=False)
        done = ((done.float() - 128.0) * scale[..., None, None]).flatten(2, 3)
        open_ = tail[:, :, side].unflatten(-1, (BLOCK, dim)) if side == 0 else _unpack_values(tail[:, :, side], dim, tail=True)
        index = pos[:, None, :, None].expand(-1, cache.kv_heads, -1, dim)
        values = torch.where((pos // BLOCK == last[:, None])[:, None, :, None], open_.float().gather(2, index % BLOCK), done.gather(2, index))
        out.append(torch.where(live[:, None, :, None], values, torch.zeros_like(values)))
    return out[0], out[1]


def attention_plain(q: torch.Tensor, cache: QuantizedKVCache, layer: int) -> torch.Tensor:
    start, count = cache.lengths.long(), cache.counts.long()
    b, hq, new, d = q.shape
    n = min(cache.held + cache.padded, cache.capacity)
    keys, values = read_plain(cache, layer, torch.zeros_like(cache.lengths), n)
    group = hq // cache.kv_heads
    scores = torch.einsum("bhgtd,bhsd->bhgts", q.float().reshape(b, cache.kv_heads, group, new, d), keys) * d ** -0.5
    t = torch.arange(new, device=q.device)
    seen = torch.arange(n, device=q.device) <= (start[:, None] + t)[..., None]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    finite = torch.isfinite(values)
    out = torch.einsum("bhgts,bhsd->bhgtd", torch.softmax(scores, -1), torch.where(finite, values, torch.zeros_like(values)))
    if not bool(finite.all()):
        # a masked probability of 0 times an infinity or a NaN would be a NaN: what is not finite is added to the rows that see it
        rest = torch.where(finite, torch.zeros_like(values), values)
        for at in (~finite).any(-1).any(1).any(0).nonzero().flatten().tolist():
            out += torch.where(seen[:, None, None, :, at, None], rest[:, :, None, None, at], torch.zeros_like(out))
    out = out.reshape(b, hq, new, d)
    live = (t < count[:, None])[:, None, :, None]
    return torch.where(live, out, torch.zeros_like(out)).to(q.dtype)
