"""The operators of one decoding step, as a program that serves a model calls them.

A decoding step appends the new tokens' keys and values to a cache that holds finished blocks of 64 tokens in 8 bits
(``kv_append``, read back with ``kv_read``), attends over that cache (``cached_attention``) and runs the mixture-of-experts
layer for the few tokens of the step (``moe_tokens``).  ``run`` is one pass of one of them: through the framework where ``own``
is true, else in elementary torch operations.
"""

import math

import torch

own = False

BLOCK = 64
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _append(name, batch, q_heads, kv_heads, dim, new, start, dtype="bf16", ragged=False):
    return {"name": name, "op": "append", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "new": new,
            "start": start, "dtype": dtype, "ragged": ragged}


def _attention(name, batch, q_heads, kv_heads, dim, new, length, dtype="bf16", ragged=False):
    return {"name": name, "op": "attention", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "new": new,
            "length": length, "dtype": dtype, "ragged": ragged}


def _moe(name, tokens, experts, top_k, hidden, inter, normalize=True):
    return {"name": name, "op": "moe", "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "inter": inter,
            "normalize": normalize}


def listed():
    return [
        # one new token of one sequence of the 12-head study model; its block closes with this token
        _append("append-token", 1, 12, 12, 64, 1, 447),
        # one new token each for 64 sequences of unlike lengths, some of them finished (no new token)
        _append("append-batch", 64, 12, 12, 64, 1, 511, ragged=True),
        # a batch of prompts of unlike lengths that fill an empty cache
        _append("append-prompt", 16, 12, 12, 64, 2048, 0, ragged=True),
        # next token at the end of the study model's 512-token window
        _attention("attend-short", 1, 12, 12, 64, 1, 512),
        # a batch that samples together, sequences of unlike lengths up to the default model's 2048 tokens
        _attention("attend-batch", 64, 12, 12, 64, 1, 2048, ragged=True),
        # shared K/V heads and wide heads over long documents
        _attention("attend-grouped", 8, 32, 8, 128, 1, 32768, ragged=True),
        # one very long document, half-precision activations; its length ends inside a block
        _attention("attend-long", 1, 16, 4, 64, 1, 131071, dtype="fp16"),
        # a short follow-up prompt of 17 tokens on conversations that are in the cache
        _attention("attend-chunk", 4, 12, 12, 64, 17, 1999, ragged=True),
        # one token through the study model's experts
        _moe("moe-token", 1, 8, 2, 768, 1024),
        # a batch of 64 tokens through the same experts
        _moe("moe-batch", 64, 8, 2, 768, 1024),
        # many small experts, each with a token or two
        _moe("moe-many", 17, 64, 8, 2048, 1024),
        # wide experts: nearly the whole time is reading their weights
        _moe("moe-wide", 8, 8, 2, 4096, 14336, normalize=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "moe", "moe"])
    if op == "moe":
        experts = _log_int(rng, 2, 64)
        hidden = 8 * _log_int(rng, 16, 512)
        inter = 8 * _log_int(rng, 16, 1792)
        while experts * hidden * inter > 8 * 4096 * 14336:
            inter = max(128, inter // 16 * 8)
            if inter == 128:
                break
        case = _moe("", _log_int(rng, 1, 64), experts, rng.randint(1, min(8, experts)), hidden, inter, rng.random() < 0.7)
    else:
        dim = rng.choice([32, 64, 64, 128])
        kv_heads = rng.choice([1, 2, 4, 6, 8, 12, 16])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        batch = _log_int(rng, 1, 64)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        ragged = rng.random() < 0.6
        if op == "append":
            if rng.random() < 0.5:      # a step, or a few tokens, anywhere
                new, start = _log_int(rng, 1, 64), rng.randint(0, 4096)
            else:                       # prompts
                new, start = _log_int(rng, 1, 4096), 0
            while batch * new * kv_heads * group * dim > 16 * 2048 * 12 * 64:
                batch, new = max(1, batch // 2), max(1, (new * 3) // 4)
            case = _append("", batch, kv_heads * group, kv_heads, dim, new, start, dtype, ragged)
        else:
            new = 1 if rng.random() < 0.6 else _log_int(rng, 2, 32)
            length = _log_int(rng, 1, 131072)
            # as many keys as the largest listed case holds, and scores that a plain form can hold
            while batch * kv_heads * length * dim > 8 * 8 * 32768 * 128 or batch * kv_heads * group * new * length > 1 << 28:
                batch, length = max(1, batch // 2), max(1, (length * 3) // 4)
            case = _attention("", batch, kv_heads * group, kv_heads, dim, new, max(length, new), dtype, ragged)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed) & 0x7FFFFFFFFFFFFFF)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _keys(gen, batch, tokens, heads, dim, dtype):
    """Keys as a trained model has them: a few channels are much larger than the others."""

    channel = torch.exp(0.5 * _randn(gen, 1, 1, heads, dim))
    return (_randn(gen, batch, tokens, heads, dim) * channel).to(dtype)


def _spans(case, gen):
    """(tokens in the cache, new tokens) of every sequence."""

    batch, new = case["batch"], case["new"]
    full = case["start"] if case["op"] == "append" else case["length"] - new
    start = torch.full((batch,), full, dtype=torch.int32, device=DEVICE)
    count = torch.full((batch,), new, dtype=torch.int32, device=DEVICE)
    if case["ragged"]:
        u = torch.rand(batch, generator=gen, device=DEVICE)
        start = (full * u).round().to(torch.int32)
        start[0] = full                                   # one sequence has the full length
        w = torch.rand(batch, generator=gen, device=DEVICE)
        some = (new * w).ceil().to(torch.int32)           # a prompt or a chunk that is shorter than the padded one
        count = some.clamp(1, new) if new > 1 else torch.where(w < 0.1, torch.zeros_like(count), count)
        count[0] = new
    return start, count


def _tables(case, positions):
    """Rotary tables in the activation type, as the framework's models keep them."""

    dim = case["dim"]
    inv = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    phase = torch.outer(torch.arange(positions, dtype=torch.float64), inv)
    phase = torch.cat((phase, phase), -1)
    return (phase.cos().to(DEVICE, DTYPES[case["dtype"]]), phase.sin().to(DEVICE, DTYPES[case["dtype"]]))


def _cache_inputs(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    batch, hq, hkv, dim, new = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], case["new"]
    start, count = _spans(case, gen)
    held = case["start"] if case["op"] == "append" else case["length"] - new
    # what a step of the model has in hand: one projection with the q, k and v heads side by side
    fused = _randn(gen, batch, new, hq + 2 * hkv, dim).to(dtype)
    fused[:, :, hq:hq + hkv] = _keys(gen, batch, new, hkv, dim, dtype)
    q, k, v = (t.transpose(1, 2) for t in (fused[:, :, :hq], fused[:, :, hq:hq + hkv], fused[:, :, hq + hkv:]))
    old_k = _keys(gen, batch, held, hkv, dim, dtype).transpose(1, 2)
    old_v = _randn(gen, batch, held, hkv, dim).to(dtype).transpose(1, 2)
    return {"q": q, "k": k, "v": v, "old_k": old_k, "old_v": old_v, "start": start, "count": count, "held": held}


def _moe_inputs(case, seed):
    gen = _generator(seed)
    t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
    return {"x": _randn(gen, t, h).to(torch.bfloat16), "router": _randn(gen, e, h) * (2.0 / math.sqrt(h)),
            "gate_up": (torch.randn(e, 2 * i, h, generator=gen, device=DEVICE, dtype=torch.bfloat16) * (1.0 / math.sqrt(h))),
            "down": (torch.randn(e, h, i, generator=gen, device=DEVICE, dtype=torch.bfloat16) * (1.0 / math.sqrt(i)))}


def _blocks(tokens):
    return -(-tokens // BLOCK)


def prepare(case, seed):
    state = {"case": dict(case)}
    if case["op"] == "moe":
        state.update(_moe_inputs(case, seed))
        if own:
            from mini_train_sys_b200.models.ops import get_ops_backend

            state["ops"] = get_ops_backend("native")
        return state
    data = _cache_inputs(case, seed)
    capacity = BLOCK * _blocks(data["held"] + case["new"])
    state.update({n: data[n] for n in ("q", "k", "v", "start", "count")})
    if case["op"] == "append":
        state["cos"], state["sin"] = _tables(case, capacity)
        state["first"] = data["start"] // BLOCK * BLOCK
        state["window"] = BLOCK * (1 + _blocks(case["new"]))
    if own:
        from mini_train_sys_b200.models.ops import get_ops_backend
        from mini_train_sys_b200.ops.kv_cache import QuantizedKVCache

        ops = get_ops_backend("native")
        cache = QuantizedKVCache(layers=1, batch=case["batch"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                                 capacity=capacity, dtype=DTYPES[case["dtype"]], device=DEVICE)
        if data["held"] > 0:
            cache.begin(data["start"], padded=data["held"])
            ops.kv_append(cache, 0, data["old_k"], data["old_v"])
            cache.commit()
        cache.begin(data["count"], padded=case["new"])
        if case["op"] == "attention":
            ops.kv_append(cache, 0, data["k"], data["v"])
        state.update(ops=ops, cache=cache)
        return state
    # plain form of the same cache: codes and scales of finished blocks, 16-bit values of the unfinished one
    total = data["start"] + (data["count"] if case["op"] == "attention" else 0)
    kept = []
    for old, new in ((data["old_k"], data["k"]), (data["old_v"], data["v"])):
        buf = torch.zeros(case["batch"], case["kv_heads"], capacity, case["dim"], dtype=DTYPES[case["dtype"]], device=DEVICE)
        buf[:, :, :data["held"]] = old
        pos = torch.arange(capacity, device=DEVICE)
        if case["op"] == "attention":
            for b, (s, c) in enumerate(zip(data["start"].tolist(), data["count"].tolist())):
                buf[b, :, s:s + c] = new[b, :, :c]
        buf *= (pos[None, :] < total[:, None])[:, None, :, None]
        codes, scale = _quantize(buf.view(*buf.shape[:2], -1, BLOCK, case["dim"]))
        last = total.long() // BLOCK * BLOCK                         # first position of the unfinished block
        rows = (last[:, None] + torch.arange(BLOCK, device=DEVICE)).clamp_max(capacity - 1)
        tail = buf.gather(2, rows[:, None, :, None].expand(-1, buf.shape[1], -1, buf.shape[3]))
        kept.append((codes.view(buf.shape), scale, tail))
    state["plain_k"], state["plain_v"] = kept
    return state


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _quantize(blocks):
    """``[..., 64, D]`` -> int8 codes and one fp32 scale a block."""

    x = blocks.float()
    amax = x.abs().amax((-1, -2), keepdim=True)
    codes = torch.where(amax > 0, torch.round(x * 127.0 / amax), torch.zeros_like(x)).to(torch.int8)
    return codes, (amax / 127.0)[..., 0, 0]


def _rotate(x, cos, sin):
    """One rounding, to the type of ``x``: in 64 bits, since a value that 32 bits put on the border would be rounded twice."""

    half = x.shape[-1] // 2
    xf, c, s = x.double(), cos.double()[..., :half], sin.double()[..., :half]
    lo, hi = xf[..., :half], xf[..., half:]
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1).to(x.dtype)


def _plain_append(state):
    start, count = state["start"].long(), state["count"].long()
    new = state["k"].shape[2]
    t = torch.arange(new, device=DEVICE)
    pos = (start[:, None] + t).clamp_max(state["cos"].shape[0] - 1)
    cos, sin = state["cos"][pos][:, None], state["sin"][pos][:, None]
    live = (t < count[:, None])[:, None, :, None]
    q = torch.where(live, _rotate(state["q"], cos, sin), torch.zeros_like(state["q"]))
    out = [q]
    window = state["window"]
    slot = torch.arange(window, device=DEVICE)
    inside = start - state["first"].long()                           # tokens that the unfinished block has
    filled = inside + count
    for fresh, (_, _, tail) in ((_rotate(state["k"], cos, sin), state["plain_k"]), (state["v"], state["plain_v"])):
        b, h, _, d = fresh.shape
        source = torch.cat((tail, fresh), 2)
        index = torch.where(slot < inside[:, None], slot, (BLOCK + slot - inside[:, None]).clamp(0, BLOCK + new - 1))
        values = source.gather(2, index[:, None, :, None].expand(-1, h, -1, d)).float()
        values = torch.where((slot < filled[:, None])[:, None, :, None], values, torch.zeros_like(values))
        blocks = values.view(b, h, -1, BLOCK, d)
        codes, scale = _quantize(blocks)
        held = (codes.float() * scale[..., None, None]).view(values.shape)
        done = ((slot // BLOCK + 1) * BLOCK <= filled[:, None])[:, None, :, None]
        out.append(torch.where(done, held, values))
    return tuple(out)


def _plain_values(kept, total):
    codes, scale, tail = kept
    b, h, capacity, d = codes.shape
    values = (codes.view(b, h, -1, BLOCK, d).float() * scale[..., None, None]).view(b, h, capacity, d)
    last = total // BLOCK * BLOCK
    pos = torch.arange(capacity, device=DEVICE)
    rows = (pos[None, :] - last[:, None]).clamp(0, BLOCK - 1)
    open_ = tail.float().gather(2, rows[:, None, :, None].expand(-1, h, -1, d))
    return torch.where((pos[None, :] < last[:, None])[:, None, :, None], values, open_)


def _plain_attention(state):
    q, start, count = state["q"], state["start"].long(), state["count"].long()
    b, hq, new, d = q.shape
    total = start + count
    keys, values = _plain_values(state["plain_k"], total), _plain_values(state["plain_v"], total)
    hkv, capacity = keys.shape[1], keys.shape[2]
    grouped = q.float().reshape(b, hkv, hq // hkv * new, d)
    scores = torch.matmul(grouped, keys.transpose(-1, -2)).view(b, hkv, hq // hkv, new, capacity) / math.sqrt(d)
    t = torch.arange(new, device=DEVICE)
    pos = torch.arange(capacity, device=DEVICE)
    seen = pos <= (start[:, None] + t)[..., None]                     # [B, new, capacity]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(scores.view(b, hkv, -1, capacity), values).view(b, hq, new, d)
    out = out / scores.sum(-1).view(b, hq, new, 1)
    live = (t < count[:, None])[:, None, :, None]
    return torch.where(live, out, torch.zeros_like(out)).to(q.dtype)


def _plain_moe(state):
    case, x = state["case"], state["x"].float()
    logits = x.double() @ state["router"].double().t()               # a choice between experts stands on these
    probs = torch.exp(logits - logits.amax(-1, keepdim=True))
    probs = probs / probs.sum(-1, keepdim=True)
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    weights = probs.gather(1, order)
    if case["normalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    mixed = torch.zeros(x.shape[0], case["experts"], dtype=torch.float32, device=DEVICE)
    mixed = mixed.scatter(1, order, weights.float())
    out = torch.zeros_like(x)
    inter = case["inter"]
    for e in range(case["experts"]):
        gate_up = x @ state["gate_up"][e].float().t()
        gate, up = gate_up[:, :inter], gate_up[:, inter:]
        out = out + mixed[:, e:e + 1] * ((gate / (1.0 + torch.exp(-gate)) * up) @ state["down"][e].float().t())
    return out.to(torch.bfloat16)


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "moe": _plain_moe}[op](state)
    ops = state["ops"]
    if op == "moe":
        return ops.moe_tokens(state["x"], state["router"], state["gate_up"], state["down"], state["case"]["top_k"],
                              normalize=state["case"]["normalize"])
    if op == "attention":
        return ops.cached_attention(state["q"], state["cache"], 0)
    q = ops.kv_append(state["cache"], 0, state["k"], state["v"], q=state["q"], cos=state["cos"], sin=state["sin"])
    k, v = ops.kv_read(state["cache"], 0, state["first"], state["window"])
    return q, k, v


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "moe":
        t, e, k, h, i = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inter"))
        used = e * (1.0 - (1.0 - k / e) ** t)                         # experts that have a token, in the mean
        return {"bytes": used * 3 * h * i * 2 + e * h * 4 + 2 * t * h * 2, "flops": 6.0 * t * k * h * i + 2.0 * t * e * h}
    b, hq, hkv, d, new = (case[n] for n in ("batch", "q_heads", "kv_heads", "dim", "new"))
    mean_new = new * 0.5 if case["ragged"] and new > 1 else new
    if case["op"] == "append":
        window = BLOCK * (1 + _blocks(new))
        fresh = b * mean_new * (2 * hq + 2 * hkv + hkv) * d * 2       # q in and out, k and v in, 1 byte each out
        return {"bytes": fresh + b * mean_new * 2 * d * 2 + b * hkv * window * d * 2 * 4, "flops": b * mean_new * (hq + hkv) * d * 3.0}
    keys = (case["length"] - new) * (0.5 if case["ragged"] else 1.0) + mean_new
    return {"bytes": b * hkv * keys * (2 * d + 8.0 / BLOCK) + 2 * b * hq * mean_new * d * 2, "flops": 4.0 * b * hq * mean_new * keys * d}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, one sequence (or one expert) at a time
# ---------------------------------------------------------------------------------------------
def _round_to(x, dtype):
    return x.to(dtype).double()


def _held64(x):
    """What the cache holds of ``[H, n, D]`` tokens that begin a block: finished blocks to 1/127 of their largest value."""

    full = x.shape[1] // BLOCK * BLOCK
    blk = x[:, :full].reshape(x.shape[0], -1, BLOCK, x.shape[2])
    most = blk.abs().flatten(2).amax(2)[:, :, None, None] if full else blk
    blk = torch.where(most > 0, torch.round(blk * 127.0 / most.clamp_min(1e-300)) * (most / 127.0), torch.zeros_like(blk))
    return torch.cat((blk.reshape(x.shape[0], full, x.shape[2]), x[:, full:]), 1)


def _turn64(x, angles_c, angles_s, dtype):
    d = x.shape[-1] // 2
    z = torch.complex(x[..., :d].contiguous(), x[..., d:].contiguous()) * torch.complex(angles_c[:, :d].contiguous(), angles_s[:, :d].contiguous())
    return _round_to(torch.cat((z.real, z.imag), -1), dtype)


def _exact_append(case, seed):
    data = _cache_inputs(case, seed)
    dtype = DTYPES[case["dtype"]]
    b, hkv, d, new = case["batch"], case["kv_heads"], case["dim"], case["new"]
    window = BLOCK * (1 + _blocks(new))
    cos, sin = (t.double() for t in _tables(case, BLOCK * _blocks(data["held"] + new)))
    q = torch.zeros(b, case["q_heads"], new, d, dtype=torch.float64, device=DEVICE)
    outs = [torch.zeros(b, hkv, window, d, dtype=torch.float64, device=DEVICE) for _ in range(2)]
    for i, (s, c) in enumerate(zip(data["start"].tolist(), data["count"].tolist())):
        base, at = s // BLOCK * BLOCK, slice(s, s + c)
        q[i, :, :c] = _turn64(data["q"][i, :, :c].double(), cos[at], sin[at], dtype)
        for out, old, fresh in ((outs[0], data["old_k"], _turn64(data["k"][i, :, :c].double(), cos[at], sin[at], dtype)),
                                (outs[1], data["old_v"], data["v"][i, :, :c].double())):
            out[i, :, :s - base + c] = _held64(torch.cat((old[i, :, base:s].double(), fresh), 1))
    return (q, *outs)


def _exact_attention(case, seed):
    data = _cache_inputs(case, seed)
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], case["q_heads"], case["new"], case["dim"], dtype=torch.float64, device=DEVICE)
    for i, (s, c) in enumerate(zip(data["start"].tolist(), data["count"].tolist())):
        for h in range(case["kv_heads"]):
            k, v = (_held64(torch.cat((old[i, h:h + 1, :s], fresh[i, h:h + 1, :c]), 1).double())[0]
                    for old, fresh in ((data["old_k"], data["k"]), (data["old_v"], data["v"])))
            for t in range(c):
                rows = data["q"][i, h * group:(h + 1) * group, t].double()
                p = torch.softmax(rows @ k[:s + t + 1].t() / math.sqrt(case["dim"]), -1)
                out[i, h * group:(h + 1) * group, t] = p @ v[:s + t + 1]
    return out


def _exact_moe(case, seed):
    data = _moe_inputs(case, seed)
    x = data["x"].double()
    probs = torch.softmax(torch.nn.functional.linear(x, data["router"].double()), -1).cpu()
    out = torch.zeros_like(x)
    routes = {}
    for t in range(x.shape[0]):
        chosen = sorted(range(case["experts"]), key=lambda e: (-float(probs[t, e]), e))[:case["top_k"]]
        total = sum(float(probs[t, e]) for e in chosen) if case["normalize"] else 1.0
        for e in chosen:
            routes.setdefault(e, []).append((t, float(probs[t, e]) / total))
    for e, taken in routes.items():
        rows = x[[t for t, _ in taken]]
        up = data["gate_up"][e].double()
        gate, lin = rows @ up[:case["inter"]].t(), rows @ up[case["inter"]:].t()
        y = (torch.sigmoid(gate) * gate * lin) @ data["down"][e].double().t()
        for j, (t, w) in enumerate(taken):
            out[t] += w * y[j]
    return out


def exact(case, seed):
    if case["op"] == "append":
        return _exact_append(case, seed)
    if case["op"] == "moe":
        return _exact_moe(case, seed)
    if case["batch"] * case["kv_heads"] * case["new"] > 8192 or case["batch"] * case["kv_heads"] * case["length"] > 1 << 24:
        return None
    return _exact_attention(case, seed)
