"""Plain forms of the decoding-step operators, their refusals and the cache's bookkeeping (no GPU)."""

import pytest
import torch

import decode_reference as dr
from mini_train_sys_b200.models.ops import get_ops_backend
from mini_train_sys_b200.models.rotary import rope_tables
from mini_train_sys_b200.ops.kv_cache import QuantizedKVCache, quantize_block


@pytest.fixture(scope="module")
def ops():
    return get_ops_backend("torch")


def make_cache(**kw):
    args = dict(layers=2, batch=3, kv_heads=2, head_dim=32, capacity=300, dtype=torch.bfloat16, device="cpu")
    args.update(kw)
    return QuantizedKVCache(**args)


def rows(batch, heads, n, dim, seed, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(batch, heads, n, dim, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("chunks", [[200], [1] * 70, [63, 1, 1, 64, 65], [130, 3]])
def test_contents_do_not_depend_on_how_the_tokens_arrive(ops, dtype, chunks):
    n = sum(chunks)
    k, v = rows(3, 2, n, 32, 1, dtype), rows(3, 2, n, 32, 2, dtype)
    cos, sin = (t.to(dtype) for t in rope_tables(32, 300, 10000.0))
    cache = make_cache(dtype=dtype)
    at = 0
    with torch.no_grad():
        for c in chunks:
            cache.begin(padded=c)
            ops.kv_append(cache, 1, k[:, :, at:at + c], v[:, :, at:at + c], cos=cos, sin=sin)
            cache.commit()
            at += c
        kr, vr = ops.kv_read(cache, 1, torch.full((3,), -5, dtype=torch.int32), n + 10)
    assert not kr[:, :, :5].any() and not kr[:, :, n + 5:].any() and not vr[:, :, n + 5:].any()
    for b in range(3):
        want_k = dr.held(dr.rotate(k[b], cos[:n], sin[:n], dtype))
        # fp32 results: one rounding of the scale and one of the product; rotations of fp32 values differ by a rounding of the sum,
        # which may move a code by one
        step = want_k.abs().max() / 127 if dtype == torch.float32 else 0.0
        assert (kr[b, :, 5:n + 5].double() - want_k).abs().max() <= 2 ** -22 * want_k.abs().max() + step
        want_v = dr.held(v[b])
        assert (vr[b, :, 5:n + 5].double() - want_v).abs().max() <= 2 ** -22 * want_v.abs().max()
    assert not ops.kv_read(cache, 0, torch.zeros(3, dtype=torch.int32), n)[0].any()      # the other layer is untouched


def test_ragged_steps_padding_and_empty_rows(ops):
    cache = make_cache()
    counts = [0, 70, 5]
    k, v, q = rows(3, 2, 70, 32, 3), rows(3, 2, 70, 32, 4), rows(3, 4, 70, 32, 5)
    for t in (k, v, q):
        t[2, :, 5:] = float("nan")                 # padding is not looked at
        t[0] = float("inf")
    cache.begin(torch.tensor(counts), padded=70)
    qo = ops.kv_append(cache, 0, k, v, q=q)
    o = ops.cached_attention(qo, cache, 0)
    assert not o[0].any() and not o[2, :, 5:].any() and torch.isfinite(o).all()
    for b, n in ((1, 70), (2, 5)):
        want, _ = dr.attend(q[b, :, :n], dr.held(k[b, :, :n]), dr.held(v[b, :, :n]), 0)
        assert (o[b, :, :n].double() - want).abs().max() <= 2 ** -8 * want.abs().max()
    cache.commit()
    assert cache.lengths.tolist() == counts and cache.held == 70


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("start", [0, 50, 100])
def test_a_later_token_that_is_not_finite_reaches_no_earlier_row(ops, dtype, start):
    """Rows before a NaN or an infinity are those of a clean step, up to the block that a finished one shares a scale in."""

    new = 20
    k, v = rows(2, 2, start + new, 32, 1, dtype), rows(2, 2, start + new, 32, 2, dtype)
    q = rows(2, 4, new, 32, 3, dtype)
    inf = float("inf")
    for name, token, value in (("v", 16, inf), ("v", 16, float("nan")), ("v", 17, -inf), ("k", 18, float("nan"))):
        outs = []
        for broken in (False, True):
            fresh = {n: t[:, :, start:].clone() for n, t in (("k", k), ("v", v))}
            if broken:
                fresh[name][0, 1, token, 3] = value
            cache = make_cache(batch=2, dtype=dtype)
            if start:
                cache.begin(padded=start)
                ops.kv_append(cache, 0, k[:, :, :start], v[:, :, :start])
                cache.commit()
            cache.begin(padded=new)
            ops.kv_append(cache, 0, fresh["k"], fresh["v"])
            outs.append(ops.cached_attention(q, cache, 0))
        clean, got = outs
        assert torch.isfinite(clean).all() and torch.equal(got[1], clean[1]) and torch.equal(got[0, :2], clean[0, :2])
        closed = (start + new) // 64 * 64 - start                 # rows of the step in finished blocks
        first = token if token >= closed else 0                   # rows from here on may see it
        torch.testing.assert_close(got[0, 2:, :first], clean[0, 2:, :first], rtol=torch.finfo(dtype).eps, atol=1e-6)
        late = got[0, 2:, token:]
        if name == "v" and token >= closed:
            assert late[..., 3].isnan().all() if value != value else (late[..., 3] == value).all()
            torch.testing.assert_close(late[..., 4:], clean[0, 2:, token:, 4:], rtol=torch.finfo(dtype).eps, atol=1e-6)
        else:
            assert late.isnan().any(-1).all()


def test_codes_are_those_of_exact_arithmetic():
    # halves: 127 x / a = n + 1/2 for x = a / 2 (63.5 -> 64, half to even), and no value between two halves is moved
    x = torch.zeros(1, 64, 32)
    x[0, 0, :4] = torch.tensor([1.5, 0.75, -0.75, 0.0])
    codes, scale = quantize_block(x)
    assert codes[0, 0, :4].tolist() == [255, 192, 64, 128] and scale.item() == (torch.tensor(1.5) / 127).item()
    zero, s0 = quantize_block(torch.zeros(1, 64, 32))
    assert (zero == 128).all() and s0.item() == 0
    bad = x.clone()
    bad[0, 3, 3] = float("inf")
    assert quantize_block(bad)[1].isnan().all()


def test_a_broken_off_step_can_be_repeated(ops):
    k, v = rows(3, 2, 90, 32, 6), rows(3, 2, 90, 32, 7)
    reads = []
    for repeat in (False, True):
        cache = make_cache()
        cache.begin(padded=60)
        ops.kv_append(cache, 0, k[:, :, :60], v[:, :, :60])
        cache.commit()
        for _ in range(2 if repeat else 1):
            cache.begin(padded=30)
            ops.kv_append(cache, 0, k[:, :, 60:], v[:, :, 60:])
        cache.commit()
        reads.append(ops.kv_read(cache, 0, torch.zeros(3, dtype=torch.int32), 90))
    assert all(torch.equal(a, b) for a, b in zip(*reads))


def test_refusals(ops):
    cache = make_cache(capacity=64)
    k, q = rows(3, 2, 4, 32, 8), rows(3, 4, 4, 32, 9)
    with pytest.raises(RuntimeError, match="begin"):
        ops.kv_append(cache, 0, k, k)
    with pytest.raises(RuntimeError, match="begin"):
        ops.cached_attention(q, cache, 0)
    with pytest.raises(RuntimeError, match="no step"):
        cache.commit()
    with pytest.raises(ValueError, match="capacity"):
        cache.begin(padded=65)
    with pytest.raises(ValueError, match="at least one"):
        cache.begin(padded=0)
    with pytest.raises(ValueError, match="one integer"):
        cache.begin(torch.ones(2, dtype=torch.int32))
    cache.begin(padded=4)
    for bad, match in ((k[:, :1], "2 heads"), (k[..., :16], "must be"), (k.float(), "activation type"), (k[:, :, :3], "padded tokens"),
                       (k[:2], "must be")):
        with pytest.raises(ValueError, match=match):
            ops.kv_append(cache, 0, k, bad)
    with pytest.raises(ValueError, match="multiple of 2 heads"):
        ops.cached_attention(rows(3, 3, 4, 32, 1), cache, 0)
    with pytest.raises(IndexError):
        ops.cached_attention(q, cache, 2)
    cos, sin = (t.to(torch.bfloat16) for t in rope_tables(32, 3, 10000.0))
    with pytest.raises(ValueError, match="positions"):
        ops.kv_append(cache, 0, k, k, cos=cos, sin=sin)
    with pytest.raises(ValueError, match="come together"):
        ops.kv_append(cache, 0, k, k, cos=cos)
    with pytest.raises(RuntimeError, match="inference"):
        ops.kv_append(cache, 0, k.clone().requires_grad_(), k)
    with pytest.raises(ValueError, match="int32"):
        ops.kv_read(cache, 0, torch.zeros(3), 4)
    with pytest.raises(ValueError, match="negative"):
        ops.kv_read(cache, 0, torch.zeros(3, dtype=torch.int32), -1)
    with pytest.raises(ValueError, match="positive"):
        make_cache(batch=0)
    with pytest.raises(ValueError, match="dtype"):
        make_cache(dtype=torch.float64)
    cache.commit()
    cache.replayed(60)
    with pytest.raises(ValueError, match="capacity"):
        cache.replayed(1)
    cache.reset()
    assert cache.held == 0 and not cache.lengths.any()


@pytest.mark.parametrize("normalize", [True, False])
def test_moe_tokens_plain(ops, normalize):
    torch.manual_seed(0)
    x, r = torch.randn(5, 24), torch.randn(6, 24)
    r[4] = r[1]                                       # ties go to the lower expert
    gu, dn = torch.randn(6, 32, 24) * 0.2, torch.randn(6, 24, 16) * 0.2
    y = ops.moe_tokens(x, r, gu, dn, 3, normalize=normalize)
    torch.testing.assert_close(y.double(), dr.moe(x, r, gu, dn, 3, normalize), rtol=1e-4, atol=1e-5)
    assert ops.moe_tokens(x[:0], r, gu, dn, 3, normalize=normalize).shape == (0, 24)
    with pytest.raises(ValueError, match="top_k"):
        ops.moe_tokens(x, r, gu, dn, 7, normalize=normalize)
    with pytest.raises(ValueError, match="do not fit"):
        ops.moe_tokens(x, r, gu, dn[:, :, :8], 3, normalize=normalize)
    with pytest.raises(RuntimeError, match="inference"):
        ops.moe_tokens(x.requires_grad_(), r, gu, dn, 3, normalize=normalize)
