"""sm_100a kernels of a decoding step against their definitions in 64 bits (``decode_reference.py``)."""

import pytest
import torch

import decode_reference as dr
from mini_train_sys_b200.models.rotary import rope_tables
from mini_train_sys_b200.ops.kv_cache import QuantizedKVCache

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from mini_train_sys_b200.ops.native_backend import NativeOpsBackend

    return NativeOpsBackend()


def rows(batch, heads, n, dim, seed, dtype=torch.bfloat16, spread=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(batch, n, heads, dim, generator=gen, device=DEV)
    if spread:
        x = x * torch.exp(0.5 * torch.randn(1, 1, heads, dim, generator=gen, device=DEV))
    return x.to(dtype).transpose(1, 2)                # strided, as slices of a fused projection are


def fill(ops, cache, layer, k, v, lengths):
    cache.begin(torch.tensor(lengths, dtype=torch.int32, device=DEV), padded=max(max(lengths), 1))
    n = cache.padded
    ops.kv_append(cache, layer, k[:, :, :n], v[:, :, :n])
    cache.commit()


def assert_attention(o, q, keys, values, starts, counts):
    """Bound per output: its own rounding (half a step), and 2^-11 (fp16 probabilities: half a step each) of sum p |v|, with a
    quarter more for the fp32 sums and exponentials behind them.  Probabilities are held times 2^14, where the smallest fp16 value
    is 2^-24: below 2^-39 of the largest one a probability is lost, which is at most 2^-39 of the largest value for each key.
    Outputs below the type's smallest normal value are rounded to half of its smallest step."""

    half = torch.finfo(o.dtype).eps / 2
    for b, (s, n) in enumerate(zip(starts, counts)):
        assert not o[b, :, n:].any()
        if n == 0:
            continue
        want, mass = dr.attend(q[b, :, :n], dr.held(keys[b, :, :s + n]), dr.held(values[b, :, :s + n]), s)
        err = (o[b, :, :n].double() - want).abs()
        bound = half * want.abs() + 1.25 * 2 ** -11 * mass + 2 ** -39 * (s + n) * values[b, :, :s + n].abs().max().double()
        bound += torch.finfo(o.dtype).tiny * half
        assert torch.isfinite(o[b, :, :n]).all() and (err <= bound).all(), (b, float((err - bound).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,heads", [(32, 3), (64, 2), (128, 1)])
@pytest.mark.parametrize("chunks", [[1], [64], [1] * 66, [63, 1, 1, 64, 65], [130, 62, 2, 129], [300]])
def test_append_and_read(ops, dtype, dim, heads, chunks):
    n = sum(chunks)
    k, v, q = (rows(2, h, n, dim, i, dtype) for i, h in enumerate((heads, heads, 2 * heads)))
    cos, sin = (t.to(DEV, dtype) for t in rope_tables(dim, 448, 10000.0))
    cache = QuantizedKVCache(layers=2, batch=2, kv_heads=heads, head_dim=dim, capacity=448, dtype=dtype, device=DEV)
    cache.tail.fill_(float("nan"))                    # nothing that was not written may be read
    at, turned = 0, []
    for c in chunks:
        cache.begin(padded=c)
        turned.append(ops.kv_append(cache, 1, k[:, :, at:at + c], v[:, :, at:at + c], q=q[:, :, at:at + c], cos=cos, sin=sin))
        cache.commit()
        at += c
    kr, vr = ops.kv_read(cache, 1, torch.tensor([-5, 3], dtype=torch.int32, device=DEV), n + 10)
    turned = torch.cat(turned, 2)
    for b, first in ((0, -5), (1, 3)):
        want_k, want_v = dr.held(dr.rotate(k[b], cos[:n], sin[:n], dtype)), dr.held(v[b])
        for got, want in ((kr[b], want_k), (vr[b], want_v)):
            expect = torch.zeros_like(got, dtype=torch.float64)
            lo = max(first, 0)
            expect[:, lo - first:max(n - first, 0)] = want[:, lo:]
            # exact codes; the scale and its product are rounded to fp32 once each
            assert ((got.double() - expect).abs() <= 2 ** -22 * expect.abs()).all()
        assert torch.equal(turned[b].double(), dr.rotate(q[b], cos[:n], sin[:n], dtype))
    assert not cache.codes[0].ne(128).any()           # the other layer
    assert ops.dispatch["kv_append:native"] and ops.dispatch["kv_read:native"] and not ops.dispatch["kv_append:fallback"]


def test_codes_of_halves_extremes_and_non_finite_blocks(ops):
    dim = 64
    cache = QuantizedKVCache(layers=1, batch=1, kv_heads=6, head_dim=dim, capacity=64, device=DEV)
    k = torch.zeros(1, 6, 64, dim, device=DEV, dtype=torch.bfloat16)
    k[0, 0, 5, :4] = torch.tensor([1.5, 0.75, -0.75, 1.5 * 2.5 / 127])
    k[0, 1, 0, 0], k[0, 1, 63, 63] = 3e38, -1.5e38    # 127 x does not fit in fp32
    k[0, 2, 0, 0], k[0, 2, 1, 1] = 1e-39, 5e-40       # subnormal
    k[0, 3, 7, 7] = float("nan")
    k[0, 4, 7, 7] = float("-inf")
    cache.begin(padded=64)
    ops.kv_append(cache, 0, k, k)
    codes = cache.codes[0, 0, :, 0, 0].view(6, 64, dim).int() - 128
    want = torch.round(k[0].double() * 127 / k[0].double().abs().amax((1, 2), keepdim=True)).nan_to_num(0.0).int()
    for h in (0, 1, 2):
        assert torch.equal(codes[h], want[h])
    kr, vr = ops.kv_read(cache, 0, torch.zeros(1, dtype=torch.int32, device=DEV), 64)
    assert kr[0, 3:5].isnan().all() and vr[0, 3:5].isnan().all() and not kr[0, 5].any() and torch.isfinite(kr[0, :3]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_for_every_mantissa_of_the_largest_value(ops, dtype):
    """Blocks whose largest value runs through the mantissas of the type, with every odd multiple of 1 / 254 of it that the type can
    express (exact halves) and random values."""

    mantissas = torch.arange(128, 256) if dtype == torch.bfloat16 else torch.arange(1024, 2048)
    heads = mantissas.numel()
    amax = (mantissas.double() / mantissas[0]).to(DEV)
    halves = (torch.arange(127, device=DEV) * 2 + 1).double()[None] * amax[:, None] / 254
    halves = torch.where(halves.to(dtype).double() == halves, halves, torch.zeros_like(halves))
    gen = torch.Generator(device=DEV).manual_seed(5)
    k = (torch.rand(heads, 64 * 32, generator=gen, device=DEV, dtype=torch.float64) * 2 - 1) * amax[:, None]
    k[:, 0], k[:, 1:128], k[:, 128:255] = amax, halves, -halves
    k = k.to(dtype).view(1, heads, 64, 32)
    cache = QuantizedKVCache(layers=1, batch=1, kv_heads=heads, head_dim=32, capacity=64, dtype=dtype, device=DEV)
    cache.begin(padded=64)
    ops.kv_append(cache, 0, k, k)
    want = torch.round(k[0].double() * 127 / k[0].double().abs().amax((1, 2), keepdim=True)).int()
    assert torch.equal(cache.codes[0, 0, :, 0, 0].reshape(heads, 64, 32).int() - 128, want)
    vr = ops.kv_read(cache, 0, torch.zeros(1, dtype=torch.int32, device=DEV), 64)[1][0]
    assert ((vr.double() - want * (amax / 127)[:, None, None]).abs() <= 2 ** -22 * want.abs() * amax[:, None, None]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,hkv,group", [(32, 3, 1), (64, 2, 1), (64, 1, 12), (128, 2, 4), (64, 2, 40)])
@pytest.mark.parametrize("new", [1, 2, 17, 65])
def test_cached_attention(ops, dtype, dim, hkv, group, new):
    lengths = [0, 1, 63, 64, 65, 700, 191]            # none, one, ends of blocks, many splits
    counts = [new, new, min(new, 1), new, 0, new, max(1, new // 2)]
    batch, most = len(lengths), max(lengths) + new
    k, v = rows(batch, hkv, most, dim, 1, dtype), rows(batch, hkv, most, dim, 2, dtype, spread=False)
    q = rows(batch, hkv * group, new, dim, 3, dtype, spread=False)
    cache = QuantizedKVCache(layers=1, batch=batch, kv_heads=hkv, head_dim=dim, capacity=1024, dtype=dtype, device=DEV)
    cache.tail.fill_(float("nan"))
    fill(ops, cache, 0, k, v, lengths)
    fresh_k = torch.stack([k[b, :, s:s + new] for b, s in enumerate(lengths)])
    fresh_v = torch.stack([v[b, :, s:s + new] for b, s in enumerate(lengths)])
    for b, n in enumerate(counts):                    # padded rows hold whatever they hold
        for t in (fresh_k, fresh_v, q):
            t[b, :, n:] = float("nan")
    cache.begin(torch.tensor(counts, device=DEV), padded=new)
    qo = ops.kv_append(cache, 0, fresh_k, fresh_v, q=q)
    o = ops.cached_attention(qo, cache, 0)
    assert_attention(o, q, k, v, lengths, counts)
    assert torch.equal(o, ops.cached_attention(qo, cache, 0))
    assert ops.dispatch["cached_attention:native"] and not ops.dispatch["cached_attention:fallback"]


@pytest.mark.parametrize("capacity,length", [(64, 3), (2048, 2047), (40000, 39999), (70000, 5)])
def test_cached_attention_over_lengths_and_capacities(ops, capacity, length):
    k, v = rows(1, 2, length + 1, 64, 4), rows(1, 2, length + 1, 64, 5, spread=False)
    q = rows(1, 4, 1, 64, 6, spread=False) * 3
    cache = QuantizedKVCache(layers=1, batch=1, kv_heads=2, head_dim=64, capacity=capacity, device=DEV)
    fill(ops, cache, 0, k, v, [length])
    cache.begin()
    ops.kv_append(cache, 0, k[:, :, length:], v[:, :, length:])
    assert_attention(ops.cached_attention(q, cache, 0), q, k, v, [length], [1])


@pytest.mark.parametrize("counted", [[0] * 63 + [1], [1] + [0] * 62 + [1], [1] * 64])
def test_cached_attention_of_many_rows(ops, counted):
    """More rows than are joined at once, of sequences that are cut into many parts or into few."""

    lengths = [9000 if n else 0 for n in counted] if sum(counted) < 64 else [17 * b for b in range(64)]
    k, v = rows(64, 2, max(lengths) + 1, 32, 11), rows(64, 2, max(lengths) + 1, 32, 12, spread=False)
    q = rows(64, 24, 1, 32, 13, spread=False)
    cache = QuantizedKVCache(layers=1, batch=64, kv_heads=2, head_dim=32, capacity=9001, device=DEV)
    fill(ops, cache, 0, k, v, lengths)
    cache.begin(torch.tensor(counted, dtype=torch.int32, device=DEV))
    fresh = [torch.stack([x[b, :, n:n + 1] for b, n in enumerate(lengths)]) for x in (k, v)]
    ops.kv_append(cache, 0, *fresh)
    assert_attention(ops.cached_attention(q, cache, 0), q, k, v, lengths, counted)


def test_scores_far_apart_and_query_scales(ops):
    """One key takes all of the mass; queries that are tiny, huge or zero."""

    k, v = rows(1, 2, 200, 64, 7), rows(1, 2, 200, 64, 8, spread=False)
    k[0, :, 150] = 20.0
    q = torch.ones(1, 2, 4, 64, device=DEV, dtype=torch.bfloat16)
    q[0, :, 1] = 1e-30
    q[0, :, 2] = 0.0
    q[0, :, 3] = 1e4
    cache = QuantizedKVCache(layers=1, batch=1, kv_heads=2, head_dim=64, capacity=256, device=DEV)
    fill(ops, cache, 0, k, v, [196])
    cache.begin(padded=4)
    ops.kv_append(cache, 0, k[:, :, 196:], v[:, :, 196:])
    assert_attention(ops.cached_attention(q, cache, 0), q, k, v, [196], [4])


def test_a_non_finite_token_stays_in_its_sequence_and_its_block(ops):
    k, v = rows(2, 1, 130, 64, 9), rows(2, 1, 130, 64, 10, spread=False)
    clean = k.clone()
    k[1, :, 70] = float("nan")
    outs = []
    for keys in (clean, k):
        cache = QuantizedKVCache(layers=1, batch=2, kv_heads=1, head_dim=64, capacity=192, device=DEV)
        cache.begin(padded=130)
        q = ops.kv_append(cache, 0, keys, v, q=v)
        outs.append(ops.cached_attention(q, cache, 0))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1, :, :64], outs[1][1, :, :64])
    assert outs[1][1, :, 70:].isnan().all()


@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_the_plan_of_an_attention_fits_on_the_machine(ops, dim, fp16):
    """As many CTAs as are resident at once: single items and lists of units, small tiles and large, few sequences and thousands."""

    from mini_train_sys_b200.ops.native_backend import ext

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    kinds = set()
    for batch in (1, 4, 17, 40, 64, 600, 660, 2048):
        for group, new in ((1, 1), (8, 1), (1, 17), (3, 9), (4, 32)):
            for blocks in (1, 8, 32, 600):
                rows_, ctas, cluster, resident = ext().cached_attention_plan(batch, 4, 4 * group, new, dim, blocks, fp16)
                assert 0 < ctas <= sms * resident, (batch, group, new, blocks)
                assert cluster == 0 or ctas % cluster == 0
                kinds.add((cluster > 0, rows_))
    assert {(True, 8), (False, 8), (False, 16 if dim == 128 else 32)} <= kinds


def test_cached_attention_of_more_sequences_than_leave_room_for_three_ctas(ops):
    lengths = [70 + 40 * (b % 5 == 0) + b % 7 for b in range(700)]
    k, v = rows(700, 1, 120, 128, 34), rows(700, 1, 120, 128, 35, spread=False)
    q = rows(700, 2, 1, 128, 36, spread=False)
    cache = QuantizedKVCache(layers=1, batch=700, kv_heads=1, head_dim=128, capacity=1024, device=DEV)
    fill(ops, cache, 0, k, v, lengths)
    cache.begin()
    ops.kv_append(cache, 0, *[torch.stack([x[b, :, n:n + 1] for b, n in enumerate(lengths)]) for x in (k, v)])
    assert_attention(ops.cached_attention(q, cache, 0), q, k, v, lengths, [1] * 700)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group,batch,capacity", [(32, 1, 1, 256), (64, 3, 2, 256), (64, 24, 3, 8192), (128, 1, 2, 256), (128, 8, 40, 4096)])
@pytest.mark.parametrize("start", [0, 70, 100])
def test_a_later_token_that_is_not_finite_reaches_no_earlier_row_of_an_open_block(ops, dtype, dim, group, batch, capacity, start):
    """Values and keys of a step whose block stays open: rows before a NaN or an infinity are those of a clean step, rows behind it hold
    it.  Both ways of sharing the work, and both halves of the block."""

    new = 20
    k, v = rows(batch, 2, start + new, dim, 31, dtype), rows(batch, 2, start + new, dim, 32, dtype, spread=False)
    q = rows(batch, 2 * group, new, dim, 33, dtype, spread=False)
    inf = float("inf")
    for name, where, token, value in (("v", 1, 5, inf), ("v", 1, 17, -inf), ("v", 0, 1, float("nan")), ("k", 1, 8, float("nan")), ("k", 0, 19, inf)):
        outs = []
        for broken in (False, True):
            fresh = {n: t[:, :, start:].clone() for n, t in (("k", k), ("v", v))}
            if broken:
                fresh[name][0, where, token, 3] = value
            cache = QuantizedKVCache(layers=1, batch=batch, kv_heads=2, head_dim=dim, capacity=capacity, dtype=dtype, device=DEV)
            if start:
                fill(ops, cache, 0, k, v, [start] * batch)
            cache.begin(padded=new)
            ops.kv_append(cache, 0, fresh["k"], fresh["v"])
            outs.append(ops.cached_attention(q, cache, 0))
        clean, got = outs
        hit = slice(where * group, (where + 1) * group)
        others = [h for h in range(2 * group) if not where * group <= h < (where + 1) * group]
        assert torch.isfinite(clean).all() and torch.equal(got[1:], clean[1:]) and torch.equal(got[0, others], clean[0, others])
        # sums in another order: the bound of the other tests, on values of this size
        early = (got[0, hit, :token].double() - clean[0, hit, :token].double()).abs()
        assert (early <= torch.finfo(dtype).eps * clean[0, hit, :token].double().abs() + 2.5 * 2 ** -11 * v.abs().max().double()).all()
        late = got[0, hit, token:]
        if name == "k":
            # a score of +inf is the row's maximum and makes a NaN of it, one of -inf is a probability of 0
            alone = value != value or q[0, hit, token:, 3].float() > 0
            assert (late.isnan().all(-1) == alone).all() and torch.isfinite(late[~late.isnan().all(-1)]).all()
        else:
            others = [d for d in range(dim) if d != 3]
            want = clean[0, hit, token:, others].double()
            assert (late[..., others].double() - want).abs().max() <= torch.finfo(dtype).eps * want.abs().max() + 2.5 * 2 ** -11 * v.abs().max().double()
            assert late[..., 3].isnan().all() if value != value else (late[..., 3] == value).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_queries_and_repeated_steps_and_copies(ops, dtype):
    """Logits of some hundreds; a step that is appended twice; a copy that goes on by itself."""

    import copy

    k, v = rows(2, 2, 700, 64, 14, dtype), rows(2, 2, 700, 64, 15, dtype, spread=False)
    q = (rows(2, 6, 20, 64, 16, torch.float32, spread=False) * 8).to(dtype)
    q[:, 2:4] = (q[:, 2:4].float() * 4).to(dtype).abs()           # no sign cancels in the sums
    cache = QuantizedKVCache(layers=1, batch=2, kv_heads=2, head_dim=64, capacity=704, dtype=dtype, device=DEV)
    fill(ops, cache, 0, k, v, [640, 597])
    fresh = [torch.stack([t[b, :, s:s + 20] for b, s in enumerate((640, 597))]) for t in (k, v)]
    other = copy.deepcopy(cache)
    for c, repeats in ((cache, 2), (other, 1)):
        for _ in range(repeats):
            c.begin(padded=20)
            ops.kv_append(c, 0, *fresh)
        assert_attention(ops.cached_attention(q, c, 0), q, k, v, [640, 597], [20, 20])
        c.commit()
    assert torch.equal(cache.records, other.records) and cache.records.data_ptr() != other.records.data_ptr()
    cache.begin(padded=20)
    ops.kv_append(cache, 0, *fresh)
    assert other.lengths.tolist() == [660, 617] and not torch.equal(cache.tail, other.tail)


def test_two_streams_and_replays(ops):
    """Two caches on two streams at once, and one captured step replayed while its lengths move on, equal the plain calls."""

    n, steps = 100, 70
    k, v = rows(2, 2, n + steps, 64, 11), rows(2, 2, n + steps, 64, 12, spread=False)
    q = rows(2, 4, n + steps, 64, 13, spread=False)

    def fresh():
        cache = QuantizedKVCache(layers=1, batch=2, kv_heads=2, head_dim=64, capacity=256, device=DEV)
        fill(ops, cache, 0, k, v, [n, n - 37])
        return cache

    def step(cache, kt, vt, qt):
        cache.begin()
        out = ops.cached_attention(ops.kv_append(cache, 0, kt, vt, q=qt), cache, 0)
        cache.commit()
        return out

    piece = [tuple(t[:, :, n + i:n + i + 1].contiguous() for t in (k, v, q)) for i in range(steps)]
    plain = fresh()
    want = [step(plain, *p) for p in piece]
    caches, streams = [fresh(), fresh()], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                got[j].append(step(caches[j], *piece[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))

    replayed = fresh()
    static = tuple(t.clone() for t in piece[0])
    warm = fresh()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(warm, *static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    held = replayed.held
    with torch.cuda.graph(graph):
        out = step(replayed, *static)
    replayed.held = held                              # the capture has run nothing
    for i in range(steps):
        for dst, src in zip(static, piece[i]):
            dst.copy_(src)
        replayed.replayed(1)
        graph.replay()
        assert torch.equal(out, want[i]), i
    assert torch.equal(replayed.codes, plain.codes) and torch.equal(replayed.lengths, plain.lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_replays_behind_the_rotary_tables_take_their_last_row(ops, dtype, dim):
    """A graph that is replayed beyond the tables it was recorded with: the codes, the open block and the queries of the plain form."""

    from mini_train_sys_b200.models.ops import get_ops_backend

    table, steps = 70, 75
    k, v, q = rows(2, 2, 3 * steps, dim, 21, dtype), rows(2, 2, 3 * steps, dim, 22, dtype), rows(2, 4, 3 * steps, dim, 23, dtype)
    cos, sin = (t.to(DEV, dtype) for t in rope_tables(dim, table, 10000.0))
    full = [torch.cat((t, t[-1:].expand(256 - table, -1))).cpu() for t in (cos, sin)]
    cache = QuantizedKVCache(layers=1, batch=2, kv_heads=2, head_dim=dim, capacity=256, dtype=dtype, device=DEV)
    plain = QuantizedKVCache(layers=1, batch=2, kv_heads=2, head_dim=dim, capacity=256, dtype=dtype, device="cpu")
    static = [t[:, :, :3].clone() for t in (k, v, q)]

    def step(backend, into, kt, vt, qt, c, s):
        into.begin(padded=3)
        out = backend.kv_append(into, 0, kt, vt, q=qt, cos=c, sin=s)
        into.commit()
        return out

    step(ops, QuantizedKVCache(layers=1, batch=2, kv_heads=2, head_dim=dim, capacity=64, dtype=dtype, device=DEV), *static, cos, sin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ops, cache, *static, cos, sin)
    cache.held = 0                                    # the capture has run nothing
    for i in range(steps):
        piece = [t[:, :, 3 * i:3 * i + 3] for t in (k, v, q)]
        for dst, src in zip(static, piece):
            dst.copy_(src)
        cache.replayed(3)
        graph.replay()
        want = step(get_ops_backend("torch"), plain, *(t.cpu() for t in piece), *full)
        # products of 16-bit factors are exact in fp32, so both forms round the same sum
        assert torch.equal(out.cpu(), want), i
    first = torch.zeros(2, dtype=torch.int32)
    got, want = ops.kv_read(cache, 0, first.to(DEV), 3 * steps), get_ops_backend("torch").kv_read(plain, 0, first, 3 * steps)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------------------------
# mixture of experts for a few tokens
# ---------------------------------------------------------------------------------------------
def moe_inputs(tokens, experts, hidden, inter, seed, router_dtype=torch.float32):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)                         # noqa: E731
    return (r(tokens, hidden).to(torch.bfloat16), (r(experts, hidden) * 2 * hidden ** -0.5).to(router_dtype),
            (r(experts, 2 * inter, hidden) * hidden ** -0.5).to(torch.bfloat16), (r(experts, hidden, inter) * inter ** -0.5).to(torch.bfloat16))


def assert_moe(y, want):
    """One rounding to bf16 (half a step, ``finfo.eps / 2`` = 2^-8 of the value); fp32 sums and the 2^-16 of the split hidden
    values are far below 2^-12 of the typical output."""

    half = torch.finfo(torch.bfloat16).eps / 2
    rms = want.pow(2).mean().sqrt()
    err = (y.double() - want).abs()
    assert (err <= (1 + 2 ** -6) * half * want.abs() + 2 ** -12 * rms).all(), float((err / rms).max())


@pytest.mark.parametrize("tokens", [1, 2, 8, 9, 17, 33, 64])
@pytest.mark.parametrize("experts,top_k,hidden,inter", [(8, 2, 768, 1024), (4, 1, 128, 128), (64, 8, 264, 72), (5, 5, 40, 8), (1, 1, 1032, 520)])
def test_moe_tokens(ops, tokens, experts, top_k, hidden, inter):
    for normalize in (True, False):
        x, r, gu, dn = moe_inputs(tokens, experts, hidden, inter, tokens + experts)
        y = ops.moe_tokens(x, r, gu, dn, top_k, normalize=normalize)
        assert_moe(y, dr.moe(x, r, gu, dn, top_k, normalize))
        assert torch.equal(y, ops.moe_tokens(x, r, gu, dn, top_k, normalize=normalize))
    assert ops.dispatch["moe_tokens:native"] and not ops.dispatch["moe_tokens:fallback"]


@pytest.mark.parametrize("tokens", [1, 3, 4, 5])
@pytest.mark.parametrize("router_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts,hidden", [(8, 768), (24, 2056)])
def test_moe_tokens_of_both_routings(ops, tokens, router_dtype, experts, hidden):
    """Few tokens and many, small routers and large ones are routed by different code."""

    x, r, gu, dn = moe_inputs(tokens, experts, hidden, 64, 7, router_dtype)
    assert_moe(ops.moe_tokens(x, r, gu, dn, 3, normalize=True), dr.moe(x, r, gu, dn, 3, True))


def test_moe_tokens_crowded_ties_strides_and_weights(ops):
    x, r, gu, dn = moe_inputs(64, 16, 256, 136, 1)
    x[:] = x[0]                                       # every token goes to the same experts
    assert_moe(ops.moe_tokens(x, r, gu, dn, 4, normalize=True), dr.moe(x, r, gu, dn, 4, True))
    x, r, gu, dn = moe_inputs(20, 48, 256, 136, 2, torch.bfloat16)
    r[40], r[33], r[7] = r[3], r[3], r[3]             # exact ties: the lower experts win
    want = dr.moe(x, r, gu, dn, 2, True)
    assert_moe(ops.moe_tokens(x, r, gu, dn, 2, normalize=True), want)
    wide = torch.full((20, 512), float("nan"), device=DEV, dtype=torch.bfloat16)
    wide[:, 8:264] = x
    assert_moe(ops.moe_tokens(wide[:, 8:264], r, gu, dn, 2, normalize=True), want)
    with torch.no_grad():                             # fp32 parameters: their bf16 copies
        assert torch.equal(ops.moe_tokens(x, r, torch.nn.Parameter(gu.float()), torch.nn.Parameter(dn.float()), 2, normalize=True),
                           ops.moe_tokens(x, r, gu, dn, 2, normalize=True))
    x[3] = float("nan")                               # a token that is not a number touches no other
    y = ops.moe_tokens(x, r, gu, dn, 2, normalize=True)
    keep = torch.arange(20, device=DEV) != 3
    assert y[3].isnan().all()
    assert_moe(y[keep], want[keep])
    assert ops.moe_tokens(x[:0], r, gu, dn, 2, normalize=True).shape == (0, 256)


def test_moe_tokens_copies_no_weights_that_it_does_not_use(ops):
    """fp32 weights and a call that the kernels do not cover: the plain form reads the weights as they are."""

    from mini_train_sys_b200.ops.native_backend import kept_bf16

    x, r, gu, dn = moe_inputs(65, 16, 256, 64, 6)
    weights = [torch.nn.Parameter(t.float()) for t in (gu, dn)]
    before = ops.dispatch["moe_tokens:fallback"]
    with torch.no_grad():
        for rows_, top_k in ((x, 2), (x[:8].float(), 2), (x[:8], 9)):
            ops.moe_tokens(rows_, r, *weights, top_k, normalize=True)
            assert all(kept_bf16(w) is None for w in weights)
        assert ops.dispatch["moe_tokens:fallback"] == before + 3
        ops.dispatch.subtract({"moe_tokens:fallback": 3})
        assert torch.equal(ops.moe_tokens(x[:8], r, *weights, 2, normalize=True), ops.moe_tokens(x[:8], r, gu, dn, 2, normalize=True))
    assert all(kept_bf16(w) is not None for w in weights)


def test_moe_tokens_on_two_streams_and_replayed(ops):
    x, r, gu, dn = moe_inputs(12, 8, 768, 1024, 3)
    want = ops.moe_tokens(x, r, gu, dn, 2, normalize=True)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.moe_tokens(x, r, gu, dn, 2, normalize=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    static = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.moe_tokens(static, r, gu, dn, 2, normalize=True)
    static.copy_(x)
    graph.replay()
    assert torch.equal(y, want)


@pytest.mark.parametrize("tokens,experts,hidden,inter", [(1, 8, 256, 128), (4, 8, 768, 1024), (12, 8, 768, 1024), (64, 64, 768, 256)])
def test_operators_that_read_what_the_one_before_wrote(ops, tokens, experts, hidden, inter):
    """Append, attention and two layers of experts in a row, each kernel started while the one before it runs: the same values as
    with the device waited for between the calls, eagerly and replayed."""

    heads = hidden // 64
    x, r, gu, dn = moe_inputs(tokens, experts, hidden, inter, 17)
    k, v = rows(tokens, heads, 150, 64, 18), rows(tokens, heads, 150, 64, 19, spread=False)
    cos, sin = (t.to(DEV, torch.bfloat16) for t in rope_tables(64, 192, 10000.0))
    cache = QuantizedKVCache(layers=1, batch=tokens, kv_heads=heads, head_dim=64, capacity=192, device=DEV)
    fill(ops, cache, 0, k, v, [149 - 2 * (b % 60) for b in range(tokens)])
    cache.begin()
    fresh = [t[:, :, 149:] for t in (k, v)]

    def chain(between):
        out = []
        q = x.view(tokens, 1, heads, 64).transpose(1, 2)
        for _ in range(3):
            out.append(ops.kv_append(cache, 0, *fresh, q=q, cos=cos, sin=sin))
            between()
            out.append(ops.cached_attention(out[-1], cache, 0))
            between()
            out.append(ops.moe_tokens(out[-1].transpose(1, 2).reshape(tokens, hidden), r, gu, dn, 2, normalize=True))
            between()
            out.append(ops.moe_tokens(out[-1], r, gu, dn, 2, normalize=False))
            between()
            q = out[-1].view(tokens, 1, heads, 64).transpose(1, 2)
        return out

    want = chain(torch.cuda.synchronize)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(lambda: None)
    for _ in range(10):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_native_and_plain_forms_share_a_cache(ops):
    """Calls whose strides send one operator of a step to the plain form, on a cache that the kernels fill and read too."""

    n, steps = 60, [1, 3, 5, 70, 2]
    total = n + sum(steps)
    k, v, q = rows(2, 2, total, 64, 41), rows(2, 2, total, 64, 42, spread=False), rows(2, 4, total, 64, 43, spread=False)
    odd = [torch.empty(2, t.shape[1], total, 66, device=DEV, dtype=t.dtype) for t in (k, v, q)]      # rows on no 16 bytes
    for dst, src in zip(odd, (k, v, q)):
        dst[..., :64] = src
    cache = QuantizedKVCache(layers=1, batch=2, kv_heads=2, head_dim=64, capacity=256, device=DEV)
    fill(ops, cache, 0, k, v, [n, n])
    before, at = dict(ops.dispatch), n
    for i, c in enumerate(steps):
        sources = odd if i % 2 else (k, v, q)
        ks, vs = (t[:, :, at:at + c, :64] for t in sources[:2])
        qs = (q if i % 2 else odd[2])[:, :, at:at + c, :64]
        cache.begin(padded=c)
        ops.kv_append(cache, 0, ks, vs)
        assert_attention(ops.cached_attention(qs, cache, 0), q[:, :, at:at + c], k, v, [at, at], [c, c])
        cache.commit()
        at += c
    for op, plain in (("kv_append", 2), ("cached_attention", 3)):
        assert ops.dispatch[f"{op}:fallback"] == before.get(f"{op}:fallback", 0) + plain
        ops.dispatch.subtract({f"{op}:fallback": plain})


def test_what_the_kernels_do_not_cover_takes_the_plain_path(ops):
    before = dict(ops.dispatch)
    cache = QuantizedKVCache(layers=1, batch=1, kv_heads=2, head_dim=48, capacity=128, device=DEV)
    k, v, q = rows(1, 2, 70, 48, 1), rows(1, 2, 70, 48, 2, spread=False), rows(1, 2, 70, 48, 3, spread=False)
    cache.begin(padded=70)
    ops.kv_append(cache, 0, k, v)
    assert_attention(ops.cached_attention(q, cache, 0), q, k, v, [0], [70])
    x, r, gu, dn = moe_inputs(65, 4, 64, 64, 4)
    assert_moe(ops.moe_tokens(x, r, gu, dn, 2, normalize=True), dr.moe(x, r, gu, dn, 2, True))
    for op in ("kv_append", "cached_attention", "moe_tokens"):
        assert ops.dispatch[f"{op}:fallback"] == before.get(f"{op}:fallback", 0) + 1
    ops.dispatch.subtract({f"{op}:fallback": 1 for op in ("kv_append", "cached_attention", "moe_tokens")})
