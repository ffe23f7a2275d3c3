"""Decoding from a cache where it is easy to be nearly right.

A rounding to bf16 is off by at most 2^-8 of the value, and so is the output's. A softmax weight enters its product as two bf16 values, the
first cut to eight bits and the rest rounded: 2^-15 of it. The f32 sums and exponentials stay below 2^-15 of the sums taken with |v|."""
import numpy as np
import pytest
import torch

import oracle
from paged_model import attention_64
from sys1_b200 import _lib, device, norm, paged, qwen35
from test_paged_gpu import DEV, _attention_case, _decoder, _linear_attention, _refused, _step_case, bf, gen, ints

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ paged attention
@pytest.mark.parametrize("lens,H,kv,dim,page", [([17], 8, 2, 256, 16), ([1, 2, 3, 700], 8, 2, 128, 16), ([40, 65, 0, 5], 6, 3, 64, 4), ([300, 33], 16, 1, 64, 16),
                                                ([128, 2500], 32, 2, 256, 64), ([513], 9, 1, 128, 32), ([9 + i % 90 for i in range(450)], 4, 1, 256, 16),
                                                ([1 + i % 70 for i in range(500)], 4, 2, 128, 16), ([3 + i % 50 for i in range(480)], 2, 2, 64, 8),
                                                ([2 + i % 130 for i in range(450)], 16, 1, 256, 16), ([2 + i % 99 for i in range(450)], 12, 1, 128, 16),
                                                ([2 + i % 99 for i in range(450)], 16, 1, 64, 16)])
@pytest.mark.parametrize("gated", [False, True])
def test_paged_attention_keeps_its_weights(ctx, lens, H, kv, dim, page, gated):
    q, kc, vc, tables, lengths, gate = _attention_case(lens, H, kv, dim, page, len(lens) + H, gated=gated)
    got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    ctx.sync()
    ref, size = attention_64(q, kc, vc, tables, lens, gate, dim ** -0.5)
    err = (got.double().unflatten(1, (-1, dim)) - ref).abs()
    assert bool((err <= 2.0 ** -8 * ref.abs() + 2.0 ** -14 * size).all()), float((err - 2.0 ** -8 * ref.abs()).div(size + 1e-30).max())


@pytest.mark.parametrize("lens,H,kv,dim", [([1, 16, 100], 4, 2, 128), ([5000, 3], 16, 1, 64), ([700], 8, 2, 256)])
def test_paged_attention_of_infinite_values(ctx, lens, H, kv, dim):
    """Weights that are all alike: one infinite value makes its column infinite, two of different sign make it no number."""
    q, kc, vc, tables, lengths, _ = _attention_case(lens, H, kv, dim, 16, 3, gated=False, poison=False)
    q.zero_()
    for b, n in enumerate(lens):
        for j, d, x in ((0, 1, "inf"), (n - 1, 2, "-inf"), (0, 3, "inf"), (n - 1, 3, "-inf"), (n // 2, 4, "nan")):
            vc[tables[b, j // 16].long(), j % 16, :, d] = float(x)
    got = paged.attention_paged(q, kc, vc, tables, lengths)
    ctx.sync()
    ref, _ = attention_64(q, kc, vc, tables, lens, None, dim ** -0.5)
    got, special = got.float().unflatten(1, (-1, dim)), ~torch.isfinite(ref)
    assert bool(special[:, :, 1:5].all()) and int(special.sum()) == 4 * len(lens) * H
    assert torch.equal(got[special].nan_to_num(7.0), ref[special].float().nan_to_num(7.0)) and bool(torch.isfinite(got[~special]).all())


def _blind(q, kc, tables, b, keys, page=16):
    """Scores of -inf for these keys of row b, for every head."""
    q[..., 0] = q[..., 0].abs() + 0.5
    j = torch.tensor(list(keys), device=DEV, dtype=torch.long)
    kc[tables[b].long()[j // page], j % page, :, 0] = float("-inf")


@pytest.mark.parametrize("lens,H,kv,dim", [([20, 100, 33, 0], 4, 2, 128), ([5000, 9000, 300, 40], 8, 2, 256), ([9000, 6000, 100], 16, 1, 64), ([70] * 450, 2, 1, 64)])
def test_paged_attention_of_scores_that_are_minus_infinity(ctx, lens, H, kv, dim):
    """A row without a finite score is no number (softmax divides nothing by nothing); keys of -inf beside others weigh nothing, also where
    they are all that a warp or a block sees. A row without a key stays zero."""
    q, kc, vc, tables, lengths, gate = _attention_case(lens, H, kv, dim, 16, 11, poison=False)
    _blind(q, kc, tables, 0, range(lens[0]))
    _blind(q, kc, tables, 1, range(lens[1] - 1))          # only the last key is left
    _blind(q, kc, tables, 2, range(1, lens[2]))           # only the first
    got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    ctx.sync()
    ref, size = attention_64(q, kc, vc, tables, lens, gate, dim ** -0.5)
    got = got.double().unflatten(1, (-1, dim))
    assert bool(torch.isnan(ref[0]).all()) and bool(torch.isnan(got[0]).all())
    assert bool(((got[1:] - ref[1:]).abs() <= 2.0 ** -8 * ref[1:].abs() + 2.0 ** -14 * size[1:]).all())


def test_paged_attention_of_a_row_whose_pages_are_all_bad(ctx):
    """Keys that are left out are no keys: zeros, and the report; a bad page beside keys of -inf does not hide them."""
    q, kc, vc, tables, lengths, _ = _attention_case([40, 40], 2, 1, 64, 16, 5, gated=False, poison=False)
    _blind(q, kc, tables, 1, range(40))
    tables[0, :3], tables[1, 1] = -1, -1
    got = paged.attention_paged(q, kc, vc, tables, lengths)
    _refused(ctx, "names page -1")
    assert bool((got[0] == 0).all()) and bool(torch.isnan(got[1]).all())


@pytest.mark.parametrize("rows,H,kv,dim,longest", [(200, 6, 3, 64, 200000), (230, 6, 2, 128, 150000), (100, 32, 2, 64, 100000), (3, 16, 1, 128, 90000), (250, 2, 2, 256, 60000),
                                                   (1, 8, 2, 256, 131071), (1, 4, 2, 128, 70001), (2, 4, 4, 64, 70001), (1, 32, 2, 256, 30001), (1, 64, 4, 64, 66164),
                                                   (160, 12, 1, 256, 20001), (300, 12, 1, 128, 20001)])
def test_paged_attention_counts_every_key_once(ctx, rows, H, kv, dim, longest):
    """Scores that are all alike, values that are 1 at the keys that a column marks and 0 elsewhere: the column's output is how many of its
    keys were seen over how many there are. A column marks at most 64 keys, so one missing or counted twice is off by 2^-6 of the
    output, and what is allowed is 2^-8 (the output's rounding) and 2^-14. Every key is marked once; neighbours have different columns."""
    lens = [int(n) for n in np.random.RandomState(9).randint(0, 60, rows)]
    b = rows // 2
    lens[b] = longest
    q, kc, vc, tables, lengths, _ = _attention_case(lens, H, kv, dim, 64, 9, gated=False, poison=False)
    kc.zero_()
    j = torch.arange(longest, device=DEV)
    page, at = tables[b].long()[j // 64], j % 64
    which = torch.arange(kv, device=DEV)[:, None] * 7 + j  # the KV heads' columns are not alike
    column, turn = which % dim, which // dim // 64
    counts = 0
    for t in range(int(turn.max()) + 1):
        vc.zero_()
        for h in range(kv):
            mine = turn[h] == t
            vc[page[mine], at[mine], h, column[h][mine]] = 1.0
        want = torch.stack([torch.bincount(column[h][turn[h] == t], minlength=dim) for h in range(kv)]).double()
        assert int(want.max()) <= 64
        got = paged.attention_paged(q, kc, vc, tables, lengths)[b].double().view(kv, H // kv, dim) * longest
        assert bool(((got - want[:, None]).abs() <= (2.0 ** -8 + 2.0 ** -14) * want[:, None]).all()), (t, float((got - want[:, None]).abs().max()))
        counts += int(want.sum())
    ctx.sync()
    assert counts == kv * longest


def test_paged_attention_refuses_a_scale_beyond_its_exponent(ctx):
    """The scores are kept in units of log 2: a scale that is finite but not times log2(e) would make every score infinite or no number."""
    q, kc, vc, tables, lengths, _ = _attention_case([20, 30], 4, 2, 64, 16, 1, gated=False)
    with pytest.raises(_lib.S1Error, match="scale"):
        paged.attention_paged(q, kc, vc, tables, lengths, scale=2.9e38)
    q.zero_()
    got = paged.attention_paged(q, kc, vc, tables, lengths, scale=2.3e38)
    ctx.sync()
    assert torch.equal(got, paged.attention_paged(q, kc, vc, tables, lengths))


# ------------------------------------------------------------------------------------------------ strides that mean nothing
def _odd(t, dims, stride=3):
    """The same values with another stride in dimensions of size 1."""
    strides = list(t.stride())
    for d in dims:
        assert t.shape[d] == 1
        strides[d] = stride
    return t.as_strided(t.shape, strides)


def test_strides_of_dimensions_of_size_one_are_of_no_account(ctx):
    """One row, one head, one page or one token: whatever a transposed or expanded tensor leaves as the stride there."""
    q, kc, vc, tables, lengths, gate = _attention_case([13], 4, 1, 128, 16, 2, poison=False)
    want = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)  # [1, 4, 128] of strides 128, 128: heads x rows turned round
    assert turned.stride(0) == 128 and torch.equal(paged.attention_paged(turned, kc, vc, tables, lengths, gate=gate), want)
    out = torch.empty(512, 1, dtype=torch.bfloat16, device=DEV).t()
    paged.attention_paged(_odd(q, [0]), _odd(kc, [2]), _odd(vc, [2], 0), _odd(tables, [0], 1), lengths, gate=_odd(gate, [0], 1), out=out)
    assert torch.equal(out, want)
    one = [torch.zeros(1, 16, 1, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    k, v = bf(gen(3), 1, 1, 128), bf(gen(4), 1, 1, 128)
    paged.cache_write(_odd(k, [0, 1], 1), _odd(v, [0, 1], 0), _odd(one[0], [0]), _odd(one[1], [0, 2], 0), ints([5]))
    ctx.sync()
    assert torch.equal(one[0][0, 5], k[0]) and torch.equal(one[1][0, 5], v[0]) and int((one[0] != 0).any(-1).sum()) == 1
    small = [torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)]  # pages of one token
    k, v = bf(gen(3), 2, 2, 64), bf(gen(4), 2, 2, 64)
    paged.cache_write(k, v, _odd(small[0], [1]), _odd(small[1], [1], 0), ints([2, 0]))
    ctx.sync()
    assert torch.equal(small[0][[2, 0], 0], k) and torch.equal(small[1][[2, 0], 0], v)
    table = ints([[4, 7]])
    r = paged.block_tables(ints([3]), _odd(table, [0], 1), ints([1, 2]), ints([2]), 4)
    ctx.sync()
    assert r.slots.tolist() == [19]
    paged.release_blocks(ints([1]), r.lengths, _odd(table, [0], 1), ints([0, 0]), r.free_count.zero_(), 4)
    ctx.sync()
    assert r.lengths.tolist() == [-1] and r.free_count.tolist() == [1]


def test_delta_step_of_one_row_of_any_stride(ctx):
    c = _step_case(1, 2, 4, 8)
    d = dict(c, state=c["state"].clone(), conv_state=c["conv_state"].clone())
    want = qwen35.gated_delta_rule_step(**c)
    for name in ("mixed", "b", "a", "z"):
        d[name] = _odd(d[name], [0], 1)
    out = torch.empty(512, 1, dtype=torch.bfloat16, device=DEV).t()
    qwen35.gated_delta_rule_step(**d, out=out)
    ctx.sync()
    assert torch.equal(out, want) and torch.equal(c["state"], d["state"]) and torch.equal(c["conv_state"], d["conv_state"])


# ------------------------------------------------------------------------------------------------ calls that fail half-way
def _fails(*a, **k):
    raise RuntimeError("no")


def _device_matches(cache):
    return cache.lengths.tolist() == cache.held.tolist() and cache.free_count.tolist() == [cache.pages_left]


def test_a_step_that_fails_half_way_is_not_gone_on_from(ctx, monkeypatch):
    """Some layers' states have the token and others do not: the rows are refused until they are released, others may come in, and nothing
    of the failed step is left."""
    cfg, w, dec = _decoder()
    cache, other = (paged.PagedCache(cfg, rows=3, num_pages=16, page_size=16, max_length=64, dev=DEV) for _ in range(2))
    ids = torch.randint(0, 500, (60,), generator=torch.Generator().manual_seed(3)).to(DEV)
    tokens = ids[:3]
    dec.prefill(ids[:47], [15, 32], cache)
    for broken in (1, 3):  # a linear-attention layer, the full-attention layer
        live = cache.active
        with monkeypatch.context() as m:
            m.setattr(dec.layers[broken].mlp, "forward", _fails)
            with pytest.raises(RuntimeError, match="no"):
                dec.step(tokens, cache)
        ctx.sync()
        assert _device_matches(cache) and not cache.fits()
        with pytest.raises(ValueError, match="release"):
            dec.step(tokens, cache)
        with pytest.raises(ValueError, match="release"):
            cache.advanced(1)
        assert _device_matches(cache)
        _, rows = dec.prefill(ids[47:], [13], cache)  # an idle row is none of its business
        with pytest.raises(ValueError, match="release"):
            dec.step(tokens, cache)
        cache.release(live[:1])
        if len(live) > 1:
            with pytest.raises(ValueError, match="release"):
                dec.step(tokens, cache)
            cache.release(live[1:])
        _, same = dec.prefill(ids[47:], [13], other)
        got, want = dec.step(tokens, cache), dec.step(tokens[rows].repeat(3), other)
        ctx.sync()
        assert torch.equal(got[rows[0]], want[same[0]]) and _device_matches(cache)
        other.release(same)
    cache.release(cache.active)
    ctx.sync()
    assert sorted(cache.free_pages.tolist()) == list(range(16)) and cache.free_count.tolist() == [16]


def test_a_capture_that_fails_has_moved_nothing(ctx, monkeypatch):
    cfg, w, dec = _decoder(layers=2)
    cache = paged.PagedCache(cfg, rows=2, num_pages=8, page_size=16, max_length=64, dev=DEV)
    ids = torch.zeros(20, dtype=torch.int64, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        dec.prefill(ids, [20], cache)
        dec.step(ids[:2], cache)
        stream.synchronize()
        with monkeypatch.context() as m:
            m.setattr(dec.layers[1].mlp, "forward", _fails)
            with pytest.raises(RuntimeError, match="no"):
                with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                    dec.step(ids[:2], cache)
        assert cache.fits()
        dec.step(ids[:2], cache)
        stream.synchronize()
        device.load(0).sync()
    assert cache.held.tolist() == [22, -1] and _device_matches(cache)


@pytest.mark.parametrize("call", ["prefill", "step", "release"])
def test_bookkeeping_that_fails_changes_nothing(ctx, monkeypatch, call):
    """The call itself is refused (no memory for its outputs, say): host and device stay as they were, and together."""
    cfg, w, dec = _decoder(layers=1)
    cache = paged.PagedCache(cfg, rows=3, num_pages=8, page_size=16, max_length=64, dev=DEV)
    ids = torch.zeros(20, dtype=torch.int64, device=DEV)
    dec.prefill(ids[:16], [16], cache)
    before = [t.clone() for t in (cache.lengths, cache.state_index, cache.free_count, cache.free_pages, cache.tables)]
    with monkeypatch.context() as m:
        m.setattr(paged, "block_tables", _fails)
        m.setattr(paged, "release_blocks", _fails)
        with pytest.raises(RuntimeError, match="no"):
            dict(prefill=lambda: dec.prefill(ids, [20], cache), step=lambda: dec.step(ids[:3], cache), release=lambda: cache.release([0]))[call]()
    ctx.sync()
    assert cache.held.tolist() == [16, -1, -1] and cache.pages_left == 7
    for t, old in zip((cache.lengths, cache.state_index, cache.free_count, cache.free_pages, cache.tables), before):
        assert torch.equal(t, old)
    dec.step(ids[:3], cache)
    ctx.sync()
    assert cache.held.tolist() == [17, -1, -1] and _device_matches(cache)


def test_replayed_steps_end_where_the_positions_do(ctx):
    """A cache that could hold longer rows than the decoder has positions: what counts the replays of a captured step stops there."""
    cfg, w, dec = _decoder(layers=1)
    dec = qwen35.Decoder(dec.w, cfg, max_positions=24)
    cache = paged.PagedCache(cfg, rows=2, num_pages=8, page_size=16, max_length=64, dev=DEV)
    ids = torch.zeros(20, dtype=torch.int64, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        dec.prefill(ids, [20], cache)
        dec.step(ids[:2], cache)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            dec.step(ids[:2], cache)
        assert cache.fits(3) and not cache.fits(4)
        with pytest.raises(ValueError, match="24"):
            cache.advanced(4)
        cache.advanced(3)
        for _ in range(3):
            graph.replay()
        stream.synchronize()
        device.load(0).sync()
        with pytest.raises(ValueError, match="24"):
            cache.advanced(1)
        with pytest.raises(ValueError, match="24 positions"):
            dec.step(ids[:2], cache)
    assert cache.held.tolist() == [24, -1] and cache.lengths.tolist() == [24, -1]


# ------------------------------------------------------------------------------------------------ operands that the call before has written
def test_weights_that_the_call_before_writes(ctx):
    """A norm weight that lies in a page and is written there by the cache write just before: the kernels overlap, and the second one's
    loads wait all the same."""
    g = gen(6)
    T, dim = 4096, 256
    kc, vc = (torch.zeros(T // 16 + 1, 16, 1, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cos, sin = torch.ones(1, 8, device=DEV), torch.zeros(1, 8, device=DEV)
    last, slots, zeros = ints([T]), torch.arange(T, device=DEV, dtype=torch.int32), torch.zeros(T, dtype=torch.int32, device=DEV)
    k = bf(g, T, 1, dim)
    weights = [bf(g, 1, 1, dim) for _ in range(6)]
    got = []
    for w in weights:
        paged.cache_write(w, w, kc, vc, last)
        paged.cache_write(k, k, kc, vc, slots, norm_weight=kc[-1, 0, 0], cos=cos, sin=sin, positions=zeros, rotary_dim=16)
        got.append(kc[:-1].clone())
    for w, x in zip(weights, got):
        want = k[:, 0].clone()
        norm.head_norm_rope_(want, 1, dim, dim, w[0, 0], 1e-6, cos, sin, zeros, 16)
        assert torch.equal(x.view(T, dim), want)
    ctx.sync()


def test_step_weights_that_the_call_before_writes(ctx):
    """The same for the delta rule's step: its norm weight and its conv taps come out of a page that is written just before."""
    c = _step_case(40, 1, 1, 12)
    kc, vc = (torch.zeros(8, 1, 1, 256, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for seed in range(6):
        g = gen(seed)
        taps, w = bf(g, 384, 4, s=0.3), 1 + bf(g, 128, s=0.1)
        rows = torch.cat([taps.flatten(), w, w]).view(7, 1, 256)  # six rows of taps, one of two norm weights
        c = dict(c, conv_weight=taps, norm_weight=w)
        d = dict(c, state=c["state"].clone(), conv_state=c["conv_state"].clone(), conv_weight=kc[:6].view(384, 4), norm_weight=kc[6].view(256)[:128])
        want = qwen35.gated_delta_rule_step(**c)
        ctx.sync()
        paged.cache_write(rows, rows, kc, vc, ints(range(7)))
        got = qwen35.gated_delta_rule_step(**d)
        assert torch.equal(got, want) and torch.equal(c["state"], d["state"])
    ctx.sync()


@pytest.mark.parametrize("name,change", [("cu_seqlens", lambda t: t[:-1]), ("cu_seqlens", lambda t: t.long()), ("cu_seqlens", lambda t: t.cpu()),
                                         ("state_index", lambda t: t[:1]), ("state_index", lambda t: t.long()), ("state_index", lambda t: t.repeat(2)[::2]),
                                         ("positions", lambda t: t[:-1]), ("positions", lambda t: t.long()), ("state", lambda t: t.to(torch.bfloat16)),
                                         ("state", lambda t: t.transpose(2, 3)), ("conv", lambda t: t.float()), ("conv", lambda t: t[::2]), ("conv", lambda t: t.cpu())])
def test_prefill_refuses_what_its_kernels_would_misread(ctx, name, change):
    """Arrays too short for the batch, of other types, elsewhere, or with gaps: before any kernel sees them."""
    m, lens = _linear_attention(7), [70, 5]
    x, cu = bf(gen(3), 75, 256), np.cumsum([0] + lens).astype(np.int32)
    pos = ints(np.concatenate([np.arange(n) for n in lens]))
    parts = dict(conv=torch.zeros(4, 4, 1024, dtype=torch.bfloat16, device=DEV), state=torch.zeros(4, 4, 128, 128, device=DEV), positions=pos,
                 state_index=ints([2, 0]), cu_seqlens=ints(cu))
    kept = lambda p: qwen35.Kept(paged.DeltaState(p["conv"], p["state"]), p["positions"], pos, p["state_index"], cu_seqlens=p["cu_seqlens"])  # noqa: E731
    with pytest.raises(ValueError, match="state|conv|positions|cu_seqlens"):
        m.mix(x, cu, pos, kept({**parts, name: change(parts[name])}))
    assert torch.equal(m.mix(x, cu, pos, kept(parts)), m.mix(x, cu, pos))
    ctx.sync()
    assert bool((parts["state"][[0, 2]] != 0).any(-1).any(-1).all()) and not parts["state"][[1, 3]].any()


def test_prefill_of_a_batch_without_sequences(ctx):
    """Only tokens behind the last sequence: no sequence leaves a state, and that is no error."""
    m, x = _linear_attention(7), bf(gen(3), 8, 256)
    conv, state, pos = torch.ones(2, 4, 1024, dtype=torch.bfloat16, device=DEV), torch.ones(2, 4, 128, 128, device=DEV), ints([0] * 8)
    m.mix(x, np.zeros(1, np.int32), pos, qwen35.Kept(paged.DeltaState(conv, state), pos, pos, ints([0]), cu_seqlens=ints([0])))
    ctx.sync()
    assert bool((conv == 1).all()) and bool((state == 1).all())


def test_the_cache_takes_every_size_that_its_kernels_do(ctx):
    """16 query heads to a KV head are one span: 8192 rows of up to 2^21 tokens are within the attention's limit, and so within the cache's."""
    cfg = oracle.DecoderConfig(vocab_size=16, hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=64, num_key_value_heads=4,
                               head_dim=256, full_attention_interval=1)
    cache = paged.PagedCache(cfg, rows=8192, num_pages=1, page_size=65536, max_length=1 << 21, dev=DEV)
    cache.lengths[:2] = ints([1, 3])
    k, v = cache.layers[0]
    k[0, :3], v[0, :3] = 0, bf(gen(1), 3, 4, 256)
    got = paged.attention_paged(torch.zeros(8192, 64, 256, dtype=torch.bfloat16, device=DEV), k, v, cache.tables, cache.lengths, workspace=cache.workspace)
    ctx.sync()
    want = torch.stack([v[0, 0].float(), v[0, :3].float().mean(0)])[:, :, None].expand(2, 4, 16, 256).reshape(2, 64 * 256)
    assert bool(((got[:2].float() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14).all()) and not got[2:].any()
    with pytest.raises(ValueError, match="below 2.31"):
        paged.PagedCache(cfg, rows=8192, num_pages=1, page_size=65536, max_length=1 << 22, dev=DEV)
