"""Decoding from a cache on the GPU: block tables, cache write, paged attention, the delta rule's step and the state that a
prompt leaves, each against 64-bit arithmetic or an integer model, then the decoder that uses them together.

Tolerances count roundings. A value rounded to bf16 is off by at most 2^-8 of itself. Paged attention rounds every softmax weight
to bf16 once (2^-8 of the weight, so 2^-8 of the output's sum taken with |v|) and its output once; its f32 sums and exponentials
stay below 2^-15 of the same sums. The step kernel is f32 throughout (`paged_model.delta_step_64` carries the bound)."""
import dataclasses

import numpy as np
import pytest
import torch

import oracle
from conftest import max_rel
from paged_model import attention_64, block_tables_model, delta_step_64, pages, release_model
from sys1_b200 import _lib, device, norm, paged, qwen35

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def bf(g, *shape, s=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * s).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ block tables
def _tables_case(rows, page, longest, added, idle, seed, spare=5):
    h = np.random.RandomState(seed)
    cached = h.randint(0, longest + 1, rows)
    cached[h.permutation(rows)[:idle]] = -1
    add = None if added is None else h.randint(0, added + 1, rows)
    new = np.ones(rows, int) if add is None else add
    held = [pages(max(c, 0), page) for c in cached]
    width = max(pages(max(c, 0) + n, page) for c, n in zip(cached, new)) + 1
    total = sum(pages(max(c, 0) + n, page) for c, n in zip(cached, new)) + spare
    pool = h.permutation(total)
    tables, at = np.full((rows, width), -1, np.int32), 0
    for b, n in enumerate(held):
        tables[b, :n] = pool[at:at + n]
        at += n
    free = np.full(total, -1, np.int32)
    free[:total - at] = pool[at:]
    tokens = rows if add is None else int(np.where(cached < 0, 0, add).sum())
    return cached, add, tables, free, total - at, tokens


def _check_tables(r, tables, want):
    assert tables.cpu().numpy().tolist() == want["tables"].tolist()
    assert r.lengths.tolist() == want["lengths"] and r.cu_seqlens.tolist() == want["cu_seqlens"]
    assert r.positions.tolist() == want["positions"] and r.slots.tolist() == want["slots"]
    assert r.free_count.tolist() == [want["left"]]


@pytest.mark.parametrize("rows,page,longest,added,idle,pad", [
    (1, 1, 0, None, 0, 0), (1, 16, 16, None, 0, 0), (7, 16, 64, None, 2, 0), (1025, 64, 300, None, 40, 0), (8192, 16, 40, None, 100, 0),
    (1, 64, 0, 1, 0, 3), (1, 16, 40, 5000, 0, 0), (31, 64, 700, 1000, 3, 57), (5, 65536, 70000, 9000, 1, 0), (2048, 16, 100, 30, 200, 8), (3, 4, 9, 0, 1, 4),
    (17, 2, 5, 7, 17, 2)])
def test_block_tables(ctx, rows, page, longest, added, idle, pad):
    cached, add, tables, free, count, tokens = _tables_case(rows, page, longest, added, idle, rows + page)
    want = block_tables_model(cached, add, page, free, count, tables, tokens + pad)
    assert not want["refused"]
    dt, dc = ints(tables), ints(cached)
    args = (dc, dt, ints(free), ints([count]), page)
    kw = dict(added=None if add is None else ints(add), max_tokens=tokens + pad)
    r = paged.block_tables(*args, **kw)
    ctx.sync()
    _check_tables(r, dt, want)
    assert dc.tolist() == list(cached)
    # in place: the same results where lengths and count are the inputs themselves
    dt2, dc2, left = ints(tables), ints(cached), ints([count])
    r = paged.block_tables(dc2, dt2, args[2], left, page, lengths=dc2, free_count_out=left, **kw)
    ctx.sync()
    assert r.lengths.data_ptr() == dc2.data_ptr()
    _check_tables(r, dt2, want)


def _refused(ctx, match):
    with pytest.raises(_lib.S1Error, match=match) as e:
        ctx.sync()
    assert e.value.code == _lib.S1_EKERNEL
    ctx.sync()  # said once


@pytest.mark.parametrize("what", ["pages", "width", "tokens", "page id"])
def test_block_tables_that_do_not_fit(ctx, what):
    cached, add, tables, free, count, tokens = _tables_case(9, 16, 60, 50, 1, 3)
    page = 16
    if what == "pages":
        count = max(1, sum(pages(max(c, 0) + (n if c >= 0 else 0), page) - pages(max(c, 0), page) for c, n in zip(cached, add)) // 2)
    elif what == "width":
        tables = np.ascontiguousarray(tables[:, :-2])
    elif what == "tokens":
        tokens -= 20
    want = block_tables_model(cached, add, page, free, count, tables, tokens)
    if what == "page id":
        free = np.full_like(free, -5)
    else:
        assert want["refused"]
    dt = ints(tables)
    r = paged.block_tables(ints(cached), dt, ints(free), ints([count]), page, added=ints(add), max_tokens=tokens)
    _refused(ctx, dict(pages="no free pages", width="more pages than", tokens="beyond max_tokens")[what] if what != "page id" else "was given page -5")
    if what == "page id":
        assert min(r.slots.tolist()) == -1
    else:
        _check_tables(r, dt, want)


def test_block_tables_up_to_the_last_length(ctx):
    """Lengths end at 2^31 - 1, also where a row's block table could hold more."""
    page, width = 65536, 32770
    tables = np.tile(np.arange(width, dtype=np.int32) % 32768, (3, 1))
    cached, add, free = [2 ** 31 - 1, 2 ** 31 - 3, 5], [3, 2, 1], [4, 9]
    want = block_tables_model(cached, add, page, free, 2, tables, 6)
    assert want["refused"] == [0] and want["lengths"][:2] == [2 ** 31 - 1] * 2
    dt = ints(tables)
    r = paged.block_tables(ints(cached), dt, ints(free), ints([2]), page, added=ints(add), max_tokens=6)
    _refused(ctx, "more pages than")
    _check_tables(r, dt, want)


@pytest.mark.parametrize("rows,page,width", [(1, 1, 3), (9, 16, 5), (1500, 16, 4), (8192, 64, 2)])
def test_release(ctx, rows, page, width):
    h = np.random.RandomState(rows)
    lengths = h.randint(-1, width * page + 1, rows)
    ended = h.randint(0, 2, rows)
    tables = np.arange(rows * width, dtype=np.int32).reshape(rows, width)
    free, count = [-7] * (rows * width + 4), 3
    for bad in (False, True):
        if bad:  # two rows that cannot be taken back: one longer than its table, and no room for the last ones
            ended[0], lengths[0] = 1, width * page + 1
            free = free[:count + max(0, sum(pages(max(n, 0), page) for n, e in zip(lengths[1:], ended[1:]) if e) - 1)]
        want = release_model(ended, lengths, tables, free, count, page)
        dl, df, dc = ints(lengths), ints(free), ints([count])
        paged.release_blocks(ints(ended), dl, ints(tables), df, dc, page)
        assert bool(want[3]) == bad
        if bad:
            _refused(ctx, "s1_release_blocks")
        else:
            ctx.sync()
        n = want[1]
        assert dc.tolist() == [n] and df.tolist()[:n] == want[0][:n] and dl.tolist() == want[2]


# ------------------------------------------------------------------------------------------------ cache write
def _rotation(g, positions, rot):
    angle = torch.rand(positions, rot // 2, device=DEV, generator=g) * 6.28
    return angle.cos().contiguous(), angle.sin().contiguous()


@pytest.mark.parametrize("T,kv,dim,rot,page,layout", [(1, 1, 64, 16, 1, "token"), (5, 2, 256, 64, 16, "token"), (33, 3, 128, 128, 64, "head"),
                                                      (1000, 4, 256, 256, 32, "head"), (513, 8, 64, 32, 128, "token")])
@pytest.mark.parametrize("normed", [False, True])
def test_cache_write(ctx, T, kv, dim, rot, page, layout, normed):
    g = gen(T + dim)
    n = pages(T + 3, page) + 1
    qkv = bf(g, T, 2 * kv * dim + 16)
    k, v = qkv[:, 8:8 + kv * dim].unflatten(1, (kv, dim)), qkv[:, 8 + kv * dim:8 + 2 * kv * dim].unflatten(1, (kv, dim))
    if layout == "token":
        kc, vc = bf(g, n, page, kv, dim), bf(g, n, page, kv, dim)
    else:  # [pages, kv, page_size, dim] in memory, a gap after every page
        kc, vc = (bf(g, n, kv * page + 1, dim)[:, :kv * page].unflatten(1, (kv, page)).transpose(1, 2) for _ in range(2))
    slots = torch.randperm(n * page, device=DEV, generator=g)[:T].to(torch.int32)
    if T > 1:
        slots[T // 2] = -1
    w, (cos, sin) = bf(g, dim, s=0.1), _rotation(g, 50, rot)
    pos = torch.randint(0, 50, (T,), device=DEV, generator=g, dtype=torch.int32)
    keep = slots >= 0
    at = slots[keep].long()
    for bf16_ops in (False, True):
        want_k, want_v, kk = kc.clone(), vc.clone(), k.clone()
        if normed:
            flat = kk.flatten(1)
            norm.head_norm_rope_(flat, kv, dim, dim, w, 1e-6, cos, sin, pos, rot, bf16_ops=bf16_ops)
        want_k[at // page, at % page], want_v[at // page, at % page] = kk[keep], v[keep]
        before = qkv.clone()
        if normed:
            paged.cache_write(k, v, kc, vc, slots, norm_weight=w, eps=1e-6, cos=cos, sin=sin, positions=pos, rotary_dim=rot, bf16_ops=bf16_ops)
        else:
            paged.cache_write(k, v, kc, vc, slots)
        ctx.sync()
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v) and torch.equal(qkv, before)
        if normed and not bf16_ops:  # and against 64 bits: the norm's rounding, the rotation's two products of it, the last rounding
            x = k[keep].double()
            y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
            c, s = (t[pos[keep].long()][:, None].double() for t in (cos, sin))
            lo, hi = y[..., :rot // 2], y[..., rot // 2:rot]
            ref = torch.cat([lo * c - hi * s, hi * c + lo * s, y[..., rot:]], -1)
            size = torch.cat([lo.abs() * c.abs() + hi.abs() * s.abs(), hi.abs() * c.abs() + lo.abs() * s.abs(), torch.zeros_like(y[..., rot:])], -1)
            err = (kc[at // page, at % page].double() - ref).abs()
            assert bool((err <= (2.0 ** -8 + 2.0 ** -14) * (size + ref.abs())).all())


def test_cache_write_of_a_batch_beyond_32_bits(ctx):
    """2^26 + 8 tokens, whose last rows lie 2^34 elements behind the first."""
    T, dim, g = 2 ** 26 + 8, 256, gen(19)
    x = torch.empty(T, 1, dim, dtype=torch.bfloat16, device=DEV)  # 34 GB, keys and values in one; only the last rows are copied
    x[-3:] = bf(g, 3, 1, dim)
    slots, positions = torch.full((T,), -1, dtype=torch.int32, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    slots[-3:] = ints([2, 0, 1])
    kc, vc = torch.zeros(2, 1, 4, 1, dim, dtype=torch.bfloat16, device=DEV)
    cos, sin = torch.ones(1, 8, device=DEV), torch.zeros(1, 8, device=DEV)
    paged.cache_write(x, x, kc, vc, slots, norm_weight=bf(g, dim), cos=cos, sin=sin, positions=positions, rotary_dim=16)
    ctx.sync()
    assert torch.equal(vc[0, [2, 0, 1]], x[-3:]) and int((kc[0, :3] != 0).any(-1).sum()) == 3 and not kc[0, 3].any() and not vc[0, 3].any()
    del x
    torch.cuda.empty_cache()


def test_cache_write_reports_slots_and_positions_outside(ctx):
    g = gen(1)
    k, v, kc = bf(g, 3, 1, 64), bf(g, 3, 1, 64), bf(g, 2, 16, 1, 64)
    vc = kc.clone()
    before = kc.clone()
    paged.cache_write(k, v, kc, vc, ints([4, 32, 5]))
    _refused(ctx, "token 1 has slot 32")
    assert torch.equal(kc[0, 4:6, 0], k[[0, 2], 0]) and torch.equal(kc[0, :4], before[0, :4]) and torch.equal(kc[1], before[1])
    cos, sin = _rotation(g, 4, 16)
    paged.cache_write(k, v, kc, vc, ints([0, 1, 2]), norm_weight=bf(g, 64), cos=cos, sin=sin, positions=ints([0, 4, 1]), rotary_dim=16)
    _refused(ctx, "row 1 has index 4")
    with pytest.raises(_lib.S1Error, match="rotary_dim"):
        paged.cache_write(k, v, kc, vc, ints([0, 1, 2]), norm_weight=bf(g, 64), cos=torch.ones(4, 12, device=DEV), sin=torch.ones(4, 12, device=DEV),
                          positions=ints([0, 0, 0]), rotary_dim=24)
    with pytest.raises(ValueError, match="shape"):
        paged.cache_write(k, v[:2], kc, vc, ints([0, 1, 2]))
    with pytest.raises(ValueError, match="same shape"):
        paged.cache_write(k, v, kc, vc[:, :8], ints([0, 1, 2]))


# ------------------------------------------------------------------------------------------------ paged attention
def _attention_case(lens, H, kv, dim, page, seed, layout="token", gated=True, poison=True, scale=1.0):
    g, h = gen(seed), np.random.RandomState(seed)
    held = [pages(max(n, 0), page) for n in lens]
    n, width = sum(held) + 2, max(held + [1]) + 1
    pool = h.permutation(n)
    tables, at = np.full((len(lens), width), 1 << 20, np.int32), 0  # entries behind a row's pages are not to be followed
    for b, m in enumerate(held):
        tables[b, :m] = pool[at:at + m]
        at += m
    shape = (n, page, kv, dim) if layout == "token" else (n, kv, page, dim)
    kc, vc = bf(g, *shape), bf(g, *shape)
    if layout != "token":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    if poison:  # what no row holds is not a number, or the largest there is
        dead = torch.ones(n * page, dtype=torch.bool, device=DEV)
        for b, m in enumerate(lens):
            for i in range(held[b]):
                dead[int(tables[b, i]) * page:int(tables[b, i]) * page + min(page, m - i * page)] = False
        dead = dead.view(n, page)
        kc[dead] = float("nan")
        vc[dead] = float("nan")
        one = torch.nonzero(dead)[:1]
        kc[one[:, 0], one[:, 1]], vc[one[:, 0], one[:, 1]] = float("inf"), float("-inf")
    qg = bf(g, len(lens), H, 2, dim, s=scale)
    return qg[:, :, 0], kc, vc, ints(tables), ints(lens), qg[:, :, 1] if gated else None


def _check_attention(got, q, kc, vc, tables, lens, gate, scale=None):
    dim = q.shape[2]
    ref, size = attention_64(q, kc, vc, tables, lens, gate, dim ** -0.5 if scale is None else scale)
    err = (got.double().unflatten(1, (-1, dim)) - ref).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -15) * size).all()), float((err / (ref.abs() + size + 1e-30)).max())


@pytest.mark.parametrize("lens,H,kv,dim,page,layout", [
    ([1], 1, 1, 64, 16, "token"), ([17], 8, 2, 256, 16, "token"), ([0, -1, 5, 16, 15], 4, 4, 128, 16, "head"),
    ([128, 129, 127, 1, 300], 6, 2, 256, 64, "token"), ([1000, 3, 0, 64, 65, 2049], 24, 4, 256, 16, "head"),
    ([255, 256, 257], 16, 1, 64, 1, "token"), ([77, 200], 9, 1, 256, 2, "token"), ([513, 40], 16, 2, 128, 8, "head"), ([3000], 34, 2, 64, 128, "token"),
    ([3000, 200], 32, 2, 256, 16, "token"), ([5000, 0, 130], 12, 1, 128, 64, "head"), ([20000, 5], 3, 1, 256, 65536, "token"), ([30000], 8, 2, 256, 64, "head")])
@pytest.mark.parametrize("gated", [False, True])
def test_paged_attention(ctx, lens, H, kv, dim, page, layout, gated):
    q, kc, vc, tables, lengths, gate = _attention_case(lens, H, kv, dim, page, sum(map(abs, lens)) + H, layout, gated)
    got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    ctx.sync()
    _check_attention(got, q, kc, vc, tables, lens, gate)
    assert torch.equal(got, paged.attention_paged(q, kc, vc, tables, lengths, gate=gate))  # the order of every sum is fixed
    # a strided output and a scale of one's own
    out = torch.full((len(lens), H * dim + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    paged.attention_paged(q, kc, vc, tables, lengths, gate=gate, scale=0.31, out=out[:, :H * dim])
    ctx.sync()
    _check_attention(out[:, :H * dim], q, kc, vc, tables, lens, gate, 0.31)
    assert bool((out[:, H * dim:] == 7).all())


@pytest.mark.parametrize("rows,H,kv,dim,longest", [(700, 4, 2, 64, 900), (250, 8, 2, 256, 900), (300, 24, 2, 128, 500), (230, 32, 2, 256, 300),
                                                   (90, 12, 6, 128, 5000), (120, 6, 1, 256, 3000)])
def test_paged_attention_many_ragged_rows(ctx, rows, H, kv, dim, longest):
    """More rows than threads in a block, and more units than CTAs: ranges that begin and end anywhere."""
    h = np.random.RandomState(5)
    lens = [int(n) for n in np.where(h.rand(rows) < 0.1, 0, np.exp(h.uniform(0, np.log(longest), rows)))]
    q, kc, vc, tables, lengths, gate = _attention_case(lens, H, kv, dim, 16, 5)
    got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    ctx.sync()
    _check_attention(got, q, kc, vc, tables, lens, gate)


@pytest.mark.parametrize("rows,H,kv,dim,longest", [(200, 6, 3, 64, 200000), (230, 6, 2, 128, 150000), (100, 32, 2, 64, 100000), (3, 16, 1, 128, 90000), (250, 2, 2, 256, 60000)])
def test_paged_attention_of_one_long_context_among_many(ctx, rows, H, kv, dim, longest):
    """More pieces of one span than the join's threads, or than its warps, among spans that are never cut; few spans of many heads."""
    lens = [int(n) for n in np.random.RandomState(9).randint(0, 60, rows)]
    lens[rows // 2] = longest
    q, kc, vc, tables, lengths, gate = _attention_case(lens, H, kv, dim, 64, 9)
    got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    ctx.sync()
    _check_attention(got, q, kc, vc, tables, lens, gate)
    assert torch.equal(got, paged.attention_paged(q, kc, vc, tables, lengths, gate=gate))


@pytest.mark.parametrize("rows,kv,page,longest", [(3, 2, 16, 112), (3, 2, 16, 128), (70, 3, 16, 112), (1, 1, 64, 64), (250, 2, 16, 48), (250, 2, 16, 64), (600, 1, 2, 62)])
@pytest.mark.parametrize("dim", [64, 256])
def test_paged_attention_of_tables_about_a_unit_wide(ctx, rows, kv, page, longest, dim):
    """Block tables of just a unit (128 keys, 64 with many rows), whose spans are never cut, and of a page more."""
    lens = [int(n) for n in np.random.RandomState(rows).randint(0, longest + 1, rows)]
    lens[0] = longest
    q, kc, vc, tables, lengths, gate = _attention_case(lens, 4 * kv, kv, dim, page, rows)
    got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    ctx.sync()
    _check_attention(got, q, kc, vc, tables, lens, gate)
    assert torch.equal(got, paged.attention_paged(q, kc, vc, torch.nn.functional.pad(tables, (0, 100)), lengths, gate=gate))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_paged_attention_of_sharp_and_flat_scores(ctx, dim):
    lens = [700, 33]
    q, kc, vc, tables, lengths, _ = _attention_case(lens, 4, 2, dim, 16, 3, gated=False, scale=30.0)  # one key takes nearly all
    got = paged.attention_paged(q, kc, vc, tables, lengths)
    # scores of up to ~30 * 5 * sqrt(dim) / sqrt(dim): f32 sums of dim products put 2^-24 * dim * |score| <= 2^-9 into the exponent
    ref, size = attention_64(q, kc, vc, tables, lens, None, dim ** -0.5)
    err = (got.double().unflatten(1, (-1, dim)) - ref).abs()
    assert bool((err <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -8) * size).all())
    q.zero_()
    got = paged.attention_paged(q, kc, vc, tables, lengths)
    ctx.sync()
    _check_attention(got, q, kc, vc, tables, lens, None)


def test_paged_attention_of_a_cache_beyond_32_bits(ctx):
    """Element offsets past 2^31 in the cache (a little over 4 GB each for keys and values)."""
    page, kv, dim = 64, 2, 256
    n = (1 << 31) // (page * kv * dim) + 40
    kc, vc = (torch.empty(n, page, kv, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lens = [500, 64]
    tables = ints([[n - 1 - 2 * i for i in range(8)], [3] + [0] * 7])
    g = gen(2)
    used = torch.unique(tables.long())
    kc[used], vc[used] = bf(g, len(used), page, kv, dim), bf(g, len(used), page, kv, dim)
    k, v = bf(g, 2, kv, dim), bf(g, 2, kv, dim)
    slots = ints([(n - 1 - 2 * (499 // page)) * page + 499 % page, 3 * page + 63])
    paged.cache_write(k, v, kc, vc, slots)
    q = bf(g, 2, 8, dim)
    got = paged.attention_paged(q, kc, vc, tables, ints(lens))
    ctx.sync()
    assert torch.equal(kc[tables[0, 7].item(), 499 % page], k[0]) and torch.equal(vc[3, 63], v[1])
    _check_attention(got, q, kc, vc, tables, lens, None)


def test_paged_attention_reports_bad_pages_and_lengths(ctx):
    lens = [100, 40, 64]
    q, kc, vc, tables, lengths, gate = _attention_case(lens, 4, 2, 128, 16, 9, poison=False)
    good = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
    for page in (-1, kc.shape[0], 2 ** 31 - 1):
        bad = tables.clone()
        bad[0, 3] = page
        got = paged.attention_paged(q, kc, vc, bad, lengths, gate=gate)
        _refused(ctx, f"row 0 names page {page}")
        assert torch.equal(got[1:], good[1:]) and bool(torch.isfinite(got).all())
        # the row's other 84 keys
        keep = [j for j in range(100) if j // 16 != 3]
        at = tables[0, [j // 16 for j in keep]].long()
        rest_k, rest_v = (c[at, [j % 16 for j in keep]].reshape(1, 84, 2, 128) for c in (kc, vc))
        _check_attention(got[:1], q[:1], rest_k, rest_v, ints([[0]]), [84], gate[:1])
    too_long = lengths.clone()
    too_long[1] = 16 * tables.shape[1] + 1
    got = paged.attention_paged(q, kc, vc, tables, too_long, gate=gate)
    _refused(ctx, "row 1 has")
    assert bool((got[1] == 0).all())


def test_paged_attention_refusals(ctx):
    q, kc, vc, tables, lengths, gate = _attention_case([20, 30], 4, 2, 64, 16, 1)
    with pytest.raises(_lib.S1Error, match="scale"):
        paged.attention_paged(q, kc, vc, tables, lengths, scale=0.0)
    with pytest.raises(_lib.S1Error, match="workspace of"):
        paged.attention_paged(q, kc, vc, tables, lengths, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    with pytest.raises(_lib.S1Error, match="multiple of kv_heads"):
        paged.attention_paged(q[:, :3], kc, vc, tables, lengths)
    with pytest.raises(ValueError, match="shape"):
        paged.attention_paged(q, kc, vc, tables, lengths[:1])
    with pytest.raises(ValueError, match="block tables"):
        paged.attention_paged(q, kc, vc, tables[:1], lengths)
    with pytest.raises(_lib.S1Error, match="head_dim"):
        paged.attention_paged(bf(gen(1), 2, 4, 96), bf(gen(1), 3, 16, 2, 96), bf(gen(1), 3, 16, 2, 96), tables, lengths)
    with pytest.raises(_lib.S1Error, match="power of two"):
        paged.attention_paged(q, bf(gen(1), 3, 24, 2, 64), bf(gen(1), 3, 24, 2, 64), tables, lengths)
    assert paged.attention_paged(q[:0], kc, vc, tables[:0], lengths[:0]).shape == (0, 256)


def test_paged_attention_captured_follows_its_lengths(ctx):
    """A captured call works from the lengths and tables that are there when it is replayed."""
    lens = [700, 30, 0, 129]
    q, kc, vc, tables, lengths, gate = _attention_case([900] * 4, 8, 2, 128, 16, 21, poison=False)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = device.load(0)
        paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate)
        for n in (lens, [1] * 4, [900] * 4, [0] * 4, [5, 800, 16, 17]):
            lengths.copy_(ints(n))
            graph.replay()
            got = out.clone()
            assert torch.equal(got, paged.attention_paged(q, kc, vc, tables, ints(n), gate=gate))
            _check_attention(got, q, kc, vc, tables, n, gate)
        other.sync()


def test_without_programmatic_serialization(ctx):
    """The context's "pdl" option off: plain launches, the same results."""
    q, kc, vc, tables, lengths, gate = _attention_case([700, 30, 0, 2000], 8, 2, 256, 16, 41)
    c = _step_case(5, 2, 4, 42)
    d = dict(c, state=c["state"].clone(), conv_state=c["conv_state"].clone())
    want = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate), qwen35.gated_delta_rule_step(**c)
    ctx.set_option("pdl", 0)
    try:
        got = paged.attention_paged(q, kc, vc, tables, lengths, gate=gate), qwen35.gated_delta_rule_step(**d)
    finally:
        ctx.set_option("pdl", 1)
    ctx.sync()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(c["state"], d["state"])


def test_two_streams_at_once(ctx):
    """Calls that run at the same time on two streams (each with its own context and workspace) give what they give alone."""
    cases = [_attention_case([3000, 1, 900], 8, 2, 128, 16, 31), _attention_case([10, 2500, 70], 8, 2, 128, 16, 32)]
    steps = [_step_case(9, 2, 4, 33), _step_case(9, 2, 4, 34)]
    alone = [paged.attention_paged(*c[:5], gate=c[5]) for c in cases]
    after = [dict(c, state=c["state"].clone(), conv_state=c["conv_state"].clone()) for c in steps]
    for _ in range(5):
        [qwen35.gated_delta_rule_step(**c) for c in after]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = paged.attention_paged(*cases[i][:5], gate=cases[i][5])
                qwen35.gated_delta_rule_step(**steps[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], alone[i]) and torch.equal(steps[i]["state"], after[i]["state"])


# ------------------------------------------------------------------------------------------------ delta rule
def _step_case(rows, keys, values, seed, states=None, fresh=(), idle=()):
    g, h = gen(seed), np.random.RandomState(seed)
    C = (2 * keys + values) * 128
    states = states or rows + 2
    index, pos = h.permutation(states)[:rows], h.randint(4, 5000, rows)
    for i, r in enumerate(fresh):
        pos[r] = i % 4
    index[list(idle)] = -1
    ba = bf(g, rows, 2 * values + 8)
    return dict(mixed=bf(g, rows, C + 8)[:, :C], conv_weight=bf(g, C, 4, s=0.3), positions=ints(pos), b=ba[:, :values], a=ba[:, values:2 * values],
                dt_bias=torch.randn(values, device=DEV, generator=g) * 0.5, neg_exp_a=-torch.exp(torch.randn(values, device=DEV, generator=g) * 0.5),
                z=bf(g, rows, values * 128), norm_weight=1 + bf(g, 128, s=0.1), eps=1e-6, conv_state=bf(g, states, 4, C),
                state=torch.randn(states, values, 128, 128, device=DEV, generator=g) * 0.1, key_heads=keys, state_index=ints(index))


def _step_reference(c):
    return delta_step_64(c["mixed"], c["conv_weight"], c["positions"].tolist(), c["b"], c["a"], c["dt_bias"], c["neg_exp_a"], c["z"], c["norm_weight"],
                         c["eps"], c["conv_state"], c["state"], c["key_heads"],
                         list(range(c["mixed"].shape[0])) if c["state_index"] is None else c["state_index"].tolist())


@pytest.mark.parametrize("rows,keys,values,fresh,idle", [(1, 1, 1, [0], []), (1, 16, 16, [], []), (6, 2, 6, [0, 1, 2, 3], [5]), (5, 4, 8, [2, 4], [0, 2]),
                                                         (40, 16, 48, [], [39])])
def test_delta_step(ctx, rows, keys, values, fresh, idle):
    c = _step_case(rows, keys, values, rows + values, fresh=fresh, idle=idle)
    if fresh:  # what a fresh sequence's state held before is of no account
        live = [int(c["state_index"][r]) for r in fresh if int(c["positions"][r]) == 0 and int(c["state_index"][r]) >= 0]
        c["state"][live], c["conv_state"][live] = float("nan"), float("nan")
    y64, yb, S64, Sb, ring = _step_reference(c)
    y = qwen35.gated_delta_rule_step(**c)
    ctx.sync()
    assert torch.equal(c["conv_state"].nan_to_num(9.0), ring.nan_to_num(9.0))
    touched = torch.tensor(sorted(int(i) for i in c["state_index"] if i >= 0), device=DEV)
    assert bool(((c["state"][touched].double() - S64[touched]).abs() <= Sb[touched]).all())
    others = torch.tensor([i for i in range(c["state"].shape[0]) if i not in touched.tolist()], device=DEV)
    assert torch.equal(c["state"][others].double(), S64[others])
    assert bool(((y.double() - y64).abs() <= yb).all())
    assert all(bool((y[r] == 0).all()) for r in idle)


def test_delta_step_without_an_index(ctx):
    c = _step_case(3, 2, 4, 8, states=3)
    c["state_index"] = None
    y64, yb, S64, Sb, _ = _step_reference(c)
    y = qwen35.gated_delta_rule_step(**c)
    ctx.sync()
    assert bool(((y.double() - y64).abs() <= yb).all()) and bool(((c["state"].double() - S64).abs() <= Sb).all())


@pytest.mark.parametrize("what", ["twice", "outside", "position"])
def test_delta_step_reports_bad_states(ctx, what):
    c = _step_case(4, 2, 2, 4)
    if what == "twice":
        c["state_index"][3] = c["state_index"][1]
    elif what == "outside":
        c["state_index"][3] = c["state"].shape[0]
    else:
        c["positions"][3] = -2
    good = dict(c, state=c["state"].clone(), conv_state=c["conv_state"].clone(), state_index=c["state_index"].clone(), positions=c["positions"].clone())
    good["state_index"][3] = -1
    y = qwen35.gated_delta_rule_step(**c)
    _refused(ctx, "position -2" if what == "position" else "row 3 has state")
    want = qwen35.gated_delta_rule_step(**good)
    ctx.sync()
    assert torch.equal(y, want) and torch.equal(c["state"], good["state"]) and torch.equal(c["conv_state"], good["conv_state"])


def test_delta_step_of_many_rows(ctx):
    """More rows than a block has threads (a state given twice is found there too), more pairs of rows and heads than blocks."""
    c = _step_case(700, 1, 1, 12, fresh=range(0, 700, 9), idle=range(3, 700, 11))
    y64, yb, S64, Sb, ring = _step_reference(c)
    y = qwen35.gated_delta_rule_step(**c)
    ctx.sync()
    assert torch.equal(c["conv_state"], ring) and bool(((y.double() - y64).abs() <= yb).all()) and bool(((c["state"].double() - S64).abs() <= Sb).all())
    c["state_index"][699] = c["state_index"][601] if int(c["state_index"][601]) >= 0 else c["state_index"][602]
    before = c["state"].clone()
    qwen35.gated_delta_rule_step(**c)
    _refused(ctx, "row 699 has state")
    assert not torch.equal(c["state"], before) and bool(torch.isfinite(c["state"]).all())


def test_delta_step_refusals(ctx):
    c = _step_case(3, 2, 4, 8)
    with pytest.raises(ValueError, match="columns"):
        qwen35.gated_delta_rule_step(**dict(c, key_heads=1))
    with pytest.raises(ValueError, match="row stride"):
        qwen35.gated_delta_rule_step(**dict(c, b=c["b"].contiguous()))
    with pytest.raises(ValueError, match="state must be"):
        qwen35.gated_delta_rule_step(**dict(c, state=c["state"].transpose(2, 3)))
    with pytest.raises(_lib.S1Error, match="states"):
        qwen35.gated_delta_rule_step(**dict(c, state_index=None, state=c["state"][:2].contiguous(), conv_state=c["conv_state"][:2].contiguous()))


def _linear_attention(seed, hidden=256, keys=2, values=4):
    cfg = oracle.DecoderConfig(vocab_size=16, hidden_size=hidden, intermediate_size=64, num_hidden_layers=1, linear_num_key_heads=keys, linear_num_value_heads=values)
    w = oracle.qwen35.init_weights(cfg, seed)
    p = "layers.0.linear_attn."
    b = {k[len(p):]: (t if k.endswith(("A_log", "dt_bias")) else t.to(torch.bfloat16)).to(DEV) for k, t in w.items() if k.startswith(p)}
    lin = lambda n: qwen35.Linear(b[n])  # noqa: E731
    return qwen35.LinearAttention(lin("in_proj_qkv"), lin("in_proj_z"), lin("in_proj_b"), lin("in_proj_a"), b["conv1d"], -torch.exp(b["A_log"]), b["dt_bias"],
                                  b["norm"], lin("out_proj"), keys, values, 1e-6)


@pytest.mark.parametrize("lens", [[1], [64, 3], [200, 65, 1, 2, 130]])
def test_prefill_leaves_the_state_of_the_recurrence(ctx, lens):
    """The chunked form on the tensor cores takes bf16 operands: its final state is held to 2e-2 of the state's scale, the bound of
    its outputs, against the step kernel (f32, held to 64 bits above) run token by token."""
    m = _linear_attention(7)
    x = bf(gen(3), sum(lens), 256)
    cu = np.cumsum([0] + lens).astype(np.int32)
    pos = ints(np.concatenate([np.arange(n) for n in lens]))
    n = len(lens)
    index = list(np.random.RandomState(1).permutation(n + 3)[:n])
    if n > 2:
        index[2] = -1
    conv, state = bf(gen(4), n + 3, 4, 1024), torch.randn(n + 3, 4, 128, 128, device=DEV, generator=gen(5))
    conv0, state0 = conv.clone(), state.clone()
    kept = qwen35.Kept(paged.DeltaState(conv, state), pos, pos, ints(index), cu_seqlens=ints(cu))
    y = m.mix(x, cu, pos, kept)
    assert torch.equal(y, m.mix(x, cu, pos))
    pre, zz, bb, aa = m._inputs(x)
    rc, rs = torch.zeros_like(conv), torch.zeros_like(state)
    steps = [qwen35.gated_delta_rule_step(pre[cu[s] + t:cu[s] + t + 1], m.conv_taps, pos[cu[s] + t:cu[s] + t + 1], bb[cu[s] + t:cu[s] + t + 1],
                                          aa[cu[s] + t:cu[s] + t + 1], m.dt_bias, m.decay, zz[cu[s] + t:cu[s] + t + 1], m.norm, m.eps, rc, rs, 2,
                                          state_index=ints([max(int(index[s]), 0)]))
             for s in range(n) if index[s] >= 0 for t in range(lens[s])]
    ctx.sync()
    outs = torch.cat([y[cu[s]:cu[s + 1]] for s in range(n) if index[s] >= 0])
    assert max_rel(outs, torch.cat(steps)) <= 2e-2
    for s in range(n):
        i = int(index[s])
        if i >= 0:
            assert max_rel(state[i], rs[i]) <= 2e-2
            for p in range(max(0, lens[s] - 4), lens[s]):
                assert torch.equal(conv[i, p % 4], pre[cu[s] + p])
    free = [i for i in range(n + 3) if i not in index]
    assert torch.equal(conv[free], conv0[free]) and torch.equal(state[free], state0[free])


def test_prefill_reports_a_state_given_twice(ctx):
    m, lens = _linear_attention(7), [70, 5, 0, 9]
    x, cu = bf(gen(3), sum(lens), 256), np.cumsum([0] + lens).astype(np.int32)
    pos = ints(np.concatenate([np.arange(n) for n in lens]))
    a, b = (paged.DeltaState(torch.zeros(4, 4, 1024, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 4, 128, 128, device=DEV)) for _ in range(2))
    m.mix(x, cu, pos, qwen35.Kept(a, pos, pos, ints([2, 2, 1, 1]), cu_seqlens=ints(cu)))  # sequence 2 is empty: state 1 is sequence 3's alone
    _refused(ctx, "row 1 has state 2")
    m.mix(x, cu, pos, qwen35.Kept(b, pos, pos, ints([2, -1, -1, 1]), cu_seqlens=ints(cu)))
    ctx.sync()
    assert torch.equal(a.state, b.state) and torch.equal(a.conv, b.conv)


# ------------------------------------------------------------------------------------------------ the decoder
def _decoder(layers=4, seed=41):
    cfg = oracle.DecoderConfig(vocab_size=500, hidden_size=256, intermediate_size=384, num_hidden_layers=layers, num_attention_heads=4,
                               num_key_value_heads=2, head_dim=256, linear_num_key_heads=4, linear_num_value_heads=8)
    keep = ("A_log", "dt_bias")
    w = {k: (t if k.endswith(keep) else t.to(torch.bfloat16).float()) for k, t in oracle.qwen35.init_weights(cfg, seed).items()}
    return cfg, w, qwen35.Decoder({k: (t.to(DEV) if k.endswith(keep) else t.to(torch.bfloat16).to(DEV)) for k, t in w.items()}, cfg, max_positions=512)


def test_decoder_goes_on_from_its_prompts(ctx):
    """Prompts of uneven length entered in two batches, steps, a row that ends and is given to another prompt: every hidden state
    against the f32 oracle run on the whole sequence, within 2e-2 or 1.5 times what the bf16 restatement of the reference is off."""
    cfg, w, dec = _decoder()
    cache = paged.PagedCache(cfg, rows=5, num_pages=40, page_size=16, max_length=256, dev=DEV)
    g = torch.Generator().manual_seed(4)
    seqs, got = {}, {}

    def enter(lens):
        prompts = [torch.randint(0, 500, (n,), generator=g) for n in lens]
        ids = torch.cat(prompts).to(DEV)
        y, rows = dec.prefill(ids, lens, cache)
        cu = np.cumsum([0] + lens).astype(np.int32)
        assert torch.equal(y, dec.forward(ids, cu, ints(np.concatenate([np.arange(n) for n in lens]))))
        for r, p, a, z in zip(rows, prompts, cu[:-1], cu[1:]):
            seqs[r], got[r] = p, [y[a:z]]
        return rows

    def finish(r):
        ids, y = seqs.pop(r), torch.cat(got.pop(r)).float().cpu()
        want, low = (oracle.decoder_forward(ids, w, cfg, dtype=d) for d in ("f32", "bf16"))
        assert y.shape == want.shape and max_rel(y, want) <= max(2e-2, 1.5 * max_rel(low, want)), r

    def steps(n):
        for _ in range(n):
            ids = torch.randint(0, 500, (5,), generator=g)
            y = dec.step(ids.to(DEV), cache)
            for r in seqs:
                seqs[r] = torch.cat([seqs[r], ids[r:r + 1]])
                got[r].append(y[r:r + 1])

    assert enter([70, 1, 33]) == [0, 1, 2]
    steps(20)
    assert enter([15]) == [3]
    steps(3)
    cache.release([1])
    finish(1)
    assert enter([130, 2]) == [1, 4]
    steps(18)
    device.load(0).sync()
    assert cache.lengths.tolist() == cache.held.tolist() and cache.free_count.tolist() == [cache.pages_left]
    in_use = [int(p) for r in range(5) for p in cache.tables[r, :pages(int(cache.held[r]), 16)]]
    assert sorted(in_use + cache.free_pages.tolist()[:cache.pages_left]) == list(range(40))
    for r in list(seqs):
        finish(r)
    cache.release(cache.active)
    ctx.sync()
    assert sorted(cache.free_pages.tolist()) == list(range(40)) and cache.lengths.tolist() == [-1] * 5


def test_a_captured_step_is_the_step(ctx):
    """Two caches filled alike: one steps eagerly, the other replays one captured step on a stream of its own. Bit-identical, and no
    host work in between."""
    cfg, w, dec = _decoder()
    ids = torch.randint(0, 500, (45,), generator=torch.Generator().manual_seed(1)).to(DEV)
    a, b = (paged.PagedCache(cfg, rows=4, num_pages=16, page_size=16, max_length=128, dev=DEV) for _ in range(2))
    for c in (a, b):
        dec.prefill(ids, [30, 15], c)
    tokens = torch.randint(0, 500, (30, 4), generator=torch.Generator().manual_seed(2)).to(DEV)
    want = [dec.step(t, a).clone() for t in tokens]
    ctx.sync()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = device.load(0)
        first = dec.step(tokens[0], b).clone()  # warm
        feed = tokens[1].clone()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = dec.step(feed, b)
        got = [first]
        b.advanced(29)
        for t in tokens[1:]:
            feed.copy_(t)
            graph.replay()
            got.append(out.clone())
        other.sync()
    for i, (x, y) in enumerate(zip(got, want)):
        assert torch.equal(x[:2], y[:2]), i
    assert torch.equal(a.lengths, b.lengths) and torch.equal(a.free_count, b.free_count) and a.held.tolist() == b.held.tolist()
    for x, y in zip(a.layers, b.layers):
        if isinstance(x, paged.DeltaState):
            assert torch.equal(x.state[:2], y.state[:2]) and torch.equal(x.conv[:2], y.conv[:2])
    with pytest.raises(ValueError, match="do not fit"):
        b.advanced(100)


def test_a_row_that_gets_no_page_keeps_its_states(ctx, monkeypatch):
    """A step that the host's mirror did not look after (a replay without `advanced`): the row without a page is reported and stays
    where it was, the others go on; once pages are free again, it goes on too."""
    cfg, w, dec = _decoder()
    cache, free = (paged.PagedCache(cfg, rows=3, num_pages=n, page_size=16, max_length=64, dev=DEV) for n in (4, 12))
    ids = torch.randint(0, 500, (47,), generator=torch.Generator().manual_seed(6)).to(DEV)
    for c in (cache, free):
        dec.prefill(ids, [10, 32, 5], c)
    tokens = torch.randint(0, 500, (2, 3), generator=torch.Generator().manual_seed(7)).to(DEV)
    before = [(t.state[1].clone(), t.conv[1].clone()) for t in cache.layers if isinstance(t, paged.DeltaState)]
    monkeypatch.setattr(cache, "fits", lambda steps=1: True)
    y = dec.step(tokens[0], cache)
    _refused(ctx, "no free pages")
    want = dec.step(tokens[0], free)
    assert torch.equal(y[[0, 2]], want[[0, 2]]) and cache.lengths.tolist() == [11, 32, 6] and cache.free_count.tolist() == [0]
    for t, (state, conv) in zip((t for t in cache.layers if isinstance(t, paged.DeltaState)), before):
        assert torch.equal(t.state[1], state) and torch.equal(t.conv[1], conv)
    monkeypatch.undo()
    cache.held[:], cache.pages_left = [11, 32, 6], 0
    cache.release([0])
    assert max_rel(dec.step(tokens[0], cache)[1], want[1]) <= 2e-2
    ctx.sync()
    assert cache.lengths.tolist() == [-1, 33, 7] == cache.held.tolist()


def test_a_prefill_that_fails_leaves_the_cache_as_it_was(ctx, monkeypatch):
    cfg, w, dec = _decoder(layers=2)
    cache = paged.PagedCache(cfg, rows=3, num_pages=8, page_size=16, max_length=64, dev=DEV)
    ids = torch.zeros(40, dtype=torch.int64, device=DEV)
    dec.prefill(ids[:20], [20], cache)
    with monkeypatch.context() as m:
        m.setattr(dec.layers[1].mlp, "forward", lambda *a, **k: (_ for _ in ()).throw(RuntimeError("no")))
        with pytest.raises(RuntimeError, match="no"):
            dec.prefill(ids, [40], cache)
    ctx.sync()
    assert cache.held.tolist() == [20, -1, -1] and cache.lengths.tolist() == [20, -1, -1] and cache.free_count.tolist() == [6] == [cache.pages_left]
    assert cache.state_index.tolist() == [0, -1, -1]


def test_the_cache_refuses_what_does_not_fit(ctx):
    cfg, w, dec = _decoder(layers=1)
    cache = paged.PagedCache(cfg, rows=2, num_pages=3, page_size=16, max_length=40, dev=DEV)
    ids = torch.zeros(64, dtype=torch.int64, device=DEV)
    for lens, match in (([41], "1 to 40"), ([20, 20], "4 pages"), ([1, 1, 1], "idle rows"), ([0], "1 to 40")):
        with pytest.raises(ValueError, match=match):
            dec.prefill(ids[:sum(lens)], lens, cache)
    with pytest.raises(ValueError, match="tokens"):
        dec.prefill(ids[:5], [6], cache)
    y, rows = dec.prefill(ids[:38], [32, 6], cache)
    with pytest.raises(ValueError, match="do not fit"):
        dec.step(ids[:2], cache)
    assert cache.held.tolist() == [32, 6] and cache.lengths.tolist() == [32, 6]
    cache.release([1])
    dec.step(ids[:2], cache)
    assert cache.held.tolist() == [33, -1]
    with pytest.raises(ValueError, match="active"):
        cache.release([1])
    with pytest.raises(ValueError, match="for every row"):
        dec.step(ids[:1], cache)
    exact = qwen35.Decoder(dec.w, cfg, max_positions=512, recurrence="exact")
    with pytest.raises(ValueError, match="chunked"):
        exact.prefill(ids[:3], [3], cache)
    short = qwen35.Decoder(dec.w, cfg, max_positions=33)
    with pytest.raises(ValueError, match="33 positions"):
        short.step(ids[:2], cache)
    ctx.sync()


@pytest.mark.parametrize("other", [dict(linear_num_value_heads=4), dict(linear_num_key_heads=2), dict(num_key_value_heads=1), dict(head_dim=128),
                                   dict(num_hidden_layers=8), dict(full_attention_interval=2)])
def test_the_decoder_refuses_the_cache_of_another(ctx, other):
    cfg, w, dec = _decoder()
    cache = paged.PagedCache(dataclasses.replace(cfg, **other), rows=2, num_pages=4, page_size=16, max_length=32, dev=DEV)
    ids = torch.zeros(5, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="other layers or heads"):
        dec.prefill(ids, [5], cache)
    with pytest.raises(ValueError, match="other layers or heads"):
        dec.step(ids[:2], cache)
    ctx.sync()
    assert cache.held.tolist() == [-1, -1] and cache.lengths.tolist() == [-1, -1]


def test_a_context_of_another_gpu_is_refused(ctx):
    other = type("Other", (), dict(ordinal=1))()
    g, i32 = gen(1), ints([0])
    kc = bf(g, 2, 16, 1, 64)
    x = bf(g, 1, 384)
    for call in (lambda: paged.block_tables(i32, ints([[0]]), ints([0]), i32, 16, ctx=other),
                 lambda: paged.release_blocks(i32, i32, ints([[0]]), ints([0]), i32, 16, ctx=other),
                 lambda: paged.cache_write(kc[:1, 0], kc[:1, 0], kc, kc, i32, ctx=other),
                 lambda: paged.attention_paged(kc[:1, 0], kc, kc, ints([[0]]), i32, ctx=other),
                 lambda: qwen35.gated_delta_rule_step(x, bf(g, 384, 4), i32, x[:, :1], x[:, :1], torch.zeros(1, device=DEV), torch.zeros(1, device=DEV),
                                                      x[:, :128], x[0, :128], 1e-6, bf(g, 1, 4, 384), torch.zeros(1, 1, 128, 128, device=DEV), 1, ctx=other)):
        with pytest.raises(ValueError, match="GPU 0, the context on GPU 1"):
            call()


def test_outputs_given_come_back(ctx):
    """The tensors of the call themselves, on every path (no rows included); whole numbers of other types are numbers too."""
    cached, left = ints([3, 15]), ints([4])
    r = paged.block_tables(cached, ints([[0, 1], [2, 3]]), ints([4, 5, 6, 7]), left, np.int64(16), lengths=cached, free_count_out=left)
    assert r.lengths is cached and r.free_count is left and cached.tolist() == [4, 16] and r.slots.tolist() == [3, 47]
    assert r.cu_seqlens.tolist() == [0, 1, 2] and r.positions.tolist() == [3, 15]
    q, kc, vc, tables, lengths, gate = _attention_case([20, 30], 4, 2, 64, 16, 1)
    wide = torch.zeros(2, 304, dtype=torch.bfloat16, device=DEV)
    for out in (wide[:, 8:264], wide[:0, 8:264]):
        n = out.shape[0]
        assert paged.attention_paged(q[:n], kc, vc, tables[:n], lengths[:n], out=out) is out
    assert torch.equal(wide[:, 8:264], paged.attention_paged(q, kc, vc, tables, lengths)) and not wide[:, :8].any() and not wide[:, 264:].any()
    c = _step_case(3, 2, 4, 8)
    y = qwen35.gated_delta_rule_step(**dict(c, state=c["state"].clone(), conv_state=c["conv_state"].clone()))
    out = torch.empty_like(y)
    assert qwen35.gated_delta_rule_step(**c, out=out) is out and torch.equal(out, y)
    with pytest.raises(ValueError, match="out must be"):
        qwen35.gated_delta_rule_step(**c, out=out[:, :-8])
    ctx.sync()


@pytest.mark.parametrize("name,change", [("mixed", lambda t: t.float()), ("conv_weight", lambda t: t[:, :3]), ("positions", lambda t: t.long()), ("b", lambda t: t[:, :-1]),
                                         ("a", lambda t: t.cpu()), ("dt_bias", lambda t: t.to(torch.bfloat16)), ("neg_exp_a", lambda t: t[:-1]),
                                         ("z", lambda t: t[:, ::2]), ("norm_weight", lambda t: t[:64]), ("state", lambda t: t.to(torch.bfloat16)),
                                         ("conv_state", lambda t: t[:, :3]), ("state_index", lambda t: t.repeat(2))])
def test_delta_step_names_the_argument_it_refuses(ctx, name, change):
    c = _step_case(3, 2, 4, 8)
    with pytest.raises(ValueError, match="mixed must|columns" if name == "mixed" else f"{name} must be"):
        qwen35.gated_delta_rule_step(**dict(c, **{name: change(c[name])}))
    ctx.sync()
