"""Cases for the operators that serve a hybrid decoder one new token at a time: block tables and slot maps from request
lengths, the write of keys and values into the paged cache, attention of one token over that cache, and the gated delta
rule's step on a carried state. Each has a plain form in elementary torch operations, the call that a program makes of
the library, and its definition in 64 bits."""
import math

import numpy as np
import torch

own = False
DEV = "cuda:0"
TAPS = 4          # causal conv of the linear-attention layers
HEAD = 128        # key and value head dimension of the gated delta rule
EPS = 1e-6


def listed():
    return [
        # eight conversations, each one token further: the bookkeeping at the head of a small decode step
        dict(name="tables one token 8", op="tables", rows=8, page=16, shortest=0, longest=2048, added=0, idle=1),
        # a thousand rows in flight, some idle
        dict(name="tables one token 1024", op="tables", rows=1024, page=64, shortest=1, longest=8192, added=0, idle=17),
        # a packed batch of prompts (16384 tokens in 31 rows of uneven length) that enters the cache
        dict(name="tables prompts 31", op="tables", rows=31, page=64, shortest=0, longest=700, added=529, idle=2),
        # keys and values of one decode step, keys normed and rotated on the way (2 KV heads of 256, 64 rotated)
        dict(name="write step 64", op="write", tokens=64, kv=2, dim=256, rot=64, page=64, norm=True, idle=3),
        # keys and values of a 16384-token prompt batch of the 27B shape, keys already normed and rotated
        dict(name="write prompts 16384", op="write", tokens=16384, kv=4, dim=256, rot=0, page=64, norm=False, idle=0),
        # the smallest call: one young conversation
        dict(name="attend 1 x 17", op="attend", rows=1, heads=8, kv=2, dim=256, shortest=17, longest=17, page=16, gate=True, idle=0),
        # an ordinary step: 32 conversations of uneven length
        dict(name="attend 32 x 2048", op="attend", rows=32, heads=8, kv=2, dim=256, shortest=1, longest=2048, page=64, gate=True, idle=1),
        # one very long context alone: the work is one row's, split over the whole GPU
        dict(name="attend 1 x 131071", op="attend", rows=1, heads=8, kv=2, dim=256, shortest=131071, longest=131071, page=64, gate=False, idle=0),
        # a full serving step of the 27B shape: 64 long conversations, six query heads to a KV head
        dict(name="attend 64 x 8192", op="attend", rows=64, heads=24, kv=4, dim=256, shortest=100, longest=8192, page=16, gate=True, idle=2),
        # linear attention, one conversation (16 + 16 heads of 128)
        dict(name="step 1", op="step", rows=1, keys=16, values=16, fresh=0, idle=0),
        # linear attention, one tensor-parallel rank's heads, an odd number of rows, new and idle ones among them
        dict(name="step 37", op="step", rows=37, keys=2, values=6, fresh=5, idle=2),
        # linear attention of the 27B shape (48 value heads on 16 key heads), 64 conversations
        dict(name="step 64", op="step", rows=64, keys=16, values=48, fresh=1, idle=1),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["tables", "write", "attend", "attend", "step", "step"])
    page = rng.choice([16, 32, 64, 128])
    if op == "tables":
        rows = _log(rng, 1, 2048)
        added = rng.choice([0, _log(rng, 1, max(1, 32768 // rows))])
        return dict(op=op, rows=rows, page=page, shortest=rng.choice([0, 1]), longest=_log(rng, 1, 16384), added=added, idle=rng.randrange(0, 1 + rows // 4))
    if op == "write":
        dim, kv, tokens = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8]), _log(rng, 1, 16384)
        norm = rng.random() < 0.6
        return dict(op=op, tokens=tokens, kv=kv, dim=dim, rot=rng.choice([16, 32, 64]) if norm else 0, page=page, norm=norm, idle=rng.randrange(0, 1 + tokens // 8))
    if op == "attend":
        dim, kv, rows = rng.choice([64, 128, 256, 256]), rng.choice([1, 2, 4, 8]), _log(rng, 1, 128)
        heads = kv * rng.choice([1, 2, 3, 4, 6, 8, 16])
        longest = min(_log(rng, 1, 131072), 64 * 8192 * 4 * 256 // (rows * kv * dim))
        return dict(op=op, rows=rows, heads=heads, kv=kv, dim=dim, shortest=rng.randint(1, longest), longest=longest, page=page,
                    gate=rng.random() < 0.5, idle=rng.randrange(0, 1 + rows // 4))
    keys = rng.choice([1, 2, 4, 16])
    values = keys * rng.choice([1, 2, 3])
    rows = _log(rng, 1, 64 * 48 // values)
    return dict(op=op, rows=rows, keys=keys, values=values, fresh=rng.randrange(0, 1 + rows // 2), idle=rng.randrange(0, 1 + rows // 4))


def _lengths(case):
    """The rows' context lengths: spread evenly from the shortest to the longest, and none for the idle rows (the last ones)."""
    n = case["rows"] - case["idle"]
    return [round(x) for x in np.linspace(case["longest"], case["shortest"], n)] + [-1] * case["idle"]


def _added(case):
    """Tokens that each row of a prompt batch adds: spread evenly around the mean, so that their sum is rows * added."""
    n = case["rows"] - case["idle"]
    return [2 * case["added"] * (i + 1) // (n + 1) for i in range(n)] + [0] * case["idle"]


def _pages(tokens, page):
    return -(-tokens // page)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = np.random.RandomState(seed % (1 << 32))
    normal = lambda *shape, s=1.0: (torch.randn(*shape, device=DEV, generator=g) * s).to(torch.bfloat16)  # noqa: E731
    ints = lambda values: torch.tensor(np.asarray(values), dtype=torch.int32, device=DEV)  # noqa: E731
    st = dict(case)
    page = case.get("page")
    if case["op"] == "tables":
        order = h.permutation(case["rows"])
        cached, added = np.array(_lengths(case))[order], np.array(_added(case))[order]
        held = [_pages(max(0, int(c)), page) for c in cached]
        width = max(_pages(max(0, int(c)) + max(1, int(a)), page) for c, a in zip(cached, added)) + 1
        total = sum(_pages(max(0, int(c)) + max(1, int(a)), page) for c, a in zip(cached, added)) + 7
        pool = h.permutation(total)
        tables = np.full((case["rows"], width), -1, np.int32)
        at = 0
        for b, n in enumerate(held):
            tables[b, :n] = pool[at:at + n]
            at += n
        free = np.full(total, -1, np.int32)
        free[:total - at] = pool[at:]
        tokens = int(added.sum()) if case["added"] else case["rows"]
        st.update(cached=ints(cached), added_each=ints(added) if case["added"] else None, tables=ints(tables), free=ints(free), count=ints([total - at]),
                  max_tokens=-(-max(tokens, 1) // 8) * 8 if case["added"] else case["rows"])
    elif case["op"] == "write":
        T, kv, dim = case["tokens"], case["kv"], case["dim"]
        pages = 1 + _pages(T, page) + 3  # page 0 stays unused
        slots = page + h.permutation((pages - 1) * page)[:T] if case["norm"] else page + np.arange(T)  # steps are scattered, prompts are not
        slots[h.permutation(T)[:case["idle"]]] = -1
        qkv = normal(T, 2 * kv * dim + 8)  # the keys' and values' columns of the stacked projection
        st.update(k=qkv[:, :kv * dim].unflatten(1, (kv, dim)), v=qkv[:, kv * dim:2 * kv * dim].unflatten(1, (kv, dim)), slots=ints(slots),
                  k_cache=normal(pages, page, kv, dim), v_cache=normal(pages, page, kv, dim))
        if case["norm"]:
            angle = torch.arange(8192, device=DEV, dtype=torch.float64)[:, None] / 1e7 ** (torch.arange(case["rot"] // 2, device=DEV, dtype=torch.float64) * 2 / case["rot"])
            st.update(weight=normal(dim, s=0.1), cos=angle.cos().float(), sin=angle.sin().float(), positions=ints(h.randint(0, 8192, T)))
    elif case["op"] == "attend":
        B, H, kv, dim = case["rows"], case["heads"], case["kv"], case["dim"]
        lengths = np.array(_lengths(case))[h.permutation(B)]
        held = [_pages(max(0, int(n)), page) for n in lengths]
        pages, width = sum(held) + 3, max(held) + 1
        pool = h.permutation(pages)
        tables = np.zeros((B, width), np.int32)
        at = 0
        for b, n in enumerate(held):
            tables[b, :n] = pool[at:at + n]
            at += n
        qg = normal(B, H, 2, dim)  # query and output gate lie side by side for each head, as the projection leaves them
        st.update(q=qg[:, :, 0], gate_in=qg[:, :, 1] if case["gate"] else None, k_cache=normal(pages, page, kv, dim), v_cache=normal(pages, page, kv, dim),
                  tables=ints(tables), lengths=ints(lengths))
    else:
        B, Hk, Hv = case["rows"], case["keys"], case["values"]
        C = (2 * Hk + Hv) * HEAD
        index = 1 + h.permutation(B)  # slot 0 belongs to nobody
        index[h.permutation(B)[:case["idle"]]] = -1
        positions = h.randint(TAPS, 8192, B)
        positions[h.permutation(B)[:case["fresh"]]] = h.randint(0, TAPS, case["fresh"])
        ba = normal(B, 2 * Hv)
        st.update(mixed=normal(B, C + 8)[:, :C], conv=normal(C, TAPS, s=0.3), positions=ints(positions), b=ba[:, :Hv], a=ba[:, Hv:],
                  dt_bias=torch.randn(Hv, device=DEV, generator=g) * 0.5, decay=-torch.exp(torch.randn(Hv, device=DEV, generator=g) * 0.5),
                  z=normal(B, Hv * HEAD), weight=1 + normal(HEAD, s=0.1), index=ints(index), conv_state=normal(B + 1, TAPS, C),
                  state=torch.randn(B + 1, Hv, HEAD, HEAD, device=DEV, generator=g) * 0.1)
    return st


def run(st):
    if own:
        from sys1_b200 import paged, qwen35
        if st["op"] == "tables":
            r = paged.block_tables(st["cached"], st["tables"], st["free"], st["count"], st["page"], added=st["added_each"], max_tokens=st["max_tokens"])
            return dict(tables=st["tables"], lengths=r.lengths, starts=r.cu_seqlens, positions=r.positions, slots=r.slots, left=r.free_count)
        if st["op"] == "write":
            if st["norm"]:
                paged.cache_write(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"], norm_weight=st["weight"], eps=EPS, cos=st["cos"], sin=st["sin"],
                                  positions=st["positions"], rotary_dim=st["rot"], bf16_ops=False)
            else:
                paged.cache_write(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"])
            return dict(k=st["k_cache"], v=st["v_cache"])
        if st["op"] == "attend":
            return paged.attention_paged(st["q"], st["k_cache"], st["v_cache"], st["tables"], st["lengths"], gate=st["gate_in"])
        y = qwen35.gated_delta_rule_step(st["mixed"], st["conv"], st["positions"], st["b"], st["a"], st["dt_bias"], st["decay"], st["z"], st["weight"], EPS,
                                         st["conv_state"], st["state"], st["keys"], state_index=st["index"])
        return dict(y=y, state=st["state"], conv=st["conv_state"])
    return dict(tables=_tables, write=_write, attend=_attend, step=_step)[st["op"]](st)


def _tables(st):
    page, idle = st["page"], st["cached"] < 0
    old = st["cached"].clamp(min=0).long()
    adds = torch.where(idle, 0, 1 if st["added_each"] is None else st["added_each"].long())
    takes = torch.ones_like(adds) if st["added_each"] is None else adds  # tokens of the batch that belong to the row
    starts = torch.nn.functional.pad(takes.cumsum(0), (1, 0))
    have, want = (old + page - 1) // page, (old + adds + page - 1) // page
    before = (want - have).cumsum(0) - (want - have)
    cols = torch.arange(st["tables"].shape[1], device=DEV)
    taken = st["count"].long() - 1 - before[:, None] - (cols - have[:, None])
    new = (cols >= have[:, None]) & (cols < want[:, None])
    tables = torch.where(new, st["free"][taken.clamp(0, st["free"].numel() - 1)], st["tables"])
    t = torch.arange(st["max_tokens"], device=DEV)
    row = torch.searchsorted(starts[1:], t, right=True).clamp(max=old.numel() - 1)
    live = (t < starts[-1]) & ~idle[row]
    positions = torch.where(live, old[row] + t - starts[row], 0)
    slots = torch.where(live, tables[row, (positions // page).clamp(max=tables.shape[1] - 1)].long() * page + positions % page, -1)
    lengths = torch.where(idle, st["cached"].long(), old + adds)
    left = st["count"].long() - (want - have).sum()
    return dict(tables=tables, lengths=lengths.int(), starts=starts.int(), positions=positions.int(), slots=slots.int(), left=left.int())


def _write(st):
    k = st["k"].float()
    if st["norm"]:
        k = k / (k.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + st["weight"].float())
        half = st["rot"] // 2
        c, s = (t[st["positions"].long()][:, None] for t in (st["cos"], st["sin"]))
        lo, hi = k[..., :half], k[..., half:2 * half]
        k = torch.cat([lo * c - hi * s, hi * c + lo * s, k[..., 2 * half:]], -1)
    at, live = st["slots"].long().clamp(min=0), (st["slots"] >= 0)[:, None, None]
    kc, vc = st["k_cache"].flatten(0, 1), st["v_cache"].flatten(0, 1)
    kc.index_copy_(0, at, torch.where(live, k.to(torch.bfloat16), kc[:1]))  # idle tokens put slot 0's own value back
    vc.index_copy_(0, at, torch.where(live, st["v"], vc[:1]))
    return dict(k=st["k_cache"], v=st["v_cache"])


def _attend(st):
    B, H, D = st["q"].shape
    kv = st["kv"]
    k = st["k_cache"][st["tables"].long()].float().flatten(1, 2).permute(0, 2, 3, 1)  # [B, kv, D, L]
    v = st["v_cache"][st["tables"].long()].float().flatten(1, 2).transpose(1, 2)      # [B, kv, L, D]
    scores = st["q"].float().reshape(B, kv, H // kv, D) @ k * D ** -0.5
    seen = (torch.arange(v.shape[2], device=DEV) < st["lengths"][:, None])[:, None, None]
    top = torch.where(seen, scores, -math.inf).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - top), 0.0)
    o = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.reshape(B, H, D)
    if st["gate_in"] is not None:
        o = o * torch.sigmoid(st["gate_in"].float())
    return o.reshape(B, H * D).to(torch.bfloat16)


def _step(st):
    B, Hk, Hv = st["rows"], st["keys"], st["values"]
    live = st["index"] >= 0
    at, pos = st["index"].long().clamp(min=0), st["positions"].long()
    ring, x, w = st["conv_state"][at].float(), st["mixed"].float(), st["conv"].float()
    back = torch.arange(1, TAPS, device=DEV)
    past = ring[torch.arange(B, device=DEV)[:, None], (pos[:, None] - back) % TAPS]  # [B, 3, C]
    past = torch.where((back <= pos[:, None])[..., None], past, 0.0)
    u = x * w[:, TAPS - 1] + (past * w.t().flip(0)[1:]).sum(1)
    u = u * torch.sigmoid(u)
    q, k, v = (t.unflatten(1, (-1, HEAD)) for t in u.split([Hk * HEAD, Hk * HEAD, Hv * HEAD], 1))
    q, k = (t.repeat_interleave(Hv // Hk, 1) / (t.square().sum(-1, keepdim=True) + EPS).sqrt().repeat_interleave(Hv // Hk, 1) for t in (q, k))
    q = q * HEAD ** -0.5
    beta = torch.sigmoid(st["b"].float())
    f = st["a"].float() + st["dt_bias"]
    gate = torch.exp((f.clamp(min=0) + torch.log1p(torch.exp(-f.abs()))) * st["decay"])
    S = torch.where((pos > 0)[:, None, None, None], st["state"][at], 0.0) * gate[..., None, None]
    delta = (v - (S * k[..., None]).sum(2)) * beta[..., None]
    S = S + k[..., None] * delta[:, :, None]
    o = (S * q[..., None]).sum(2)
    z = st["z"].float().unflatten(1, (Hv, HEAD))
    y = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * st["weight"].float() * z * torch.sigmoid(z)
    y = torch.where(live[:, None, None], y, 0.0).flatten(1).to(torch.bfloat16)
    st["state"].index_copy_(0, at, torch.where(live[:, None, None, None], S, st["state"][:1]))  # idle rows put slot 0's own value back
    cs = st["conv_state"].flatten(0, 1)
    cs.index_copy_(0, torch.where(live, at * TAPS + pos % TAPS, 0), torch.where(live[:, None], st["mixed"], cs[:1]))
    return dict(y=y, state=st["state"], conv=st["conv_state"])


def work(case):
    page = case.get("page")
    if case["op"] == "tables":
        lengths = _lengths(case)
        added = _added(case) if case["added"] else [int(n >= 0) for n in lengths]
        tokens = sum(added) if case["added"] else case["rows"]
        new = sum(_pages(max(n, 0) + a, page) - _pages(max(n, 0), page) for n, a in zip(lengths, added))
        return dict(bytes=4 * (case["rows"] * (4 if case["added"] else 3) + 2 * new + 2 * tokens), flops=0)
    if case["op"] == "write":
        n = (case["tokens"] - case["idle"]) * case["kv"] * case["dim"]
        rope = (case["tokens"] - case["idle"]) * (4 * case["rot"] + 4) if case["norm"] else 0
        return dict(bytes=8 * n + rope + 4 * case["tokens"], flops=8 * n if case["norm"] else 0)
    if case["op"] == "attend":
        tokens = sum(max(0, n) for n in _lengths(case))
        own_rows = case["rows"] * case["heads"] * case["dim"] * (6 if case["gate"] else 4)
        return dict(bytes=4 * tokens * case["kv"] * case["dim"] + own_rows + 4 * tokens // page, flops=4 * tokens * case["heads"] * case["dim"])
    live, Hv = case["rows"] - case["idle"], case["values"]
    C = (2 * case["keys"] + Hv) * HEAD
    return dict(bytes=live * (8 * Hv * HEAD * HEAD + 2 * C * (TAPS + 1) + 4 * Hv * HEAD) + 2 * TAPS * C, flops=live * Hv * HEAD * HEAD * 7)


def exact(case, seed):
    """The definitions, one row after the other, in 64 bits. Whole numbers have no rounding and are not given."""
    if case["op"] == "tables":
        return None
    st = prepare(case, seed)
    f = lambda t: t.double()  # noqa: E731
    if case["op"] == "write":
        K, V = f(st["k_cache"]).flatten(0, 1), f(st["v_cache"]).flatten(0, 1)
        keep = torch.nonzero(st["slots"] >= 0).flatten()
        k, slots = f(st["k"][keep]), st["slots"][keep].long()
        if case["norm"]:
            k = k * torch.rsqrt(torch.mean(k * k, -1, keepdim=True) + EPS) * (f(st["weight"]) + 1)
            p = st["positions"][keep].long()
            turn = torch.complex(f(st["cos"])[p], f(st["sin"])[p])[:, None]
            half = case["rot"] // 2
            both = torch.complex(k[..., :half], k[..., half:2 * half]) * turn
            k = torch.cat([both.real, both.imag, k[..., 2 * half:]], -1)
        K[slots], V[slots] = k, f(st["v"][keep])
        return dict(k=K.unflatten(0, (-1, case["page"])), v=V.unflatten(0, (-1, case["page"])))
    if case["op"] == "attend":
        out = torch.zeros(case["rows"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
        for b, n in enumerate(st["lengths"].tolist()):
            if n <= 0:
                continue
            at = st["tables"][b, :_pages(n, case["page"])].long()
            k, v = (f(st[c][at].flatten(0, 1)[:n]) for c in ("k_cache", "v_cache"))  # [n, kv, D]
            each = case["heads"] // case["kv"]
            for j in range(case["kv"]):
                q = f(st["q"][b, j * each:(j + 1) * each])
                p = torch.softmax(q @ k[:, j].t() / math.sqrt(case["dim"]), -1)
                out[b, j * each:(j + 1) * each] = p @ v[:, j]
            if case["gate"]:
                out[b] /= 1 + torch.exp(-f(st["gate_in"][b]))
        return out.reshape(case["rows"], -1)
    Hk, Hv = case["keys"], case["values"]
    state, ring = f(st["state"]), f(st["conv_state"])
    y = torch.zeros(case["rows"], Hv, HEAD, dtype=torch.float64, device=DEV)
    index, positions = st["index"].tolist(), st["positions"].tolist()
    w = f(st["conv"])
    for r in range(case["rows"]):
        i, p = index[r], positions[r]
        if i < 0:
            continue
        ring[i, p % TAPS] = f(st["mixed"][r])
        u = sum(ring[i, (p - back) % TAPS] * w[:, TAPS - 1 - back] for back in range(min(p, TAPS - 1) + 1))
        u = (u / (1 + torch.exp(-u))).reshape(-1, HEAD)
        heads = torch.arange(Hv, device=DEV) // (Hv // Hk)
        q, k, v = u[heads], u[Hk + heads], u[2 * Hk:]
        q = q / torch.sqrt((q * q).sum(1, keepdim=True) + EPS) / math.sqrt(HEAD)
        k = k / torch.sqrt((k * k).sum(1, keepdim=True) + EPS)
        beta = 1 / (1 + torch.exp(-f(st["b"][r])))
        keep = torch.exp(f(st["decay"]) * torch.nn.functional.softplus(f(st["a"][r]) + f(st["dt_bias"]), threshold=100.0))
        S = state[i] * keep[:, None, None] if p > 0 else torch.zeros_like(state[i])
        d = (v - torch.bmm(k[:, None], S)[:, 0]) * beta[:, None]
        S = S + torch.bmm(k[:, :, None], d[:, None])
        state[i] = S
        o = torch.bmm(q[:, None], S)[:, 0]
        z = f(st["z"][r]).reshape(Hv, HEAD)
        y[r] = o * torch.rsqrt((o * o).mean(1, keepdim=True) + EPS) * f(st["weight"]) * z / (1 + torch.exp(-z))
    return dict(y=y.flatten(1), state=state, conv=ring)
