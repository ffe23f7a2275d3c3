"""What the decode operators compute, in plain integers and 64-bit floating point."""
import math

import torch


def pages(tokens, page):
    return -(-tokens // page)


def block_tables_model(cached, added, page, free, count, tables, max_tokens):
    tables = tables.copy()
    rows, width = tables.shape
    cu, lengths, refused, positions, slots, taken = [0], [], [], [0] * max_tokens, [-1] * max_tokens, 0
    wanted = 0
    for b in range(rows):
        idle = cached[b] < 0
        add = 0 if idle else 1 if added is None else max(int(added[b]), 0)
        cu.append(cu[-1] + (1 if added is None else add))
        old = max(int(cached[b]), 0)
        need = pages(old + add, page) - pages(old, page)
        if pages(old + add, page) > width or old + add >= 2 ** 31 or cu[-1] > max_tokens:
            refused.append(b)
            lengths.append(int(cached[b]))
            continue
        wanted += need
        if need and wanted > count:
            refused.append(b)
            lengths.append(int(cached[b]))
            continue
        for i in range(need):
            tables[b, pages(old, page) + i] = free[count - 1 - (wanted - need + i)]
        taken = max(taken, wanted) if need else taken
        lengths.append(int(cached[b]) if idle else old + add)
        for j in range(add):
            p = old + j
            positions[cu[b] + j], slots[cu[b] + j] = p, int(tables[b, p // page]) * page + p % page
    return dict(tables=tables, lengths=lengths, cu_seqlens=cu, positions=positions, slots=slots, left=count - taken, refused=refused)


def release_model(ended, lengths, tables, free, count, page):
    free, lengths, refused, put, offered = list(free), [int(n) for n in lengths], [], 0, 0
    for b in range(len(lengths)):
        if not ended[b]:
            continue
        n = pages(max(lengths[b], 0), page)
        if n > tables.shape[1]:
            refused.append(b)
            continue
        offered += n
        if n and count + offered > len(free):
            refused.append(b)
            continue
        free[count + offered - n:count + offered] = [int(x) for x in tables[b, :n]]
        put = max(put, offered) if n else put
        lengths[b] = -1
    return free, count + put, lengths, refused


def attention_64(q, k_cache, v_cache, tables, lengths, gate, scale):
    """The output [rows, heads, dim] and, for the error bound, the same sum with |v| for v."""
    B, H, D = q.shape
    kv, page = k_cache.shape[2], k_cache.shape[1]
    out, size = torch.zeros(B, H, D, dtype=torch.float64, device=q.device), torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        at = tables[b, :pages(n, page)].long()
        k, v = (c[at].flatten(0, 1)[:n].double() for c in (k_cache, v_cache))
        for h in range(H):
            p = torch.softmax(k[:, h // (H // kv)] @ q[b, h].double() * scale, 0)
            out[b, h], size[b, h] = p @ v[:, h // (H // kv)], p @ v[:, h // (H // kv)].abs()
    if gate is not None:
        out, size = out * torch.sigmoid(gate.double()), size * torch.sigmoid(gate.double())
    return out, size


TAU = 2.0 ** -19  # 32 roundings of f32: sums of a few terms or in trees, exp and sqrt with errors of a few units


def delta_step_64(mixed, conv_w, pos, b, a, dt_bias, neg_exp_a, z, w, eps, conv_state, state, key_heads, index):
    """Outputs and updated states in 64 bits, with a bound on the error of an f32 evaluation rounded once: every sum is bounded by
    TAU times the sum of its terms' sizes, carried through the formula. Returns (y, y_bound, state, state_bound, conv_state)."""
    f = lambda t: t.double()  # noqa: E731
    rows, Hv = mixed.shape[0], state.shape[1]
    y, yb = (torch.zeros(rows, Hv, 128, dtype=torch.float64, device=mixed.device) for _ in range(2))
    S_all, Sb = f(state).clone(), torch.zeros_like(f(state))
    ring = conv_state.clone()
    heads = torch.arange(Hv, device=mixed.device) // (Hv // key_heads)
    for r in range(rows):
        i, p = int(index[r]), int(pos[r])
        if i < 0:
            continue
        ring[i, p % 4] = mixed[r]
        terms = [f(ring[i, (p - back) % 4]) * f(conv_w)[:, 3 - back] for back in range(min(p, 3) + 1)]
        u, size = sum(terms), sum(t.abs() for t in terms)
        size = torch.maximum(1.1 * size, u.abs())  # |silu'| < 1.1
        u = u * torch.sigmoid(u)
        u, size = u.reshape(-1, 128), size.reshape(-1, 128)
        nq, nk = (torch.sqrt((u[s + heads] ** 2).sum(1, keepdim=True) + 1e-6) for s in (0, key_heads))
        q, qs = u[heads] / nq / math.sqrt(128), size[heads] / nq / math.sqrt(128)
        k, ks = u[key_heads + heads] / nk, size[key_heads + heads] / nk
        # the norm's own error is that of the vector: |delta n| / n <= TAU |size| / n
        qs, ks = qs + q.abs() * (qs.norm(dim=1, keepdim=True) * math.sqrt(128)), ks + k.abs() * ks.norm(dim=1, keepdim=True)
        v, vs = u[2 * key_heads:], size[2 * key_heads:]
        beta = torch.sigmoid(f(b[r]))[:, None]
        g = torch.nn.functional.softplus(f(a[r]) + f(dt_bias), threshold=100.0) * f(neg_exp_a)
        keep, grow = torch.exp(g)[:, None, None], (1 + g.abs())[:, None, None]  # exp of g(1 + e): relative error |g| e
        S = f(state[i]) * keep if p > 0 else torch.zeros_like(f(state[i]))
        sk = torch.einsum("hkv,hk->hv", S, k)
        sks = torch.einsum("hkv,hk->hv", S.abs() * grow, ks)
        d, ds = beta * (v - sk), beta * (vs + sks)
        new = S + k[:, :, None] * d[:, None]
        S_all[i], Sb[i] = new, TAU * (S.abs() * grow + ks[:, :, None] * ds[:, None])
        o = torch.einsum("hkv,hk->hv", new, q)
        os_ = TAU * (torch.einsum("hkv,hk->hv", S.abs() * grow, qs) + ds * (qs * ks).sum(1, keepdim=True))
        zz = f(z[r]).reshape(Hv, 128)
        norm = torch.rsqrt((o * o).mean(1, keepdim=True) + eps)
        last = f(w) * zz * torch.sigmoid(zz)
        y[r] = o * norm * last
        yb[r] = os_ * norm * last.abs() + y[r].abs() * (2.0 ** -8 + TAU * (1 + zz.abs()) + os_.norm(dim=1, keepdim=True) * norm / math.sqrt(128))
    return y.flatten(1), yb.flatten(1), S_all, Sb, ring
