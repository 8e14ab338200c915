"""The operators of fermix_amd.network from their definitions, in 64 bits on the CPU, with the
gradients written out: what the GPU tests compare with."""

import math

import torch


def bucket_of(buckets, num, q_pos, k_pos):
    R = buckets.numel() // 2
    d = k_pos.long()[..., None, :] - q_pos.long()[..., :, None]
    return buckets.long()[d.clamp(-R, R) + R].clamp(max=num - 1)


def relative_bias(table, buckets, q_pos, k_pos):
    return table.double()[bucket_of(buckets, table.shape[0], q_pos, k_pos)].movedim(-1, -3)


def bucket_sums(g, bucket, num):
    """g (B, H, Q, K), bucket (B, Q, K) -> (num, H)"""
    out = torch.zeros(num, g.shape[1], dtype=torch.float64)
    for h in range(g.shape[1]):
        out[:, h].index_add_(0, bucket.flatten(), g[:, h].flatten())
    return out


def attention(q, k, v, table=None, buckets=None, q_pos=None, k_pos=None, lengths=None, q_lengths=None, mask=None,
              causal=False, offset=0, scale=None, grad=None):
    """out, and with grad (the cotangent) also dq, dk, dv, dtable and by bucket the magnitudes that its terms
    P (dP - delta) are made of, P (|dP| + |delta|): a term's error goes by them, not by what is left of it."""
    B, N, H, D = q.shape
    K, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    rows, keys = torch.arange(N) + offset, torch.arange(K)
    key_ok = torch.ones(B, K, dtype=torch.bool)
    if lengths is not None:
        key_ok &= keys < lengths[:, None]
    if mask is not None:
        key_ok &= mask
    ok = key_ok[:, None, :].expand(B, N, K).clone()
    if causal:
        ok &= keys <= rows[:, None]
    if q_lengths is not None:
        ok &= (torch.arange(N) < q_lengths[:, None])[:, :, None]
    ok = ok[:, None]
    zero = lambda t: torch.where(key_ok[:, :, None, None], t.double(), 0.0).transpose(1, 2).repeat_interleave(G, 1)
    q64, k64, v64 = q.double().transpose(1, 2), zero(k), zero(v)
    if q_lengths is not None:
        q64 = torch.where((torch.arange(N) < q_lengths[:, None])[:, None, :, None], q64, 0.0)
    S = scale * q64 @ k64.transpose(2, 3)
    if table is not None:
        if q_pos is None:
            q_pos, k_pos = rows.expand(B, N), keys.expand(B, K)
        bucket = bucket_of(buckets, table.shape[0], q_pos, k_pos)
        S = S + table.double()[bucket].movedim(-1, 1)
    S = torch.where(ok, S, -math.inf)
    top = S.amax(-1, keepdim=True) if K else torch.full((B, H, N, 1), -math.inf, dtype=torch.float64)
    P = torch.exp(S - torch.where(torch.isinf(top), 0.0, top))
    total = P.sum(-1, keepdim=True)
    P = P / torch.where(total == 0, 1.0, total)
    out = (P @ v64).transpose(1, 2)
    if grad is None:
        return out
    g = grad.double().transpose(1, 2)
    if q_lengths is not None:
        g = torch.where((torch.arange(N) < q_lengths[:, None])[:, None, :, None], g, 0.0)
    dP = g @ v64.transpose(2, 3)
    delta = (P * dP).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    dq = scale * dS @ k64
    dk, dv = scale * dS.transpose(2, 3) @ q64, P.transpose(2, 3) @ g
    dk, dv = (t.reshape(B, Hkv, G, K, D).sum(2).transpose(1, 2) for t in (dk, dv))
    dt = size = None
    if table is not None:
        dt = bucket_sums(dS, bucket, table.shape[0])
        size = bucket_sums(P * (dP.abs() + delta.abs()), bucket, table.shape[0])
    return out, dq.transpose(1, 2), dk, dv, dt, size


def attention_step(q, k_cache, v_cache, pages, lengths, k=None, v=None, table=None, buckets=None, scale=None):
    """out; the caches are written in place."""
    B, H, D = q.shape
    P, page, Hkv, _ = k_cache.shape
    G = H // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, H, D, dtype=torch.float64)
    n_of = lambda b: max(int(lengths[b]) + (k is not None), 0) if int(lengths[b]) >= 0 else 0
    good = []
    for b in range(B):
        n = n_of(b)
        used = pages[b, : -(-n // page)] if n <= pages.shape[1] * page else None
        good.append(used is not None and bool(((used >= 0) & (used < P)).all()))
        if k is not None and n and used is not None and 0 <= int(pages[b, (n - 1) // page]) < P:
            at = int(pages[b, (n - 1) // page])
            k_cache[at, (n - 1) % page], v_cache[at, (n - 1) % page] = k[b], v[b]
    for b in range(B):
        n = n_of(b)
        if n == 0:
            continue
        if not good[b]:
            out[b] = math.nan
            continue
        rows = pages[b, : -(-n // page)].long()
        kk, vv = (t[rows].flatten(0, 1)[:n].double().repeat_interleave(G, 1) for t in (k_cache, v_cache))
        S = scale * torch.einsum("hd,nhd->hn", q[b].double(), kk)
        if table is not None:
            bucket = bucket_of(buckets, table.shape[0], torch.tensor([n - 1]), torch.arange(n))[0]
            S = S + table.double()[bucket].t()
        top = S.amax(-1, keepdim=True)
        p = torch.exp(S - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(-1, keepdim=True)
        out[b] = torch.einsum("hn,nhd->hd", p / torch.where(total == 0, 1.0, total), vv)
    return out


def residual_norm(x, h, post_weight=None, post_bias=None, gate=None, scale=None, pre_weight=None, pre_bias=None,
                  norm="rms", eps=1e-6, post_norm=True, pre_norm=True, grads=None):
    """(y, z), and with grads = (dy, dz) the gradients by name, and as size_<name> the magnitudes that each is
    made of: those of the addends of dx = dy + r (dn - n mean(n dn) - mean(dn)) and of what follows from it."""
    wide = lambda t: None if t is None else (t.double() if isinstance(t, torch.Tensor) else t)
    x, h, w1, b1, g, s, w2, b2 = (wide(t) for t in (x, h, post_weight, post_bias, gate, scale, pre_weight, pre_bias))
    s, g = 1.0 if s is None else s, 1.0 if g is None else g

    def normed(t, size):
        """the normed row, its divisor's reciprocal, and the magnitudes it is made of"""
        mean = t.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(t[..., :1])
        c = t - mean
        r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        return c * r, r, r * (size + mean.abs())

    def back(n, r, dn, size):
        d = dn - n * (n * dn).mean(-1, keepdim=True)
        d = r * (d - dn.mean(-1, keepdim=True) if norm == "layer" else d)
        s = size + n.abs() * (n.abs() * size).mean(-1, keepdim=True)
        return d, r * (s + size.mean(-1, keepdim=True) if norm == "layer" else s)

    mag = lambda t: t.abs() if isinstance(t, torch.Tensor) else abs(t)
    n1, r1, o1 = normed(h, h.abs()) if post_norm else (h, None, h.abs())
    a = n1 * (1.0 if w1 is None else w1) + (0.0 if b1 is None else b1)
    y = x + s * g * a
    m1 = o1 * (1.0 if w1 is None else w1.abs()) + (0.0 if b1 is None else b1.abs())  # of a
    n2, r2, o2 = normed(y, x.abs() + mag(s) * mag(g) * m1) if pre_norm else (y, None, None)
    z = n2 * (1.0 if w2 is None else w2) + (0.0 if b2 is None else b2) if pre_norm else None
    if grads is None:
        return y, z
    dy, dz = grads
    dx = torch.zeros_like(y) if dy is None else dy.double()
    mx = dx.abs()
    got = {}
    if pre_norm and dz is not None:
        dz = dz.double()
        got["pre_weight"], got["pre_bias"] = dz * n2, dz
        dn2 = dz * (1.0 if w2 is None else w2)
        more, size = back(n2, r2, dn2, dn2.abs())
        dx, mx = dx + more, mx + size
    else:
        got["pre_weight"] = got["pre_bias"] = torch.zeros_like(dx)
    da, ma = dx * s * g, mx * mag(s) * mag(g)
    sizes = dict(got, scale=mx * m1 * mag(g), gate=mx * m1 * mag(s), post_weight=ma * o1, post_bias=ma)
    if pre_norm and dz is not None:
        sizes["pre_weight"] = dz.abs() * o2
    got.update(scale=dx * a * g, gate=dx * a * s, post_weight=da * n1, post_bias=da)
    w = 1.0 if w1 is None else w1
    C = x.shape[-1]
    out = {"x": dx, "size_x": mx}
    out["h"], out["size_h"] = back(n1, r1, da * w, ma * mag(w)) if post_norm else (da * w, ma * mag(w))
    for name, t in got.items():
        if name != "gate":
            out[name] = t.reshape(-1, C).sum(0)
            out["size_" + name] = sizes[name].abs().reshape(-1, C).sum(0)
    if gate is not None:
        out["gate"] = torch.zeros(gate.shape, dtype=torch.float64) + got["gate"].sum_to_size(gate.shape)
        out["size_gate"] = sizes["gate"].sum_to_size(gate.shape)
    return y, z, out
