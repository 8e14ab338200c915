"""The operators of the network in front of the determinants, as a user's program calls them:
the relative position bias by distance buckets, attention with that bias, its step of one
token over a paged cache (autoregressive sampling), and the norms around a block fused with
its gate and residual scale.

A case names the operator ("op"), the element type ("dtype"), whether gradients are taken
("grad") and the sizes. Without ``own`` the operators run in their plain form, elementary
torch operations in 32 bits (64 for float64 inputs), rounded once at the end.
"""

import math

import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ the cases


def _bias(name=None, **c):
    case = {"op": "relative_bias", "dtype": "f32", "grad": True, "B": 1, "H": 1, "Q": 128, "K": 128, "buckets": 32, "distance": 128}
    return {**({"name": name} if name else {}), **case, **c}


def _attention(name=None, **c):
    case = {
        "op": "attention", "dtype": "bf16", "grad": True, "B": 1, "N": 128, "K": 128, "H": 8, "Hkv": 8, "D": 64, "causal": False,
        "positions": False, "ragged": False, "masked": False, "buckets": 32, "distance": 128,
    }
    return {**({"name": name} if name else {}), **case, **c}


def _step(name=None, **c):
    case = {"op": "attention_step", "dtype": "bf16", "B": 1, "H": 8, "Hkv": 8, "D": 64, "longest": 128, "page": 16, "buckets": 32, "distance": 128}
    return {**({"name": name} if name else {}), **case, **c}


def _norm(name=None, **c):
    case = {"op": "residual_norm", "dtype": "bf16", "grad": True, "B": 1, "N": 128, "C": 512, "norm": "rms", "gate": "sample"}
    return {**({"name": name} if name else {}), **case, **c}


def listed():
    return [
        # pairing functions of the electrons' distance, on their way into slogpf: the
        # benchmark's batch and order, each walker with its own positions
        _bias("bias_walkers_4096x128", B=4096, H=1, Q=128, K=128),
        # one dense bias for all samples of a long chain of sites, in double precision
        _bias("bias_chain_f64_2048", dtype="f64", H=8, Q=2048, K=2048, distance=512),
        # values for a few walkers of a small system: one call's latency
        _attention("attn_values_f32_16x12", dtype="f32", grad=False, B=16, N=12, K=12, H=4, Hkv=4, D=16),
        # training on the benchmark's order, all walkers of one batch
        _attention("attn_train_1024x128", B=1024, N=128, K=128),
        # training in float32: electrons with positions of their own, shared heads, padded samples
        _attention("attn_train_f32_48x302", dtype="f32", B=48, N=302, K=302, H=6, Hkv=2, D=40, positions=True, ragged=True, masked=True),
        # training on long chains, causal, heads shared by four
        _attention("attn_train_causal_2x8192", B=2, N=8192, K=8192, H=16, Hkv=4, D=128, causal=True),
        # sampling: one step of all walkers of the benchmark's batch, part of the way through
        _step("step_walkers_4096x128", B=4096, D=32, longest=128, page=16),
        # sampling a few long sequences, heads shared by four
        _step("step_long_4x65536", B=4, H=32, Hkv=8, D=128, longest=65536, page=64),
        # float32, ragged, an odd page size, heads shared by three
        _step("step_f32_48x2000", dtype="f32", B=48, H=6, Hkv=2, D=64, longest=2000, page=24),
        # values for a few walkers of a small system: one call's latency
        _norm("norm_values_f32_16x12", dtype="f32", grad=False, B=16, N=12, C=64, gate="none"),
        # training on the benchmark's batch and order, the gate from the sample's condition
        _norm("norm_train_4096x128", B=4096, N=128, C=512),
        # training in float32, layer norm, a gate per element, an odd width
        _norm("norm_train_f32_2000x90", dtype="f32", B=2000, N=90, C=333, norm="layer", gate="full"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("relative_bias", "attention", "attention", "attention_step", "residual_norm"))
    buckets, distance = rng.choice(((32, 128), (16, 64), (32, 512), (20, 100)))
    if op == "relative_bias":
        Q, H = _log_int(rng, 12, 2048), rng.choice((1, 2, 3, 8))
        K = rng.choice((Q, _log_int(rng, 12, 2048)))
        dtype = rng.choice(("f32", "f32", "f64", "bf16", "f16"))
        most = 2**26 // (H * Q * K)
        B = _log_int(rng, 1, max(1, min(4096, most)))
        return _bias(dtype=dtype, grad=rng.random() < 0.7, B=B, H=H, Q=Q, K=K, buckets=buckets, distance=distance)
    if op == "attention":
        grad, dtype = rng.random() < 0.7, rng.choice(("bf16", "f16", "f32"))
        Hkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 3, 4))
        D, N = rng.choice((16, 32, 40, 64, 80, 128)), _log_int(rng, 1, 4096)
        causal = rng.random() < 0.4
        K = N if rng.random() < 0.7 else N + _log_int(rng, 1, 1000)
        B = _log_int(rng, 1, max(1, min(1024, int(1.2e8 / (Hkv * group * N * K)), int(1.3e8 / (Hkv * group * N * D)))))
        c = {"positions": not causal and rng.random() < 0.4, "ragged": rng.random() < 0.5, "masked": rng.random() < 0.3}
        return _attention(
            dtype=dtype, grad=grad, B=B, N=N, K=K, H=Hkv * group, Hkv=Hkv, D=D, causal=causal, buckets=buckets, distance=distance, **c
        )
    if op == "attention_step":
        dtype = rng.choice(("bf16", "f16", "f32"))
        Hkv, group, D = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8)), rng.choice((16, 32, 64, 80, 128))
        longest, page = _log_int(rng, 1, 65536), rng.choice((8, 16, 24, 64, 100))
        B = _log_int(rng, 1, max(1, min(4096, int(2.6e8 / (Hkv * D * (longest + page))))))
        return _step(
            dtype=dtype, B=B, H=Hkv * group, Hkv=Hkv, D=D, longest=longest, page=page, buckets=buckets, distance=distance
        )
    C, N = _log_int(rng, 16, 8192), _log_int(rng, 1, 512)
    B = _log_int(rng, 1, max(1, min(4096, 2**27 // (C * N))))
    return _norm(
        dtype=rng.choice(("bf16", "f16", "f32")), grad=rng.random() < 0.7, B=B, N=N, C=C, norm=rng.choice(("rms", "layer")),
        gate=rng.choice(("none", "channel", "token", "sample", "full")),
    )


# ------------------------------------------------------------------ inputs


def _bucket_map(buckets, distance):
    """Bucket of each distance -distance .. distance: half the buckets for either sign, of
    which half hold one distance each and the others grow by a constant factor. The limits
    are found in whole numbers."""
    half = buckets // 2
    single = half // 2
    row = []
    for n in range(distance + 1):
        b = n
        if n >= single:
            b = single  # the largest bucket whose lower end, single (distance / single)^(t / (half - single)), is at most n
            while b + 1 < half and n ** (half - single) >= single ** (half - b - 1) * distance ** (b + 1 - single):
                b += 1
        row.append(b)
    return [row[-d] for d in range(-distance, 0)] + [row[0]] + [half + row[d] for d in range(1, distance + 1)]


def _map(case):
    m = _bucket_map(case["buckets"], case["distance"])
    return torch.tensor(m, dtype=torch.uint8, device="cuda")


def _sites(gen, shape, sites):
    """Sites that the electrons of each sample occupy, in order."""
    return torch.randint(0, sites, shape, generator=gen, device="cuda").sort(-1).values.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        return (torch.randn(shape, generator=gen, device="cuda", dtype=wide) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "relative_bias":
        B, H, Q, K = (case[k] for k in "BHQK")
        s["table"] = normal(case["buckets"], H)
        s["buckets"] = _map(case)
        if B > 1:
            s["q_pos"], s["k_pos"] = _sites(gen, (B, Q), 2 * Q), _sites(gen, (B, K), 2 * Q)
        else:
            s["q_pos"] = torch.arange(Q, device="cuda", dtype=torch.int32)
            s["k_pos"] = torch.arange(K, device="cuda", dtype=torch.int32)
        s["leaves"] = ["table"]
        s["cotangents"] = (normal(*((B,) if B > 1 else ()), H, Q, K),) if case["grad"] else ()
    elif case["op"] == "attention":
        B, N, K, H, Hkv, D = (case[k] for k in ("B", "N", "K", "H", "Hkv", "D"))
        s["q"], s["k"], s["v"] = normal(B, N, H, D), normal(B, K, Hkv, D), normal(B, K, Hkv, D)
        s["table"] = normal(case["buckets"], H, dtype=torch.float32)
        s["buckets"] = _map(case)
        s["kw"] = {"causal": case["causal"], "offset": K - N if case["causal"] else 0}
        if case["positions"]:
            s["kw"]["q_pos"], s["kw"]["k_pos"] = _sites(gen, (B, N), 2 * N), _sites(gen, (B, K), 2 * N)
        if case["ragged"]:
            s["kw"]["lengths"] = torch.randint(0, K + 1, (B,), generator=gen, device="cuda").to(torch.int32)
        if case["masked"]:
            s["kw"]["mask"] = torch.rand((B, K), generator=gen, device="cuda") < 0.9
        s["leaves"] = ["q", "k", "v", "table"]
        s["cotangents"] = (normal(B, N, H, D),) if case["grad"] else ()
    elif case["op"] == "attention_step":
        B, H, Hkv, D, page = (case[k] for k in ("B", "H", "Hkv", "D", "page"))
        M = case["longest"] // page + 1
        s["q"], s["k"], s["v"] = normal(B, H, D), normal(B, Hkv, D), normal(B, Hkv, D)
        s["k_cache"], s["v_cache"] = normal(B * M, page, Hkv, D), normal(B * M, page, Hkv, D)
        s["pages"] = torch.randperm(B * M, generator=gen, device="cuda").reshape(B, M).to(torch.int32)
        # samples are anywhere in their last half; every 16th has only begun
        lengths = torch.randint(case["longest"] // 2, case["longest"] + 1, (B,), generator=gen, device="cuda")
        s["lengths"] = torch.where(torch.arange(B, device="cuda") % 16 == 15, 0, lengths).to(torch.int32)
        s["table"] = normal(case["buckets"], H, dtype=torch.float32)
        s["buckets"] = _map(case)
        s["leaves"] = []
        s["cotangents"] = ()
    else:
        B, N, C = case["B"], case["N"], case["C"]
        s["x"], s["h"] = normal(B, N, C), normal(B, N, C, scale=2.0)
        s["post_weight"], s["pre_weight"] = 1 + normal(C, scale=0.1, dtype=torch.float32), 1 + normal(C, scale=0.1, dtype=torch.float32)
        s["scale"] = 0.5 + normal(C, scale=0.1, dtype=torch.float32)
        s["leaves"] = ["x", "h", "post_weight", "pre_weight", "scale"]
        shape = {"none": None, "channel": (C,), "token": (B, N, 1), "sample": (B, 1, C), "full": (B, N, C)}[case["gate"]]
        s["gate"] = None if shape is None else normal(*shape)
        if shape is not None:
            s["leaves"].append("gate")
        s["post_bias"] = s["pre_bias"] = None
        if case["norm"] == "layer":
            s["post_bias"], s["pre_bias"] = normal(C, scale=0.1, dtype=torch.float32), normal(C, scale=0.1, dtype=torch.float32)
            s["leaves"] += ["post_bias", "pre_bias"]
        s["cotangents"] = (normal(B, N, C), normal(B, N, C)) if case["grad"] else ()
    if s["cotangents"]:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------ the framework's calls


def _own(s):
    import fermix_amd

    op = s["case"]["op"]
    if op == "relative_bias":
        outs = (fermix_amd.relative_bias(s["table"], s["buckets"], s["q_pos"], s["k_pos"]),)
    elif op == "attention":
        outs = (fermix_amd.attention(s["q"], s["k"], s["v"], table=s["table"], buckets=s["buckets"], **s["kw"]),)
    elif op == "attention_step":
        out = fermix_amd.attention_step(
            s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], k=s["k"], v=s["v"], table=s["table"], buckets=s["buckets"]
        )
        return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    else:
        outs = fermix_amd.residual_norm(
            s["x"], s["h"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], scale=s["scale"],
            pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], norm=s["case"]["norm"],
        )
    got = {"out%d" % i: o.detach() for i, o in enumerate(outs)}
    if s["cotangents"]:
        grads = torch.autograd.grad(outs, [s[k] for k in s["leaves"]], s["cotangents"])
        got.update(("d_" + k, g) for k, g in zip(s["leaves"], grads))
    return got


# ------------------------------------------------------------------ the plain forms


def _bucket_of(buckets, q_pos, k_pos):
    """(.., Q, K) bucket of each pair."""
    R = buckets.numel() // 2
    d = k_pos[..., None, :] - q_pos[..., :, None]
    return buckets.long()[d.clamp(-R, R).long() + R]


def _bucket_sums(d, bucket, count):
    """Sums of d (B, H, Q, K) over the pairs in each bucket (B or 1, Q, K): (count, H). A
    product with the buckets' indicator, the samples that share their positions summed first."""
    if bucket.shape[0] == 1:
        d = d.sum(0, keepdim=True)
    ids = torch.arange(count, device=d.device)
    hot = (bucket[..., None] == ids).to(d.dtype)
    return torch.matmul(d.transpose(1, 2).contiguous(), hot).sum((0, 1)).t().contiguous()


def _plain_bias(s):
    wide = torch.float64 if s["table"].dtype == torch.float64 else torch.float32
    bucket = _bucket_of(s["buckets"], s["q_pos"], s["k_pos"])
    table = s["table"].detach()
    got = {"out0": table.to(wide)[bucket].movedim(-1, -3).contiguous().to(table.dtype)}
    if s["cotangents"]:
        (g,) = s["cotangents"]
        Q, K = g.shape[-2:]
        d = _bucket_sums(g.to(wide).reshape(-1, g.shape[-3], Q, K), bucket.reshape(-1, Q, K), table.shape[0])
        got["d_table"] = d.to(table.dtype)
    return got


def _plain_attention(s):
    c, kw = s["case"], s["kw"]
    B, N, K, H, Hkv, D = (c[k] for k in ("B", "N", "K", "H", "Hkv", "D"))
    group = H // Hkv
    q, k, v = (s[n].detach().float().transpose(1, 2) for n in "qkv")
    keys = torch.arange(K, device="cuda")
    rows = torch.arange(N, device="cuda") + kw["offset"]
    left = torch.ones((1, 1, 1, 1), dtype=torch.bool, device="cuda")
    if "lengths" in kw:
        left = left & (keys < kw["lengths"][:, None])[:, None, None]
    if "mask" in kw:
        left = left & kw["mask"][:, None, None]
    if c["causal"]:
        left = left & (keys <= rows[:, None])
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    bucket = _bucket_of(s["buckets"], kw["q_pos"], kw["k_pos"]) if "q_pos" in kw else _bucket_of(s["buckets"], rows, keys)[None]
    scale = 1.0 / math.sqrt(D)
    S = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    S += s["table"].detach()[bucket].movedim(-1, 1)
    S.masked_fill_(~left, -math.inf)
    top = S.amax(-1, keepdim=True)
    P = (S - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = P.sum(-1, keepdim=True)
    P /= torch.where(total == 0, 1.0, total)
    out = torch.matmul(P, v).transpose(1, 2).contiguous()
    got = {"out0": out.to(s["q"].dtype)}
    if s["cotangents"]:
        g = s["cotangents"][0].float().transpose(1, 2).contiguous()
        dP = torch.matmul(g, v.transpose(2, 3).contiguous())
        dS = P * (dP - (P * dP).sum(-1, keepdim=True))
        dv = torch.matmul(P.transpose(2, 3).contiguous(), g)
        dq = torch.matmul(dS, k) * scale
        dk = torch.matmul(dS.transpose(2, 3).contiguous(), q) * scale
        dk, dv = (t.reshape(B, Hkv, group, K, D).sum(2) for t in (dk, dv))
        for n, t in (("q", dq), ("k", dk), ("v", dv)):
            got["d_" + n] = t.transpose(1, 2).contiguous().to(s[n].dtype)
        got["d_table"] = _bucket_sums(dS, bucket, s["table"].shape[0])
    return got


def _plain_step(s):
    c = s["case"]
    B, H, Hkv, D, page = (c[k] for k in ("B", "H", "Hkv", "D", "page"))
    pages, lengths = s["pages"].long(), s["lengths"].long()
    at = pages.gather(1, (lengths // page)[:, None])[:, 0]
    s["k_cache"][at, lengths % page] = s["k"]
    s["v_cache"][at, lengths % page] = s["v"]
    k, v = (s[n][pages].reshape(B, -1, Hkv, D).float().transpose(1, 2) for n in ("k_cache", "v_cache"))
    keys = torch.arange(k.shape[2], device="cuda")
    q = s["q"].float().reshape(B, Hkv, H // Hkv, D)
    S = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    bucket = _bucket_of(s["buckets"], lengths[:, None], keys.expand(B, -1))[:, 0]
    S += s["table"][bucket].movedim(-1, 1).reshape(S.shape)
    S.masked_fill_((keys > lengths[:, None])[:, None, None], -math.inf)
    P = (S - S.amax(-1, keepdim=True)).exp_()
    P /= P.sum(-1, keepdim=True)
    out = torch.matmul(P, v.contiguous()).reshape(B, H, D)
    return {"out": out.to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


EPS = 1e-6


def _normed(x, layer):
    """x centred (layer) and divided by its deviation, and that divisor's reciprocal."""
    if layer:
        x = x - x.mean(-1, keepdim=True)
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return x * r, r


def _normed_grad(n, r, dn, layer):
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    if layer:
        d -= dn.mean(-1, keepdim=True)
    return r * d


def _plain_norm(s):
    layer, dt = s["case"]["norm"] == "layer", s["x"].dtype
    x, h = s["x"].detach().float(), s["h"].detach().float()
    w, b, pw, pb, scale, gate = (
        None if s[n] is None else s[n].detach().float() for n in ("post_weight", "post_bias", "pre_weight", "pre_bias", "scale", "gate")
    )
    n1, r1 = _normed(h, layer)
    a = n1 * w if b is None else n1 * w + b
    u = scale if gate is None else scale * gate
    y = x + u * a
    n2, r2 = _normed(y, layer)
    z = n2 * pw if pb is None else n2 * pw + pb
    got = {"out0": y.to(dt), "out1": z.to(dt)}
    if s["cotangents"]:
        dy, dz = (t.float() for t in s["cotangents"])
        rows = (0, 1)
        dx = dy + _normed_grad(n2, r2, dz * pw, layer)
        da = dx * u
        got["d_x"] = dx.to(dt)
        got["d_h"] = _normed_grad(n1, r1, da * w, layer).to(dt)
        got["d_post_weight"] = (da * n1).sum(rows)
        got["d_pre_weight"] = (dz * n2).sum(rows)
        du = dx * a
        got["d_scale"] = (du if gate is None else du * gate).sum(rows)
        if gate is not None:
            dg = du * scale
            kept = [i for i in range(3) if (1,) * (3 - gate.dim()) + gate.shape != dg.shape and ((1,) * (3 - gate.dim()) + gate.shape)[i] == 1]
            got["d_gate"] = (dg.sum(kept, keepdim=True) if kept else dg).reshape(gate.shape).to(dt)
        if layer:
            got["d_post_bias"] = da.sum(rows)
            got["d_pre_bias"] = dz.sum(rows)
    return got


_PLAIN = {"relative_bias": _plain_bias, "attention": _plain_attention, "attention_step": _plain_step, "residual_norm": _plain_norm}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    e, train = SIZE[case["dtype"]], case.get("grad", False)
    if case["op"] == "relative_bias":
        pairs = case["B"] * case["H"] * case["Q"] * case["K"]
        return {"bytes": pairs * e * (2 if train else 1), "flops": pairs if train else 0}
    if case["op"] == "attention":
        B, N, K, H, Hkv, D = (case[k] for k in ("B", "N", "K", "H", "Hkv", "D"))
        pairs = N * (K - (N - 1) / 2) if case["causal"] else N * K
        if case["ragged"]:
            pairs /= 2  # lengths are spread evenly over 0 .. K
        # q, out; k, v; in training the cotangent and three gradients besides
        tensors = B * N * H * D * (4 if train else 2) + B * K * Hkv * D * (4 if train else 2)
        return {"bytes": tensors * e, "flops": B * H * pairs * D * (14 if train else 4)}
    if case["op"] == "attention_step":
        B, H, Hkv, D = (case[k] for k in ("B", "H", "Hkv", "D"))
        tokens = 1 + (B - B // 16) * (0.75 * case["longest"] + 1)
        return {"bytes": 2 * e * D * (Hkv * tokens + B * (H + Hkv)), "flops": 4 * H * D * tokens}
    elements = case["B"] * case["N"] * case["C"]
    gate = {"none": 0, "channel": 0, "token": case["B"] * case["N"], "sample": case["B"] * case["C"], "full": elements}[case["gate"]]
    # x, h, y, z; in training two cotangents and two gradients besides
    return {"bytes": e * (elements * (8 if train else 4) + gate * (2 if train else 1)), "flops": elements * (50 if train else 15)}


# ------------------------------------------------------------------ 64 bits, from the definitions


def _exact_map(buckets, R, pairs):
    return torch.take(buckets.to(torch.int64), torch.clip(pairs.to(torch.int64), -R, R) + R)


def _exact_bias(s):
    R, table = s["buckets"].numel() // 2, s["table"].detach().double()
    lead = s["q_pos"].shape[:-1]
    q, k = (p.long().reshape(-1, p.shape[-1]) for p in (s["q_pos"], s["k_pos"]))
    outs, grad = [], torch.zeros_like(table)
    g = s["cotangents"][0].reshape(-1, *s["cotangents"][0].shape[-3:]) if s["cotangents"] else None
    step = max(1, 2**25 // (q.shape[1] * k.shape[1] * table.shape[1]))
    for at in range(0, len(q), step):
        which = _exact_map(s["buckets"], R, k[at : at + step, None, :] - q[at : at + step, :, None])
        # one head at a time: the table's column laid out over the pairs
        for b in range(table.shape[1]) if g is not None else ():
            grad[:, b] += torch.bincount(which.flatten(), g[at : at + step, b].double().flatten(), minlength=len(table))
        outs.append(torch.stack([torch.take(col, which) for col in table.unbind(1)], 1))
    out = torch.cat(outs)
    return {"out0": out.reshape(*lead, *out.shape[1:])} | ({"d_table": grad} if g is not None else {})


def _exact_attention(s):
    """Each sample's shared heads by themselves through torch's own differentiation of the
    definition."""
    c, kw = s["case"], s["kw"]
    B, N, K, H, Hkv, D = (c[k] for k in ("B", "N", "K", "H", "Hkv", "D"))
    group, R = H // Hkv, s["buckets"].numel() // 2
    rows, keys = torch.arange(N, device="cuda") + kw["offset"], torch.arange(K, device="cuda")
    table = s["table"].detach().double()
    names = ["out0"] + (["d_q", "d_k", "d_v"] if s["cotangents"] else [])
    parts = {n: [] for n in names}
    d_table = torch.zeros_like(table)
    step = max(1, 2**26 // (N * K * H))
    for at in range(0, B, step):
        b = slice(at, at + step)
        heads = []
        for j in range(Hkv) if N * K * H > 2**27 else (slice(None),):
            j = slice(j, j + 1) if isinstance(j, int) else j
            n = len(range(Hkv)[j])
            hs = slice((j.start or 0) * group, (j.start or 0) * group + n * group)
            q = s["q"].detach()[b, :, hs].double().reshape(-1, N, n, group, D).permute(0, 2, 3, 1, 4).contiguous().requires_grad_(True)
            k, v = (s[t].detach()[b, :, j].double().permute(0, 2, 1, 3).unsqueeze(2).contiguous().requires_grad_(True) for t in "kv")
            if "q_pos" in kw:
                which = _exact_map(s["buckets"], R, kw["k_pos"][b].long()[:, None, :] - kw["q_pos"][b].long()[:, :, None])
            else:
                which = _exact_map(s["buckets"], R, keys[None, None, :] - rows[None, :, None])
            bias = torch.stack([torch.take(column, which) for column in table[:, hs].unbind(1)], 1)
            bias = bias.reshape(-1, n, group, N, K).expand(len(q), -1, -1, -1, -1).contiguous().requires_grad_(True)
            allowed = torch.ones((len(q), 1, 1, N, K), dtype=torch.bool, device="cuda")
            if "lengths" in kw:
                allowed &= (keys[None] < kw["lengths"][b].long()[:, None])[:, None, None, None]
            if "mask" in kw:
                allowed &= kw["mask"][b][:, None, None, None]
            if c["causal"]:
                allowed &= (rows[:, None] >= keys[None])[None, None, None]
            # a finite stand-in for what is left out, so that rows without a key differentiate to zero
            weight = torch.softmax(torch.where(allowed, torch.matmul(q, k.transpose(3, 4)) / math.sqrt(D) + bias, -1e300), -1) * allowed
            out = torch.matmul(weight, v)
            got = [out.detach()]
            if s["cotangents"]:
                g = s["cotangents"][0][b, :, hs].double().reshape(-1, N, n, group, D).permute(0, 2, 3, 1, 4)
                *grads, db = torch.autograd.grad(out, [q, k, v, bias], g)
                got += grads
                for i in range(len(table)):
                    d_table[i, hs] += torch.where((which == i)[:, None, None], db, 0.0).sum((0, 3, 4)).flatten()
                del db, grads
            del out, weight, bias
            heads.append([t.permute(0, 3, 1, 2, 4).reshape(len(t), t.shape[3], -1, D) for t in got])
        for name, *t in zip(names, *heads):
            parts[name].append(torch.cat(t, 2))
    got = {n: torch.cat(t) for n, t in parts.items()}
    return got | ({"d_table": d_table} if s["cotangents"] else {})


def _exact_step(s):
    """Sample by sample over its own tokens."""
    c = s["case"]
    page, R, group = c["page"], s["buckets"].numel() // 2, c["H"] // c["Hkv"]
    outs, k_cache, v_cache = [], s["k_cache"].double(), s["v_cache"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        own_pages = s["pages"][b, : n // page + 1].long()
        k_cache[own_pages[-1], n % page] = s["k"][b].double()
        v_cache[own_pages[-1], n % page] = s["v"][b].double()
        k, v = (t[own_pages].flatten(0, 1)[: n + 1].repeat_interleave(group, 1) for t in (k_cache, v_cache))
        which = _exact_map(s["buckets"], R, torch.arange(-n, 1, device="cuda"))
        score = (k * s["q"][b].double()).sum(-1) / math.sqrt(c["D"]) + s["table"].double()[which]
        outs.append((torch.softmax(score, 0)[..., None] * v).sum(0))
    return {"out": torch.stack(outs), "k_cache": k_cache, "v_cache": v_cache}


def _exact_norm(s):
    """The composition of the definitions, differentiated by torch, in parts of the batch."""
    names = ("x", "h", "post_weight", "post_bias", "pre_weight", "pre_bias", "scale", "gate")
    whole = {n: None if s[n] is None else s[n].detach() for n in names}
    B, layer = s["case"]["B"], s["case"]["norm"] == "layer"
    ys, zs, grads = [], [], {}

    def norm(t, w, b):
        mean = t.mean(-1, keepdim=True) if layer else 0.0
        t = (t - mean) / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + EPS)
        return t * w + (0.0 if b is None else b)

    step = max(1, 2**27 // (s["case"]["N"] * s["case"]["C"]))
    for at in range(0, B, step):
        t = {}
        for n, x in whole.items():
            split = x is not None and x.dim() == 3
            t[n] = None if x is None else (x[at : at + step] if split else x).double().requires_grad_(bool(s["cotangents"]))
        branch = t["scale"] * norm(t["h"], t["post_weight"], t["post_bias"])
        y = t["x"] + (branch if t["gate"] is None else t["gate"] * branch)
        z = norm(y, t["pre_weight"], t["pre_bias"])
        ys.append(y.detach())
        zs.append(z.detach())
        if s["cotangents"]:
            cots = [g[at : at + step].double() for g in s["cotangents"]]
            for n, g in zip(s["leaves"], torch.autograd.grad((y, z), [t[n] for n in s["leaves"]], cots)):
                grads.setdefault(n, []).append(g)
    got = {"out0": torch.cat(ys), "out1": torch.cat(zs)}
    for n, parts in grads.items():
        got["d_" + n] = torch.cat(parts) if parts[0].dim() == 3 else torch.stack(parts).sum(0)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    f = {"relative_bias": _exact_bias, "attention": _exact_attention, "attention_step": _exact_step, "residual_norm": _exact_norm}
    return f[case["op"]](s)
