"""Cases of the attention-input and optimizer operators, in plain form and through the package.

Operators: the per-head norm of queries and keys with the position rotation ("qk"), the learned
relative position bias by buckets ("distance" and "grid"), and the Newton-Schulz
orthogonalisation alone ("orthogonalize") and inside the optimizer step ("muon").

`run(state)` makes one pass; with `own` set it calls the package, otherwise it evaluates the same
formulas with elementary torch operations.  `exact` evaluates the definitions in 64 bits.
"""

import math

import torch

own = False

NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
NS_STEPS = 5
MOMENTUM, LR, WEIGHT_DECAY = 0.95, 1e-3, 0.1
NORM_EPS = 1e-6
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One new token of each of 16 sequences at far positions, grouped key heads: latency.
        dict(name="qk decode", op="qk", batch=16, tokens=1, q_heads=32, k_heads=8, head_dim=128,
             rot_dim=128, interleaved=False, packed=False, positions=True, dtype="bf16",
             backward=False),
        # The attention block of the ViT-B/16 training step: packed qkv, batch 128, 197 tokens.
        dict(name="qk vit train", op="qk", batch=128, tokens=197, q_heads=12, k_heads=12,
             head_dim=64, rot_dim=64, interleaved=False, packed=True, positions=False,
             dtype="bf16", backward=True),
        # A long sequence of odd length with grouped key heads, forward and backward.
        dict(name="qk long train", op="qk", batch=2, tokens=8191, q_heads=32, k_heads=8,
             head_dim=128, rot_dim=128, interleaved=False, packed=False, positions=False,
             dtype="bf16", backward=True),
        # Neighbouring pairs, part of the head rotated, a head size that is no power of two.
        dict(name="qk odd partial", op="qk", batch=3, tokens=1021, q_heads=6, k_heads=2,
             head_dim=80, rot_dim=48, interleaved=True, packed=False, positions=True,
             dtype="fp16", backward=True),
        # One query over a long key range, as a decoder asks for it.
        dict(name="distance one query", op="distance", heads=16, lq=1, lk=4097, offset=4096,
             buckets=32, max_distance=128, causal=True, dtype="bf16", backward=False),
        # A long training sequence, both directions of distance, with the table's gradient.
        dict(name="distance long train", op="distance", heads=16, lq=4096, lk=4096, offset=0,
             buckets=32, max_distance=128, causal=False, dtype="bf16", backward=True),
        # The 14 x 14 patch grid and class token of the ViT-B/16 blocks.
        dict(name="grid vit train", op="grid", heads=12, rows=14, cols=14, prefix=1,
             dtype="bf16", backward=True),
        # A 512 x 512 image's patch grid, 32-bit bias.
        dict(name="grid large train", op="grid", heads=16, rows=32, cols=32, prefix=1,
             dtype="fp32", backward=True),
        # One projection's update.
        dict(name="orthogonalize one", op="orthogonalize", count=1, rows=768, cols=768,
             dtype="bf16"),
        # The attention projections of all twelve ViT-B/16 blocks, 32-bit weights.
        dict(name="muon vit proj", op="muon", count=12, rows=768, cols=768, dtype="fp32"),
        # The qkv weights of the same blocks, 16-bit weights.
        dict(name="muon vit qkv", op="muon", count=12, rows=2304, cols=768, dtype="bf16"),
        # Odd sizes, as patch embeddings and heads have them.
        dict(name="muon odd", op="muon", count=3, rows=197, cols=1000, dtype="fp32"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["qk", "qk", "distance", "grid", "orthogonalize", "muon"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "qk":
        head_dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        k_heads = rng.choice([1, 2, 3, 4, 8, 12])
        q_heads = k_heads * rng.choice([1, 1, 2, 4])
        width = (q_heads + k_heads) * head_dim
        backward = rng.random() < 0.6
        total = _log_int(rng, 1, max(1, 60_000_000 // width))
        batch = _log_int(rng, 1, min(128, total))
        rot = head_dim if rng.random() < 0.6 else 2 * rng.randint(1, head_dim // 2)
        return dict(op="qk", batch=batch, tokens=max(1, total // batch), q_heads=q_heads,
                    k_heads=k_heads, head_dim=head_dim, rot_dim=rot,
                    interleaved=rng.random() < 0.4, packed=rng.random() < 0.4,
                    positions=rng.random() < 0.5, dtype=dtype, backward=backward)
    if op == "distance":
        heads = rng.choice([1, 4, 8, 12, 16])
        lk = _log_int(rng, 1, 4000)
        lq = 1 if rng.random() < 0.3 else _log_int(rng, 1, 4000)
        causal = rng.random() < 0.5
        buckets = rng.choice([8, 32, 64])
        return dict(op="distance", heads=heads, lq=lq, lk=lk,
                    offset=lk - lq if rng.random() < 0.5 else rng.randint(-5, 5),
                    buckets=buckets, max_distance=rng.choice([buckets * 2, 128, 500]),
                    causal=causal, dtype=dtype, backward=rng.random() < 0.6)
    if op == "grid":
        return dict(op="grid", heads=rng.choice([3, 6, 12, 16]), rows=_log_int(rng, 1, 32),
                    cols=_log_int(rng, 2, 32), prefix=rng.choice([0, 1, 5]), dtype=dtype,
                    backward=rng.random() < 0.6)
    count, rows, cols = rng.choice([1, 2, 3, 6]), _log_int(rng, 8, 1500), _log_int(rng, 8, 1500)
    if op == "orthogonalize":
        return dict(op=op, count=count, rows=rows, cols=cols, dtype=rng.choice(["bf16", "fp16"]))
    return dict(op=op, count=count, rows=rows, cols=cols, dtype=rng.choice(["bf16", "fp32"]))


def work(case):
    op = case["op"]
    if op == "qk":
        rows = case["batch"] * case["tokens"]
        size = 4 if case["dtype"] == "fp32" else 2
        qk = rows * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        v = rows * case["k_heads"] * case["head_dim"] if case["packed"] else 0
        # the table rows in use, or one row a token where positions pick them
        tables = case["tokens"] * (case["batch"] if case["positions"] else 1) * case["rot_dim"] * 4
        passes = 5 if case["backward"] else 2
        moved = passes * qk * size + tables * (2 if case["backward"] else 1)
        if case["backward"]:
            moved += 2 * v * size  # dv into the packed gradient
        return {"bytes": moved, "flops": qk * (18 if case["backward"] else 7)}
    if op in ("distance", "grid"):
        size = 4 if case["dtype"] == "fp32" else 2
        if op == "distance":
            cells, index = case["lq"] * case["lk"], 0
        else:
            cells = (case["rows"] * case["cols"] + case["prefix"]) ** 2
            index = 4 * cells
        n = case["heads"] * cells
        both = 2 if case["backward"] else 1
        return {"bytes": both * (n * size + index), "flops": n if case["backward"] else 0}
    m, n = sorted((case["rows"], case["cols"]))
    # Symmetric products count by halves; iterating on the m x m Gram matrix alone costs less
    # where the matrix is wide.
    direct = NS_STEPS * (3 * m * m * n + m ** 3)
    gram = 3 * m * m * n + (4 * NS_STEPS - 3) * m ** 3
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "orthogonalize":
        moved = 2 * size * m * n
    else:
        moved = (3 * size + 8) * m * n  # read w, g, momentum; write w, momentum
    return {"bytes": case["count"] * moved, "flops": case["count"] * min(direct, gram)}


# ---------------------------------------------------------------------------------- inputs


def _bucket_borders(buckets, max_distance):
    """Distances at which the log-spaced half of the buckets begins, from integers alone.

    The first half of the buckets holds one distance each; bucket half + k starts at the least n
    with (n / half) ** rest >= (max_distance / half) ** k."""
    half = buckets // 2
    rest = buckets - half
    found, n = [], half
    for k in range(rest):
        while n ** rest * half ** k < max_distance ** k * half ** rest:
            n += 1
        found.append(n)
    return found


def _grid_index(rows, cols, prefix):
    """Bucket of each pair of tokens: one for each (dy, dx) of two patches, then one each for
    prefix to patch, patch to prefix and prefix to prefix."""
    y = torch.arange(rows).repeat_interleave(cols)
    x = torch.arange(cols).repeat(rows)
    dy = y[:, None] - y[None, :] + rows - 1
    dx = x[:, None] - x[None, :] + cols - 1
    pairs = (2 * rows - 1) * (2 * cols - 1)
    n = rows * cols + prefix
    index = torch.empty(n, n, dtype=torch.int64)
    index[prefix:, prefix:] = dy * (2 * cols - 1) + dx
    index[:prefix, prefix:] = pairs
    index[prefix:, :prefix] = pairs + 1
    index[:prefix, :prefix] = pairs + 2
    return index, pairs + (3 if prefix else 0)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "qk":
        B, L, Hq, Hk, D = (case[k] for k in ("batch", "tokens", "q_heads", "k_heads", "head_dim"))
        back = case["backward"]
        span = 32768 if case["positions"] else L
        freq = 10000.0 ** (-torch.arange(case["rot_dim"] // 2, device=dev, dtype=torch.float64)
                           * 2 / case["rot_dim"])
        angle = torch.arange(span, device=dev, dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = None
        if case["positions"]:
            start = torch.randint(0, span - L + 1, (B, 1), generator=gen, device=dev)
            s["positions"] = start + torch.arange(L, device=dev)
        s["wq"] = (1 + normal(D, scale=0.1)).requires_grad_(back)
        s["wk"] = (1 + normal(D, scale=0.1)).requires_grad_(back)
        if case["packed"]:
            s["qkv"] = normal(B, L, (Hq + 2 * Hk) * D, dtype=dtype).requires_grad_(back)
        else:
            s["q"] = normal(B, L, Hq, D, dtype=dtype).requires_grad_(back)
            s["k"] = normal(B, L, Hk, D, dtype=dtype).requires_grad_(back)
        if back:
            s["dq"] = normal(B, L, Hq, D, dtype=dtype)
            s["dk"] = normal(B, L, Hk, D, dtype=dtype)
            if case["packed"]:
                s["dv"] = normal(B, L, Hk, D, dtype=dtype)
        return s
    if op in ("distance", "grid"):
        if op == "distance":
            lq, lk, count = case["lq"], case["lk"], case["buckets"]
            side = count if case["causal"] else count // 2
            s["borders"] = torch.tensor(_bucket_borders(side, case["max_distance"]), device=dev)
            if own:
                import rational_kat_cu_b200 as kat

                s["plan"] = kat.DistanceBuckets(count, case["max_distance"],
                                                bidirectional=not case["causal"])
        else:
            index, count = _grid_index(case["rows"], case["cols"], case["prefix"])
            lq = lk = index.shape[0]
            s["index"] = index.to(dev)
            if own:
                import rational_kat_cu_b200 as kat

                s["plan"] = kat.IndexBuckets(s["index"], count)
        s["table"] = normal(count, case["heads"], scale=0.5).requires_grad_(case["backward"])
        if case["backward"]:
            s["dout"] = normal(case["heads"], lq, lk, dtype=dtype, scale=0.1)
        return s
    # Updates as training meets them: a few strong directions above noise.
    shape = (case["rows"], case["cols"])
    rank = max(1, min(shape) // 16)
    make = lambda: (normal(shape[0], rank) @ normal(rank, shape[1], scale=rank ** -0.5)  # noqa: E731
                    + normal(*shape, scale=0.5)) * 1e-4
    s["grads"] = [make().to(dtype) for _ in range(case["count"])]
    if op == "orthogonalize":
        s["grads"] = torch.stack(s["grads"])
    else:
        s["weights"] = [normal(*shape, dtype=dtype, scale=0.02) for _ in range(case["count"])]
        s["momenta"] = [make() * 5 for _ in range(case["count"])]
    return s


# ---------------------------------------------------------------------------------- passes


def run(s):
    op = s["case"]["op"]
    if op == "qk":
        return _qk_own(s) if own else _qk_plain(s)
    if op in ("distance", "grid"):
        return _bias_own(s) if own else _bias_plain(s)
    if op == "orthogonalize":
        if own:
            import rational_kat_cu_b200 as kat

            return kat.orthogonalize(s["grads"], steps=NS_STEPS)
        return _newton_schulz(s["grads"].float()).to(s["grads"].dtype)
    if own:
        import rational_kat_cu_b200 as kat

        kat.muon_step(s["weights"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM,
                      nesterov=True, weight_decay=WEIGHT_DECAY, steps=NS_STEPS)
    else:
        scale = 0.2 * math.sqrt(max(s["case"]["rows"], s["case"]["cols"]))
        grads = torch.stack(s["grads"]).float()
        momenta = torch.stack(s["momenta"]) * MOMENTUM + grads
        ortho = _newton_schulz(grads + MOMENTUM * momenta)
        weights = torch.stack(s["weights"]).float()
        weights = weights * (1 - LR * WEIGHT_DECAY) - LR * scale * ortho
        for i in range(len(s["weights"])):
            s["weights"][i].copy_(weights[i])
            s["momenta"][i].copy_(momenta[i])
    return {"weights": s["weights"], "momenta": s["momenta"]}


def _newton_schulz(u):
    """Five quintic steps on u / |u|_F, on the side with fewer rows; zeros stay zeros."""
    wide = u.shape[-2] <= u.shape[-1]
    x = u if wide else u.transpose(-1, -2)
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = (x.double() / torch.where(norm > 0, norm, 1.0)).float()
    for _ in range(NS_STEPS):
        a = x @ x.transpose(-1, -2)
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    return x if wide else x.transpose(-1, -2)


def _split(s):
    """q and k [B, L, H, D] of the state, and v where it is packed."""
    c = s["case"]
    B, L, Hq, Hk, D = (c[k] for k in ("batch", "tokens", "q_heads", "k_heads", "head_dim"))
    if not c["packed"]:
        return s["q"].detach(), s["k"].detach(), None
    x = s["qkv"].detach().view(B, L, Hq + 2 * Hk, D)
    return x[:, :, :Hq], x[:, :, Hq:Hq + Hk], x[:, :, Hq + Hk:]


def _angles(s):
    c = s["case"]
    if s["positions"] is None:
        return s["cos"][: c["tokens"], None], s["sin"][: c["tokens"], None]
    return s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]


def _turn(x, cos, sin, rot, interleaved):
    """The first `rot` values turned by the angles, pair by pair; the others as they are."""
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = r[..., : rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([r, rest], -1)


def _qk_plain(s):
    c = s["case"]
    q, k, v = _split(s)
    cos, sin = _angles(s)
    rot, inter = c["rot_dim"], c["interleaved"]
    outs, grads, dws = [], [], []
    for x, w, name in ((q, s["wq"].detach(), "dq"), (k, s["wk"].detach(), "dk")):
        f = x.float()
        r = (f * f).mean(-1, keepdim=True).add(NORM_EPS).rsqrt()
        hat = f * r
        outs.append(_turn(hat * w, cos, sin, rot, inter).to(x.dtype))
        if c["backward"]:
            dn = _turn(s[name].float(), cos, -sin, rot, inter)
            dws.append((dn * hat).double().sum((0, 1, 2)).float())
            g = dn * w
            grads.append((r * (g - hat * (g * hat).mean(-1, keepdim=True))).to(x.dtype))
    if not c["backward"]:
        return outs + ([v] if c["packed"] else [])
    if c["packed"]:
        grads = [torch.cat(grads + [s["dv"]], 2).flatten(2)]
        outs.append(v)
    return outs + grads + dws


def _qk_own(s):
    import rational_kat_cu_b200 as kat

    c = s["case"]
    keys = dict(positions=s["positions"], eps=NORM_EPS, interleaved=c["interleaved"])
    if c["packed"]:
        leaves = [s["qkv"], s["wq"], s["wk"]]
        outs = kat.qkv_norm_rope(s["qkv"], c["q_heads"], c["k_heads"], s["wq"], s["wk"], s["cos"],
                                 s["sin"], **keys)
    else:
        leaves = [s["q"], s["k"], s["wq"], s["wk"]]
        outs = kat.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], **keys)
    outs = list(outs)
    if not c["backward"]:
        return outs
    up = [s["dq"], s["dk"]] + ([s["dv"]] if c["packed"] else [])
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, up))


def _buckets_plain(s, d):
    """Bucket of each distance d = key - query, and where a causal decoder may look."""
    c = s["case"]
    side = c["buckets"] if c["causal"] else c["buckets"] // 2
    n = (-d).clamp(min=0) if c["causal"] else d.abs()
    half = side // 2
    far = half - 1 + torch.bucketize(n, s["borders"], right=True)
    b = torch.where(n < half, n, far)
    return (b, d <= 0) if c["causal"] else (b + (d > 0) * side, None)


def _bias_plain(s):
    c = s["case"]
    table, dtype = s["table"].detach(), DTYPES[c["dtype"]]
    dev = table.device
    if c["op"] == "grid":
        bucket, seen = s["index"], None
    else:
        i = torch.arange(c["lq"], device=dev)[:, None] + c["offset"]
        bucket, seen = _buckets_plain(s, torch.arange(c["lk"], device=dev)[None, :] - i)
    out = table.t().to(dtype)[:, bucket]
    if seen is not None:
        out = out.masked_fill(~seen, -math.inf)
    if not c["backward"]:
        return out
    grad, cells = s["dout"].float(), bucket.reshape(-1)
    if seen is not None:
        grad = grad.masked_fill(~seen, 0.0)
    if c["op"] == "distance":
        # One sum for each distance first: rows, the last one first, each shifted by one more
        # place, put equal distances into one column.
        lq, lk = c["lq"], c["lk"]
        grad = torch.cat([grad.flip(1), grad.new_zeros(c["heads"], lq, lq)], 2).flatten(1)
        grad = grad[:, : lq * (lk + lq - 1)].view(-1, lq, lk + lq - 1)
        grad = grad.sum(1, dtype=torch.float64)
        cells, _ = _buckets_plain(s, torch.arange(lk + lq - 1, device=dev) - lq + 1 - c["offset"])
    d = torch.zeros(c["heads"], table.shape[0], device=dev, dtype=torch.float64)
    d.index_add_(1, cells, grad.flatten(1).double())
    return out, d.t().float()


def _bias_own(s):
    import rational_kat_cu_b200 as kat

    c = s["case"]
    if c["op"] == "grid":
        out = kat.index_bias(s["table"], s["plan"], dtype=DTYPES[c["dtype"]])
    else:
        out = kat.distance_bias(s["table"], s["plan"], c["lq"], c["lk"], offset=c["offset"],
                                causal=c["causal"], dtype=DTYPES[c["dtype"]])
    if not c["backward"]:
        return out
    return out.detach(), *torch.autograd.grad(out, s["table"], s["dout"])


# ---------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk":
        return _qk_exact(s)
    if case["op"] in ("distance", "grid"):
        return _bias_exact(s)
    if case["op"] == "orthogonalize":
        return torch.stack([_polar_exact(g.double()) for g in s["grads"]])
    scale = 0.2 * max(case["rows"], case["cols"]) ** 0.5
    momenta = [g.double() + MOMENTUM * m.double() for g, m in zip(s["grads"], s["momenta"])]
    weights = []
    for w, g, m in zip(s["weights"], s["grads"], momenta):
        o = _polar_exact(torch.add(g.double(), m, alpha=MOMENTUM))
        weights.append(w.double() - LR * (WEIGHT_DECAY * w.double() + scale * o))
    return {"weights": weights, "momenta": momenta}


def _polar_exact(u):
    """The five steps as a function of the squared singular values, by an eigenbasis."""
    if u.shape[0] > u.shape[1]:
        return _polar_exact(u.t()).t()
    if not u.any():
        return u
    x = u / torch.linalg.matrix_norm(u)
    lam, v = torch.linalg.eigh(x @ x.t())
    lam = lam.clamp(min=0)
    total = torch.ones_like(lam)
    for _ in range(NS_STEPS):
        p = NS_A + lam * (NS_B + lam * NS_C)
        total, lam = total * p, lam * p * p
    return (v * total) @ (v.t() @ x)


def _qk_exact(s):
    """With complex numbers: a pair is one number and a rotation one product."""
    c = s["case"]
    rot = c["rot_dim"]
    pos = s["positions"] if s["positions"] is not None else torch.arange(
        c["tokens"], device=s["cos"].device)[None]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos].unsqueeze(2)

    def spin(x, t):
        z = x[..., :rot].reshape(*x.shape[:-1], *((-1, 2) if c["interleaved"] else (2, -1)))
        axis = -1 if c["interleaved"] else -2
        z = torch.complex(z.select(axis, 0), z.select(axis, 1)) * t
        z = torch.stack([z.real, z.imag], axis).flatten(-2)
        return torch.cat([z, x[..., rot:]], -1)

    q, k, v = _split(s)
    outs, dxs, dws = [], [], []
    for x, w, up in ((q, s["wq"], s.get("dq")), (k, s["wk"], s.get("dk"))):
        x, w = x.double(), w.detach().double()
        size = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + NORM_EPS) ** 0.5
        outs.append(spin(x / size * w, turn))
        if up is not None:
            back = spin(up.double(), turn.conj())
            dws.append(torch.einsum("blhd,blhd->d", back, x / size))
            along = torch.einsum("blhd,blhd,d->blh", back, x, w).unsqueeze(-1)
            dxs.append(back * w / size - x * along / (x.shape[-1] * size ** 3))
    if v is not None:
        outs.append(v.double())
        if dxs:
            dxs = [torch.cat(dxs + [s["dv"].double()], 2).flatten(2)]
    return outs + dxs + dws


def _bias_exact(s):
    c = s["case"]
    table = s["table"].detach().double()
    H, dev = c["heads"], table.device
    back = c["backward"]
    if c["op"] == "grid":
        out = table[s["index"]].permute(2, 0, 1)
        if not back:
            return out
        cells, weights = s["index"].cpu().flatten(), s["dout"].double().cpu().flatten(1)
        return out, torch.stack([torch.bincount(cells, weights=weights[h],
                                                minlength=table.shape[0])
                                 for h in range(H)], 1).to(dev)
    # The bucket of each distance from the integers' definition, then diagonal by diagonal.
    side = c["buckets"] if c["causal"] else c["buckets"] // 2
    half, start = side // 2, _bucket_borders(side, c["max_distance"])
    first = -(c["lq"] - 1) - c["offset"]
    row = []
    for d in range(first, c["lk"] - c["offset"]):
        n = max(0, -d) if c["causal"] else abs(d)
        b = n if n < half else half - 1 + sum(1 for t in start if t <= n)
        row.append(b + (side if d > 0 and not c["causal"] else 0))
    values = table[torch.tensor(row, device=dev)].t().contiguous()
    if c["causal"]:
        values[:, max(0, 1 - first):] = -math.inf
    out = torch.stack([values.unfold(1, c["lk"], 1)[h].flip(0) for h in range(H)])
    if not back:
        return out
    grad = s["dout"].double()
    sums = torch.zeros(table.shape[0], H, device=dev, dtype=torch.float64)
    for k, b in enumerate(row):
        if not c["causal"] or first + k <= 0:
            sums[b] += grad.diagonal(k - (c["lq"] - 1), 1, 2).sum(-1)
    return out, sums
