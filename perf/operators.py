"""The encoder operators in front of the alignment: what is timed, and their plain forms.

Four operators, as a training step or a serving loop calls them:

* ``attention``: softmax attention over a ragged batch, q [B, Lq, H, D] against k, v [B, Lk, Hkv, D] with
  ``lengths`` [B, 2] as the alignment operators take them, shared heads, a causal form (rows right-aligned
  to the keys) and a learned relative position bias by buckets; one pass forward ("infer"), or forward and
  gradients ("train"), among them the bias table's;
* the same for single tokens over a long cache ("token");
* ``qk_norm_rope``: RMS norms of queries and keys for each head with the position rotation;
* ``dropout_add``: residual + dropout(x) from a counter-based generator, the mask never stored.

``own`` False runs the plain forms (elementary torch in 32 bits, rounded once), True the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def _attend(name, mode, B, Lq, Lk, H, Hkv, D, dtype, causal=False, buckets=0, max_distance=128, ragged=False,
            packed=False):
    return dict(name=name, op="attend", mode=mode, B=B, Lq=Lq, Lk=Lk, H=H, Hkv=Hkv, D=D, dtype=dtype, causal=causal,
                buckets=buckets, max_distance=max_distance, ragged=ragged, packed=packed)


def _rope(name, mode, B, L, H, Hkv, D, R, dtype):
    return dict(name=name, op="rope", mode=mode, B=B, L=L, H=H, Hkv=Hkv, D=D, R=R, dtype=dtype)


def _drop(name, mode, rows, width, dtype, p):
    return dict(name=name, op="drop", mode=mode, rows=rows, width=width, dtype=dtype, p=p)


def listed():
    return [
        # one generated token per sequence: the norms and rotation of a serving step, all latency
        _rope("rope_token", "infer", 32, 1, 16, 4, 128, 128, "bf16"),
        # an encoder's training step at the ragged batches' 512 positions, queries and keys inside one projection
        _rope("rope_batch_train", "train", 64, 512, 8, 8, 64, 64, "bf16"),
        # long sequences (4096 positions less a few, an odd count), shared key heads, half of each head rotated
        _rope("rope_long_train", "train", 2, 4093, 16, 4, 128, 64, "fp16"),
        # the smallest training step (2 x 100 positions of an odd width), full precision
        _drop("drop_small_train", "train", 200, 333, "fp32", 0.1),
        # the residual stream of 256 sequences of 512 positions, embedding width 256
        _drop("drop_batch_train", "train", 256 * 512, 256, "bf16", 0.1),
        # one token of one sequence over a short cache: latency alone
        _attend("token_single", "token", 1, 1, 513, 8, 2, 64, "bf16", causal=True),
        # one token for each of 32 sequences over caches of up to 4096, with the position bias
        _attend("token_batch", "token", 32, 1, 4096, 16, 16, 64, "bf16", causal=True, buckets=32, ragged=True),
        # the smallest pair of sequences (100 against 120): cross attention with its gradients
        _attend("pair_train", "train", 2, 100, 120, 4, 4, 64, "bf16", buckets=32, ragged=True),
        # inference of an encoder layer on a large ragged batch of 512 positions, q, k and v inside one projection
        _attend("batch_infer", "infer", 256, 512, 512, 8, 8, 64, "bf16", buckets=32, ragged=True, packed=True),
        # cross attention of odd lengths and head size, shared heads, no bias
        _attend("cross_odd_infer", "infer", 8, 1021, 777, 12, 3, 80, "fp16"),
        # an encoder layer's training step on a ragged batch of 512 positions, with the bias table's gradient
        _attend("batch_train", "train", 64, 512, 512, 8, 8, 64, "bf16", buckets=32, ragged=True),
        # long causal training, 4096 positions, shared key heads of 128
        _attend("long_train", "train", 2, 4096, 4096, 16, 4, 128, "bf16", causal=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    kind = rng.choice(["rope", "drop", "token", "attend", "attend", "attend"])
    if kind == "drop":
        return _drop(None, "train", _log(rng, 50, 256 * 512), _log(rng, 33, 512), rng.choice(["bf16", "fp16", "fp32"]),
                     rng.choice([0.0, 0.1, 0.25, 0.5]))
    group = rng.choice([1, 1, 2, 4])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rope":
        D = rng.choice([32, 64, 80, 128])
        R = rng.choice([D, D, 16 * max(1, D // 32)])
        return _rope(None, rng.choice(["infer", "train"]), _log(rng, 1, 64), _log(rng, 1, 4096), Hkv * group, Hkv, D, R, dtype)
    D = rng.choice([32, 64, 64, 80, 128, 128])
    buckets = rng.choice([0, 16, 32])
    distance = rng.choice([64, 128, 200])
    ragged = rng.random() < 0.5
    if kind == "token":
        return _attend(None, "token", _log(rng, 1, 32), 1, _log(rng, 64, 32768), Hkv * group, Hkv, D, dtype, True,
                       buckets, distance, ragged)
    own_keys = rng.random() < 0.5
    Lq = _log(rng, 16, 4096)
    Lk = Lq if own_keys else _log(rng, 16, 4096)
    return _attend(None, rng.choice(["infer", "train"]), _log(rng, 1, 128), Lq, Lk, Hkv * group, Hkv, D, dtype,
                   own_keys and rng.random() < 0.4, buckets, distance, ragged)


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    planes = max(c["B"] * c["H"] * c["Lq"] * c["Lk"] for c in listed() if c["op"] == "attend")
    while True:
        c = _draw_one(rng)
        del c["name"]
        if _cost(c) <= most[c["op"]] and (c["op"] != "attend" or c["B"] * c["H"] * c["Lq"] * c["Lk"] <= planes):
            return c


def _lengths(case):
    """[(lq, lk)] of the problems: None where all are full.  They go by the case alone; evenly spread from an
    eighth of the padded length (a batch of eight or more also holds an empty problem) in a fixed order."""
    if not case["ragged"]:
        return None
    B = case["B"]

    def spread(L):
        lo = max(1, L // 8)
        ls = [lo + (L - lo) * (b + 1) // B for b in range(B)]
        if B >= 8:
            ls[0] = 0
        return ls

    order = list(range(B))
    random.Random(B).shuffle(order)
    q, k = spread(case["Lq"]), spread(case["Lk"])
    if case["mode"] == "token":
        return [(1 if k[o] else 0, k[o]) for o in order]
    if case["Lq"] == case["Lk"]:
        return [(q[o], k[o]) for o in order]
    turned = order[1:] + order[:1]
    return [(q[o], k[t]) for o, t in zip(order, turned)]


def work(case):
    e = SIZE[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "drop":
        n = case["rows"] * case["width"]
        # x and the residual read, y written; the gradient read and dx written (the residual's is dy itself)
        return {"bytes": n * e * (5 if train else 3), "flops": n * (5 if train else 3)}
    if case["op"] == "rope":
        rows = case["B"] * case["L"] * (case["H"] + case["Hkv"])
        n = rows * case["D"]
        tables = case["B"] * case["L"] * case["R"] * 4 + 2 * case["D"] * 4
        # forward: q, k read, written; backward: their gradients and q, k read, dq, dk written
        return {"bytes": n * e * (5 if train else 2) + tables, "flops": n * (22 if train else 8)}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    lens = _lengths(case) or [(case["Lq"], case["Lk"])] * case["B"]
    cells = rows_q = rows_k = 0
    for lq, lk in lens:
        if case["causal"]:
            cells += sum(max(0, min(lk, i + lk - lq + 1)) for i in range(lq))
        else:
            cells += lq * lk
        rows_q, rows_k = rows_q + lq, rows_k + lk
    read = rows_q * H * D * e + 2 * rows_k * Hkv * D * e
    out = case["B"] * case["Lq"] * H * D * e   # padded rows are written as zeros
    table = case["buckets"] * H * e
    if not train:
        return {"bytes": read + out + table, "flops": 4 * cells * H * D + 5 * cells * H}
    grads = out + 2 * case["B"] * case["Lk"] * Hkv * D * e + table
    # two products forward; the recomputed scores and four products backward
    return {"bytes": read + out + table + rows_q * H * D * e + grads, "flops": 14 * cells * H * D + 12 * cells * H}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    st = {"case": case, "train": case["mode"] == "train"}
    if case["op"] == "drop":
        shape = (case["rows"], case["width"])
        st["x"], st["residual"], st["grad"] = (normal(*shape).to(dt) for _ in range(3))
        st["seed"], st["offset"], st["p"] = seed * 1000003 + 17, 5, case["p"]
        if st["train"]:
            st["x"].requires_grad_(True)
            st["residual"].requires_grad_(True)
        return st
    if case["op"] == "rope":
        B, L, H, Hkv, D, R = (case[n] for n in ("B", "L", "H", "Hkv", "D", "R"))
        # q, k (and v) come out of one projection
        qkv = normal(B, L, H + 2 * Hkv, D, scale=1.7).to(dt)
        st["q"], st["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
        st["qw"], st["kw"] = ((1.0 + normal(D, scale=0.1)).to(dt) for _ in range(2))
        most = 8192
        inv = 10000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)
        angle = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * inv
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        start = torch.randint(0, most - L, (B, 1), generator=g, device=dev)
        st["positions"] = (start + torch.arange(L, device=dev)).to(torch.int32)
        st["dq"], st["dk"] = normal(B, L, H, D).to(dt), normal(B, L, Hkv, D).to(dt)
        if st["train"]:
            for n in ("q", "k", "qw", "kw"):
                st[n] = st[n].detach().requires_grad_(True)
        return st
    B, Lq, Lk, H, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    if case["packed"]:
        qkv = normal(B, Lq, H + 2 * Hkv, D).to(dt)
        st["q"], st["k"], st["v"] = qkv[:, :, :H], qkv[:, :, H:H + Hkv], qkv[:, :, H + Hkv:]
    else:
        st["q"] = normal(B, Lq, H, D).to(dt)
        st["k"], st["v"] = (normal(B, Lk, Hkv, D).to(dt) for _ in range(2))
    st["bias"] = normal(case["buckets"], H, scale=0.5).to(dt) if case["buckets"] else None
    lens = _lengths(case)
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev) if lens else None
    st["grad"] = normal(B, Lq, H, D).to(dt) if st["train"] else None
    if st["train"]:
        for n in ("q", "k", "v", "bias"):
            if st[n] is not None:
                st[n].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        return {"attend": _own_attend, "rope": _own_rope, "drop": _own_drop}[op](st)
    with torch.no_grad():
        return {"attend": _plain_attend, "rope": _plain_rope, "drop": _plain_drop}[op](st)


def _own_attend(st):
    import d2p_b200 as d2p

    c = st["case"]
    out = d2p.attention(st["q"], st["k"], st["v"], bias=st["bias"], lengths=st["lengths"], causal=c["causal"],
                        max_distance=c["max_distance"])
    if not st["train"]:
        return [out]
    leaves = [st[n] for n in ("q", "k", "v", "bias") if st[n] is not None]
    return [out.detach(), *torch.autograd.grad(out, leaves, st["grad"])]


def _own_rope(st):
    import d2p_b200 as d2p

    q, k = d2p.qk_norm_rope(st["q"], st["k"], st["qw"], st["kw"], st["cos"], st["sin"], positions=st["positions"])
    if not st["train"]:
        return [q, k]
    grads = torch.autograd.grad((q, k), [st[n] for n in ("q", "k", "qw", "kw")], (st["dq"], st["dk"]))
    return [q.detach(), k.detach(), *grads]


def _own_drop(st):
    import d2p_b200 as d2p

    y = d2p.dropout_add(st["x"], st["residual"], st["p"], st["seed"], st["offset"])
    if not st["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [st["x"], st["residual"]], st["grad"])]


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------
def _thresholds(buckets, max_distance, two_sided):
    """Smallest distance of each bucket but the first, on one side, in whole numbers: distances below `exact`
    have a bucket each; bucket exact + t starts at the first n with (n / exact)^c >= (max_distance / exact)^t,
    c = side - exact."""
    side = buckets // 2 if two_sided else buckets
    exact = side // 2
    c = side - exact
    edges = list(range(1, exact + 1))
    n = exact
    for t in range(1, c):
        while n ** c * exact ** t < max_distance ** t * exact ** c:
            n += 1
        edges.append(n)
    return edges


def _bucket(d, buckets, max_distance, two_sided):
    """Bucket of each key position less query position in d."""
    edges = torch.tensor(_thresholds(buckets, max_distance, two_sided), device=d.device)
    n = d.abs() if two_sided else (-d).clamp(min=0)
    b = torch.bucketize(n, edges, right=True)
    return b + (d > 0) * (buckets // 2) if two_sided else b


def _plain_attend(st):
    c = st["case"]
    q, k, v = (st[n].float().transpose(1, 2) for n in ("q", "k", "v"))   # [B, heads, L, D]
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    dev, dt = q.device, st["q"].dtype
    scale = 1.0 / math.sqrt(D)
    if st["lengths"] is None:
        lq = torch.full((1, 1, 1), Lq, device=dev)
        lk = torch.full((1, 1, 1), Lk, device=dev)
    else:
        lq, lk = st["lengths"].long()[:, :1, None], st["lengths"].long()[:, 1:, None]
    i = torch.arange(Lq, device=dev)[None, :, None]
    j = torch.arange(Lk, device=dev)[None, None, :]
    d = j - i - (lk - lq if c["causal"] else 0)
    allowed = (i < lq) & (j < lk)
    if c["causal"]:
        allowed = allowed & (d <= 0)
    allowed = allowed[:, None]                                           # [1 or B, 1, Lq, Lk]
    qg = q.reshape(B, Hkv, H // Hkv, Lq, D)
    s = torch.matmul(qg, k[:, :, None].transpose(-1, -2)).reshape(B, H, Lq, Lk) * scale
    bucket = None
    if st["bias"] is not None:
        bucket = _bucket(d, c["buckets"], c["max_distance"], not c["causal"])
        s = s + st["bias"].float()[bucket].permute(0, 3, 1, 2)
    s = torch.where(allowed, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    del s
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    pg = p.reshape(B, Hkv, H // Hkv, Lq, Lk)
    o = torch.matmul(pg, v[:, :, None]).reshape(B, H, Lq, D)
    outs = [o.transpose(1, 2).contiguous().to(dt)]
    if not st["train"]:
        return outs
    g = st["grad"].float().transpose(1, 2)
    gg = g.reshape(B, Hkv, H // Hkv, Lq, D)
    dv = torch.matmul(pg.transpose(-1, -2), gg).sum(2)
    dp = torch.matmul(gg, v[:, :, None].transpose(-1, -2)).reshape(B, H, Lq, Lk)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    del p, dp, pg
    dsg = ds.reshape(B, Hkv, H // Hkv, Lq, Lk)
    dq = torch.matmul(dsg, k[:, :, None]).reshape(B, H, Lq, D) * scale
    dk = torch.matmul(dsg.transpose(-1, -2), qg).sum(2) * scale
    outs += [t.transpose(1, 2).contiguous().to(dt) for t in (dq, dk, dv)]
    if st["bias"] is not None:
        if bucket.shape[0] == 1:   # the same buckets for every problem
            ds, flat = ds.sum(0, keepdim=True), bucket
        else:
            flat = bucket
        n = ds.shape[0]
        sums = torch.zeros(n, H, c["buckets"], device=dev)
        sums.scatter_add_(2, flat.reshape(n, 1, -1).expand(n, H, -1), ds.reshape(n, H, -1))
        outs.append(sums.sum(0).t().contiguous().to(dt))
    return outs


def _plain_rope(st):
    R = st["case"]["R"]
    pos = st["positions"].long()
    cos, sin = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]    # [B, L, 1, R / 2]

    def rotate(y, sin):
        a, b = y[..., :R // 2], y[..., R // 2:R]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., R:]], -1)

    outs, grads = [], []
    for x0, w0, g0 in ((st["q"], st["qw"], st["dq"]), (st["k"], st["kw"], st["dk"])):
        x, w = x0.float(), w0.float()
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        xhat = x * rstd
        outs.append(rotate(xhat * w, sin).to(x0.dtype))
        if st["train"]:
            gy = rotate(g0.float(), -sin)
            gw = gy * w
            grads.append(((rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))).to(x0.dtype),
                          (gy * xhat).sum((0, 1, 2)).to(w0.dtype)))
    if not st["train"]:
        return outs
    return [*outs, grads[0][0], grads[1][0], grads[0][1], grads[1][1]]


def _words(n, seed, offset, dev):
    """32-bit words of the counter-based generator Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
    numbers: as easy as 1, 2, 3", 2011): counter (element / 4, offset), key the seed, one word per element."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=dev)
    a, b = block & low, block >> 32
    x, y = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)
    k0, k1 = seed & low, (seed >> 32) & low
    for r in range(10):
        p, q = a * 0xD2511F53, x * 0xCD9E8D57
        a, b, x, y = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ y ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([a, b, x, y], 1).reshape(-1)[:n]


def _plain_drop(st):
    x, p = st["x"], st["p"]
    keep = (_words(x.numel(), st["seed"], st["offset"], x.device) >= int(p * 2 ** 32)).reshape(x.shape)
    scale = 1.0 / (1.0 - p)
    y = (st["residual"].float() + torch.where(keep, x.float() * scale, 0.0)).to(x.dtype)
    if not st["train"]:
        return [y]
    return [y, torch.where(keep, st["grad"].float() * scale, 0.0).to(x.dtype), st["grad"].clone()]


# ---------------------------------------------------------------------------------------------------------
# in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        return {"attend": _exact_attend, "rope": _exact_rope, "drop": _exact_drop}[case["op"]](case, st)


def _side_bucket(n, side, max_distance):
    """Bucket of distance n >= 0 among `side`, by the definition in whole numbers."""
    e = side // 2
    if n < e:
        return n
    c = side - e
    t = 0
    while t + 1 < c and n ** c * e ** (t + 1) >= max_distance ** (t + 1) * e ** c:
        t += 1
    return e + t


def _exact_attend(case, st):
    B, Lq, Lk, H, Hkv, D = (case[n] for n in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    train, causal, nb = st["train"], case["causal"], case["buckets"]
    lens = _lengths(case) or [(Lq, Lk)] * B
    out = torch.zeros(B, Lq, H, D, dtype=torch.float64, device="cuda")
    grads = None
    if train:
        grads = [torch.zeros(st[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v", "bias") if st[n] is not None]
    if nb:
        side = nb if causal else nb // 2
        far = max(Lq, Lk) + 1
        one = [_side_bucket(min(n, case["max_distance"]), side, case["max_distance"]) for n in range(far)]
        lut = [(one[-d] if d <= 0 else (0 if causal else side + one[d])) for d in range(-far + 1, far)]
        lut = torch.tensor(lut, device="cuda")
    for b, (lq, lk) in enumerate(lens):
        if lq == 0 or lk == 0:
            continue
        q, k, v = (st[n][b, :l].detach().double().requires_grad_(train) for n, l in (("q", lq), ("k", lk), ("v", lk)))
        leaves = [q, k, v]
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(H // Hkv, 1)) / math.sqrt(D)
        rel = torch.arange(lk, device="cuda")[None] - torch.arange(lq, device="cuda")[:, None] - (lk - lq if causal else 0)
        if nb:
            table = st["bias"].detach().double().requires_grad_(train)
            leaves.append(table)
            s = s + table.index_select(0, lut[rel.clamp(-far + 1, far - 1) + far - 1].reshape(-1)).reshape(lq, lk, H).permute(2, 0, 1)
        if causal:
            s = s.masked_fill(rel > 0, -math.inf)
            empty = (rel > 0).all(1)
            s = s.masked_fill(empty[None, :, None], 0.0)
        p = torch.softmax(s, -1)
        if causal:
            p = p.masked_fill(empty[None, :, None], 0.0)
        o = torch.einsum("hij,jhd->ihd", p, v.repeat_interleave(H // Hkv, 1))
        out[b, :lq] = o.detach()
        if train:
            got = torch.autograd.grad(o, leaves, st["grad"][b, :lq].double())
            for t, x, l in zip(grads, got[:3], (lq, lk, lk)):
                t[b, :l] = x
            if nb:
                grads[3] += got[3]
            del got
        del s, p, o
    return [out, *grads] if train else [out]


def _exact_rope(case, st):
    R = case["R"]
    pos = st["positions"].long().reshape(-1)
    turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double()).reshape(case["B"], case["L"], 1, R // 2)
    outs, dx, dw = [], [], []
    for x0, w0, g in ((st["q"], st["qw"], st["dq"]), (st["k"], st["kw"], st["dk"])):
        x = x0.detach().double().requires_grad_(st["train"])
        w = w0.detach().double().requires_grad_(st["train"])
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * turn
        y = torch.cat([z.real, z.imag, y[..., R:]], -1)
        outs.append(y.detach())
        if st["train"]:
            a, b = torch.autograd.grad(y, [x, w], g.double())
            dx.append(a)
            dw.append(b)
    return [*outs, *dx, *dw]


def _exact_drop(case, st):
    x, n = st["x"].detach(), st["x"].numel()
    import numpy as np

    u32, u64 = np.uint32, np.uint64
    blocks = np.arange((n + 3) // 4, dtype=u64)
    ctr = [(blocks & u64(0xFFFFFFFF)).astype(u32), (blocks >> u64(32)).astype(u32),
           np.full(blocks.size, st["offset"] & 0xFFFFFFFF, u32), np.full(blocks.size, st["offset"] >> 32, u32)]
    key = [st["seed"] & 0xFFFFFFFF, (st["seed"] >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p0 = ctr[0].astype(u64) * u64(0xD2511F53)
        p1 = ctr[2].astype(u64) * u64(0xCD9E8D57)
        ctr = [(p1 >> u64(32)).astype(u32) ^ ctr[1] ^ u32(key[0]), p1.astype(u32),
               (p0 >> u64(32)).astype(u32) ^ ctr[3] ^ u32(key[1]), p0.astype(u32)]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    kept = np.stack(ctr, 1).reshape(-1)[:n].astype(u64) >= u64(int(case["p"] * 2 ** 32))
    keep = torch.from_numpy(kept).reshape(x.shape).to(x.device).double() / (1.0 - case["p"])
    y = st["residual"].detach().double() + x.double() * keep
    return [y, st["grad"].double() * keep, st["grad"].double()]
