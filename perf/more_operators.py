"""Workloads of the 4-bit and router operators: what is timed, on which inputs.

A case is one pass through an operator as a program calls it.  ``own = False`` computes it
with elementary torch operations in 32 bits, ``own = True`` with this package's operators;
``exact`` gives the definition's value in 64 bits.

Kinds of case:

* ``quantize``  a weight matrix to 4 bits with group scales, and read back; the result is
  returned as the values it stands for.
* ``int4``      product of 16-bit tokens with a 4-bit weight matrix.
* ``grouped``   the same with one weight matrix per expert over rows sorted by expert.
* ``route``     a router's scores to each token's experts and weights; with ``train`` the
  scores' gradient too.
* ``balance``   the balance loss of a router, its counts, and with ``train`` its gradient.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SZ = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # weights prepared once when a model is loaded: bandwidth
        dict(name="quantize_weights", kind="quantize", N=4096, K=14336, dtype="bf16", group=128, scale="f32"),
        # fp32 weights whose rows are no multiple of anything, small groups
        dict(name="quantize_odd", kind="quantize", N=1001, K=4099, dtype="f32", group=32, scale="f16"),
        # one token through a feed-forward projection: the weights' bytes
        dict(name="int4_token", kind="int4", M=1, K=4096, N=14336, dtype="bf16", group=128, scale="bf16", zero=False,
             bias=False),
        # one decode step of 16 sequences through the projection back
        dict(name="int4_step", kind="int4", M=16, K=14336, N=4096, dtype="f16", group=128, scale="f16", zero=False,
             bias=False),
        # a few tokens, nothing a multiple of a tile, zero points, small groups and a bias
        dict(name="int4_odd", kind="int4", M=5, K=4100, N=2051, dtype="bf16", group=32, scale="f32", zero=True,
             bias=True),
        # a prompt through the same projection: tensor cores
        dict(name="int4_prompt", kind="int4", M=4096, K=4096, N=14336, dtype="bf16", group=128, scale="bf16",
             zero=False, bias=False),
        # 8 tokens decoded through 2 of 8 experts each: the bytes of the experts in use
        dict(name="grouped_decode", kind="grouped", T=8, k=2, E=8, K=4096, N=14336, dtype="bf16", group=128,
             scale="bf16", zero=False, skew=0.5, drop=0.0),
        # many small experts, uneven, some entries dropped by a capacity limit
        dict(name="grouped_many", kind="grouped", T=1000, k=8, E=64, K=2048, N=1536, dtype="f16", group=64,
             scale="f16", zero=True, skew=0.5, drop=0.05),
        # the router of one decode step: latency
        dict(name="route_decode", kind="route", T=16, E=64, k=8, dtype="bf16", normalize=True, masked=0.0,
             train=False),
        # the router of a training step, with its gradient
        dict(name="route_train", kind="route", T=65536, E=128, k=8, dtype="f32", normalize=False, masked=0.0,
             train=True),
        # the balance of a small batch with padded tokens
        dict(name="balance_small", kind="balance", T=1000, E=60, k=4, dtype="bf16", pad=0.2, drop=0.05, train=True),
        # the balance of a training step
        dict(name="balance_train", kind="balance", T=65536, E=128, k=8, dtype="f32", pad=0.0, drop=0.0, train=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi):  # a power of two, an odd number of 16s, or odd
        n, how = log(lo, hi), rng.randrange(3)
        if how == 0:
            return max(lo, 1 << (n.bit_length() - 1))
        return n // 32 * 32 + 16 if how == 1 else n | 1

    kind = rng.choice(["quantize", "int4", "int4", "int4", "grouped", "grouped", "route", "balance"])
    if kind == "quantize":
        dtype = rng.choice(["bf16", "f16", "f32"])
        N, K = log(1, 16384), size(64, 16384)
        return dict(kind=kind, N=max(1, min(N, 4096 * 14336 // K)), K=K, dtype=dtype,
                    group=rng.choice([32, 64, 128, 256]), scale=rng.choice(["f32", dtype]))
    if kind in ("int4", "grouped"):
        dtype = rng.choice(["bf16", "bf16", "f16"])
        more = dict(dtype=dtype, group=rng.choice([32, 64, 128, 128, 256]), scale=rng.choice(["f32", dtype]),
                    zero=rng.random() < 0.3)
    if kind == "int4":
        M, K, N = log(1, 4096), size(64, 16384), size(64, 16384)
        M = max(1, min(M, 4096 * 4096 * 14336 // (K * N)))
        return dict(kind=kind, M=M, K=K, N=N, bias=rng.random() < 0.3, **more)
    k = rng.choice([1, 2, 4, 8])
    E = rng.choice([e for e in (4, 8, 16, 60, 64, 128, 256) if e >= k])
    if kind == "grouped":
        T = min(log(1, 4096), 8192 // k)
        K = size(128, 4096)
        N = max(128, min(size(128, 14336), 8 * 4096 * 14336 // (E * K) // 32 * 32 - 16))
        return dict(kind=kind, T=T, k=k, E=E, K=K, N=N, skew=rng.choice([0.0, 0.5, 1.5]),
                    drop=rng.choice([0.0, 0.0, 0.05, 0.3]), **more)
    T, dtype = min(log(1, 131072), 65536 * 128 // E), rng.choice(["bf16", "f32", "f32", "f16"])
    if kind == "route":
        return dict(kind=kind, T=T, E=E, k=k, dtype=dtype, normalize=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.0, 0.1, 0.9]), train=rng.random() < 0.7)
    return dict(kind=kind, T=T, E=E, k=k, dtype=dtype, pad=rng.choice([0.0, 0.0, 0.3]),
                drop=rng.choice([0.0, 0.05]), train=rng.random() < 0.7)


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _floats(shape, dtype, g):
    """Activations: N(0, 1) with some strong channels."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    strong = torch.rand(shape[-1], generator=g, device="cuda") < 0.002
    return (x * torch.where(strong, 20.0, 1.0)).to(dtype)


def _route(case, g):
    """Distinct experts of each token by a router's scores; an entry that its expert has no
    room for has the number -1."""
    T, k, E = case["T"], case["k"], case["E"]
    score = torch.randn((T, E), generator=g, device="cuda")
    score = score + case["skew"] * torch.randn(E, generator=g, device="cuda")
    ids = torch.topk(score, k, dim=1).indices
    lost = torch.rand((T, k), generator=g, device="cuda") < case["drop"]
    return torch.where(lost, -1, ids)


def _weights(lead, case, g):
    """4-bit weights as they are kept: two to a byte, rows on 16-byte boundaries, a scale and
    with ``zero`` a zero point for each group of columns."""
    K, G = case["K"], case["group"]
    cols, groups = (K + 1) // 2, (K + G - 1) // G
    n = math.prod(lead)
    u = torch.empty((n, (cols + 15) // 16 * 16), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 28) // u.shape[1])
    for i in range(0, n, step):
        part = u[i:i + step]
        lo = torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float16).mul_(2.6).round_().clamp_(-7, 7)
        hi = torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float16).mul_(2.6).round_().clamp_(-7, 7)
        part.copy_((hi + 8) * 16 + (lo + 8))
    s = {"w": u.reshape(*lead, u.shape[1])[..., :cols],
         "scale": (torch.rand((*lead, groups), generator=g, device="cuda") * 4e-3 + 8e-3).to(DT[case["scale"]])}
    s["zero"] = torch.randint(5, 12, (*lead, groups), generator=g, device="cuda",
                              dtype=torch.uint8) if case["zero"] else None
    return s


def prepare(case, seed):
    g = _gen(seed)
    kind, s = case["kind"], {"case": case}
    if kind == "quantize":
        s["x"] = (torch.randn((case["N"], case["K"]), generator=g, device="cuda") * 0.02).to(DT[case["dtype"]])
        return s
    if kind == "int4":
        s.update(_weights((case["N"],), case, g))
        s["x"] = _floats((case["M"], case["K"]), DT[case["dtype"]], g)
        s["bias"] = _floats((case["N"],), DT[case["dtype"]], g) if case["bias"] else None
        return s
    if kind == "grouped":
        flat = _route(case, g).reshape(-1)
        E = case["E"]
        key = torch.where((flat >= 0) & (flat < E), flat, E)
        s["offsets"] = (key[:, None] < torch.arange(E + 1, device="cuda")[None, :]).sum(0).to(torch.int32)
        s.update(_weights((E, case["N"]), case, g))
        s["x"] = _floats((flat.numel(), case["K"]), DT[case["dtype"]], g)
        return s
    T, E, k = case["T"], case["E"], case["k"]
    logits = torch.randn((T, E), generator=g, device="cuda") * 2 + torch.randn(E, generator=g, device="cuda") * 0.5
    if kind == "route":
        # experts that a token may not use
        off = torch.rand((T, E), generator=g, device="cuda") < case["masked"]
        s["logits"] = torch.where(off, -math.inf, logits).to(DT[case["dtype"]])
        s["grad"] = torch.randn((T, k), generator=g, device="cuda")
        return s
    ids = torch.topk(logits + torch.randn((T, E), generator=g, device="cuda"), k, dim=1).indices
    lost = torch.rand((T, k), generator=g, device="cuda") < case["drop"]
    s["experts"] = torch.where(lost, -1, ids).to(torch.int32)
    s["logits"] = logits.to(DT[case["dtype"]])
    s["mask"] = torch.rand(T, generator=g, device="cuda") >= case["pad"] if case["pad"] else None
    s["grad"] = torch.rand((), generator=g, device="cuda") * 0.1 + 0.01
    return s


# ------------------------------------------------------------------------------ plain forms
def _plain_weights(s):
    """The weights' values in 32 bits: [..., N, K]."""
    K, G = s["case"]["K"], s["case"]["group"]
    w = s["w"]
    u = torch.stack((w & 15, w >> 4), dim=-1).reshape(*w.shape[:-1], -1)[..., :K].float()
    zero = 8.0 if s["zero"] is None else s["zero"].float().repeat_interleave(G, -1)[..., :K]
    return (u - zero) * s["scale"].float().repeat_interleave(G, -1)[..., :K]


def _plain_quantize(s):
    c = s["case"]
    G, K = c["group"], c["K"]
    groups = (K + G - 1) // G
    x = s["x"].float()
    padded = torch.zeros((c["N"], groups * G), device=x.device)
    padded[:, :K] = x
    parts = padded.reshape(c["N"], groups, G)
    # in 64 bits: quotients next to a half, where the last bit of a scale or of a quotient decides
    scale = (parts.abs().amax(2).double() / 7).float().to(DT[c["scale"]])
    step = torch.where(scale == 0, 1.0, scale.float())[..., None]
    q = torch.round(parts.double() / step.double()).clamp(-7, 7).float()
    q = torch.where(scale[..., None] == 0, 0.0, q)
    values = (q * scale.float()[..., None]).reshape(c["N"], -1)[:, :K]
    return {"values": values.to(s["x"].dtype), "scale": scale}


def _plain_grouped(s):
    c = s["case"]
    offsets, x = s["offsets"], s["x"].float()
    row = torch.arange(x.shape[0], device=x.device)
    e = (row[:, None] >= offsets[None, 1:]).sum(1)  # E for a dropped entry
    room = max(1, int((offsets[1:] - offsets[:-1]).max()))
    kept = e < c["E"]
    e = torch.where(kept, e, 0)
    r = torch.where(kept, row - offsets[e], room)   # the spare row takes the dropped ones
    padded = torch.zeros((c["E"], room + 1, x.shape[1]), device=x.device)
    padded[e, r] = x
    y = torch.bmm(padded, _plain_weights(s).transpose(1, 2))[e, r]
    return torch.where(kept[:, None], y, 0.0).to(s["x"].dtype)


def _softmax(x):
    """Softmax over the finite scores of each row; zeros where there is none."""
    top = x.amax(1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_route(s):
    c = s["case"]
    x = s["logits"].float()
    p = _softmax(x)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["k"]]
    ids = torch.where(torch.gather(x, 1, ids) > -math.inf, ids, -1)
    chosen = ids >= 0
    at = torch.where(chosen, ids, 0)
    picked = torch.where(chosen, torch.gather(p, 1, at), 0.0)
    total = picked.sum(1, keepdim=True)
    w = picked / torch.where(total == 0, 1.0, total) if c["normalize"] else picked
    out = {"weights": w, "experts": ids.to(torch.int32)}
    if c["train"]:
        g = torch.where(chosen, s["grad"], 0.0)
        mine = w * (g - (w * g).sum(1, keepdim=True)) if c["normalize"] else w * g
        d = torch.zeros_like(p).scatter_add(1, at, torch.where(chosen, mine, 0.0))
        if not c["normalize"]:
            d = d - p * (w * g).sum(1, keepdim=True)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_balance(s):
    c = s["case"]
    E = c["E"]
    p = _softmax(s["logits"].float())
    ids = s["experts"]
    if s["mask"] is not None:
        p = torch.where(s["mask"][:, None], p, 0.0)
        ids = torch.where(s["mask"][:, None], ids, -1)
    counts = torch.zeros(E + 1, dtype=torch.int32, device=ids.device)
    flat = torch.where(ids < 0, E, ids).reshape(-1).long()
    counts = counts.scatter_add(0, flat, torch.ones_like(flat, dtype=torch.int32))[:E]
    tokens = s["mask"].sum() if s["mask"] is not None else torch.full((), c["T"], device=ids.device)
    # the sums over the tokens in 64 bits: they are long
    share = counts.double() / counts.sum().clamp_min(1)
    load = p.double().sum(0) / tokens.clamp_min(1)
    out = {"loss": (E * (share * load).sum()).float(), "counts": counts}
    if c["train"]:
        a = (s["grad"] * E * share / tokens.clamp_min(1)).float()
        out["dlogits"] = (p * (a - (p * a).sum(1, keepdim=True))).to(s["logits"].dtype)
    return out


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "quantize":
        return _plain_quantize(s)
    if kind == "int4":
        y = s["x"].float() @ _plain_weights(s).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(s["x"].dtype)
    if kind == "grouped":
        return _plain_grouped(s)
    return _plain_route(s) if kind == "route" else _plain_balance(s)


# ------------------------------------------------------------------------------ this package
def _own(s):
    import metalblas_b200 as mb
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        q, scale = mb.quantize_int4(s["x"], c["group"], scale_dtype=DT[c["scale"]])
        return {"values": mb.dequantize_int4(q, scale, c["group"], cols=c["K"], out_dtype=s["x"].dtype),
                "scale": scale}
    if kind == "int4":
        return mb.int4_mm(s["x"], s["w"], s["scale"], c["group"], zero=s["zero"], bias=s["bias"])
    if kind == "grouped":
        return mb.grouped_int4_mm(s["x"], s["w"], s["scale"], s["offsets"], c["group"], zero=s["zero"])
    if kind == "route":
        weights, experts = mb.expert_route(s["logits"], c["k"], normalize=c["normalize"])
        out = {"weights": weights, "experts": experts}
        if c["train"]:
            out["dlogits"] = mb.expert_route_backward(s["grad"], s["logits"], experts, normalize=c["normalize"])
        return out
    b = mb.expert_balance(s["logits"], s["experts"], mask=s["mask"])
    out = {"loss": b.loss, "counts": b.counts}
    if c["train"]:
        out["dlogits"] = mb.expert_balance_backward(s["grad"], s["logits"], b, mask=s["mask"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------ 64 bits
def _exact_weights(w, scale, zero, K, G):
    rows = w.reshape(-1, w.shape[-1])
    out = torch.empty((rows.shape[0], 2 * w.shape[-1]), dtype=torch.float64, device=w.device)
    out[:, 0::2] = torch.remainder(rows, 16).double()
    out[:, 1::2] = torch.div(rows, 16, rounding_mode="floor").double()
    group = torch.div(torch.arange(K, device=w.device), G, rounding_mode="floor")
    z = torch.full_like(scale, 8, dtype=torch.float64) if zero is None else zero.double()
    out = out[:, :K].reshape(*w.shape[:-1], K)
    return (out - z.index_select(-1, group)) * scale.double().index_select(-1, group)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        K, G = case["K"], case["group"]
        x = s["x"].double()
        values = torch.empty_like(x)
        scales = []
        for k in range(0, K, G):
            part = x[:, k:k + G]
            # the scale is what the type holds of amax / 7
            one = (part.abs().max(dim=1).values / 7).float().to(DT[case["scale"]]).double()
            q = torch.round(part / one.clamp_min(1e-300)[:, None]).clamp(-7, 7)
            values[:, k:k + G] = q * one[:, None]
            scales.append(one)
        return {"values": values, "scale": torch.stack(scales, 1)}
    if kind == "int4":
        w = _exact_weights(s["w"], s["scale"], s["zero"], case["K"], case["group"])
        y = torch.matmul(s["x"].double(), w.t())
        return y if s["bias"] is None else y.add_(s["bias"].double())
    if kind == "grouped":
        ends = s["offsets"].tolist()
        y = torch.zeros((s["x"].shape[0], case["N"]), dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            lo, hi = ends[e], ends[e + 1]
            if hi > lo:
                zero = None if s["zero"] is None else s["zero"][e]
                w = _exact_weights(s["w"][e], s["scale"][e], zero, case["K"], case["group"])
                y[lo:hi] = torch.matmul(s["x"][lo:hi].double(), w.t())
        return y
    x = s["logits"].double()
    p = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
    if kind == "route":
        k = case["k"]
        order = torch.argsort(-x, dim=1, stable=True)[:, :k]
        usable = torch.isfinite(torch.gather(x, 1, order))
        hot = torch.nn.functional.one_hot(order, case["E"]).double() * usable[..., None]   # [T, k, E]
        q = torch.einsum("tke,te->tk", hot, p)
        total = q.sum(1, keepdim=True)
        w = torch.where(total > 0, q / total.clamp_min(1e-300), 0.0) if case["normalize"] else q
        out = {"weights": w, "experts": torch.where(usable, order, -1).to(torch.int32)}
        if case["train"]:
            g = s["grad"].double()
            mean = (w * g).sum(1, keepdim=True)
            if case["normalize"]:
                out["dlogits"] = torch.einsum("tke,tk->te", hot, w * (g - mean))
            else:
                out["dlogits"] = torch.einsum("tke,tk->te", hot, w * g) - p * mean
        return out
    on = torch.ones(case["T"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    kept = s["experts"][on]
    counts = torch.bincount(kept[kept >= 0].long(), minlength=case["E"])
    n, total = int(on.sum()), int(counts.sum())
    got = {"loss": torch.zeros((), dtype=torch.float64, device="cuda"), "counts": counts.to(torch.int32)}
    slope = torch.zeros(case["E"], dtype=torch.float64, device="cuda")
    if n and total:
        slope = case["E"] * counts.double() / (float(total) * n)
        got["loss"] = torch.dot(slope, p[on].sum(0))
    if case["train"]:
        a = slope * s["grad"].double()
        got["dlogits"] = torch.where(on[:, None], p * (a[None, :] - torch.mv(p, a)[:, None]), 0.0)
    return got


# ------------------------------------------------------------------------------ floors
def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n, es = case["N"] * case["K"], SZ[case["dtype"]]
        scales = case["N"] * math.ceil(case["K"] / case["group"]) * SZ[case["scale"]]
        return {"bytes": 2 * n * es + scales, "flops": 4 * n}
    if kind in ("int4", "grouped"):
        K, N, G = case["K"], case["N"], math.ceil(case["K"] / case["group"])
        one = N * ((K + 1) // 2 + G * (SZ[case["scale"]] + (1 if case["zero"] else 0)))
        if kind == "int4":
            M = case["M"]
            more = 2 * N if case["bias"] else 0
            return {"bytes": one + more + 2 * M * (K + N), "flops": 2 * M * N * K}
        n, E = case["T"] * case["k"], case["E"]
        used = E * (1 - (1 - case["k"] / E) ** case["T"])  # experts that some token chose, at even odds
        return {"bytes": int(used * one) + 4 * E + 2 * n * (K + N), "flops": 2 * n * K * N}
    T, E, k, es = case["T"], case["E"], case["k"], SZ[case["dtype"]]
    if kind == "route":
        grads = 4 * T * k + T * E * es if case["train"] else 0
        return {"bytes": T * E * es + 8 * T * k + grads, "flops": (8 if case["train"] else 5) * T * E}
    # the loss needs every row before the first gradient; the scores are counted once
    grads = T * E * es if case["train"] else 0
    return {"bytes": T * E * es + 4 * T * k + (T if case["pad"] else 0) + grads,
            "flops": (8 if case["train"] else 5) * T * E}
