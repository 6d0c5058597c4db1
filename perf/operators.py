"""Workloads of the int8 and expert-routing operators: what is timed, on which inputs.

A case is one pass through an operator as a program calls it.  ``own = False`` computes it
with elementary torch operations in 32 bits, ``own = True`` with this package's operators;
``exact`` gives the definition's value in 64 bits.

Kinds of case:

* ``quantize``  rows of floats to int8 rows with one scale each; the result is returned as
  the values it stands for.
* ``scaled``    int8 product with a scale for each token and each output channel; from int8
  tokens, or from float tokens that the pass quantizes first.
* ``grouped``   the same with one weight matrix per expert over rows sorted by expert; from
  sorted int8 rows, or from routed float tokens (sort, gather with quantization, product).
* ``dispatch``  tokens sorted by expert and gathered in that order.
* ``combine``   expert rows back to their tokens, weighted.
* ``train``     combine, its gradients, and the gradient of the gather.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SZ = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decode step's activations of 16 sequences: latency
        dict(name="quantize_decode", kind="quantize", rows=16, cols=4096, dtype="bf16"),
        # the activations of a long prefill, or a weight matrix: bandwidth
        dict(name="quantize_prefill", kind="quantize", rows=16384, cols=8192, dtype="bf16"),
        # one token through a feed-forward projection, quantized on the way
        dict(name="scaled_decode", kind="scaled", M=1, K=4096, N=14336, tokens="bf16", out="bf16", layout="nk",
             bias=False),
        # nothing aligned: row pitches that are no multiple of 16 bytes, a ragged tile on each side
        dict(name="scaled_odd", kind="scaled", M=777, K=4100, N=2051, tokens="int8", out="f32", layout="kn", bias=True),
        # a prefill's projection on int8 operands: tensor cores
        dict(name="scaled_8192", kind="scaled", M=8192, K=8192, N=8192, tokens="int8", out="bf16", layout="nk",
             bias=False),
        # 8 tokens decoded through 2 of 8 experts each: the weights' bytes
        dict(name="grouped_decode", kind="grouped", T=8, k=2, E=8, K=4096, N=14336, tokens="bf16", out="bf16",
             skew=0.5, drop=0.0),
        # many small experts, uneven, some entries dropped by a capacity limit
        dict(name="grouped_many", kind="grouped", T=1000, k=8, E=64, K=2048, N=1536, tokens="f16", out="f16",
             skew=0.5, drop=0.05),
        # a prefill through 8 large experts on rows sorted beforehand
        dict(name="grouped_prefill", kind="grouped", T=8192, k=2, E=8, K=4096, N=14336, tokens="int8", out="bf16",
             skew=0.5, drop=0.0),
        # one decode step's routing
        dict(name="dispatch_decode", kind="dispatch", T=16, k=2, E=8, H=4096, dtype="bf16", skew=0.5, drop=0.0),
        # a prefill's or training step's routing
        dict(name="dispatch_prefill", kind="dispatch", T=8192, k=8, E=64, H=4096, dtype="bf16", skew=0.5, drop=0.02),
        # the experts' answers of one decode step, summed into their tokens
        dict(name="combine_decode", kind="combine", T=16, k=2, E=8, H=4096, dtype="bf16", skew=0.5, drop=0.0),
        # the same in training, with every gradient
        dict(name="train_8192", kind="train", T=8192, k=8, E=64, H=4096, dtype="bf16", skew=0.5, drop=0.02),
    ]


def draw(rng):
    def log(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return n if n < 64 else n | 1

    def size(lo, hi):  # a power of two, an odd number of 16s, or odd
        n, how = log(lo, hi), rng.randrange(3)
        if how == 0:
            return max(lo, 1 << (n.bit_length() - 1))
        return n // 32 * 32 + 16 if how == 1 else n | 1

    kind = rng.choice(["quantize", "scaled", "scaled", "grouped", "grouped", "dispatch", "combine", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "quantize":
        rows, cols = log(1, 16384), size(64, 16384)
        return dict(kind=kind, rows=max(1, min(rows, 16384 * 8192 // cols)), cols=cols, dtype=dtype)
    if kind == "scaled":
        M, K, N = log(1, 8192), size(64, 16384), size(64, 16384)
        M = max(1, min(M, 8192 ** 3 // (K * N)))
        return dict(kind=kind, M=M, K=K, N=N, tokens=rng.choice(["int8", "bf16", "f16", "f32"]), out=dtype,
                    layout=rng.choice(["nk", "nk", "kn"]), bias=rng.random() < 0.3)
    skew, drop = rng.choice([0.0, 0.5, 1.5]), rng.choice([0.0, 0.0, 0.05, 0.3])
    T, k = log(1, 8192), rng.choice([1, 2, 4, 8])
    E = rng.choice([e for e in (4, 8, 16, 60, 64, 128) if e >= k])
    if kind == "grouped":
        T = min(T, 16384 // k)
        K = size(128, 4096)
        N = max(128, min(size(128, 14336), 8 * 4096 * 14336 // (E * K) // 32 * 32 - 16))
        return dict(kind=kind, T=T, k=k, E=E, K=K, N=N, tokens=rng.choice(["int8", "bf16", "f16"]), out=dtype,
                    skew=skew, drop=drop)
    H = size(64, 8192)
    es = SZ[dtype]
    T = max(1, min(T, 8192 * 8 * 4096 * 2 // (k * H * es)))
    return dict(kind=kind, T=T, k=k, E=E, H=H, dtype=dtype, skew=skew, drop=drop)


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


def _ints(shape, g):
    """Quantized normal values: a row's largest of a few thousand lies near four deviations."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    return (x * 32).round_().clamp_(-127, 127).to(torch.int8)


def _route(case, g):
    """Distinct experts of each token by its router's scores, their weights, and the order by
    expert; an entry that its expert has no room for has the number -1."""
    T, k, E = case["T"], case["k"], case["E"]
    score = torch.randn((T, E), generator=g, device="cuda")
    score = score + case["skew"] * torch.randn(E, generator=g, device="cuda")
    top, ids = torch.topk(score, k, dim=1)
    weights = torch.softmax(top, dim=1)
    lost = torch.rand((T, k), generator=g, device="cuda") < case["drop"]
    return torch.where(lost, -1, ids), weights


def prepare(case, seed):
    g = _gen(seed)
    kind, s = case["kind"], {"case": case}
    if kind == "quantize":
        s["x"] = _floats((case["rows"], case["cols"]), DT[case["dtype"]], g)
        return s
    if kind == "scaled":
        M, K, N = case["M"], case["K"], case["N"]
        if case["tokens"] == "int8":
            s["a"] = _ints((M, K), g)
            s["sa"] = torch.rand(M, generator=g, device="cuda") * 0.02 + 0.01
        else:
            s["x"] = _floats((M, K), DT[case["tokens"]], g)
        s["w"] = _ints((N, K), g).t() if case["layout"] == "nk" else _ints((K, N), g)
        s["sw"] = torch.rand(N, generator=g, device="cuda") * 2e-4 + 5e-4
        s["bias"] = _floats((N,), DT[case["out"]], g) if case["bias"] else None
        return s
    s["ids"], s["weights"] = _route(case, g)
    n = case["T"] * case["k"]
    if kind == "grouped":
        K, N, E = case["K"], case["N"], case["E"]
        if case["tokens"] == "int8":
            s["a"] = _ints((n, K), g)
            s["sa"] = torch.rand(n, generator=g, device="cuda") * 0.02 + 0.01
            s["order"], s["position"], s["offsets"] = _sorted(s["ids"], E)
        else:
            s["x"] = _floats((case["T"], K), DT[case["tokens"]], g)
        s["w"] = _ints((E, N, K), g).transpose(1, 2)
        s["sw"] = torch.rand((E, N), generator=g, device="cuda") * 2e-4 + 5e-4
        return s
    dt = DT[case["dtype"]]
    if kind == "dispatch":
        s["x"] = _floats((case["T"], case["H"]), dt, g)
        return s
    s["order"], s["position"], s["offsets"] = _sorted(s["ids"], case["E"])
    s["y"] = _floats((n, case["H"]), dt, g)
    if kind == "train":
        s["dout"] = _floats((case["T"], case["H"]), dt, g)
        s["dxs"] = _floats((n, case["H"]), dt, g)
    return s


# ------------------------------------------------------------------------------ plain forms
def _sorted(ids, E):
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    upto = (key[:, None] < torch.arange(E + 1, device=key.device)[None, :]).sum(0)
    return order.to(torch.int32), position.to(torch.int32).reshape(ids.shape), upto.to(torch.int32)


def _quantized(x):
    xf = x.float()
    amax = xf.abs().amax(1, keepdim=True)
    q = torch.round(xf * 127 / torch.where(amax == 0, 1.0, amax))
    return q, amax[:, 0] / 127


def _plain_scaled(s):
    c = s["case"]
    q, sa = (s["a"].float(), s["sa"]) if c["tokens"] == "int8" else _quantized(s["x"])
    y = (q @ s["w"].float()) * sa[:, None] * s["sw"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DT[c["out"]])


def _plain_grouped(s):
    c = s["case"]
    E = c["E"]
    if c["tokens"] == "int8":
        q, sa, offsets = s["a"].float(), s["sa"], s["offsets"]
    else:
        order, _, offsets = _sorted(s["ids"], E)
        q, sa = _quantized(s["x"])
        at = (order // c["k"]).long()
        q, sa = q[at], sa[at]
    row = torch.arange(q.shape[0], device=q.device)
    e = (row[:, None] >= offsets[None, 1:]).sum(1)  # E for a dropped entry
    room = max(1, int((offsets[1:] - offsets[:-1]).max()))
    kept = e < E
    e = torch.where(kept, e, 0)
    r = torch.where(kept, row - offsets[e], room)   # the spare row takes the dropped ones
    padded = torch.zeros((E, room + 1, q.shape[1]), device=q.device)
    padded[e, r] = q
    y = torch.bmm(padded, s["w"].float())[e, r]
    y = y * sa[:, None] * s["sw"][e]
    return {"y": torch.where(kept[:, None], y, 0.0).to(DT[c["out"]]), "offsets": offsets}


def _taken(rows, s):
    """The rows of each token's entries in 32 bits, zero for dropped ones: [T, k, H]."""
    kept = s["position"] < s["offsets"][-1]
    return torch.where(kept[..., None], rows[s["position"].long()].float(), 0.0)


def _plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        q, scale = _quantized(s["x"])
        return {"values": q * scale[:, None], "scale": scale}
    if kind == "scaled":
        return _plain_scaled(s)
    if kind == "grouped":
        return _plain_grouped(s)
    if kind == "dispatch":
        order, position, offsets = _sorted(s["ids"], c["E"])
        kept = torch.arange(order.numel(), device=order.device) < offsets[-1]
        rows = torch.where(kept[:, None], s["x"][(order // c["k"]).long()].float(), 0.0)
        return {"rows": rows.to(s["x"].dtype), "order": order, "position": position, "offsets": offsets}
    y = _taken(s["y"], s)
    out = {"out": (y * s["weights"][..., None]).sum(1).to(s["y"].dtype)}
    if kind == "train":
        dout = s["dout"].float()
        kept = s["position"] < s["offsets"][-1]
        dy = torch.zeros_like(s["y"])
        dy[s["position"].long()] = torch.where(kept[..., None], dout[:, None] * s["weights"][..., None],
                                               0.0).to(s["y"].dtype)
        out["dy"] = dy
        out["dweights"] = (y * dout[:, None]).sum(-1)
        out["dx"] = _taken(s["dxs"], s).sum(1).to(s["dxs"].dtype)
    return out


# ------------------------------------------------------------------------------ this package
def _own(s):
    import metalblas_b200 as mb
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        q, scale = mb.quantize(s["x"])
        return {"values": q * scale[:, None], "scale": scale}
    if kind == "scaled":
        q, sa = (s["a"], s["sa"]) if c["tokens"] == "int8" else mb.quantize(s["x"])
        return mb.scaled_mm(q, s["w"], sa, s["sw"], bias=s["bias"], out_dtype=DT[c["out"]])
    if kind == "grouped":
        if c["tokens"] == "int8":
            q, sa, offsets = s["a"], s["sa"], s["offsets"]
        else:
            order = mb.expert_sort(s["ids"], c["E"])
            q, sa = mb.expert_gather_quantize(s["x"], order)
            offsets = order.offsets
        y = mb.grouped_scaled_mm(q, s["w"], sa, s["sw"], offsets, out_dtype=DT[c["out"]])
        return {"y": y, "offsets": offsets}
    if kind == "dispatch":
        order = mb.expert_sort(s["ids"], c["E"])
        rows = mb.expert_gather(s["x"], order)
        return {"rows": rows, "order": order.order, "position": order.position, "offsets": order.offsets}
    order = mb.ExpertOrder(s["order"], s["position"], s["offsets"])
    out = {"out": mb.expert_combine(s["y"], s["weights"], order)}
    if kind == "train":
        out["dy"], out["dweights"] = mb.expert_combine_backward(s["dout"], s["y"], s["weights"], order)
        out["dx"] = mb.expert_gather_backward(s["dxs"], order)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------ 64 bits
def _exact_rows(x):
    x = x.double()
    largest = x.abs().max(dim=1).values
    scale = largest / 127
    steps = x * 127 / largest.clamp_min(1e-300)[:, None]
    return steps.round(), scale


def _exact_order(ids, E):
    """Entries of expert 0 in their order, then of expert 1, ..., then the dropped ones."""
    flat = ids.reshape(-1)
    lists = [torch.nonzero(flat == e).reshape(-1) for e in range(E)]
    ends, n = [0], 0
    for one in lists:
        n += one.numel()
        ends.append(n)
    order = torch.cat(lists + [torch.nonzero((flat < 0) | (flat >= E)).reshape(-1)])
    position = torch.empty(flat.numel(), dtype=torch.int64, device=flat.device)
    position.scatter_(0, order, torch.arange(flat.numel(), device=flat.device))
    return order, position, ends


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        q, scale = _exact_rows(s["x"])
        return {"values": q * scale[:, None], "scale": scale}
    if kind == "scaled":
        q, sa = (s["a"].double(), s["sa"].double()) if "a" in s else _exact_rows(s["x"])
        y = torch.matmul(q * sa[:, None], s["w"].double() * s["sw"].double())
        return y if s["bias"] is None else y.add_(s["bias"].double())
    order, position, ends = _exact_order(s["ids"], case["E"])
    n, k = order.numel(), case["k"]
    i32 = dict(dtype=torch.int32, device="cuda")
    if kind == "grouped":
        q, sa = (s["a"].double(), s["sa"].double()) if "a" in s else _exact_rows(s["x"])
        y = torch.zeros((n, case["N"]), dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            lo, hi = ends[e], ends[e + 1]
            if hi > lo:
                at = slice(lo, hi) if "a" in s else torch.div(order[lo:hi], k, rounding_mode="floor")
                y[lo:hi] = torch.matmul(q[at] * sa[at][:, None], s["w"][e].double()) * s["sw"][e].double()
        return {"y": y, "offsets": torch.tensor(ends, **i32)}
    if kind == "dispatch":
        rows = torch.zeros((n, case["H"]), dtype=torch.float64, device="cuda")
        m = ends[-1]
        rows[:m] = s["x"].double().index_select(0, torch.div(order[:m], k, rounding_mode="floor"))
        return {"rows": rows, "order": order.to(torch.int32), "position": position.to(torch.int32).reshape(-1, k),
                "offsets": torch.tensor(ends, **i32)}
    T, H, m = case["T"], case["H"], ends[-1]
    token = torch.div(order[:m], k, rounding_mode="floor")
    w = s["weights"].double().reshape(-1).index_select(0, order[:m])
    out = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    out.index_add_(0, token, s["y"][:m].double() * w[:, None])
    got = {"out": out}
    if kind == "train":
        d = s["dout"].double().index_select(0, token)
        dw = torch.zeros(n, dtype=torch.float64, device="cuda")
        dw[order[:m]] = torch.linalg.vecdot(d, s["y"][:m].double())
        dy = torch.zeros((n, H), dtype=torch.float64, device="cuda")
        dy[:m] = d.mul_(w[:, None])
        dx = torch.zeros((T, H), dtype=torch.float64, device="cuda")
        dx.index_add_(0, token, s["dxs"][:m].double())
        got.update(dy=dy, dweights=dw.reshape(T, k), dx=dx)
    return got


# ------------------------------------------------------------------------------ floors
def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SZ[case["dtype"]] + 1) + 4 * case["rows"], "flops": 3 * n}
    if kind == "scaled":
        M, K, N = case["M"], case["K"], case["N"]
        a = M * (K + 4) if case["tokens"] == "int8" else M * K * SZ[case["tokens"]]
        b = K * N + 4 * N + (N * SZ[case["out"]] if case["bias"] else 0)
        return {"bytes": a + b + M * N * SZ[case["out"]], "flops": 2 * M * N * K}
    T, k, E = case["T"], case["k"], case["E"]
    n = T * k
    if kind == "grouped":
        K, N = case["K"], case["N"]
        a = n * (K + 4) if case["tokens"] == "int8" else T * K * SZ[case["tokens"]] + 8 * n
        used = E * (1 - (1 - k / E) ** T)  # experts that some token chose, at even odds
        return {"bytes": int(a + used * (K * N + 4 * N) + 4 * E + n * N * SZ[case["out"]]), "flops": 2 * n * K * N}
    H, es = case["H"], SZ[case["dtype"]]
    if kind == "dispatch":
        return {"bytes": 16 * n + 4 * E + (T + n) * H * es, "flops": n}
    if kind == "combine":
        return {"bytes": 8 * n + 4 * E + (n + T) * H * es, "flops": 2 * n * H}
    # y, dout and dxs once; out, dy, dx and the weights' gradient
    return {"bytes": 12 * n + 4 * E + (3 * n + 3 * T) * H * es, "flops": 6 * n * H}
