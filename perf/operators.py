"""Cases, plain forms and measured calls of the framework's dot-product attention, node embedding and orthogonalised
updates.

`run` computes an operator on the inputs that `prepare` made: with `own` false in its plain form, elementary torch
operations in 32 bits rounded once at the end; with `own` true through the calls of `gat_amd.ops` that a user makes.
`exact` states the same operators in 64 bits, one graph, one table row or one matrix at a time.

The operators
    attend   out[b,i,h] = sum_j P_ij v[b,j,g],  P = softmax_j(scale <q[b,i,h], k[b,j,g]> + bias_mat[b,i,j]),
             g = h // (H / Hkv), over the keys j < key_sizes[b] whose bias is above -1e8; a query without such a key, or
             behind query_sizes[b], gives zeros.  "train" cases also return the gradients of q, k and v.
    embed    out[t] = scale table[ids[t]]; an id outside [0, rows) stands for padding: a row of zeros, no gradient.
             Returned with the gradient of the table.
    ortho    five steps X <- a X + b (X X^T) X + c (X X^T)^2 X of each matrix, from X = x / (|x|_F + 1e-7).
"""
import math

import torch

own = False

NS_STEPS, NS_EPS, NS_ABC = 5, 1e-7, (3.4445, -4.7750, 2.0315)
MASK = -1e9                 # what adj_to_bias puts where there is no edge
ATTENDED = -1e8             # an entry whose bias is not above this is not attended
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _attend(name, train, B, Nq, Nk, H, Hkv, D, dtype, density, ragged):
    return dict(name=name, op="attend", train=train, B=B, Nq=Nq, Nk=Nk, H=H, Hkv=Hkv, D=D, dtype=dtype, density=density, ragged=ragged)


def listed():
    return [
        # one node's answer from a trained model: one query row of a 246-node atlas; only latency counts
        _attend("serve-atlas-1", False, 1, 1, 246, 8, 8, 8, "f32", 0.1, False),
        # one new node per graph against long stored key and value rows of unequal lengths, eight query heads on two shared ones
        _attend("serve-long", False, 2, 1, 131072, 8, 2, 64, "bf16", 0.0, True),
        # a training step's attention at the brain-network autoencoder's sizes: batch 50, 246 nodes, 6 heads of 64
        _attend("train-atlas-50", True, 50, 246, 246, 6, 6, 64, "f32", 0.1, False),
        # the Cora graph through its dense mask, 8 heads of 8: nearly every entry is masked
        _attend("train-cora", True, 1, 2708, 2708, 8, 8, 8, "f32", 0.0015, False),
        # a large batch of small graphs, 8 heads of 8
        _attend("train-atlas-1024", True, 1024, 246, 246, 8, 8, 8, "f32", 0.1, False),
        # a few large padded graphs without a mask, wide shared heads, 16-bit rows
        _attend("train-wide", True, 4, 4096, 4096, 16, 4, 128, "bf16", 0.0, True),
        # one learned row per node of Cora, looked up for all nodes once
        dict(name="embed-cora", op="embed", tokens=2708, rows=2708, width=64, dtype="f32", skew=0.0, pad=0.0),
        # one learned row per region of the atlas, looked up by 1024 graphs of 246 nodes: every row is hit a thousand times
        dict(name="embed-atlas", op="embed", tokens=251904, rows=246, width=64, dtype="bf16", skew=0.0, pad=0.02),
        # four million sampled neighbours of a products-shaped graph, hubs sampled far more often than the rest
        dict(name="embed-products", op="embed", tokens=4000037, rows=2449029, width=100, dtype="f32", skew=0.8, pad=0.0),
        # the attention kernels of the brain-network autoencoder: 2 branches x 5 rounds x 6 heads, 64 x 64 each
        dict(name="ortho-atlas", op="ortho", batch=60, m=64, n=64, dtype="f32"),
        # the eight head kernels of Cora's first layer
        dict(name="ortho-cora", op="ortho", batch=8, m=1433, n=8, dtype="f32"),
        # one large dense layer with a 16-bit gradient
        dict(name="ortho-wide", op="ortho", batch=1, m=2048, n=4096, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("serve", "train", "embed", "ortho"))
    dtype = rng.choice(("f32", "bf16"))
    if kind == "serve":
        Hkv, group = rng.choice((1, 2, 4)), rng.choice((1, 2, 3, 4))
        D = rng.choice((8, 16, 24, 32, 64, 100, 128))
        Nk = _log(rng, 1, 131072)
        cap = max(1, min(16, 2 * 131072 * 2 * 64 // (Nk * Hkv * D)))
        B, Nq = rng.randint(1, cap), rng.choice((1, 1, 1, 2, 5))
        density = rng.choice((0.0, 0.1, 0.5)) if Nk <= 8192 else 0.0
        return {k: v for k, v in _attend("", False, B, Nq, Nk, Hkv * group, Hkv, D, dtype, density, rng.random() < 0.5).items() if k != "name"}
    if kind == "train":
        Hkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 3))
        D = rng.choice((8, 16, 20, 32, 64, 96, 128))
        N = _log(rng, 16, 4096)
        cap = 4 * 16 * 4096 * 4096 * 128 // 4                       # a quarter of the largest listed case's products
        B = max(1, min(1024, _log(rng, 1, 1024), cap // (N * N * Hkv * group * max(D, 32))))
        return {k: v for k, v in _attend("", True, B, N, N, Hkv * group, Hkv, D, dtype, rng.choice((0.0, 0.02, 0.1, 0.5)), rng.random() < 0.5).items() if k != "name"}
    if kind == "embed":
        width = rng.choice((7, 8, 33, 64, 100, 128, 256, 500))
        tokens = min(_log(rng, 1, 4000037), 100 * 4000037 // width)
        rows = min(_log(rng, 1, 2449029), 100 * 2449029 // width)
        return dict(op="embed", tokens=tokens, rows=rows, width=width, dtype=dtype, skew=rng.choice((0.0, 0.5, 0.8)), pad=rng.choice((0.0, 0.1)))
    m, n = _log(rng, 4, 4096), _log(rng, 4, 4096)
    if m * n > 2048 * 4096:
        n = 2048 * 4096 // m
    batch = max(1, min(64, _log(rng, 1, 64), 2048 * 2048 * 4096 // (m * n * max(32, min(m, n)))))
    return dict(op="ortho", batch=batch, m=m, n=n, dtype=dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if case["op"] == "attend":
        B, Nq, Nk, H, Hkv, D = (case[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "D"))
        s = {"case": case, "scale": D ** -0.5, "q": normal(B, Nq, H, D).to(dt), "k": normal(B, Nk, Hkv, D).to(dt), "v": normal(B, Nk, Hkv, D).to(dt),
             "bias": None, "key_sizes": None, "query_sizes": None, "dout": None}
        if case["density"] > 0.0:
            edge = torch.rand((B, Nq, Nk), generator=gen, device=dev) < case["density"]
            if Nq == Nk:                                            # self-loops, but for every 97th node, whose row stays as drawn
                i = torch.arange(Nq, device=dev)
                i = i[i % 97 != 5]
                edge[:, i, i] = True
            s["bias"] = torch.where(edge, 0.0, MASK).to(torch.float32)
        if case["ragged"]:
            s["key_sizes"] = torch.randint(max(1, Nk // 2), Nk + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            if Nq == Nk:
                s["query_sizes"] = s["key_sizes"]
        if case["train"]:
            s["dout"] = normal(B, Nq, H, D).to(dt)
        return s
    if case["op"] == "embed":
        t, rows, width = case["tokens"], case["rows"], case["width"]
        u = torch.rand(t, generator=gen, device=dev, dtype=torch.float64)
        rank = (u ** (1.0 / (1.0 - case["skew"])) * rows).long().clamp_(max=rows - 1)
        rank = torch.randperm(rows, generator=gen, device=dev)[rank]               # which rows are the frequent ones is not their order in the table
        if case["pad"] > 0.0:
            rank = torch.where(torch.rand(t, generator=gen, device=dev) < case["pad"], -1, rank)
        return {"case": case, "ids": rank, "table": (0.05 * normal(rows, width)).to(dt), "dout": normal(t, width).to(dt), "scale": float(width) ** 0.5}
    b, m, n = case["batch"], case["m"], case["n"]
    r = max(1, min(m, n) // 8)                                      # a gradient: a few strong directions and noise
    x = normal(b, m, r) @ normal(b, r, n) / r ** 0.5 + 0.3 * normal(b, m, n)
    return {"case": case, "x": (1e-3 * x).to(dt)}


def _attend_plain(s):
    q, k, v = (s[x].float().transpose(1, 2) for x in ("q", "k", "v"))                      # [B, heads, N, D]
    dt, (B, H, Nq, D), (Hkv, Nk) = s["q"].dtype, q.shape, k.shape[1:3]
    G = H // Hkv
    q = q.reshape(B, Hkv, G * Nq, D)
    k, v = k.contiguous(), v.contiguous()
    z = (q @ k.transpose(2, 3)).mul_(s["scale"]).reshape(B, H, Nq, Nk)
    seen = None
    if s["bias"] is not None:
        z += s["bias"][:, None]
        seen = s["bias"][:, None] > ATTENDED
    if s["key_sizes"] is not None:
        inside = torch.arange(Nk, device=z.device)[None, None, None] < s["key_sizes"][:, None, None, None]
        seen = inside if seen is None else seen & inside
    if s["query_sizes"] is not None:
        seen = seen & (torch.arange(Nq, device=z.device)[None, None, :, None] < s["query_sizes"][:, None, None, None])
    if seen is not None:
        z = torch.where(seen, z, -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True).clamp_(min=-3e38))
    p /= p.sum(-1, keepdim=True).clamp_(min=1e-30)
    p = p.reshape(B, Hkv, G * Nq, Nk)
    o = p @ v
    rows = lambda x, heads: x.reshape(B, heads, -1, D).transpose(1, 2).to(dt)
    if s["dout"] is None:
        return rows(o, H)
    do = s["dout"].float().transpose(1, 2).reshape(B, Hkv, G * Nq, D)
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    return rows(o, H), rows(ds @ k, H), rows(ds.transpose(2, 3) @ q, Hkv), rows(dv, Hkv)


def _embed_plain(s):
    ids, table = s["ids"], s["table"]
    ok = ((ids >= 0) & (ids < table.shape[0]))[:, None]
    at = ids.clamp(0, table.shape[0] - 1)
    out = torch.where(ok, table[at].float() * s["scale"], 0.0).to(table.dtype)
    grad = torch.zeros(table.shape, device=table.device).index_add_(0, at, torch.where(ok, s["dout"].float(), 0.0))
    return out, (grad * s["scale"]).to(table.dtype)


def _ortho_plain(s):
    x = s["x"].float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.double().pow(2).sum((1, 2), keepdim=True).sqrt() + NS_EPS).float()
    a, b, c = NS_ABC
    for _ in range(NS_STEPS):
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.transpose(1, 2) if tall else x).to(s["x"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attend": _attend_plain, "embed": _embed_plain, "ortho": _ortho_plain}[op](s)
    from gat_amd import ops
    if op == "attend":
        if s["dout"] is None:
            return ops.dot_attention(s["q"], s["k"], s["v"], s["bias"], key_sizes=s["key_sizes"], query_sizes=s["query_sizes"], scale=s["scale"])
        leaves = [s[x].detach().requires_grad_() for x in ("q", "k", "v")]
        out = ops.dot_attention(*leaves, s["bias"], key_sizes=s["key_sizes"], query_sizes=s["query_sizes"], scale=s["scale"])
        return (out.detach(), *torch.autograd.grad(out, leaves, s["dout"]))
    if op == "embed":
        table = s["table"].detach().requires_grad_()
        out = ops.embedding(s["ids"], table, scale=s["scale"])
        return out.detach(), torch.autograd.grad(out, table, s["dout"])[0]
    return ops.newton_schulz(s["x"], steps=NS_STEPS, eps=NS_EPS, coefficients=NS_ABC)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "attend":
        B, Nq, Nk, H, Hkv, D = (case[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "D"))
        q, kv = B * Nq * H * D * size, B * Nk * Hkv * D * size
        share = 0.75 if case["ragged"] else 1.0                                    # sizes are even between half and all of the rows
        pairs = B * H * Nq * Nk * (share * share if case["ragged"] and Nq == Nk else share)
        bias = 0
        if case["density"] > 0.0:                                                  # a mask is read whole, the products are those of the entries that it leaves
            bias, pairs = 4 * B * Nq * Nk, pairs * case["density"]
        if not case["train"]:
            return {"bytes": 2 * q + share * 2 * kv + bias, "flops": 4 * pairs * D}
        return {"bytes": 4 * q + 4 * kv + bias, "flops": 14 * pairs * D}           # 2 products forward, 5 backward
    if case["op"] == "embed":
        t, rows, width = case["tokens"], case["rows"], case["width"]
        looked_up = min(t, rows)                                                   # the rows in use are read once, the gradient is written whole
        return {"bytes": 8 * t + 2 * t * width * size + (looked_up + rows) * width * size, "flops": 2 * t * width}
    b, m, n = case["batch"], max(case["m"], case["n"]), min(case["m"], case["n"])
    step = m * n * (n + 1) + n * n * (n + 1) + 2 * m * n * n                       # the Gram product and its square are symmetric: half of each
    return {"bytes": 2 * b * m * n * size, "flops": NS_STEPS * b * step}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        B, Nq, Nk, H, Hkv, D = (case[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "D"))
        dev, G = s["q"].device, H // Hkv
        out = torch.zeros((B, Nq, H, D), dtype=torch.float64, device=dev)
        dq, dk, dv = torch.zeros_like(out), *(torch.zeros((2, B, Nk, Hkv, D), dtype=torch.float64, device=dev))
        for b in range(B):
            nk = Nk if s["key_sizes"] is None else int(s["key_sizes"][b])
            nq = Nq if s["query_sizes"] is None else int(s["query_sizes"][b])
            allowed = torch.ones((nq, nk), dtype=torch.bool, device=dev) if s["bias"] is None else s["bias"][b, :nq, :nk] > ATTENDED
            plus = 0.0 if s["bias"] is None else s["bias"][b, :nq, :nk].double()
            live = allowed.any(1, keepdim=True)
            for g in range(Hkv):
                q = s["q"][b, :nq, g * G:(g + 1) * G].double().transpose(0, 1)      # [G, nq, D]
                k, v = s["k"][b, :nk, g].double(), s["v"][b, :nk, g].double()
                z = (torch.matmul(q, k.t()) * s["scale"] + plus).masked_fill(~allowed, -math.inf)
                p = torch.softmax(z, dim=-1)
                p = torch.where(live, p, torch.zeros((), dtype=p.dtype, device=dev))
                o = torch.matmul(p, v)
                out[b, :nq, g * G:(g + 1) * G] = o.transpose(0, 1)
                if case["train"]:
                    do = s["dout"][b, :nq, g * G:(g + 1) * G].double().transpose(0, 1)
                    dp = torch.matmul(do, v.t())
                    dz = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
                    dq[b, :nq, g * G:(g + 1) * G] = torch.matmul(dz, k).transpose(0, 1)
                    dk[b, :nk, g] = torch.matmul(dz.transpose(1, 2), q).sum(0)
                    dv[b, :nk, g] = torch.matmul(p.transpose(1, 2), do).sum(0)
        return (out, dq, dk, dv) if case["train"] else out
    if case["op"] == "embed":
        rows, width = s["table"].shape
        pad = torch.zeros((1, width), dtype=torch.float64, device=s["table"].device)
        at = torch.where((s["ids"] < 0) | (s["ids"] >= rows), rows, s["ids"])
        out = torch.cat([s["table"].double(), pad])[at] * s["scale"]
        order = torch.argsort(at, stable=True)                                     # tokens of one row side by side: its sum is a difference
        ends = torch.cumsum(torch.bincount(at, minlength=rows + 1), 0)[:rows]
        grad = torch.empty((rows, width), dtype=torch.float64, device=at.device)
        for c in range(0, width, 16):
            total = torch.cumsum(s["dout"][:, c:c + 16].double()[order], 0)
            upto = torch.cat([torch.zeros_like(total[:1]), total])[ends]
            grad[:, c:c + 16] = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1]))
        return out, grad * s["scale"]
    a, b, c = NS_ABC
    out = torch.empty(s["x"].shape, dtype=torch.float64, device=s["x"].device)
    for i, x in enumerate(s["x"].double()):
        x = x / (torch.linalg.vector_norm(x) + NS_EPS)
        for _ in range(NS_STEPS):                                                  # a X + b X (X^T X) + c X (X^T X)^2, from the right
            if x.shape[0] >= x.shape[1]:
                gram = x.t() @ x
                x = a * x + b * (x @ gram) + c * (x @ gram @ gram)
            else:
                gram = x @ x.t()
                x = a * x + b * (gram @ x) + c * (gram @ (gram @ x))
        out[i] = x
    return out
