"""Dense attention with a learned bias by buckets, and the buckets of molecules: the calls that programs make of them, as cases.

Attention layers of the trunk (8 heads of 64 channels) see all atoms of a molecule or all tokens of a cell in sorted order; sequence models of
generic widths beside them share key heads, look back only and step one token at a time behind the keys they keep.

Dense attention: out_i = sum_j p_ij v_j, p_i = softmax_j(scale q_i . k_j + bias[bucket(i, j)]) over the keys that query i sees; a query that sees
none returns zeros.  The last query of an entry stands at its last key.  The learned table has one row for each bucket and one column for each head.  The bucket of
a pair goes by the offset j - i (a map of 2 L + 1 entries from -L to L, whose ends stand for all beyond) or is given for every pair.
Distance buckets: how many of the ascending edges lie at or below the distance of two atoms.
"""
from __future__ import annotations

import math

import torch

own = False  # True: the package's operators; False: their plain form

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _attn(batch, queries, keys, heads, head_dim, *, kv_heads=0, dtype="bf16", form="heads", causal=False, bias="none", buckets=32, reach=128,
          fill=1.0, holes=0.0, train=False):  # fmt: skip
    """``fill``: the shortest entry of a batch, as a part of the padded length; ``holes``: the part of the keys that the key mask hides."""
    return {"kind": "attn", "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads or heads, "head_dim": head_dim,
            "dtype": dtype, "form": form, "causal": causal, "bias": bias, "buckets": buckets, "reach": reach, "fill": fill, "holes": holes,
            "train": train}  # fmt: skip


def listed():
    return [
        # one molecule of 29 atoms in a sampling loop, biased by distances: launches and the host path count
        {"name": "attn_molecule", **_attn(1, 29, 29, 8, 64, form="packed", bias="pair")},
        # an attention layer of the training step on 1024 QM9-sized molecules: output, gradients of the projection and of the table
        {"name": "attn_qm9_train", **_attn(1024, 29, 29, 8, 64, form="packed", bias="pair", fill=0.31, train=True)},
        # the same on 64 drug-sized molecules, with a finer table
        {"name": "attn_drug_train", **_attn(64, 192, 192, 8, 64, form="packed", bias="pair", buckets=64, fill=0.1, train=True)},
        # two large cells in sorted order, biased by the offset: the largest call
        {"name": "attn_cells_train", **_attn(2, 4096, 4096, 8, 64, bias="offset", train=True)},
        # a prompt in half precision that looks back, shared key heads
        {"name": "attn_prompt", **_attn(1, 4111, 4111, 16, 128, kv_heads=4, dtype="f16", causal=True, bias="offset")},
        # a training step on four such sequences without a bias
        {"name": "attn_causal_train", **_attn(4, 1024, 1024, 16, 128, kv_heads=4, causal=True, train=True)},
        # queries of one set on the keys of another, some of which are hidden, narrow heads
        {"name": "attn_holes_train", **_attn(8, 577, 1000, 4, 32, dtype="f16", holes=0.2, fill=0.3, train=True)},
        # single tokens of 64 sequences behind caches of different lengths
        {"name": "attn_tokens", **_attn(64, 1, 4096, 32, 128, kv_heads=8, causal=True, bias="offset", fill=0.1)},
        # a single token behind one long cache
        {"name": "attn_token_long", **_attn(1, 1, 32771, 32, 128, kv_heads=8, causal=True)},
        # buckets for all layers of the training step on 1024 molecules
        {"name": "buckets_qm9", "kind": "buckets", "batch": 1024, "tokens": 29, "buckets": 32, "fill": 0.31},
        # buckets of two cells
        {"name": "buckets_cells", "kind": "buckets", "batch": 2, "tokens": 4096, "buckets": 64, "fill": 1.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more call of the listed ranges."""
    pairs = 2 * 8 * 4096 * 4096
    if rng.random() < 0.2:
        while True:
            batch, tokens = _log(rng, 1, 1024), _log(rng, 12, 4096)
            if batch * tokens * tokens <= 2 * 4096 * 4096:
                return {"kind": "buckets", "batch": batch, "tokens": tokens, "buckets": rng.choice([8, 32, 64, 128]), "fill": rng.choice([0.2, 1.0])}
    while True:
        head_dim = rng.choice([32, 64, 64, 64, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        train = rng.random() < 0.5
        batch, keys = _log(rng, 1, 1024), _log(rng, 1, 32768)
        single = not train and rng.random() < 0.4
        queries = rng.choice([1, 1, 1, 2, 4]) if single else keys if rng.random() < 0.7 else _log(rng, 1, 4096)
        causal = single or (queries <= keys and rng.random() < 0.3)
        bias = rng.choice(["none", "offset", "pair"])
        values = batch * keys * kv_heads * head_dim
        if batch * heads * queries * keys * head_dim * (3.5 if train else 1) <= pairs * 64 * 3.5 and batch * heads * queries * keys <= pairs and (
            values <= 2**28 and batch * queries * heads * head_dim <= 2**27 and (bias != "pair" or batch * queries * keys <= 2**26)):  # fmt: skip
            break
    packed = queries == keys and heads == kv_heads and rng.random() < 0.5
    return _attn(batch, queries, keys, heads, head_dim, kv_heads=kv_heads, dtype=rng.choice(["bf16", "bf16", "f16"]), form="packed" if packed else "heads",
                 causal=causal, bias=bias, buckets=rng.choice([8, 32, 64]), reach=rng.choice([20, 128, 500]), fill=rng.choice([0.2, 0.5, 1.0]),
                 holes=0.0 if causal else rng.choice([0.0, 0.0, 0.2]), train=train)  # fmt: skip


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _counts(g, batch, most, fill):
    """Lengths from ``fill`` of the padded one up, one of them whole."""
    least = max(1, round(most * fill))
    n = torch.randint(least, most + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = most
    return n


def _edges(buckets):
    """Borders of the buckets of a distance, evenly spaced up to 12 units, on the host in 64 bits."""
    return torch.linspace(0.0, 12.0, buckets, dtype=torch.float64)[1:]


def _coords(g, batch, tokens):
    """Atoms spread at the density of a molecule."""
    return _randn(g, batch, tokens, 3, scale=0.9 * tokens ** (1 / 3))


def _bucket_of(xyz, edges):
    """(B, N, N): in 64 bits, for distances next to an edge."""
    x = xyz.double()
    d2 = sum((x[:, :, None, a] - x[:, None, :, a]).square() for a in range(3))
    out = torch.zeros(d2.shape, dtype=torch.uint8, device=x.device)
    for e in edges.tolist():
        out += d2 >= e * e
    return out


def _offset_map(case):
    """Buckets of the offsets -L..L: half of them for each side (all for the past, where later keys are not seen), the near half of those one for each
    offset, the far half evenly over the logarithm."""
    L, total = case["reach"], case["buckets"]
    side = total if case["causal"] else total // 2
    near = max(1, side // 2)

    def rank(n):
        if n < near:
            return n
        return min(side - 1, near + int(math.log(n / near) / math.log(max(2.0, L / near)) * (side - near)))

    return torch.tensor([rank(-o) if o <= 0 else (0 if case["causal"] else side + rank(o)) for o in range(-L, L + 1)], dtype=torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "buckets":
        B, N = case["batch"], case["tokens"]
        return {"case": case, "xyz": _coords(g, B, N), "num": _counts(g, B, N, case["fill"]), "edges": _edges(case["buckets"])}
    dtype = _TYPES[case["dtype"]]
    B, M, N, H, K, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    s = {"case": case, "mask": None, "table": None, "buckets": None}
    s["num_k"] = _counts(g, B, N, case["fill"]) if case["fill"] < 1 else None
    if M == N:
        s["num_q"] = s["num_k"]
    else:  # no more than there are keys, where queries look back
        s["num_q"] = torch.minimum(_counts(g, B, M, case["fill"]), s["num_k"]) if case["fill"] < 1 and M > 1 else None
    if case["holes"]:
        s["mask"] = torch.rand(B, N, generator=g, device="cuda") >= case["holes"]
    if case["form"] == "packed":
        s["qkv"] = _randn(g, B, N, 3 * H * D, dtype=dtype)
        s["leaves"] = [s["qkv"]]
    else:
        s["q"], s["k"], s["v"] = _randn(g, B, H, M, D, dtype=dtype), _randn(g, B, K, N, D, dtype=dtype), _randn(g, B, K, N, D, dtype=dtype)
        s["leaves"] = [s["q"], s["k"], s["v"]]
    if case["bias"] != "none":
        s["table"] = _randn(g, case["buckets"], H, dtype=dtype)
        s["leaves"] = s["leaves"] + [s["table"]]
        if case["bias"] == "offset":
            s["buckets"] = _offset_map(case).cuda()
        elif M == N:
            s["buckets"] = _bucket_of(_coords(g, B, N), _edges(case["buckets"]))
        else:
            s["buckets"] = torch.randint(0, case["buckets"], (B, M, N), generator=g, device="cuda", dtype=torch.uint8)
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_(True)
        s["grad"] = _randn(g, *((B, N, H * D) if case["form"] == "packed" else (B, H, M, D)), dtype=dtype)
    return s


def _operands(s, wide):
    """q (B, K, G, M, D), k and v (B, K, 1, N, D) in the wide type, dout beside q."""
    case = s["case"]
    B, M, N, H, K, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    if case["form"] == "packed":
        q, k, v = s["qkv"].detach().to(wide).view(B, N, 3, H, D).permute(2, 0, 3, 1, 4)
        grad = s["grad"].to(wide).view(B, N, H, D).transpose(1, 2) if case["train"] else None
    else:
        q, k, v = (s[n].detach().to(wide) for n in "qkv")
        grad = s["grad"].to(wide) if case["train"] else None
    grouped = (B, K, H // K, M, D)
    return q.reshape(grouped), k.unsqueeze(2), v.unsqueeze(2), None if grad is None else grad.reshape(grouped)


def _visible(s):
    """(B, M, N) truth values."""
    case = s["case"]
    B, M, N = case["batch"], case["queries"], case["keys"]
    i, j = torch.arange(M, device="cuda")[:, None], torch.arange(N, device="cuda")
    nq = s["num_q"][:, None, None] if s["num_q"] is not None else torch.full((1, 1, 1), M, device="cuda")
    nk = s["num_k"][:, None, None] if s["num_k"] is not None else torch.full((1, 1, 1), N, device="cuda")
    see = (i < nq) & (j < nk)
    if case["causal"]:
        see = see & (j - i <= nk - nq)
    if s["mask"] is not None:
        see = see & s["mask"][:, None, :]
    return see.expand(B, M, N)


def _pair_buckets(s):
    """(1 or B, M, N) int64."""
    case = s["case"]
    if case["bias"] == "pair":
        return s["buckets"].long()
    M, N, L = case["queries"], case["keys"], case["reach"]
    nq = s["num_q"].long()[:, None, None] if s["num_q"] is not None else torch.full((1, 1, 1), M, device="cuda")
    nk = s["num_k"].long()[:, None, None] if s["num_k"] is not None else torch.full((1, 1, 1), N, device="cuda")
    offset = torch.arange(N, device="cuda") - torch.arange(M, device="cuda")[:, None] - (nk - nq)
    return s["buckets"].long()[offset.clamp(-L, L) + L]


def _plain_attn(s):
    case = s["case"]
    B, M, N, H, K, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    q, k, v, grad = _operands(s, torch.float32)
    scale = D**-0.5
    logits = scale * (q @ k.transpose(-1, -2))
    if s["table"] is not None:
        which = _pair_buckets(s)
        table = s["table"].detach().float()
        for h in range(H):
            logits[:, h // (H // K), h % (H // K)] += table[:, h][which]
    see = _visible(s)[:, None, None]
    logits = torch.where(see, logits, -math.inf)
    top = logits.max(dim=-1, keepdim=True).values
    p = torch.exp(logits - torch.where(top > -math.inf, top, 0.0))
    del logits
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    # what is hidden may hold anything
    shown = see.any(3).unsqueeze(-1)
    v = torch.where(shown, v, 0.0)
    out = p @ v
    dtype = s["leaves"][0].dtype

    def merged(t):
        return t.transpose(1, 2).reshape(B, N, H * D) if case["form"] == "packed" else t

    made = [merged(out.reshape(B, H, M, D)).to(dtype)]
    if not case["train"]:
        return made[0]
    dv = (p.transpose(-1, -2) @ grad).sum(2)
    ds = grad @ v.transpose(-1, -2)
    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
    del p
    dq, dk = (scale * (ds @ k)).reshape(B, H, M, D), scale * (ds.transpose(-1, -2) @ q).sum(2)
    if case["form"] == "packed":
        made.append(torch.stack([dq, dk, dv]).permute(1, 3, 0, 2, 4).reshape(B, N, 3 * H * D).to(dtype))
    else:
        made += [t.to(dtype) for t in (dq, dk, dv)]
    if s["table"] is not None:
        ds = ds.reshape(B, H, M * N)
        which = which.expand(B, M, N).reshape(B, M * N)
        dtable = torch.zeros(case["buckets"], H, dtype=torch.float64, device="cuda")  # a long sum
        for b in range(case["buckets"]):
            dtable[b] = torch.einsum("bhp,bp->bh", ds, (which == b).float()).double().sum(0)
        made.append(dtable.to(dtype))
    return made


def _own_attn(s):
    import matterformer_b200 as mfb

    case = s["case"]
    with torch.set_grad_enabled(case["train"]):
        common = {"key_mask": s["mask"], "causal": case["causal"], "bias": s["table"], "buckets": s["buckets"]}
        if case["form"] == "packed":
            out = mfb.dense_attention_packed(s["qkv"], case["heads"], s["num_k"], **common)
        else:
            out = mfb.dense_attention(s["q"], s["k"], s["v"], s["num_k"], s["num_q"], **common)
    return [out, *torch.autograd.grad(out, s["leaves"], s["grad"])] if case["train"] else out


def _real_pairs(s, buckets):
    """Padded atoms have the first bucket."""
    real = torch.arange(s["case"]["tokens"], device="cuda") < s["num"][:, None]
    return torch.where(real[:, :, None] & real[:, None, :], buckets, 0)


def run(state):
    if state["case"]["kind"] == "buckets":
        if own:
            import matterformer_b200 as mfb

            return mfb.distance_buckets(state["xyz"], state["edges"], state["num"])
        return _real_pairs(state, _bucket_of(state["xyz"], state["edges"])).to(torch.uint8)
    if own:
        return _own_attn(state)
    with torch.no_grad():
        return _plain_attn(state)


def work(case):
    """Inputs read once and outputs written once; two products of every visible pair forward and five more backward, which forms the logits again."""
    if case["kind"] == "buckets":
        B, N = case["batch"], case["tokens"]
        return {"bytes": B * N * 12 + B * N * N + 4 * B, "flops": 8 * B * N * N}
    B, M, N, H, K, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    lo = max(1, round(N * case["fill"]))
    mean = (lo + N) / 2  # lengths are spread evenly
    square = sum(n * n for n in range(lo, N + 1)) / (N - lo + 1)
    pairs = square if M == N else mean * (1 if M == 1 else (max(1, round(M * case["fill"])) + M) / 2)
    if case["causal"] and M > 1:
        pairs = pairs / 2
    pairs, rows_k = pairs * (1 - case["holes"]), mean / N
    rows_q = rows_k if M == N else 1.0
    size = 2
    q, kv = B * M * H * D, 2 * B * N * K * D
    bias = 0
    if case["bias"] != "none":
        bias = size * case["buckets"] * H + (B * pairs if case["bias"] == "pair" else 2 * case["reach"] + 1)
    read = size * (q * rows_q + kv * rows_k) + bias
    if not case["train"]:
        return {"bytes": int(read + size * q), "flops": int(4 * B * H * pairs * D)}
    return {"bytes": int(2 * read + size * (q * rows_q + 2 * q + kv)), "flops": int(14 * B * H * pairs * D)}


def exact(case, seed):
    """The definitions in 64 bits, entry by entry; gradients by differentiating the output."""
    s = prepare(case, seed)
    if case["kind"] == "buckets":
        x, n = s["xyz"].double(), s["num"].tolist()
        out = torch.zeros(case["batch"], case["tokens"], case["tokens"], dtype=torch.uint8, device="cuda")
        inner = (s["edges"] ** 2).cuda()
        for b in range(case["batch"]):
            d = x[b, : n[b], None] - x[b, None, : n[b]]
            out[b, : n[b], : n[b]] = torch.searchsorted(inner, (d * d).sum(-1).contiguous(), right=True).to(torch.uint8)
        return out
    B, M, N, H, K, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    wide = [t.detach().double().requires_grad_(case["train"]) for t in s["leaves"]]
    nq = s["num_q"].tolist() if s["num_q"] is not None else [M] * B
    nk = s["num_k"].tolist() if s["num_k"] is not None else [N] * B
    dtable = torch.zeros(case["buckets"], H, dtype=torch.float64, device="cuda")
    outs, grads = [], []
    for b in range(B):
        m, n = nq[b], nk[b]
        part = [t.detach()[b].requires_grad_(case["train"]) for t in (wide[:1] if case["form"] == "packed" else wide[:3])]
        table = wide[-1].detach().requires_grad_(case["train"]) if s["table"] is not None else None
        with torch.set_grad_enabled(case["train"]):
            if case["form"] == "packed":
                q, k, v = part[0].view(N, 3, H, D).permute(1, 2, 0, 3)
            else:
                q, k, v = part[0], part[1].repeat_interleave(H // K, 0), part[2].repeat_interleave(H // K, 0)
            q, k, v = q[:, :m], k[:, :n], v[:, :n]
            logits = torch.einsum("hmd,hnd->hmn", q, k) / math.sqrt(D)
            delta = torch.arange(n, device="cuda") - torch.arange(m, device="cuda")[:, None] - (n - m)
            if table is not None:
                which = s["buckets"][b, :m, :n] if case["bias"] == "pair" else s["buckets"][delta.clamp(-case["reach"], case["reach"]) + case["reach"]]
                logits = logits + torch.nn.functional.embedding(which.long(), table).permute(2, 0, 1)
            hidden = (delta > 0) if case["causal"] else torch.zeros_like(delta, dtype=torch.bool)
            if s["mask"] is not None:
                hidden = hidden | ~s["mask"][b, :n]
            blind = hidden.all(-1, keepdim=True)
            p = torch.softmax(logits.masked_fill(hidden & ~blind, -math.inf), -1).masked_fill(hidden | blind, 0.0)
            out = torch.nn.functional.pad(p @ v, (0, 0, 0, M - m))  # (H, M, D)
            if case["form"] == "packed":
                out = out.transpose(0, 1).reshape(N, H * D)
        outs.append(out.detach())
        if case["train"]:
            made = torch.autograd.grad(out, part + ([table] if table is not None else []), s["grad"][b].double())
            if table is not None:
                dtable += made[-1]
            grads.append(made[: len(part)])
    if not case["train"]:
        return torch.stack(outs)
    made = [torch.stack(outs), *(torch.stack(t) for t in zip(*grads))]
    return made + ([dtable] if s["table"] is not None else [])
