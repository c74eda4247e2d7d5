"""The gated feed-forward block and rotary positions: the calls that programs make of them, as cases that can be timed and compared.

Three kinds of programs make these calls: molecule models that train or sample with the trunk (d_model 512, 8 heads of 64 channels,
QM9-sized molecules of up to 29 atoms and drug-sized ones padded to 192), crystal models over cells of 4096 atoms, and sequence
models of generic widths beside them, which also step one token at a time.

Gated feed-forward block: y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo, with Wg above Wu in one matrix.
Rotary positions: pairs of channels of every head turn by the angle position * frequency; the table of frequencies has one row for
each axis of the position (one for places in a sequence, three for coordinates).
"""
from __future__ import annotations

import math

import torch

own = False  # True: the package's operators; False: their plain form

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ffn(tokens, dim, hidden, act="silu", dtype="bf16", bias=True, train=False):
    return {"kind": "ffn", "tokens": tokens, "dim": dim, "hidden": hidden, "act": act, "dtype": dtype, "bias": bias, "train": train}


def _rope(form, batch, tokens, heads, head_dim, rotary_dim, *, kv_heads=0, axes=1, layout="half", dtype="bf16", scaling="none",
          first=0, train=False):  # fmt: skip
    return {"kind": "rope", "form": form, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads or heads,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "axes": axes, "layout": layout, "dtype": dtype, "scaling": scaling,
            "first": first, "train": train}  # fmt: skip


def listed():
    return [
        # one molecule of 29 atoms in a sampling loop: a call of a few microseconds, launches and the host path count
        {"name": "ffn_molecule", **_ffn(29, 512, 2048)},
        # the denoiser of a sampling run of 64 molecules
        {"name": "ffn_sample", **_ffn(64 * 29, 512, 2048)},
        # one block of the training step on 1024 QM9-sized molecules: output and all gradients
        {"name": "ffn_qm9_train", **_ffn(1024 * 29, 512, 2048, train=True)},
        # the same on 64 drug-sized molecules with a hidden width that keeps the parameters of the plain block (8/3 of the width, an
        # odd multiple of 8), in half precision
        {"name": "ffn_drug_train", **_ffn(64 * 192, 512, 1368, act="gelu_tanh", dtype="f16", train=True)},
        # a wide trunk on two large cells, without biases: the largest call
        {"name": "ffn_wide_train", **_ffn(2 * 4096, 2048, 5464, bias=False, train=True)},
        # a wide model that steps one token: reading the weights is all there is to it
        {"name": "ffn_wide_token", **_ffn(1, 4096, 10928, bias=False)},
        # one molecule in a sampling loop: coordinates turn three quarters of every head of the packed projection
        {"name": "rope_molecule", **_rope("packed", 1, 29, 8, 64, 48, axes=3)},
        # an attention layer of the training step on 1024 QM9-sized molecules
        {"name": "rope_qm9_train", **_rope("packed", 1024, 29, 8, 64, 48, axes=3, train=True)},
        # queries and keys of large cells in sorted order, neighbouring channels paired, frequencies scaled by parts
        {"name": "rope_cells_train", **_rope("heads", 32, 4096, 8, 64, 64, layout="interleaved", scaling="parts", train=True)},
        # a long prompt in 32 bits with shared key heads that continues a million tokens further on
        {"name": "rope_long_f32", **_rope("heads", 1, 32771, 16, 128, 128, kv_heads=4, dtype="f32", scaling="linear", first=1_000_003)},
        # single tokens of 64 sequences, each at a place of its own
        {"name": "rope_tokens", **_rope("heads", 64, 1, 32, 128, 128, kv_heads=8, dtype="f16", first=5000)},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more call of the listed ranges."""
    if rng.random() < 0.5:
        most = 18 * 8192 * 2048 * 5464
        while True:
            dim = 8 * _log(rng, 16, 512)
            hidden = 8 * _log(rng, dim // 8, dim // 2)
            train = rng.random() < 0.5
            tokens = _log(rng, 1, 32768)
            if (18 if train else 6) * tokens * dim * hidden <= most:
                break
        return _ffn(tokens, dim, hidden, act=rng.choice(["silu", "silu", "gelu_tanh"]), dtype=rng.choice(["bf16", "bf16", "f16"]),
                    bias=rng.random() < 0.5, train=train)  # fmt: skip
    most = 32 * 4096 * 8 * 64
    while True:
        form = rng.choice(["packed", "heads"])
        head_dim = rng.choice([32, 40, 64, 64, 80, 128])
        axes = rng.choice([1, 1, 3])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * (1 if form == "packed" else rng.choice([1, 2, 4]))
        batch, tokens = _log(rng, 1, 1024), _log(rng, 1, 32768)
        if batch * tokens * heads * head_dim <= most and batch * tokens <= 32 * 4096:
            break
    pairs = rng.choice([head_dim // 2, head_dim // 4, rng.randint(axes, head_dim // 2)])
    return _rope(form, batch, tokens, heads, head_dim, 2 * axes * max(1, pairs // axes), kv_heads=kv_heads, axes=axes,
                 layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                 scaling="none" if axes == 3 else rng.choice(["none", "linear", "parts"]),
                 first=0 if axes == 3 else rng.choice([0, 0, 777, 200_001]), train=rng.random() < 0.5)  # fmt: skip


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _table(case):
    """Frequencies in radians per unit of the position, (pairs,) or (axes, pairs), on the host in 64 bits."""
    axes = case["axes"]
    pairs = case["rotary_dim"] // (2 * axes)
    base = 10000.0 if axes == 1 else 100.0  # coordinates of molecules span a few units
    theta = base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    if case["scaling"] == "linear":
        theta = theta / 8.0
    elif case["scaling"] == "parts":  # four times the length: what turns often within 1024 places stays, what hardly turns is stretched
        kept = ((1024.0 * theta / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        theta = kept * theta + (1 - kept) * theta / 4.0
    return theta if axes == 1 else theta.repeat(axes, 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    if case["kind"] == "ffn":
        T, C, F = case["tokens"], case["dim"], case["hidden"]
        s = {"x": _randn(g, T, C, dtype=dtype), "w_in": _randn(g, 2 * F, C, scale=C**-0.5, dtype=dtype),
             "w_out": _randn(g, C, F, scale=F**-0.5, dtype=dtype), "b_in": None, "b_out": None}  # fmt: skip
        if case["bias"]:
            s.update(b_in=_randn(g, 2 * F, scale=0.1, dtype=dtype), b_out=_randn(g, C, scale=0.1, dtype=dtype))
        s["leaves"] = [s[n] for n in ("x", "w_in", "w_out", "b_in", "b_out") if s[n] is not None]
        shape = (T, C)
    else:
        B, N, H, K, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        s = {"table": _table(case)}
        if case["axes"] == 3:
            s["positions"] = _randn(g, B, N, 3, scale=1.5)
        elif N == 1:  # every sequence is at a place of its own
            s["positions"] = case["first"] + torch.randint(0, 4096, (B, 1), generator=g, device="cuda")
        else:
            s["positions"] = case["first"] + torch.arange(N, device="cuda")
        if case["form"] == "packed":
            s["qkv"] = _randn(g, B, N, 3 * H * D, dtype=dtype)
            s["leaves"], shape = [s["qkv"]], (B, N, 3 * H * D)
        else:
            s["q"], s["k"] = _randn(g, B, H, N, D, dtype=dtype), _randn(g, B, K, N, D, dtype=dtype)
            s["leaves"], shape = [s["q"], s["k"]], None
    s["case"] = case
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_(True)
        s["grad"] = [_randn(g, *shape, dtype=dtype)] if shape else [_randn(g, *t.shape, dtype=dtype) for t in s["leaves"]]
    return s


def _activation(name, z):
    """act(z) and its derivative."""
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    b, c = math.sqrt(2 / math.pi), 0.044715
    e = torch.exp(-2 * torch.abs(b * (z + c * z * z * z)))
    t = torch.sign(z) * (1 - e) / (1 + e)  # tanh
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * b * (1 + 3 * c * z * z)


def _plain_ffn(s):
    case = s["case"]
    dtype, F = s["x"].dtype, case["hidden"]
    x, w_in, w_out = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    pre = x @ w_in.t()
    if case["bias"]:
        pre = pre + s["b_in"].float()
    up = pre[:, F:]
    act, slope = _activation(case["act"], pre[:, :F])
    hidden = act * up
    y = hidden @ w_out.t()
    if case["bias"]:
        y = y + s["b_out"].float()
    if not case["train"]:
        return y.to(dtype)
    dy = s["grad"][0].float()
    dhidden = dy @ w_out
    dpre = torch.cat([dhidden * up * slope, dhidden * act], dim=1)
    out = [y, dpre @ w_in, dpre.t() @ x, dy.t() @ hidden]
    if case["bias"]:
        out += [dpre.sum(0), dy.sum(0)]
    return [t.to(dtype) for t in out]


def _cos_sin(s, dtype):
    """(B or 1, N, axes * pairs) each; the angles of far positions need 64 bits."""
    table, positions = s["table"].to("cuda"), s["positions"].double()
    angle = positions[..., None] * table if table.ndim == 1 else (positions[..., None] * table).flatten(-2)
    if angle.ndim == 2:
        angle = angle[None]
    return torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)


def _turn(x, cos, sin, layout):
    """x (..., D) with the angles along its last axis; the channels behind the last pair stay."""
    P = cos.shape[-1]
    if layout == "half":
        a, b = x[..., :P], x[..., P : 2 * P]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * P :]], dim=-1)
    a, b = x[..., 0 : 2 * P : 2], x[..., 1 : 2 * P : 2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2), x[..., 2 * P :]], dim=-1)


def _plain_rope(s):
    case = s["case"]
    cos, sin = _cos_sin(s, torch.float32)
    if case["form"] == "packed":
        B, N, H, D = case["batch"], case["tokens"], case["heads"], case["head_dim"]
        at = (slice(None), slice(None), None, None)  # angles beside (B, N, 2, H, D)

        def whole(t, sign):
            v = t.view(B, N, 3, H, D)
            qk = _turn(v[:, :, :2].float(), cos[at], sign * sin[at], case["layout"])
            return torch.cat([qk.to(t.dtype), v[:, :, 2:]], dim=2).view(B, N, 3 * H * D)

        given = [s["qkv"]]
    else:
        at = (slice(None), None)  # angles beside (B, H, N, D)

        def whole(t, sign):
            return _turn(t.float(), cos[at], sign * sin[at], case["layout"]).to(t.dtype)

        given = [s["q"], s["k"]]
    out = [whole(t, 1) for t in given]
    return out + [whole(t, -1) for t in s["grad"]] if case["train"] else out


def _own_ffn(s):
    import matterformer_b200 as mfb

    with torch.set_grad_enabled(s["case"]["train"]):
        y = mfb.gated_mlp(s["x"], s["w_in"], s["w_out"], s["b_in"], s["b_out"], activation=s["case"]["act"])
    return [y, *torch.autograd.grad(y, s["leaves"], s["grad"])] if s["case"]["train"] else y


def _own_rope(s):
    import matterformer_b200 as mfb

    case = s["case"]
    with torch.set_grad_enabled(case["train"]):
        if case["form"] == "packed":
            out = [mfb.rotary_packed(s["qkv"], case["heads"], s["positions"], s["table"], layout=case["layout"])]
        else:
            out = list(mfb.rotary_embedding(s["q"], s["k"], s["positions"], s["table"], layout=case["layout"]))
    return [*out, *torch.autograd.grad(out, s["leaves"], s["grad"])] if case["train"] else out


def run(state):
    if own:
        return _own_ffn(state) if state["case"]["kind"] == "ffn" else _own_rope(state)
    with torch.no_grad():
        return _plain_ffn(state) if state["case"]["kind"] == "ffn" else _plain_rope(state)


def work(case):
    """Inputs read once, outputs written once; the products of the block, six operations a pair for a rotation."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "ffn":
        T, C, F = case["tokens"], case["dim"], case["hidden"]
        weights = 3 * C * F + (2 * F + C if case["bias"] else 0)
        if case["train"]:
            return {"bytes": size * (4 * T * C + 2 * weights), "flops": 18 * T * C * F}
        return {"bytes": size * (2 * T * C + weights), "flops": 6 * T * C * F}
    B, N, H, K, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    values = B * N * D * (3 * H if case["form"] == "packed" else H + K)
    places = (B * N * 3 * 4 if case["axes"] == 3 else 8 * (B if N == 1 else N))
    passes = 2 if case["train"] else 1
    return {"bytes": passes * (2 * size * values + places), "flops": passes * 3 * B * N * (H + K) * case["rotary_dim"]}


def exact(case, seed):
    """The definitions in 64 bits; gradients by differentiating the output."""
    s = prepare(case, seed)
    with torch.set_grad_enabled(case["train"]):
        leaves = [t.detach().double().requires_grad_(case["train"]) for t in s["leaves"]]
        if case["kind"] == "ffn":
            bias = leaves[3:] if case["bias"] else [None, None]
            pre = torch.nn.functional.linear(leaves[0], leaves[1], bias[0])
            gate, up = pre.chunk(2, dim=-1)
            act = gate * torch.sigmoid(gate) if case["act"] == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
            out = [torch.nn.functional.linear(act * up, leaves[2], bias[1])]
        else:
            out = _exact_rope(case, s, leaves)
    if not case["train"]:
        return [t.detach() for t in out] if case["kind"] == "rope" else out[0].detach()
    grads = torch.autograd.grad(out, leaves, [t.double() for t in s["grad"]])
    return [*(t.detach() for t in out), *grads]


def _exact_rope(case, s, leaves):
    """As products of complex numbers."""
    B, N, H, D, R = case["batch"], case["tokens"], case["heads"], case["head_dim"], case["rotary_dim"]
    table = s["table"].reshape(case["axes"], -1).to("cuda")
    positions = s["positions"].double().reshape(-1, N, case["axes"])
    unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.einsum("bna,ap->bnap", positions, table)).flatten(2)[:, None]

    def turned(x):  # (B, heads, N, D)
        head, rest = x[..., :R], x[..., R:]
        if case["layout"] == "half":
            z = torch.complex(*(t.contiguous() for t in head.chunk(2, dim=-1))) * unit
            return torch.cat([z.real, z.imag, rest], dim=-1)
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], R // 2, 2).contiguous()) * unit
        return torch.cat([torch.view_as_real(z).flatten(-2), rest], dim=-1)

    if case["form"] == "heads":
        return [turned(t) for t in leaves]
    q, k, v = leaves[0].view(B, N, 3, H, D).permute(2, 0, 3, 1, 4)
    return [torch.stack([turned(q), turned(k), v]).permute(1, 3, 0, 2, 4).reshape(B, N, 3 * H * D)]
