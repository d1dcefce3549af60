"""The operators of a memory that overwrites (flyguy_b200.delta) and of the layers around it (flyguy_b200.layers) as cases:
sizes, inputs, one pass, its work, and the definitions in 64 bits.

  delta_attention   the gated delta rule over whole recordings (chunked form), with the gradients of all its inputs
  delta_step        the same for a single tick, the states updated in place (recurrent form)
  layer_norm        the norm of rows, with the gradients of rows, weight and bias
  dropout           values dropped by a counter-based generator, added to a residual; the mask is made again going back

`own` false: elementary torch operations in 32 bits. `own` true: the framework's entry points.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
DEV = "cuda"


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a training batch: 64 recordings of 1,024 ticks, with gradients
        {"name": "delta_train", "op": "delta_attention", "type": "bfloat16", "batch": 64, "ticks": 1024, "heads": 8,
         "query_heads": 8, "key_heads": 8, "value_heads": 8, "dim": 128, "value_dim": 128, "ragged": False,
         "state": False, "train": True},
        # one recording of 9 minutes at 120 ticks a second taken in at once: few rows, a long axis
        {"name": "delta_long", "op": "delta_attention", "type": "bfloat16", "batch": 1, "ticks": 65536, "heads": 8,
         "query_heads": 8, "key_heads": 8, "value_heads": 8, "dim": 128, "value_dim": 128, "ragged": False,
         "state": True, "train": False},
        # recordings of unequal lengths packed end to end, four query heads on each key head, with gradients
        {"name": "delta_ragged", "op": "delta_attention", "type": "bfloat16", "batch": 130, "ticks": 1500, "heads": 8,
         "query_heads": 8, "key_heads": 2, "value_heads": 2, "dim": 64, "value_dim": 64, "ragged": True,
         "state": True, "train": True},
        # the framework's training type, an odd length, from and to states, with gradients
        {"name": "delta_train_fp32", "op": "delta_attention", "type": "float32", "batch": 32, "ticks": 509, "heads": 4,
         "query_heads": 4, "key_heads": 4, "value_heads": 4, "dim": 64, "value_dim": 64, "ragged": False,
         "state": True, "train": True},
        # a few ticks of 8 cars carried on from their states, two value heads on each key head
        {"name": "delta_short_fp16", "op": "delta_attention", "type": "float16", "batch": 8, "ticks": 37, "heads": 4,
         "query_heads": 2, "key_heads": 2, "value_heads": 4, "dim": 64, "value_dim": 64, "ragged": False,
         "state": True, "train": False},
        # one tick of 8 cars; latency
        {"name": "delta_step_play", "op": "delta_step", "type": "bfloat16", "batch": 8, "slots": 8, "heads": 8,
         "query_heads": 8, "key_heads": 2, "value_heads": 2, "dim": 64, "value_dim": 64},
        # one tick of 2,048 games, their states in a larger pool
        {"name": "delta_step_serve", "op": "delta_step", "type": "bfloat16", "batch": 2048, "slots": 2100, "heads": 8,
         "query_heads": 8, "key_heads": 8, "value_heads": 8, "dim": 128, "value_dim": 128},
        # the observations of 8 cars at one tick; latency
        {"name": "norm_play", "op": "layer_norm", "type": "float32", "rows": 8, "dim": 517, "weight": True,
         "bias": True, "train": False},
        # the observations of a teaching batch, with gradients
        {"name": "norm_obs_fp32", "op": "layer_norm", "type": "float32", "rows": 16384, "dim": 517, "weight": True,
         "bias": True, "train": True},
        # 65,536 ticks, the outputs of 8 heads of 128 side by side, with gradients
        {"name": "norm_train", "op": "layer_norm", "type": "bfloat16", "rows": 65536, "dim": 1024, "weight": True,
         "bias": True, "train": True},
        # the same ticks' values dropped on their way to the residual, with gradients
        {"name": "dropout_train", "op": "dropout", "type": "bfloat16", "rows": 65536, "dim": 1024, "p": 0.1,
         "add": True, "train": True},
        # a short recording, odd sizes
        {"name": "dropout_short_fp16", "op": "dropout", "type": "float16", "rows": 37, "dim": 517, "p": 0.25,
         "add": False, "train": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["delta_attention", "delta_attention", "delta_attention", "delta_step", "layer_norm", "dropout"])
    typ = rng.choice(["bfloat16", "bfloat16", "float32", "float16"])
    if kind == "layer_norm":
        dim = _log_int(rng, 16, 8192)
        return {"op": kind, "type": typ, "rows": _log_int(rng, 1, max(1, (1 << 25) // dim)), "dim": dim,
                "weight": rng.random() < 0.8, "bias": rng.random() < 0.6, "train": rng.random() < 0.6}
    if kind == "dropout":
        dim = _log_int(rng, 1, 8192)
        return {"op": kind, "type": typ, "rows": _log_int(rng, 1, max(1, (1 << 25) // dim)), "dim": dim,
                "p": rng.choice([0.0, 0.05, 0.1, 0.25, 0.5]), "add": rng.random() < 0.5, "train": rng.random() < 0.6}
    dim = rng.choice([64, 64, 128, 128, 96, 80, 40])
    few = rng.choice([1, 2, 3, 4, 8])
    heads = few * rng.choice([1, 1, 2, 4])
    shared = rng.choice(["none", "keys", "values"])        # many queries to a key and value, or many values to a key
    c = {"op": kind, "type": typ, "heads": heads, "query_heads": few if shared == "values" else heads,
         "key_heads": heads if shared == "none" else few, "value_heads": few if shared == "keys" else heads,
         "dim": dim, "value_dim": rng.choice([dim, dim, 64, 128])}
    if kind == "delta_step":
        batch = _log_int(rng, 1, max(1, (1 << 27) // (heads * dim * c["value_dim"])))
        return c | {"batch": batch, "slots": batch + rng.randrange(0, 9)}
    ticks = _log_int(rng, 1, 16384)
    most = max(1, min(512, (1 << 25) // (ticks * max(dim, c["value_dim"]) * heads)))
    return c | {"batch": _log_int(rng, 1, most), "ticks": ticks, "ragged": rng.random() < 0.4,
                "state": rng.random() < 0.6, "train": rng.random() < 0.5}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lengths(c, seed):
    """Lengths of the recordings of a ragged batch: none up to all of `ticks`, two of them empty where there is room;
    the same lengths for every seed, in another order."""
    g = torch.Generator().manual_seed(c["batch"] * 65537 + c["ticks"])
    n = torch.randint(0, c["ticks"] + 1, (c["batch"],), generator=g)
    if len(n) > 3:
        n[1] = n[-1] = 0
    n[0] = c["ticks"]
    return n[torch.randperm(len(n), generator=torch.Generator().manual_seed(seed))].tolist()


def prepare(case, seed):
    c, typ = case, DTYPES[case["type"]]
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0, typ=typ):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(typ)

    s = {"case": c}
    if c["op"] == "layer_norm":
        # channels of unlike means and widths, as activations have them
        wide = torch.exp(0.5 * torch.randn(c["dim"], generator=g, device=DEV))
        s["x"] = (torch.randn(c["rows"], c["dim"], generator=g, device=DEV) * wide
                  + torch.randn(c["dim"], generator=g, device=DEV)).to(typ)
        if c["weight"]:
            s["weight"] = 1 + normal(c["dim"], scale=0.2, typ=torch.float32)
        if c["bias"]:
            s["bias"] = normal(c["dim"], scale=0.2, typ=torch.float32)
        if c["train"]:
            s["gy"] = normal(c["rows"], c["dim"])
        return s
    if c["op"] == "dropout":
        s["x"] = normal(c["rows"], c["dim"])
        s["seed"] = torch.randint(0, 1 << 62, (1,), generator=g, device=DEV)
        s["call"] = seed % 1000                            # the training step and layer that asks
        if c["add"]:
            s["add"] = normal(c["rows"], c["dim"])
        if c["train"]:
            s["gy"] = normal(c["rows"], c["dim"])
        return s

    B, H, D, E = c["batch"], c["heads"], c["dim"], c["value_dim"]
    if c["op"] == "delta_step":
        lead = (B,)
    elif c["ragged"]:
        s["lengths"] = _lengths(c, seed)
        s["offsets"] = torch.tensor([0] + s["lengths"], device=DEV).cumsum(0)
        lead = (sum(s["lengths"]),)
    else:
        lead = (B, c["ticks"])

    def unit(heads):                                       # unit vectors that share a direction, as neighbouring ticks do
        x = torch.randn(*lead, heads, D, generator=g, device=DEV) + 0.5 * torch.randn(heads, D, generator=g, device=DEV)
        return (x / x.square().sum(-1, keepdim=True).sqrt()).to(typ)

    s["q"], s["k"] = unit(c["query_heads"]), unit(c["key_heads"])
    s["v"] = normal(*lead, c["value_heads"], E, scale=0.5)
    # gates made from each tick: memories from some 20 ticks to thousands, as spread over the heads of one layer
    span = torch.exp2(-4.5 - 7.0 * torch.arange(H, device=DEV) / max(1, H - 1))
    s["log_decay"] = -span * torch.nn.functional.softplus(1 + torch.randn(*lead, H, generator=g, device=DEV))
    s["beta"] = torch.sigmoid(torch.randn(*lead, H, generator=g, device=DEV))
    if c["op"] == "delta_step":
        s["state"] = normal(c["slots"], H, D, E, scale=0.3, typ=torch.float32)
        s["slots"] = torch.randperm(c["slots"], generator=g, device=DEV)[:B]
        return s
    if c["state"]:
        s["state"] = normal(B, H, D, E, scale=0.3, typ=torch.float32)
    if c["train"]:
        s["go"] = normal(*lead, H, E)
        s["gs"] = normal(B, H, D, E, scale=0.05, typ=torch.float32)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"delta_attention": _plain_delta_attention, "delta_step": _plain_delta_step,
            "layer_norm": _plain_layer_norm, "dropout": _plain_dropout}[state["case"]["op"]](state)


def _run_own(s):
    from flyguy_b200 import delta, layers
    c, op = s["case"], s["case"]["op"]
    if op == "layer_norm":
        names = [n for n in ("x", "weight", "bias") if n in s]
        if not c["train"]:
            return layers.layer_norm(s["x"], s.get("weight"), s.get("bias"), eps=1e-5)
        ins = {n: s[n].detach().requires_grad_() for n in names}
        y = layers.layer_norm(ins["x"], ins.get("weight"), ins.get("bias"), eps=1e-5)
        return y.detach(), *torch.autograd.grad(y, [ins[n] for n in names], s["gy"])
    if op == "dropout":
        if not c["train"]:
            return layers.dropout(s["x"], c["p"], s["seed"], call=s["call"], add=s.get("add"))
        x = s["x"].detach().requires_grad_()
        y = layers.dropout(x, c["p"], s["seed"], call=s["call"], add=s.get("add"))
        return y.detach(), *torch.autograd.grad(y, x, s["gy"])
    five = ("q", "k", "v", "log_decay", "beta")
    if op == "delta_step":
        return delta.delta_step(*(s[n] for n in five), s["state"], slots=s["slots"]), s["state"]
    if not c["train"]:
        return delta.delta_attention(*(s[n] for n in five), s.get("state"), offsets=s.get("offsets"))
    ins = [s[n].detach().requires_grad_() for n in (*five, "state") if n in s]
    o, end = delta.delta_attention(*ins, offsets=s.get("offsets"))
    return o.detach(), end.detach(), *torch.autograd.grad((o, end), ins, (s["go"], s["gs"]))


CHUNK = 64


def _inverse(a):
    """(1 + a)^-1 of strictly lower triangular a [.., CHUNK, CHUNK], by blocks that double."""
    n = a.shape[-1]
    inv = torch.ones(*a.shape[:-2], n, 1, 1, device=a.device)
    m = 1
    while m < n:
        blocks = a.unflatten(-1, (n // (2 * m), 2 * m)).unflatten(-3, (n // (2 * m), 2 * m))
        below = blocks.diagonal(dim1=-4, dim2=-2).movedim(-1, -3)[..., m:, :m]            # [.., blocks, m, m]
        first, second = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        low = -(second @ below @ first)
        inv = torch.cat((torch.cat((first, torch.zeros_like(first)), -1), torch.cat((low, second), -1)), -2)
        m *= 2
    return inv.squeeze(-3)


def _chunked_delta(q, k, v, g, beta, S):
    """o_t and the last S of S_t = e^g_t S_{t-1} + k_t u_t^T, u_t = beta_t (v_t - e^g_t k_t S_{t-1}), o_t = q_t S_t, in
    chunks of ticks. [B, T, H, .] in 32 bits; ticks with k, g and beta of 0 change nothing."""
    B, T, H, D = q.shape
    n = -(-max(T, 1) // CHUNK)

    def rows(x):                                                                           # [B, H, n, CHUNK, ..]
        x = torch.cat((x, x.new_zeros(B, n * CHUNK - T, *x.shape[2:])), 1)
        return x.unflatten(1, (n, CHUNK)).movedim(3, 1)

    q, k, v, beta = rows(q), rows(k), rows(v), rows(beta).unsqueeze(-1)
    G = rows(g.double()).cumsum(-1)
    there = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((G.unsqueeze(-1) - G.unsqueeze(-2)).masked_fill(~there, -math.inf).float())
    P = q @ k.transpose(-1, -2) * decay
    inv = _inverse((k @ k.transpose(-1, -2) * decay).tril(-1) * beta)
    from0, toend = torch.exp(G.float()).unsqueeze(-1), torch.exp((G[..., -1:] - G).float()).unsqueeze(-1)
    whole = from0[..., -1:, :]
    u0, w, qs, ke = inv @ (beta * v), inv @ (beta * from0 * k), q * from0, (k * toend).transpose(-1, -2)
    o = []
    for i in range(n):
        u = u0[:, :, i] - w[:, :, i] @ S
        o.append(qs[:, :, i] @ S + P[:, :, i] @ u)
        S = S * whole[:, :, i] + ke[:, :, i] @ u
    return torch.stack(o, 2).movedim(1, 3).flatten(1, 2)[:, :T], S


def _plain_delta_attention(s):
    c, typ = s["case"], s["q"].dtype
    B, T, H, D, E = c["batch"], c["ticks"], c["heads"], c["dim"], c["value_dim"]
    names = [n for n in ("q", "k", "v", "log_decay", "beta", "state") if n in s]
    ins = {n: s[n].detach().float().requires_grad_(c["train"]) for n in names}
    if "offsets" in s:
        off = s["offsets"]
        at = off[:-1, None] + torch.arange(T, device=DEV)
        there = at < off[1:, None]
        at = at.clamp(max=max(0, s["q"].shape[0] - 1))

    def rows(x):                                           # [B, T, ..] of recordings, zeros after their ends
        if "offsets" in s:
            x = torch.where(there.view(B, T, *[1] * (x.dim() - 1)), x[at], 0.0)
        return x if x.shape[2] == H else x.repeat_interleave(H // x.shape[2], 2)

    with torch.set_grad_enabled(c["train"]):
        first = ins["state"] if "state" in s else torch.zeros(B, H, D, E, device=DEV)
        o, end = _chunked_delta(rows(ins["q"]) * D ** -0.5, rows(ins["k"]), rows(ins["v"]), rows(ins["log_decay"]),
                                rows(ins["beta"]), first)
        o = o[there] if "offsets" in s else o
    if not c["train"]:
        return o.to(typ), end
    grads = torch.autograd.grad((o, end), [ins[n] for n in names], (s["go"].float(), s["gs"]))
    return o.detach().to(typ), end.detach(), *(g.to(s[n].dtype) for n, g in zip(names, grads))


def _plain_delta_step(s):
    c, at, H = s["case"], s["slots"], s["case"]["heads"]
    q, k, v = (s[n].float().repeat_interleave(H // s[n].shape[1], 1) for n in ("q", "k", "v"))
    S = s["state"][at] * torch.exp(s["log_decay"])[..., None, None]
    u = s["beta"].unsqueeze(-1) * (v - (k.unsqueeze(-2) @ S).squeeze(-2))
    S = S + k.unsqueeze(-1) * u.unsqueeze(-2)
    s["state"][at] = S
    o = (q.unsqueeze(-2) @ S).squeeze(-2) * c["dim"] ** -0.5
    return o.to(s["q"].dtype), s["state"]


def _plain_layer_norm(s):
    c, typ, x = s["case"], s["x"].dtype, s["x"].float()
    d = x - x.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xh = d * r
    y = xh * s["weight"] if c["weight"] else xh
    y = (y + s["bias"] if c["bias"] else y).to(typ)
    if not c["train"]:
        return y
    gy = s["gy"].float()
    g = gy * s["weight"] if c["weight"] else gy
    out = [y, (r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))).to(typ)]
    if c["weight"]:
        out.append((gy * xh).sum(0))
    if c["bias"]:
        out.append(gy.sum(0))
    return tuple(out)


LOW = 0xffffffff


def _kept(s):
    """Which values stay: value i of the tensor takes 16 bits of block i / 8 of the counter-based generator Philox4x32-10
    (key: the seed, counter: block and call), and stays where they are at least round(65536 p)."""
    n = s["x"].numel()
    block = torch.arange(-(-n // 8), device=DEV)
    c0, c1 = block & LOW, block >> 32
    c2, c3 = torch.full_like(c0, s["call"] & LOW), torch.full_like(c0, s["call"] >> 32)
    k0, k1 = s["seed"] & LOW, (s["seed"] >> 32) & LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32) & LOW ^ c1 ^ k0, b & LOW, (a >> 32) & LOW ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack((c0, c1, c2, c3), -1).unsqueeze(-1)
    bits = torch.cat((words & 0xffff, words >> 16), -1).flatten()[:n]
    return (bits >= round(s["case"]["p"] * 65536)).view(s["x"].shape)


def _plain_dropout(s):
    c, typ, kept = s["case"], s["x"].dtype, _kept(s)
    by = 65536 / (65536 - round(c["p"] * 65536))
    y = torch.where(kept, s["x"].float() * by, 0.0)
    y = (y + s["add"].float() if c["add"] else y).to(typ)
    return (y, torch.where(kept, s["gy"].float() * by, 0.0).to(typ)) if c["train"] else y


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    c, e = case, SIZE[case["type"]]
    if c["op"] == "layer_norm":
        values = c["rows"] * c["dim"]
        return {"bytes": (5.0 if c["train"] else 2.0) * values * e, "flops": (20.0 if c["train"] else 7.0) * values}
    if c["op"] == "dropout":
        values = c["rows"] * c["dim"]
        return {"bytes": (2.0 + c["add"] + 2 * c["train"]) * values * e, "flops": 2.0 * (1 + c["train"]) * values}
    H, D, E = c["heads"], c["dim"], c["value_dim"]
    ins = e * (c["query_heads"] * D + c["key_heads"] * D + c["value_heads"] * E) + 8.0 * H
    if c["op"] == "delta_step":
        return {"bytes": c["batch"] * (8.0 * H * D * E + ins + e * H * E), "flops": 7.0 * c["batch"] * H * D * E}
    rows = sum(_lengths(c, 0)) if c["ragged"] else c["batch"] * c["ticks"]
    states = 4.0 * c["batch"] * H * D * E
    if not c["train"]:
        return {"bytes": rows * (ins + e * H * E) + states * (2 if c["state"] else 1), "flops": 6.0 * rows * H * D * E}
    return {"bytes": 2 * rows * (ins + e * H * E) + states * (4 if c["state"] else 2), "flops": 18.0 * rows * H * D * E}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        return _exact_dropout(case, s)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] == "layer_norm":
        return _exact_norm(case, s)
    if case["op"] == "delta_step":
        return _exact_step(case, s)
    return _exact_delta(case, s)


def _exact_norm(c, s):
    """From the sums of values and squares of the values less their first, rows a piece at a time."""
    ys, gxs, gw, gb = [], [], 0.0, 0.0
    n = c["dim"]
    for lo in range(0, c["rows"], 4096):
        x = s["x"][lo:lo + 4096]
        z = x - x[:, :1]
        mean = z.sum(1, keepdim=True) / n
        std = torch.sqrt((z * z).sum(1, keepdim=True) / n - mean * mean + 1e-5)
        xh = (z - mean) / std
        y = xh
        if c["weight"]:
            y = y * s["weight"]
        if c["bias"]:
            y = y + s["bias"]
        ys.append(y)
        if c["train"]:
            gy = s["gy"][lo:lo + 4096]
            g = gy * s["weight"] if c["weight"] else gy
            along = torch.einsum("rd,rd->r", g, xh)[:, None]
            gxs.append((n * g - g.sum(1, keepdim=True) - xh * along) / (n * std))
            gw, gb = gw + torch.einsum("rd,rd->d", gy, xh), gb + gy.sum(0)
    y = torch.cat(ys)
    if not c["train"]:
        return y
    return (y, torch.cat(gxs), *([gw] if c["weight"] else []), *([gb] if c["bias"] else []))


def _exact_dropout(c, s):
    """The generator on the host, in unsigned 64-bit integers."""
    n, seed, u = c["rows"] * c["dim"], int(s["seed"].item()), np.uint64
    if n > 1 << 27:
        return None
    low, half = u(LOW), u(32)
    block = np.arange(-(-n // 8), dtype=u)
    x = [block & low, block >> half, np.full_like(block, s["call"] & LOW), np.full_like(block, s["call"] >> 32)]
    key = [seed & LOW, (seed >> 32) & LOW]
    for _ in range(10):
        p, r = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [(r >> half) ^ x[1] ^ u(key[0]), r & low, (p >> half) ^ x[3] ^ u(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
    bits = np.empty((len(block), 8), np.uint16)
    for i in range(4):
        bits[:, 2 * i], bits[:, 2 * i + 1] = (x[i] & u(0xffff)).astype(np.uint16), (x[i] >> u(16)).astype(np.uint16)
    least = int(math.floor(c["p"] * 65536 + 0.5))
    by = torch.from_numpy((bits.reshape(-1)[:n] >= least).astype(np.float32)).to(DEV).view(c["rows"], c["dim"]).double()
    by *= 65536 / (65536 - least)
    y = s["x"].double() * by
    if c["add"]:
        y += s["add"].double()
    return (y, s["gy"].double() * by) if c["train"] else y


def _exact_step(c, s):
    H, at = c["heads"], s["slots"]
    o = torch.empty(c["batch"], H, c["value_dim"], dtype=torch.float64, device=DEV)
    for h in range(H):
        q, k, v = (s[n][:, h // (H // s[n].shape[1])] for n in ("q", "k", "v"))
        old = s["state"][at, h] * s["log_decay"][:, h].exp()[:, None, None]
        miss = v - torch.einsum("bd,bde->be", k, old)
        new = old + torch.einsum("b,bd,be->bde", s["beta"][:, h], k, miss)
        s["state"][at, h] = new
        o[:, h] = torch.einsum("bd,bde->be", q, new) / math.sqrt(c["dim"])
    return o, s["state"]


def _exact_delta(c, s):
    """Tick by tick, forward and back; going back, the states of a stretch of ticks are made again from its first."""
    B, T, H, D, E = c["batch"], c["ticks"], c["heads"], c["dim"], c["value_dim"]
    size = B * H * D * E * 8
    if T * (5 if c["train"] else 1) * max(2e-4, size * 6 / 2e12) > 16:
        return None
    scale = 1 / math.sqrt(D)
    heads = {n: s[n].shape[-2] for n in ("q", "k", "v")}
    if c["ragged"]:
        off = s["offsets"].tolist()
        spans = [(b, off[b], off[b + 1]) for b in range(B) if off[b + 1] > off[b]]

    def rows(x, per=1):                                    # [T, B, H, ..], ticks after a recording's end zero
        if c["ragged"]:
            y = x.new_zeros(T, B, *x.shape[1:])
            for b, lo, hi in spans:
                y[:hi - lo, b] = x[lo:hi]
        else:
            y = x.transpose(0, 1)
        return y.repeat_interleave(per, 2) if per > 1 else y

    def back(y, per=1):
        if per > 1:
            y = y.unflatten(2, (-1, per)).sum(3)
        return torch.cat([y[:hi - lo, b] for b, lo, hi in spans]) if c["ragged"] else y.transpose(0, 1)

    per = {n: H // heads[n] for n in heads}
    q, k, v = (rows(s[n], per[n]) for n in ("q", "k", "v"))
    decay, beta = rows(s["log_decay"]).exp(), rows(s["beta"])

    def tick(S, t):
        old = S * decay[t][..., None, None]
        miss = v[t] - torch.einsum("bhd,bhde->bhe", k[t], old)
        return old, miss, old + k[t].unsqueeze(-1) * (beta[t].unsqueeze(-1) * miss).unsqueeze(-2)

    S = s["state"] if c["state"] else torch.zeros(B, H, D, E, dtype=torch.float64, device=DEV)
    stretch = max(1, min(64, int(1.2e10 / size)))
    o, marks = torch.empty_like(v), []
    for t in range(T):
        if c["train"] and t % stretch == 0:
            marks.append(S.to("cpu") if size * (T / stretch) > 3e10 else S)
        S = tick(S, t)[2]
        o[t] = torch.einsum("bhd,bhde->bhe", q[t], S) * scale
    if not c["train"]:
        return back(o), S
    end, R, go = S, s["gs"].clone(), rows(s["go"])
    gq, gk, gv, gg, gb = (torch.empty_like(x) for x in (q, k, v, decay, beta))
    for i in reversed(range(len(marks))):
        S, steps = marks.pop().to(DEV), []
        for t in range(i * stretch, min(T, (i + 1) * stretch)):
            steps.append(S)
            S = tick(S, t)[2]
        for t in reversed(range(i * stretch, min(T, (i + 1) * stretch))):
            before = steps.pop()
            old, miss, now = tick(before, t)
            gq[t] = torch.einsum("bhde,bhe->bhd", now, go[t]) * scale
            R = R + q[t].unsqueeze(-1) * go[t].unsqueeze(-2) * scale
            gu = torch.einsum("bhde,bhd->bhe", R, k[t])
            gb[t] = (gu * miss).sum(-1)
            gv[t] = gu * beta[t].unsqueeze(-1)
            gk[t] = torch.einsum("bhde,bhe->bhd", R, beta[t].unsqueeze(-1) * miss) - torch.einsum("bhde,bhe->bhd", old, gv[t])
            R = R - k[t].unsqueeze(-1) * gv[t].unsqueeze(-2)
            gg[t] = (R * old).sum((-2, -1))
            R = R * decay[t][..., None, None]
    grads = (back(gq, per["q"]), back(gk, per["k"]), back(gv, per["v"]), back(gg), back(gb))
    return (back(o), end, *grads, R) if c["state"] else (back(o), end, *grads)
