"""The operators of the memory over ticks (flyguy_b200.memory) as cases: sizes, inputs, one pass, its work, and the
definitions in 64 bits.

  rotate            rotary positions: pairs of a head's values turned by position * frequency
  norm_rotate       the norms of queries and keys for each head with the rotation in the same pass
  decay_attention   linear attention with a decay for each head over whole recordings (chunked form)
  decay_step        the same for a single tick, the states updated in place (recurrent form)

`own` false: elementary torch operations in 32 bits. `own` true: the framework's entry points.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
DEV = "cuda"


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one tick of the 8 cars of a playing call: the queries of one memory layer; latency
        {"name": "rotate_play", "op": "rotate", "type": "bfloat16", "batch": 8, "ticks": 1, "heads": 8, "dim": 64,
         "turned": 64, "layout": "half", "scaling": "none", "first": 40000, "train": False},
        # whole recordings far into a session, half of each head turned, slowed frequencies, with gradients
        {"name": "rotate_train_fp32", "op": "rotate", "type": "float32", "batch": 16, "ticks": 2047, "heads": 8,
         "dim": 128, "turned": 64, "layout": "interleaved", "scaling": "parts", "first": 1000000, "train": True},
        # one tick of 8 cars, queries and fewer key heads out of one projection's result; latency
        {"name": "norm_rotate_play", "op": "norm_rotate", "type": "bfloat16", "batch": 8, "ticks": 1, "heads": 8,
         "key_heads": 2, "dim": 64, "turned": 64, "layout": "half", "scaling": "none", "first": 40000, "each": False,
         "train": False},
        # a training batch of 16,384 ticks (128 recordings of 128), with gradients of inputs and weights
        {"name": "norm_rotate_train", "op": "norm_rotate", "type": "bfloat16", "batch": 128, "ticks": 128, "heads": 16,
         "key_heads": 4, "dim": 128, "turned": 128, "layout": "half", "scaling": "none", "first": 0, "each": False,
         "train": True},
        # 65,536 ticks a call, weights of their own for each head
        {"name": "norm_rotate_large_fp16", "op": "norm_rotate", "type": "float16", "batch": 32, "ticks": 2048,
         "heads": 8, "key_heads": 8, "dim": 128, "turned": 96, "layout": "interleaved", "scaling": "linear",
         "first": 0, "each": True, "train": False},
        # one recording of 9 minutes at 120 ticks a second taken in at once: few rows, a long axis
        {"name": "attention_long", "op": "decay_attention", "type": "bfloat16", "batch": 1, "ticks": 65536, "heads": 8,
         "key_heads": 8, "dim": 128, "value_dim": 128, "ragged": False, "state": True, "train": False},
        # a training batch: 64 recordings of 1,024 ticks, with gradients
        {"name": "attention_train", "op": "decay_attention", "type": "bfloat16", "batch": 64, "ticks": 1024, "heads": 8,
         "key_heads": 8, "dim": 128, "value_dim": 128, "ragged": False, "state": False, "train": True},
        # recordings of unequal lengths packed end to end, four query heads on each key head, with gradients
        {"name": "attention_ragged", "op": "decay_attention", "type": "bfloat16", "batch": 130, "ticks": 1500,
         "heads": 8, "key_heads": 2, "dim": 64, "value_dim": 64, "ragged": True, "state": True, "train": True},
        # the framework's training type, an odd length, from and to states, with gradients
        {"name": "attention_train_fp32", "op": "decay_attention", "type": "float32", "batch": 32, "ticks": 509,
         "heads": 4, "key_heads": 4, "dim": 64, "value_dim": 64, "ragged": False, "state": True, "train": True},
        # a few ticks of 8 cars carried on from their states
        {"name": "attention_short_fp16", "op": "decay_attention", "type": "float16", "batch": 8, "ticks": 37,
         "heads": 4, "key_heads": 4, "dim": 64, "value_dim": 64, "ragged": False, "state": True, "train": False},
        # one tick of 8 cars; latency
        {"name": "step_play", "op": "decay_step", "type": "bfloat16", "batch": 8, "slots": 8, "heads": 8,
         "key_heads": 2, "dim": 64, "value_dim": 64},
        # one tick of 2,048 games, their states in a larger pool
        {"name": "step_serve", "op": "decay_step", "type": "bfloat16", "batch": 2048, "slots": 2100, "heads": 8,
         "key_heads": 8, "dim": 128, "value_dim": 128},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "norm_rotate", "decay_attention", "decay_attention", "decay_step"])
    typ = rng.choice(["bfloat16", "bfloat16", "float32", "float16"])
    dim = rng.choice([64, 64, 128, 128, 96, 80])
    key_heads = rng.choice([1, 2, 3, 4, 8])
    heads = key_heads * rng.choice([1, 1, 2, 4])
    if kind in ("rotate", "norm_rotate"):
        ticks = _log_int(rng, 1, 4096)
        most = max(1, min(4096, (1 << 25) // (ticks * dim * (heads + key_heads))))
        batch = _log_int(rng, 1, most)
        c = {"op": kind, "type": typ, "batch": batch, "ticks": ticks, "heads": heads, "dim": dim,
             "turned": rng.choice([dim, dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
             "scaling": rng.choice(["none", "linear", "parts"]), "first": rng.choice([0, 0, rng.randrange(1 << 20)]),
             "train": rng.random() < 0.5}
        if kind == "norm_rotate":
            c |= {"key_heads": key_heads, "each": rng.random() < 0.3}
        return c
    if kind == "decay_step":
        batch = _log_int(rng, 1, max(1, (1 << 27) // (heads * dim * dim)))
        return {"op": kind, "type": typ, "batch": batch, "slots": batch + rng.randrange(0, 9), "heads": heads,
                "key_heads": key_heads, "dim": dim, "value_dim": rng.choice([dim, 64, 128])}
    train = rng.random() < 0.5
    ticks = _log_int(rng, 1, 16384)
    most = max(1, min(512, (1 << 25) // (ticks * dim * heads)))
    batch = _log_int(rng, 1, most)
    return {"op": kind, "type": typ, "batch": batch, "ticks": ticks, "heads": heads, "key_heads": key_heads,
            "dim": dim, "value_dim": rng.choice([dim, dim, 64]), "ragged": rng.random() < 0.4,
            "state": rng.random() < 0.6, "train": train}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _frequencies(c):
    """Radians a tick for each turned pair, in 64 bits: 10000^(-2i / turned), for longer recordings divided by 8
    ("linear"), or divided by 8 only where the wave is long against 1,024 ticks ("parts": kept above 32 turns in 1,024
    ticks, divided below 1, between the two in proportion)."""
    n = c["turned"] // 2
    f = [10000.0 ** (-i / n) for i in range(n)]
    if c["scaling"] == "linear":
        f = [x / 8 for x in f]
    elif c["scaling"] == "parts":
        keep = [min(1.0, max(0.0, (1024 * x / (2 * math.pi) - 1) / 31)) for x in f]
        f = [x * a + x / 8 * (1 - a) for x, a in zip(f, keep)]
    return f


def _amplitude(c):
    return 0.1 * math.log(8.0) + 1.0 if c["scaling"] == "parts" else 1.0


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
    if c["op"] in ("rotate", "norm_rotate"):
        B, T, H, D, hk = c["batch"], c["ticks"], c["heads"], c["dim"], c.get("key_heads", 0)
        turns = [int(round(f / (2 * math.pi) * 2.0 ** 64)) for f in _frequencies(c)]
        s["turns"] = torch.tensor(turns, dtype=torch.int64, device=DEV)
        first = torch.randint(0, c["first"] + 1, (B, 1), generator=g, device=DEV)
        s["positions"] = first + torch.arange(T, device=DEV)
        if c["op"] == "rotate":
            s["x"] = normal(B, T, H, D)
        else:                                              # one projection's result: queries, keys, values side by side
            packed = normal(B, T, H + 2 * hk, D, scale=2.0)
            s["q"], s["k"] = packed[:, :, :H], packed[:, :, H:H + hk]
            shape = (H, D) if c["each"] else (D,)
            s["wq"] = 1 + normal(*shape, scale=0.2, typ=torch.float32)
            s["wk"] = 1 + normal(*((hk, D) if c["each"] else (D,)), scale=0.2, typ=torch.float32)
        if c["train"]:
            s["gy"] = normal(B, T, H, D)
            if hk:
                s["gk"] = normal(B, T, hk, D)
        return s
    B, H, hk, D, E = c["batch"], c["heads"], c["key_heads"], c["dim"], c["value_dim"]
    # decays from a memory of some 20 ticks to one of thousands, as spread over the heads of one layer
    s["log_decay"] = torch.log1p(-torch.exp2(-4.5 - 7.0 * torch.arange(H, device=DEV) / max(1, H - 1)))
    if c["op"] == "decay_step":
        s["q"], s["k"], s["v"] = normal(B, H, D), normal(B, hk, D), normal(B, hk, E, scale=0.5)
        s["state"] = normal(c["slots"], H, D, E, scale=3.0, typ=torch.float32)
        s["slots"] = torch.randperm(c["slots"], generator=g, device=DEV)[:B]
        return s
    if c["ragged"]:
        s["lengths"] = _lengths(c, seed)
        s["offsets"] = torch.tensor([0] + s["lengths"], device=DEV).cumsum(0)
        lead = (sum(s["lengths"]),)
    else:
        lead = (B, c["ticks"])
    s["q"], s["k"], s["v"] = normal(*lead, H, D), normal(*lead, hk, D), normal(*lead, hk, E, scale=0.5)
    if c["state"]:
        s["state"] = normal(B, H, D, E, scale=3.0, typ=torch.float32)
    if c["train"]:
        s["go"] = normal(*lead, H, E)
        s["gs"] = normal(B, H, D, E, scale=0.05, typ=torch.float32)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"rotate": _plain_rotate, "norm_rotate": _plain_norm_rotate, "decay_attention": _plain_decay_attention,
            "decay_step": _plain_decay_step}[state["case"]["op"]](state)


def _run_own(s):
    from flyguy_b200 import memory
    c, op = s["case"], s["case"]["op"]
    if op == "rotate":
        kw = dict(positions=s["positions"], layout=c["layout"], amplitude=_amplitude(c))
        if not c["train"]:
            return memory.rotate(s["x"], s["turns"], **kw)
        x = s["x"].detach().requires_grad_()
        y = memory.rotate(x, s["turns"], **kw)
        return y.detach(), *torch.autograd.grad(y, x, s["gy"])
    if op == "norm_rotate":
        kw = dict(positions=s["positions"], layout=c["layout"], amplitude=_amplitude(c), eps=1e-6)
        if not c["train"]:
            return memory.norm_rotate(s["q"], s["k"], s["turns"], s["wq"], s["wk"], **kw)
        q, k, wq, wk = (s[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk"))
        y, z = memory.norm_rotate(q, k, s["turns"], wq, wk, **kw)
        return y.detach(), z.detach(), *torch.autograd.grad((y, z), (q, k, wq, wk), (s["gy"], s["gk"]))
    if op == "decay_step":
        o = memory.decay_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"])
        return o, s["state"]
    kw = dict(offsets=s.get("offsets"))
    if not c["train"]:
        return memory.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], s.get("state"), **kw)
    ins = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "state") if n in s]
    o, end = memory.decay_attention(*ins[:3], s["log_decay"], *ins[3:], **kw)
    return o.detach(), end.detach(), *torch.autograd.grad((o, end), ins, (s["go"], s["gs"]))


def _angles(s):
    """cos and sin, [B, T, 1, turned / 2]: the turns in fixed point (64-bit products wrap), rounded to 32 bits once."""
    at = (s["positions"].unsqueeze(-1) * s["turns"]) >> 32
    a = at.float() * (2 * math.pi / 2.0 ** 32)
    return a.cos().unsqueeze(2) * _amplitude(s["case"]), a.sin().unsqueeze(2) * _amplitude(s["case"])


def _turn(x, cos, sin, c):
    """x in 32 bits with its first `turned` values turned, pair by pair."""
    n = c["turned"]
    if c["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., n:]), -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((y, x[..., n:]), -1)


def _plain_rotate(s):
    c, x = s["case"], s["x"]
    cos, sin = _angles(s)
    y = _turn(x.float(), cos, sin, c).to(x.dtype)
    if not c["train"]:
        return y
    return y, _turn(s["gy"].float(), cos, -sin, c).to(x.dtype)


def _plain_norm(x, w, cos, sin, c, gy):
    xf = x.float()
    r = (xf.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    y = _turn(xf * r * w, cos, sin, c).to(x.dtype)
    if gy is None:
        return y, None, None
    g = _turn(gy.float(), cos, -sin, c)
    xh = xf * r
    gw = (g * xh).sum((0, 1) if w.dim() == 2 else (0, 1, 2))
    gx = g * w
    return y, (r * (gx - xh * (gx * xh).mean(-1, keepdim=True))).to(x.dtype), gw


def _plain_norm_rotate(s):
    c = s["case"]
    cos, sin = _angles(s)
    y, gq, gwq = _plain_norm(s["q"], s["wq"], cos, sin, c, s.get("gy"))
    z, gk, gwk = _plain_norm(s["k"], s["wk"], cos, sin, c, s.get("gk"))
    return (y, z, gq, gk, gwq, gwk) if c["train"] else (y, z)


CHUNK = 128


def _chunked(q, k, v, g, first, steps, lead):
    """o_t = q_t S_t and the last S, S_t = e^g S_{t-1} + k_t v_t^T, in chunks of ticks. [B, T, H, .] in 32 bits, each
    row's ticks at the end of T with zeros before them; `first` (or None) enters `steps` ticks before the end, and
    counts e^(g * lead) at its first tick."""
    B, T, H, D = q.shape
    n = -(-max(T, 1) // CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, n * CHUNK - T, 0)).view(B, n, CHUNK, H, -1).permute(0, 3, 1, 2, 4)
               for x in (q, k, v))                                                     # [B, H, n, CHUNK, .]
    t = torch.arange(CHUNK, device=q.device, dtype=torch.float32)
    dt = t[:, None] - t
    within = torch.where(dt >= 0, torch.exp(g[:, None, None] * dt.clamp(min=0)), 0.0)   # [H, CHUNK, CHUNK]
    o = (q @ k.transpose(-1, -2) * within[:, None]) @ v
    part = (k * torch.exp(g[:, None] * (CHUNK - 1 - t))[:, None, :, None]).transpose(-1, -2) @ v   # [B, H, n, D, E]
    m = torch.arange(n + 1, device=q.device, dtype=torch.float32)
    dm = m[:, None] - 1 - m[:n]
    across = torch.where(dm >= 0, torch.exp(g[:, None, None] * CHUNK * dm.clamp(min=0)), 0.0)   # [H, n + 1, n]
    into = (across @ part.flatten(-2)).unflatten(-1, part.shape[-2:])                  # the state into each chunk
    o = o + (q @ into[:, :, :n]) * torch.exp(g[:, None] * (t + 1))[:, None, :, None]
    end = into[:, :, n]
    o = o.permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, -1)[:, n * CHUNK - T:]
    if first is not None:
        q = q.permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, -1)[:, n * CHUNK - T:]
        age = torch.arange(T, device=q.device) - (T - steps[:, None]) + lead               # [B, T]
        f = torch.where(age[..., None] >= lead, torch.exp(g * age[..., None].clamp(min=0)), 0.0)
        o = o + torch.einsum("bthd,bhde->bthe", q, first) * f[..., None]
        last = torch.exp(g * (steps[:, None] - 1 + lead).clamp(min=0))                     # [B, H]
        end = end + first * last[..., None, None]
    return o, end


def _plain_decay_attention(s):
    c, typ = s["case"], s["q"].dtype
    B, T, H, hk = c["batch"], c["ticks"], c["heads"], c["key_heads"]
    ragged = "offsets" in s
    if ragged:
        off = s["offsets"]
        steps = off[1:] - off[:-1]
        at = off[1:, None] - T + torch.arange(T, device=DEV)
        there = at >= off[:-1, None]
        at = at.clamp(min=0)
    else:
        steps = torch.full((B,), T, device=DEV)

    def rows(x):                                           # [B, T, H, .] in 32 bits, ticks at the end of T
        x = x.float()
        if ragged:
            x = torch.where(there[..., None, None], x[at], 0.0)
        return x if x.shape[2] == H else x.repeat_interleave(H // hk, 2)

    def back(x, shared=False):
        if shared:
            x = x.unflatten(2, (hk, H // hk)).sum(3)
        return (x[there] if ragged else x).to(typ)

    scale, g, first = c["dim"] ** -0.5, s["log_decay"], s.get("state")
    q, k, v = rows(s["q"]), rows(s["k"]), rows(s["v"])
    o, end = _chunked(q * scale, k, v, g, first, steps, 1)
    if not c["train"]:
        return back(o), end
    go = rows(s["go"]) * scale
    gq, _ = _chunked(go, v, k, g, None if first is None else first.transpose(-1, -2), steps, 1)

    def turned(x):                                         # ticks from last to first, still at the end of T
        x = x.flip(1)
        i = (torch.arange(T, device=DEV) - (T - steps[:, None])) % max(T, 1)
        return x.gather(1, i[..., None, None].expand(-1, -1, *x.shape[2:])) if ragged else x

    qr, kr, vr, gr = turned(q), turned(k), turned(v), turned(go)
    gv, r = _chunked(kr, qr, gr, g, s["gs"], steps, 0)
    gk, _ = _chunked(vr, gr, qr, g, s["gs"].transpose(-1, -2), steps, 0)
    if ragged:                                             # rows without ticks hand the state's gradient through
        r = torch.where((steps > 0)[:, None, None, None], r * torch.exp(g)[:, None, None], s["gs"])
    else:
        r = r * torch.exp(g)[:, None, None]
    out = (back(o), end, back(gq), back(turned(gk), True), back(turned(gv), True))
    return out if first is None else (*out, r)


def _plain_decay_step(s):
    c, at = s["case"], s["slots"]
    n = c["heads"] // c["key_heads"]
    q, k, v = s["q"].float(), s["k"].float().repeat_interleave(n, 1), s["v"].float().repeat_interleave(n, 1)
    S = s["state"][at] * torch.exp(s["log_decay"])[:, None, None] + k.unsqueeze(-1) * v.unsqueeze(-2)
    s["state"][at] = S
    o = (q.unsqueeze(-2) @ S).squeeze(-2) * c["dim"] ** -0.5
    return o.to(s["q"].dtype), s["state"]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    c, e = case, SIZE[case["type"]]
    if c["op"] in ("rotate", "norm_rotate"):
        values = c["batch"] * c["ticks"] * (c["heads"] + c.get("key_heads", 0)) * c["dim"]
        times = 2 if c["train"] else 1
        return {"bytes": 2.0 * times * values * e + 8 * c["batch"] * c["ticks"], "flops": 8.0 * times * values}
    H, hk, D, E = c["heads"], c["key_heads"], c["dim"], c["value_dim"]
    if c["op"] == "decay_step":
        return {"bytes": c["batch"] * (8.0 * H * D * E + e * (H * (D + E) + hk * (D + E))),
                "flops": 5.0 * c["batch"] * H * D * E}
    rows = sum(_lengths(c, 0)) if c["ragged"] else c["batch"] * c["ticks"]
    tick = e * (H * D + hk * (D + E) + H * E)
    states = 4.0 * c["batch"] * H * D * E
    if not c["train"]:
        return {"bytes": rows * tick + states * (2 if c["state"] else 1), "flops": 4.0 * rows * H * D * E}
    return {"bytes": 2 * rows * tick + states * (4 if c["state"] else 2), "flops": 12.0 * rows * H * D * E}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] in ("rotate", "norm_rotate"):
        return _exact_rotations(case, s)
    if case["op"] == "decay_step":
        return _exact_step(case, s)
    return _exact_attention(case, s)


def _exact_rotations(c, s):
    """The pairs as complex numbers times a e^(i angle)."""
    f = torch.tensor(_frequencies(c), dtype=torch.float64, device=DEV)
    angle = (s["positions"].double().unsqueeze(-1) * f).unsqueeze(2)
    unit = torch.polar(torch.full_like(angle, _amplitude(c)), angle)
    n = c["turned"]
    if c["layout"] == "half":
        first, second = torch.arange(n // 2, device=DEV), torch.arange(n // 2, n, device=DEV)
    else:
        first, second = torch.arange(0, n, 2, device=DEV), torch.arange(1, n, 2, device=DEV)

    def turn(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if c["op"] == "rotate":
        return (turn(s["x"], unit), turn(s["gy"], unit.conj())) if c["train"] else turn(s["x"], unit)
    ys, gxs, gws = [], [], []
    for x, w, gy in (("q", "wq", "gy"), ("k", "wk", "gk")):
        x, w = s[x], s[w]
        norm = torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
        ys.append(turn(x / norm * w, unit))
        if c["train"]:
            g = turn(s[gy], unit.conj())
            gw = g * (x / norm)
            gws.append(gw.sum((0, 1)) if c["each"] else gw.sum((0, 1, 2)))
            gw = None
            g = g * w
            gxs.append(g / norm - x * (g * x).sum(-1, keepdim=True) / (norm ** 3 * x.shape[-1]))
    return (*ys, *gxs, *gws)


def _exact_step(c, s):
    q, k, v, S, at = s["q"], s["k"], s["v"], s["state"], s["slots"]
    decay = s["log_decay"].exp()
    n = c["heads"] // c["key_heads"]
    o = torch.empty(c["batch"], c["heads"], c["value_dim"], dtype=torch.float64, device=DEV)
    for h in range(c["heads"]):
        new = decay[h] * S[at, h] + torch.einsum("bd,be->bde", k[:, h // n], v[:, h // n])
        S[at, h] = new
        o[:, h] = torch.einsum("bd,bde->be", q[:, h], new) / math.sqrt(c["dim"])
    return o, S


def _exact_attention(c, s):
    """Tick by tick, forward and back."""
    B, T, H, hk, D, E = c["batch"], c["ticks"], c["heads"], c["key_heads"], c["dim"], c["value_dim"]
    if T * (3 if c["train"] else 1) * max(2e-4, B * H * D * E * 8 * 4 / 2e12) > 16:
        return None
    n, scale = H // hk, 1 / math.sqrt(D)
    q, k, v = s["q"], s["k"], s["v"]
    decay = s["log_decay"].exp()[:, None, None]
    if c["ragged"]:
        off = s["offsets"].tolist()
        order = sorted(range(B), key=lambda b: off[b] - off[b + 1])     # longest first: those still running are a prefix
        ends = [off[b + 1] - off[b] for b in order]
        base = torch.tensor([off[b] for b in order], device=DEV)
        running = [sum(1 for e in ends if e > t) for t in range(T)]

        def take(x, t):
            return x[base[:running[t]] + t]

        def put(x, t, y):
            x[base[:running[t]] + t] = y
    else:
        order, running = list(range(B)), [B] * T

        def take(x, t):
            return x[:, t]

        def put(x, t, y):
            x[:, t] = y
    sort = torch.tensor(order, device=DEV)
    wide = lambda x: x.repeat_interleave(n, 1)             # noqa: E731  key heads as the query heads see them
    S = s["state"][sort].clone() if c["state"] else torch.zeros(B, H, D, E, dtype=torch.float64, device=DEV)
    o, gq = torch.empty_like(s["q"][..., :1].expand(*s["q"].shape[:-1], E)).contiguous(), torch.empty_like(q)
    for t in range(T):
        r = running[t]
        now = S[:r].mul_(decay).add_(wide(take(k, t)).unsqueeze(-1) * wide(take(v, t)).unsqueeze(-2))
        put(o, t, torch.einsum("bhd,bhde->bhe", take(q, t), now) * scale)
        if c["train"]:
            put(gq, t, torch.einsum("bhde,bhe->bhd", now, take(s["go"], t)) * scale)
    end = torch.empty_like(S)
    end[sort] = S
    if not c["train"]:
        return o, end
    R, gk, gv = s["gs"][sort].clone(), torch.empty_like(k), torch.empty_like(v)
    for t in reversed(range(T)):
        r = running[t]
        now = R[:r].add_((take(q, t) * scale).unsqueeze(-1) * take(s["go"], t).unsqueeze(-2))
        put(gk, t, torch.einsum("bhde,bhe->bhd", now, wide(take(v, t))).unflatten(1, (hk, n)).sum(2))
        put(gv, t, torch.einsum("bhde,bhd->bhe", now, wide(take(k, t))).unflatten(1, (hk, n)).sum(2))
        now.mul_(decay)
    first = torch.empty_like(R)
    first[sort] = R
    return (o, end, gq, gk, gv, first) if c["state"] else (o, end, gq, gk, gv)
