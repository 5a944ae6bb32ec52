"""Timed cases of the decoder-block operators: rotary positions, counter-based dropout (alone, and
inside the residual add + LayerNorm), and attention with a per-head decay (prompts, training, single
tokens).

``run`` computes one pass of a case: in plain torch operations where ``own`` is false, through
``nexar_b200.ops`` where it is true. Both start from what ``prepare`` returns.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one new token of 16 sequences at positions of their own, 12 heads of 64 (the GPT-2 layer's heads)
        dict(name="rotary-step", op="rotary", B=16, T=1, Hq=12, Hk=12, D=64, R=64, layout="half", dtype="bf16",
             scaling="none", own_positions=True, packed=False, train=False),
        # one layer's packed QKV projection in a GPT-2 training step (8 x 1024 tokens), both directions
        dict(name="rotary-train", op="rotary", B=8, T=1024, Hq=12, Hk=12, D=64, R=64, layout="half", dtype="bf16",
             scaling="none", own_positions=False, packed=True, train=True),
        # a long prompt past the trained length, shared key heads, part of the head rotated
        dict(name="rotary-long", op="rotary", B=1, T=65537, Hq=32, Hk=8, D=128, R=96, layout="interleaved",
             dtype="bf16", scaling="yarn", own_positions=False, packed=False, train=False),
        # a small odd tensor: latency, and a tail that ends inside a block of draws
        dict(name="dropout-odd", op="dropout", rows=7, cols=1001, dtype="fp16", p=0.1),
        # activations of 16384 tokens at width 4096, both directions
        dict(name="dropout-wide", op="dropout", rows=16384, cols=4096, dtype="bf16", p=0.2),
        # residual add + dropout + LayerNorm of one GPT-2 layer (8 x 1024 tokens of 768), both directions
        dict(name="residual-gpt2", op="residual", rows=8192, cols=768, p=0.1, bias=True),
        # the same at width 2048 and 32768 tokens
        dict(name="residual-wide", op="residual", rows=32768, cols=2048, p=0.1, bias=True),
        # one new token of one sequence
        dict(name="decay-step", op="step", B=1, H=12, D=64),
        # one new token of many sequences, heads of 128
        dict(name="decay-step-batch", op="step", B=192, H=32, D=128),
        # prompts of different lengths (an empty one among them) that go on from a state
        dict(name="decay-prompts", op="decay", B=5, T=1000, H=12, D=64, ragged=True, state=True, train=False),
        # one GPT-2-sized layer in training, both directions
        dict(name="decay-train", op="decay", B=8, T=1024, H=12, D=64, ragged=False, state=False, train=True),
        # few long sequences, heads of 128, from a state, both directions
        dict(name="decay-train-long", op="decay", B=1, T=16385, H=16, D=128, ragged=False, state=True, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "dropout", "residual", "step", "decay", "decay"])
    if op == "rotary":
        D = rng.choice([32, 64, 80, 128])
        Hk = rng.choice([1, 2, 4, 8, 12])
        Hq = Hk * rng.choice([1, 2, 4])
        B = _log(rng, 1, 32)
        T = _log(rng, 1, max(1, min(65536, 3 * 10 ** 8 // (B * (Hq + 2 * Hk) * D))))
        return dict(op=op, B=B, T=T, Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D, D // 2, D // 4 * 3]),
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    scaling=rng.choice(["none", "linear", "ntk", "bands", "yarn"]), own_positions=rng.random() < 0.5,
                    packed=rng.random() < 0.5, train=rng.random() < 0.5)
    if op == "dropout":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, cols=_log(rng, 1, 4096), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    p=rng.choice([0.05, 0.1, 0.2, 0.5]))
    if op == "residual":
        return dict(op=op, rows=_log(rng, 1, 32768), cols=8 * rng.randint(2, 256), p=rng.choice([0.05, 0.1, 0.2]),
                    bias=rng.random() < 0.7)
    if op == "step":
        return dict(op=op, B=_log(rng, 1, 160), H=rng.randint(1, 32), D=rng.choice([64, 128]))
    D = rng.choice([64, 64, 128])
    B, H = _log(rng, 1, 16), rng.randint(1, 16)
    T = _log(rng, 1, max(1, min(16384, 2 * 10 ** 7 // (B * H * D))))
    train = rng.random() < 0.5
    return dict(op=op, B=B, T=T, H=H, D=D, ragged=not train and B > 1 and rng.random() < 0.7, state=rng.random() < 0.5,
                train=train)


# ---------------------------------------------------------------- inputs
SCALING = {  # name -> (factor, original length); the remaining constants are the operator's defaults
    "none": None, "linear": (4.0, 2048), "ntk": (4.0, 2048), "bands": (8.0, 8192), "yarn": (16.0, 4096)}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return (std * torch.randn(*shape, device=dev, generator=g)).to(dtype)

    s = dict(case=case, dev=dev)
    op = case["op"]
    if op == "rotary":
        dt, B, T, Hq, Hk, D = DTYPES[case["dtype"]], case["B"], case["T"], case["Hq"], case["Hk"], case["D"]
        reach = T + 4096
        first = int(torch.randint(0, 4096, (1,), device=dev, generator=g)) if not case["own_positions"] else 0
        s["start"] = first
        s["positions"] = torch.randint(0, reach, (B, T), device=dev, generator=g) if case["own_positions"] else None
        qkv = normal(B, T, Hq + 2 * Hk, D, dtype=dt)
        s["qkv"] = qkv.requires_grad_(case["train"])
        # the pair form reads the query and key heads where the projection left them
        s["q"], s["k"] = qkv.detach()[:, :, :Hq].requires_grad_(case["train"]), qkv.detach()[:, :, Hq:Hq + Hk].requires_grad_(case["train"])
        if case["train"]:
            s["dqkv"] = normal(B, T, Hq + 2 * Hk, D, dtype=dt)
            s["dq"], s["dk"] = s["dqkv"][:, :, :Hq].contiguous(), s["dqkv"][:, :, Hq:Hq + Hk].contiguous()
        if own:  # the table of cosines and sines that a program builds once
            from nexar_b200 import ops
            sc = SCALING[case["scaling"]]
            s["table"] = ops.rotary_table(reach, case["R"], scaling=None if sc is None else ops.RotaryScaling(
                case["scaling"], factor=sc[0], original_length=sc[1]), device=dev)
    elif op in ("dropout", "residual"):
        if op == "dropout":
            dt = DTYPES[case["dtype"]]
            s["x"] = normal(case["rows"], case["cols"], dtype=dt).requires_grad_(True)
            s["dy"] = normal(case["rows"], case["cols"], dtype=dt)
        else:
            R, C = case["rows"], case["cols"]
            for n in ("x", "r"):
                s[n] = normal(R, C).requires_grad_(True)
            s["ds"], s["dy"] = normal(R, C), normal(R, C)
            s["w"] = (1 + 0.1 * torch.randn(C, device=dev, generator=g)).to(torch.bfloat16).requires_grad_(True)
            s["b"] = normal(C, std=0.1).requires_grad_(True)
            s["rb"] = normal(C, std=0.1).requires_grad_(True) if case["bias"] else None
        # (seed, step) of the generator on the device, and the call's number within the step
        s["rng"] = torch.tensor([(seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), seed % 1000], device=dev)
        s["site"] = 3 + seed % 17
        if own:
            from nexar_b200 import ops
            s["dropout"] = ops.DropoutState(0, device=dev)
            s["dropout"].tensor.copy_(s["rng"])
    else:
        B, H, D = case["B"], case["H"], case["D"]
        # decays from about 1 - 2^-5 to 1 - 2^-9 over the heads, one head without decay
        lam = 1 - 2.0 ** -(5 + 4 * torch.rand(H, device=dev, generator=g))
        lam[0] = 1.0
        s["log_decay"] = lam.log()
        if op == "step":
            s["q"], s["k"], s["v"] = (normal(B, H, D) for _ in range(3))
            s["state"] = normal(B, H, D, D, dtype=torch.float32, std=4.0)
        else:
            T, tr = case["T"], case["train"]
            s["qkv"] = normal(B, T, 3, H, D).requires_grad_(tr)
            s["state"] = normal(B, H, D, D, dtype=torch.float32, std=4.0).requires_grad_(tr) if case["state"] else None
            s["lengths"] = None
            if case["ragged"]:
                n = torch.randint(0, T + 1, (B,), device=dev, generator=g, dtype=torch.int32)
                n[0], n[-1] = T, 0
                s["lengths"] = n
            if tr:
                s["do"] = normal(B, T, H, D)
                s["dstate"] = normal(B, H, D, D, dtype=torch.float32) if case["state"] else None
    return s


# ---------------------------------------------------------------- plain forms
def _frequencies(case, dev):
    """Turns per token of each pair, in 64 bits, and the factor on cosine and sine."""
    R, base, m = case["R"], 10000.0, 1.0
    i = torch.arange(R // 2, dtype=torch.float64, device=dev)
    f = base ** (-2.0 * i / R)
    kind = case["scaling"]
    if kind != "none":
        factor, length = SCALING[kind]
        if kind == "linear":
            f = f / factor
        elif kind == "ntk":
            f = (base * factor ** (R / (R - 2.0))) ** (-2.0 * i / R)
        elif kind == "bands":
            turns = length * f / (2 * math.pi)
            keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
            f = f / factor * (1 - keep) + f * keep
        else:
            def pair_of(turns):
                return R * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
            low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), R // 2 - 1)
            far = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
            f = f / factor * far + f * (1 - far)
            m = 0.1 * math.log(factor) + 1.0
    return f, m


def _angles(s):
    case = s["case"]
    f, m = _frequencies(case, s["dev"])
    pos = s["positions"] if s["positions"] is not None else s["start"] + torch.arange(case["T"], device=s["dev"])[None]
    a = pos.double()[..., None, None] * f
    return (m * a.cos()).float(), (m * a.sin()).float()


def _rotate(x, cos, sin, R, layout, dtype):
    x = x.float()
    head, rest = x[..., :R], x[..., R:]
    if layout == "half":
        a, b = head[..., :R // 2], head[..., R // 2:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([head, rest], dim=-1).to(dtype)


def _plain_rotary(s):
    case = s["case"]
    cos, sin = _angles(s)
    dt, R, lay, n = DTYPES[case["dtype"]], case["R"], case["layout"], case["Hq"] + case["Hk"]
    with torch.no_grad():
        if case["packed"]:
            out = torch.cat([_rotate(s["qkv"][:, :, :n], cos, sin, R, lay, dt), s["qkv"][:, :, n:]], dim=2)
            if not case["train"]:
                return [out]
            return [out, torch.cat([_rotate(s["dqkv"][:, :, :n], cos, -sin, R, lay, dt), s["dqkv"][:, :, n:]], dim=2)]
        out = [_rotate(s["q"], cos, sin, R, lay, dt), _rotate(s["k"], cos, sin, R, lay, dt)]
        if case["train"]:
            out += [_rotate(s["dq"], cos, -sin, R, lay, dt), _rotate(s["dk"], cos, -sin, R, lay, dt)]
        return out


def _draws(n, rng, site):
    """16-bit draws of elements 0 .. n-1: Philox4x32-10 (Salmon et al., 2011), one 128-bit block per 8 elements.
    Counter (block low, block high, site, step), key = the seed."""
    low = 0xFFFFFFFF
    b = torch.arange((n + 7) // 8, device=rng.device)
    c0, c1, c2, c3 = b & low, b >> 32, torch.full_like(b, site), (rng[1] & low).expand_as(b)
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    w = torch.stack([c0, c1, c2, c3], dim=-1)
    return torch.stack([w & 0xFFFF, w >> 16], dim=-1).reshape(-1)[:n]


def _keep(s, rows, cols):
    t = round(s["case"]["p"] * 65536)
    return (_draws(rows * cols, s["rng"], s["site"]) >= t).view(rows, cols), 65536.0 / (65536 - t)


def _plain_dropout(s):
    case = s["case"]
    keep, scale = _keep(s, case["rows"], case["cols"])
    with torch.no_grad():
        return [torch.where(keep, t.float() * scale, 0.0).to(t.dtype) for t in (s["x"], s["dy"])]


def _plain_residual(s):
    case = s["case"]
    R, C = case["rows"], case["cols"]
    keep, scale = _keep(s, R, C)
    bf = torch.bfloat16
    with torch.no_grad():
        r = s["r"].float() + (s["rb"].float() if case["bias"] else 0.0)
        # the stored sum is what the norm reads, as in the operator without dropout
        st = (s["x"].float() + torch.where(keep, r * scale, 0.0)).to(bf)
        f, w, dy = st.float(), s["w"].float(), s["dy"].float()
        mean = f.mean(-1, keepdim=True)
        rstd = ((f - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        xh = (f - mean) * rstd
        y = xh * w + s["b"].float()
        gw = dy * w
        dx = s["ds"].float() + rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
        dr = torch.where(keep, dx * scale, 0.0)
        out = [st, y.to(bf), dx.to(bf), dr.to(bf), (dy * xh).sum(0).to(bf), dy.sum(0).to(bf)]
        return out + ([dr.sum(0).to(bf)] if case["bias"] else [])


def _plain_decay(qkv, g, scale, state, lengths):
    """o, final state: blocks of 128 tokens; inside a block the decayed scores, across blocks the decayed states."""
    B, T, _, H, D = qkv.shape
    n, C = -(-T // 128), 128
    x = qkv.float()
    pos = torch.arange(T, device=qkv.device)
    length = lengths if lengths is not None else torch.full((B,), T, device=qkv.device)
    live = pos[None] < length[:, None]
    if lengths is not None:
        x = torch.where(live[:, :, None, None, None], x, 0.0)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, 0, 0, n * C - T)).view(B, n, C, 3, H, D).permute(3, 0, 4, 1, 2, 5)
    q, k, v = x[0] * scale, x[1], x[2]                      # [B, H, n, C, D]
    g = g.double()[:, None, None]
    i = torch.arange(C, device=qkv.device, dtype=torch.float64)
    gap = i[:, None] - i[None]
    inside = torch.where(gap >= 0, (g * gap.clamp(min=0)).exp(), 0.0).float()          # [H, C, C]
    o = ((q @ k.transpose(-1, -2)) * inside[None, :, None]) @ v
    tail = (g * (C - 1 - i)[None, :, None]).exp().float()                              # [H, C, 1]
    part = (k * tail[None, :, None]).transpose(-1, -2) @ v                             # [B, H, n, D, D]
    m = torch.arange(n, device=qkv.device, dtype=torch.float64)
    gap = m[:, None] - 1 - m[None]
    across = torch.where(gap >= 0, (g * C * gap.clamp(min=0)).exp(), 0.0).float()      # [H, n, n]
    before = (across @ part.flatten(3)).view_as(part)
    if state is not None:
        before = before + (g * C * m[None, :, None]).exp().float()[..., None] * state[:, :, None]
    o = o + (q * (g * (i + 1)[None, :, None]).exp().float()[None, :, None]) @ before
    o = o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, D)[:, :T]
    left = (length[:, None] - 1 - pos[None]).double()                                  # [B, T]
    w = torch.where(live[:, None], (g[None, :, :, 0] * left.clamp(min=0)[:, None]).exp(), 0.0).float()  # [B, H, T]
    w = torch.nn.functional.pad(w, (0, n * C - T))
    final = (k.flatten(2, 3) * w[..., None]).transpose(-1, -2) @ v.flatten(2, 3)
    if state is not None:
        final = final + (g[None] * length.double()[:, None, None, None]).exp().float() * state
    return o, final


def _run_plain_decay(s):
    case = s["case"]
    scale = case["D"] ** -0.5
    if not case["train"]:
        o, final = _plain_decay(s["qkv"], s["log_decay"], scale, s["state"], s["lengths"])
        return [o.to(torch.bfloat16), final]
    x = s["qkv"].detach().float().requires_grad_(True)
    st = s["state"].detach().clone().requires_grad_(True) if case["state"] else None
    o, final = _plain_decay(x, s["log_decay"], scale, st, None)
    if not case["state"]:
        (dx,) = torch.autograd.grad(o, x, s["do"].float())
        return [o.detach().to(torch.bfloat16), dx.to(torch.bfloat16)]
    dx, dst = torch.autograd.grad((o, final), (x, st), (s["do"].float(), s["dstate"]))
    return [o.detach().to(torch.bfloat16), final.detach(), dx.to(torch.bfloat16), dst]


def _plain_step(s):
    lam = s["log_decay"].double().exp().float()[:, None, None]
    st = lam * s["state"] + s["k"].float()[..., :, None] * s["v"].float()[..., None, :]
    s["state"].copy_(st)
    o = (s["q"].float()[..., None, :] @ st)[..., 0, :] * s["case"]["D"] ** -0.5
    return [o.to(torch.bfloat16), s["state"]]


# ---------------------------------------------------------------- the framework's calls
def _own(s):
    from nexar_b200 import ops
    case = s["case"]
    op = case["op"]
    if op == "rotary":
        kw = dict(positions=s["positions"], start=s["start"], layout=case["layout"])
        if case["packed"]:
            out = ops.rotary(s["qkv"], s["table"], heads=case["Hq"] + case["Hk"], **kw)
            return [out, *torch.autograd.grad(out, s["qkv"], s["dqkv"])] if case["train"] else [out]
        out = ops.rotary_qk(s["q"], s["k"], s["table"], **kw)
        return [*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))] if case["train"] else list(out)
    if op == "dropout":
        y = ops.dropout(s["x"], case["p"], s["dropout"], site=s["site"])
        return [y, *torch.autograd.grad(y, s["x"], s["dy"])]
    if op == "residual":
        out = ops.residual_layer_norm(s["x"], s["r"], s["w"], s["b"], 1e-5, rbias=s["rb"], p=case["p"],
                                      dropout=s["dropout"], site=s["site"])
        leaves = [s["x"], s["r"], s["w"], s["b"]] + ([s["rb"]] if case["bias"] else [])
        return [*out, *torch.autograd.grad(out, leaves, (s["ds"], s["dy"]))]
    if op == "step":
        o = ops.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        return [o, s["state"]]
    if not case["train"]:
        q, k, v = s["qkv"].unbind(2)
        return list(ops.decay_attention(q, k, v, s["log_decay"], state=s["state"], lengths=s["lengths"],
                                        return_state=True))
    if not case["state"]:
        o = ops.decay_attention_qkv(s["qkv"], s["log_decay"])
        return [o, *torch.autograd.grad(o, s["qkv"], s["do"])]
    out = ops.decay_attention_qkv(s["qkv"], s["log_decay"], state=s["state"], return_state=True)
    return [*out, *torch.autograd.grad(out, (s["qkv"], s["state"]), (s["do"], s["dstate"]))]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "dropout": _plain_dropout, "residual": _plain_residual, "step": _plain_step,
            "decay": _run_plain_decay}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "rotary":
        width = {"fp32": 4}.get(case["dtype"], 2)
        tokens, ways = case["B"] * case["T"], 2 if case["train"] else 1
        heads = case["Hq"] + case["Hk"] * (2 if case["packed"] else 1)
        turned = tokens * (case["Hq"] + case["Hk"]) * case["R"]
        return {"bytes": ways * 2 * tokens * heads * case["D"] * width, "flops": ways * 3 * turned}
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n * (4 if case["dtype"] == "fp32" else 2), "flops": 2 * n}
    if op == "residual":
        n = case["rows"] * case["cols"]
        # forward: x, r in and s, y out; backward: ds, dy, s in and dx, dr out
        return {"bytes": 9 * n * 2, "flops": 30 * n}
    B, H, D = case["B"], case["H"], case["D"]
    if op == "step":
        return {"bytes": B * H * (2 * D * D * 4 + 4 * D * 2), "flops": 5 * B * H * D * D}
    rows, st = B * case["T"] * H, B * H * D * D * 4
    if not case["train"]:
        read = 0.5 if case["ragged"] else 1.0  # rows behind the last token of a sequence are not read
        return {"bytes": rows * D * 2 * (3 * read + 1) + st * (1 + case["state"]), "flops": 4 * rows * D * D * read}
    return {"bytes": rows * D * 2 * (4 + 7) + st * 4 * case["state"], "flops": 12 * rows * D * D}


# ---------------------------------------------------------------- 64-bit values from the definitions
def _exact_turn(x, pos, case, back):
    """Each pair as a complex number times exp(i pos f), in 64 bits; ``back`` turns the other way."""
    R = case["R"]
    j = np.arange(0, R, 2, dtype=np.float64)
    f, m, kind = 10000.0 ** (-j / R), 1.0, case["scaling"]
    if kind != "none":
        factor, length = SCALING[kind]
        if kind == "linear":
            f = f / factor
        elif kind == "ntk":
            f = (10000.0 * factor ** (R / (R - 2))) ** (-j / R)
        elif kind == "bands":
            wave = 2 * np.pi / f
            blend = (length / wave - 1) / 3
            mid = (1 - blend) * f / factor + blend * f
            f = np.where(wave > length, f / factor, np.where(wave < length / 4, f, mid))
        else:
            at = [R / 2 * math.log(length / (2 * math.pi * t)) / math.log(10000.0) for t in (32, 1)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), R // 2 - 1)
            far = np.clip((j / 2 - lo) / max(hi - lo, 1e-3), 0, 1)
            f, m = f * (1 + far * (1 / factor - 1)), 1 + math.log(factor) / 10
    angle = pos[..., None] * torch.from_numpy(f).to(pos.device)
    turn = torch.polar(torch.full_like(angle, m), -angle if back else angle)[:, :, None]
    x = x.detach().double()
    head = x[..., :R]
    pairs = head.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["layout"] == "half" else head.unflatten(-1, (R // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else z.flatten(-2)
    return torch.cat([z, x[..., R:]], dim=-1)


def _exact_keep(n, rng, site, p):
    """Philox4x32-10 on the host in unsigned 64-bit arithmetic."""
    seed, step = (int(v) & (2 ** 64 - 1) for v in rng.tolist())
    u, m32 = np.uint64, np.uint64(0xFFFFFFFF)
    idx = np.arange(-(-n // 8), dtype=np.uint64)
    x = [idx & m32, idx >> u(32), np.full_like(idx, site), np.full_like(idx, step & 0xFFFFFFFF)]
    for r in range(10):
        ka = u((seed + r * 0x9E3779B9) & 0xFFFFFFFF)
        kb = u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [(b >> u(32)) ^ x[1] ^ ka, b & m32, (a >> u(32)) ^ x[3] ^ kb, a & m32]
    words = np.stack(x, axis=1).astype(np.uint32)
    return words.view(np.uint16).reshape(-1)[:n] >= round(p * 65536)  # little-endian: the low half first


def _exact_decay(case, s):
    """The sums over earlier tokens written out, a block of queries at a time."""
    B, T, H, D = case["B"], case["T"], case["H"], case["D"]
    q, k, v = (t.detach().double().transpose(1, 2) for t in s["qkv"].unbind(2))         # [B, H, T, D]
    g, c = s["log_decay"].double().view(1, H, 1, 1), D ** -0.5
    n = (s["lengths"].double() if s["lengths"] is not None else torch.full((B,), float(T), device=q.device, dtype=torch.float64)).view(B, 1, 1, 1)
    t = torch.arange(T, device=q.device, dtype=torch.float64)
    live = t.view(1, 1, T, 1) < n
    q, k, v = q * live, k * live, v * live
    s0 = s["state"].detach().double() if s["state"] is not None else q.new_zeros(B, H, D, D)
    do = s["do"].double().transpose(1, 2) if case["train"] else None
    d1 = s["dstate"].double() if case["train"] and s["dstate"] is not None else torch.zeros_like(s0)
    o = torch.empty_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.exp(g * (t + 1).view(1, 1, T, 1))                 # of the first state at token t
    step = max(1, min(512, (1 << 29) // (B * H * T)))
    for a in range(0, T, step):
        e = min(T, a + step)
        gap = (t[a:e, None] - t[None, :e])[None, None]
        w = torch.exp(g * gap.clamp(min=0)) * (gap >= 0) * c
        sc = torch.einsum("bhid,bhjd->bhij", q[:, :, a:e], k[:, :, :e]) * w
        o[:, :, a:e] = sc @ v[:, :, :e] + c * reach[:, :, a:e] * (q[:, :, a:e] @ s0)
        if do is not None:
            dv[:, :, :e] += sc.transpose(-1, -2) @ do[:, :, a:e]
            dp = torch.einsum("bhid,bhjd->bhij", do[:, :, a:e], v[:, :, :e]) * w
            dq[:, :, a:e] = dp @ k[:, :, :e] + c * reach[:, :, a:e] * (do[:, :, a:e] @ s0.transpose(-1, -2))
            dk[:, :, :e] += dp.transpose(-1, -2) @ q[:, :, a:e]
    left = torch.exp(g * (n - 1 - t.view(1, 1, T, 1)).clamp(min=0)) * live                # of token t in the last state
    final = (k * left).transpose(-1, -2) @ v + torch.exp(g * n) * s0
    if do is None:
        return [o.transpose(1, 2), final]
    dk += left * (v @ d1.transpose(-1, -2))
    dv += left * (k @ d1)
    ds0 = c * (q * reach).transpose(-1, -2) @ do + torch.exp(g * n) * d1
    dqkv = torch.stack([x.transpose(1, 2) for x in (dq, dk, dv)], dim=2)
    return [o.transpose(1, 2), final, dqkv, ds0] if case["state"] else [o.transpose(1, 2), dqkv]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "rotary":
            B, T, n = case["B"], case["T"], case["Hq"] + case["Hk"]
            pos = s["positions"].double() if s["positions"] is not None else \
                s["start"] + torch.arange(T, device=s["dev"], dtype=torch.float64).expand(B, T)
            if case["packed"]:
                def turn(x, back):
                    return torch.cat([_exact_turn(x[:, :, :n], pos, case, back), x[:, :, n:].double()], dim=2)
                return [turn(s["qkv"], False)] + ([turn(s["dqkv"], True)] if case["train"] else [])
            out = [_exact_turn(s[x], pos, case, False) for x in ("q", "k")]
            return out + ([_exact_turn(s[x], pos, case, True) for x in ("dq", "dk")] if case["train"] else [])
        if op in ("dropout", "residual"):
            R, C = case["rows"], case["cols"]
            keep = torch.from_numpy(_exact_keep(R * C, s["rng"], s["site"], case["p"])).to(s["dev"]).view(R, C).double()
            keep /= 1 - round(case["p"] * 65536) / 65536
            if op == "dropout":
                return [s["x"].double() * keep, s["dy"].double() * keep]
            r = s["r"].double() + (s["rb"].double() if case["bias"] else 0)
            total = s["x"].double() + keep * r
            st = total.to(torch.bfloat16).double()  # the norm is that of the stored sum
            sd = (st.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
            xh = (st - st.mean(-1, keepdim=True)) / sd
            w, dy = s["w"].double(), s["dy"].double()
            # the normalised row's Jacobian: remove the mean and the part along xh
            gw = dy * w
            inner = gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True)
            dx = s["ds"].double() + inner / sd
            dr = dx * keep
            out = [total, xh * w + s["b"].double(), dx, dr, (dy * xh).sum(0), dy.sum(0)]
            return out + ([dr.sum(0)] if case["bias"] else [])
        if op == "step":
            lam = torch.exp(s["log_decay"].double()).view(1, -1, 1, 1)
            st = lam * s["state"].double() + torch.einsum("bhi,bhj->bhij", s["k"].double(), s["v"].double())
            return [torch.einsum("bhi,bhij->bhj", s["q"].double(), st) / math.sqrt(case["D"]), st]
        return _exact_decay(case, s)
