"""The decayed linear attention, the norms around a block and gradient clipping, case by case.

A case is a dict of plain values.  Its "kind" names the call:

* train    linear_attn_fn, forward and backward: one layer of a training step;
* prompt   linear_attn_fn without autograd: a prompt that fills the decode state;
* step     linear_attn_update: one token per sequence, the state advancing in place;
* border   block_norm_fn: the norm after a block, its gate and residual scale, and the norm in front of the next one;
* heads    gated_rms_norm_fn: the gated norm of each head inside a block;
* clip     clip_grads: the norm over all gradients of a model and the clipped gradients.

With ``own`` false the plain forms below run, elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
CHUNK = 64          # tokens per chunk of the plain linear attention


# ---------------------------------------------------------------- cases --
def listed():
    return [
        # one token of one conversation in a 768-wide model: launches and latency
        {"name": "step_single", "kind": "step", "batch": 1, "heads": 24, "groups": 24, "dk": 64, "dv": 64, "dtype": "bf16"},
        # one token of a full serving batch of a 1024-wide model
        {"name": "step_batch", "kind": "step", "batch": 64, "heads": 16, "groups": 16, "dk": 128, "dv": 128, "dtype": "bf16"},
        # one long document read by a single user: few rows, a long axis
        {"name": "prompt_long", "kind": "prompt", "batch": 1, "len": 32768, "heads": 24, "groups": 24, "dk": 64, "dv": 64,
         "dtype": "bf16", "ragged": False, "initial": False, "decay": "token"},
        # prompts of different lengths continued from earlier turns, keys shared by several heads, fp32
        {"name": "prompt_ragged", "kind": "prompt", "batch": 5, "len": 1021, "heads": 24, "groups": 4, "dk": 64, "dv": 64,
         "dtype": "f32", "ragged": True, "initial": True, "decay": "token"},
        # one layer of a 768-wide model's training step
        {"name": "train_layer", "kind": "train", "batch": 8, "len": 2048, "heads": 24, "groups": 24, "dk": 64, "dv": 64,
         "dtype": "bf16", "ragged": False, "initial": False, "decay": "token"},
        # a small fp32 model with one fixed decay per head, odd head sizes, states carried between segments
        {"name": "train_odd", "kind": "train", "batch": 2, "len": 515, "heads": 6, "groups": 2, "dk": 96, "dv": 80,
         "dtype": "f32", "ragged": False, "initial": True, "decay": "head"},
        # the border between two blocks in a decode step
        {"name": "border_step", "kind": "border", "rows": 16, "dim": 768, "dtype": "bf16", "gate": True, "scale": True, "grad": False},
        # the same in a training step
        {"name": "border_train", "kind": "border", "rows": 16384, "dim": 768, "dtype": "bf16", "gate": True, "scale": True, "grad": True},
        # rows of an odd width in fp16, without a gate
        {"name": "border_odd", "kind": "border", "rows": 2047, "dim": 1001, "dtype": "f16", "gate": False, "scale": True, "grad": True},
        # every head's output normalised and gated before the output projection of a training step
        {"name": "heads_train", "kind": "heads", "rows": 16384, "dim": 1536, "groups": 24, "dtype": "bf16", "grad": True},
        # the gradients of a 24-layer 768-wide model with a 50280-word embedding
        {"name": "clip_model", "kind": "clip", "layers": 24, "width": 768, "vocab": 50280, "dtype": "bf16"},
        # a unit-test-size model of an odd width
        {"name": "clip_small", "kind": "clip", "layers": 2, "width": 65, "vocab": 301, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _near(rng, v, unit):
    """v itself, or v rounded to the unit (half of the draws each)."""
    return v if rng.random() < 0.5 else max(unit, unit * round(v / unit))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["train", "train", "train", "prompt", "prompt", "step", "border", "border", "heads", "clip"])
        c = {"kind": kind, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
        if kind in ("train", "prompt", "step"):
            c["groups"] = _log(rng, 1, 24)
            c["heads"] = c["groups"] * rng.choice([1, 1, 1, 2, 3])
            c["dk"], c["dv"] = _near(rng, _log(rng, 16, 128), 16), _near(rng, _log(rng, 16, 128), 16)
            c["batch"] = _log(rng, 1, 64 if kind == "step" else 8)
        if kind in ("train", "prompt"):
            c["len"] = _near(rng, _log(rng, 2, 4096 if kind == "train" else 32768), 64)
            c["ragged"], c["initial"] = rng.random() < 0.3, rng.random() < 0.3
            c["decay"] = rng.choice(["token", "token", "head"])
        if kind == "border":
            c.update(rows=_log(rng, 1, 16384), dim=_near(rng, _log(rng, 64, 5120), 64), gate=rng.random() < 0.7,
                     scale=rng.random() < 0.5, grad=rng.random() < 0.7)
        if kind == "heads":
            c["groups"] = _log(rng, 1, 40)
            c.update(rows=_log(rng, 1, 16384), dim=c["groups"] * _near(rng, _log(rng, 16, 256), 16), grad=rng.random() < 0.7)
        if kind == "clip":
            c.update(layers=_log(rng, 1, 24), width=_near(rng, _log(rng, 32, 768), 64), vocab=_log(rng, 256, 50280))
        if _cost(c) <= top:
            return c


# --------------------------------------------------------------- inputs --
def _shapes(c):
    """Parameter shapes of a model as the framework's: embedding, then per layer its norm, projections and state parameters."""
    w = c["width"]
    i, r = 2 * w, -(-w // 16)
    layer = [(w,), (2 * i, w), (i, 1, 4), (r + 32, i), (i, r), (i,), (i, 16), (i,), (w, i)]
    return [(c["vocab"], w)] + layer * c["layers"] + [(w,)]


def _decays(c, gen, shape, dev):
    """Log decays -dt * A: dt spread over [1e-3, 0.1], A over [1, 16]."""
    A = 1 + 15 * torch.rand(c["heads"], generator=gen, device=dev)
    if c.get("decay") == "head":
        return -A * 0.01
    dt = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(shape, generator=gen, device=dev))
    return -dt * A


def prepare(case, seed):
    dev = torch.device("cuda")
    c, dt = case, DT[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, dtype=dt, mul=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * mul).to(dtype)

    if c["kind"] in ("train", "prompt"):
        B, L, H, G, K, V = (c[n] for n in ("batch", "len", "heads", "groups", "dk", "dv"))
        s = {"q": rand(B, L, G, K), "k": rand(B, L, G, K), "v": rand(B, L, H, V), "g": _decays(c, gen, (B, L, H), dev),
             "initial": rand(B, H, K, V, dtype=torch.float32) if c["initial"] else None, "lengths": None}
        if c["ragged"]:       # one row of a ragged batch has nothing to read
            n = torch.randint(1, L + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            n[B // 2] = 0 if B > 1 else max(1, L // 2)
            s["lengths"] = n
        if c["kind"] == "train":
            s["dout"] = rand(B, L, H, V)
            s["dlast"] = rand(B, H, K, V, dtype=torch.float32) if c["initial"] else None
            s["leaves"] = [s[n].requires_grad_() for n in ("q", "k", "v", "g")]
            if c["initial"]:
                s["leaves"].append(s["initial"].requires_grad_())
    elif c["kind"] == "step":
        B, H, G, K, V = (c[n] for n in ("batch", "heads", "groups", "dk", "dv"))
        s = {"q": rand(B, G, K), "k": rand(B, G, K), "v": rand(B, H, V), "g": _decays(c, gen, (B, H), dev),
             "state": rand(B, H, K, V, dtype=torch.float32, mul=3.0)}
    elif c["kind"] == "border":
        R, D = c["rows"], c["dim"]
        s = {"x": rand(R, D), "residual": rand(R, D, mul=2.0), "post": rand(D, mul=0.1), "pre": rand(D, mul=0.1),
             "gate": rand(R, D) if c["gate"] else None, "scale": rand(D, mul=0.3) if c["scale"] else 0.5}
        if c["grad"]:
            s["dout"], s["ds"] = rand(R, D), rand(R, D)
            s["leaves"] = [s[n].requires_grad_() for n in ("x", "residual", "post", "pre", "gate", "scale")
                           if isinstance(s[n], torch.Tensor)]
    elif c["kind"] == "heads":
        R, D = c["rows"], c["dim"]
        s = {"x": rand(R, D), "gate": rand(R, D), "weight": rand(D, mul=0.1)}
        if c["grad"]:
            s["dout"] = rand(R, D)
            s["leaves"] = [s[n].requires_grad_() for n in ("x", "gate", "weight")]
    else:
        shapes = _shapes(c)
        # gradients of a model have sizes of their own in each tensor
        grads = [rand(*sh, mul=10.0 ** (-3 + 2 * ((7 * i) % 11) / 10)) for i, sh in enumerate(shapes)]
        flat = torch.empty(sum(g.numel() for g in grads), device=dev, dtype=dt)
        out = [t.view(sh) for t, sh in zip(flat.split([g.numel() for g in grads]), shapes)]
        s = {"grads": grads, "flat": flat, "out": out}
    s["case"] = c
    return s


# --------------------------------------------------------- plain forms --
def _plain_attn(s):
    """Chunks of CHUNK tokens: the masked product inside a chunk, and the states that the chunks before it leave."""
    q, k, v, g = s["q"].float(), s["k"].float(), s["v"].float(), s["g"].double()
    B, L, G, K = q.shape
    H, V = v.shape[2:]
    g = g.expand(B, L, H)
    if s["lengths"] is not None:
        live = (torch.arange(L, device=q.device) < s["lengths"][:, None])[:, :, None]
        g = torch.where(live, g, 0.0)
        q, k, v = (torch.where(live[..., None], t, 0.0) for t in (q, k, v))
    n = -(-L // CHUNK)
    pad = n * CHUNK - L

    def cut(t):                                   # (B, L, heads, X) -> (B, H, n, CHUNK, X)
        t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad)).view(B, n, CHUNK, t.shape[2], t.shape[3])
        return t.permute(0, 3, 1, 2, 4).repeat_interleave(H // t.shape[3], dim=1)

    q, k, v = cut(q) * K ** -0.5, cut(k), cut(v)
    G1 = cut(g[..., None])[..., 0].cumsum(-1)     # within the chunk, 64 bits
    ones = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    w = torch.exp(torch.where(ones, G1[..., :, None] - G1[..., None, :], -math.inf).float())
    inside = (q @ k.transpose(-1, -2).contiguous() * w) @ v
    total = G1[..., -1]                           # (B, H, n)
    kd = k * torch.exp(total[..., None] - G1).float()[..., None]
    local = (kd.transpose(-1, -2).contiguous() @ v).view(B, H, n, K * V)
    G2 = torch.nn.functional.pad(total.cumsum(-1), (1, 0))         # up to the start of chunk 0 .. n
    start = torch.ones(n + 1, n, dtype=torch.bool, device=q.device).tril(-1)
    hop = torch.exp(torch.where(start, G2[..., :, None] - G2[..., None, 1:], -math.inf).float())
    states = hop @ local                          # (B, H, n + 1, K * V)
    if s["initial"] is not None:
        states = states + torch.exp(G2).float()[..., None] * s["initial"].view(B, H, 1, K * V)
    states = states.view(B, H, n + 1, K, V)
    o = inside + (q * torch.exp(G1).float()[..., None]) @ states[:, :, :-1]
    o = o.permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, V)[:, :L]
    return o.to(s["v"].dtype), states[:, :, -1]


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    r = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(r, 1) * q.shape[-1] ** -0.5, k.repeat_interleave(r, 1)
    s["state"].mul_(torch.exp(s["g"])[..., None, None]).add_(k[..., :, None] * v[..., None, :])
    o = (q[..., :, None] * s["state"]).sum(-2)
    return o.to(s["v"].dtype)


def _plain_norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + w)


def _plain_border(s):
    t = _plain_norm(s["x"].float(), s["post"].float())
    if s["gate"] is not None:
        z = s["gate"].float()
        t = t * z * torch.sigmoid(z)
    scale = s["scale"].float() if isinstance(s["scale"], torch.Tensor) else s["scale"]
    r = s["residual"].float() + scale * t
    out = _plain_norm(r, s["pre"].float())
    return out.to(s["x"].dtype), r.to(s["x"].dtype)


def _plain_heads(s):
    x, z, G = s["x"].float(), s["gate"].float(), s["case"]["groups"]
    R, D = x.shape
    t = _plain_norm(x.view(R, G, D // G), s["weight"].float().view(G, D // G)).view(R, D)
    return (t * z * torch.sigmoid(z)).to(s["x"].dtype)


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).double().sum().sqrt().float()
    coef = torch.clamp(1.0 / (norm + EPS), max=1.0)
    [o.copy_(g.float() * coef) for o, g in zip(s["out"], s["grads"])]
    return norm


# ------------------------------------------------------------- one pass --
def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        from mamba_amd.ops.block_norm import block_norm_fn, gated_rms_norm_fn
        from mamba_amd.ops.clip_grads import clip_grads
        from mamba_amd.ops.linear_attn import linear_attn_fn, linear_attn_update
    if kind == "prompt":
        if not own:
            return _plain_attn(s)
        return linear_attn_fn(s["q"], s["k"], s["v"], s["g"], initial_state=s["initial"], lengths=s["lengths"],
                              return_last_state=True)
    if kind == "train":
        if own:
            o, last = linear_attn_fn(s["q"], s["k"], s["v"], s["g"], initial_state=s["initial"], lengths=s["lengths"],
                                     return_last_state=True)
        else:
            o, last = _plain_attn(s)
        if s["dlast"] is None:
            return [o.detach()] + list(torch.autograd.grad(o, s["leaves"], s["dout"]))
        return [o.detach(), last.detach()] + list(torch.autograd.grad([o, last], s["leaves"], [s["dout"], s["dlast"]]))
    if kind == "step":
        o = linear_attn_update(s["state"], s["q"], s["k"], s["v"], s["g"]) if own else _plain_step(s)
        return [o, s["state"]]
    if kind == "border":
        if own:
            o, r = block_norm_fn(s["x"], s["residual"], s["post"], s["pre"], gate=s["gate"], scale=s["scale"], eps=EPS)
        else:
            o, r = _plain_border(s)
        if not s["case"]["grad"]:
            return [o, r]
        return [o.detach(), r.detach()] + list(torch.autograd.grad([o, r], s["leaves"], [s["dout"], s["ds"]]))
    if kind == "heads":
        if own:
            o = gated_rms_norm_fn(s["x"], s["gate"], s["weight"], n_groups=s["case"]["groups"], eps=EPS)
        else:
            o = _plain_heads(s)
        if not s["case"]["grad"]:
            return o
        return [o.detach()] + list(torch.autograd.grad(o, s["leaves"], s["dout"]))
    norm = clip_grads(s["grads"], 1.0, out=s["out"], eps=EPS) if own else _plain_clip(s)
    return [norm, s["flat"]]


# ----------------------------------------------------------------- work --
def work(case):
    """Bytes: every input read once, every output written once.  FLOPs of the linear attention: its recurrence, 4 dk dv a
    token forward (the state's update and its product with the query) and 10 dk dv backward."""
    c, e = case, SIZE[case["dtype"]]
    if c["kind"] in ("train", "prompt"):
        n = c["batch"] * c["len"]
        qk, v, st = n * c["groups"] * c["dk"] * e, n * c["heads"] * c["dv"] * e, c["batch"] * c["heads"] * c["dk"] * c["dv"] * 4
        g = 4 * (c["heads"] if c["decay"] == "head" else n * c["heads"])
        mac = n * c["heads"] * c["dk"] * c["dv"]
        b = 2 * qk + 2 * v + g + st * (1 + c["initial"])
        if c["kind"] == "prompt":
            return {"bytes": b, "flops": 4 * mac}
        b -= 0 if c["initial"] else st
        # backward: q, k, v, dout, g in, their gradients out, and the states' where they are carried
        return {"bytes": b + 4 * qk + 3 * v + 2 * g + 3 * st * c["initial"], "flops": 14 * mac}
    if c["kind"] == "step":
        n = c["batch"]
        st = n * c["heads"] * c["dk"] * c["dv"]
        return {"bytes": 8 * st + n * (2 * c["groups"] * c["dk"] + 2 * c["heads"] * c["dv"]) * e + 4 * n * c["heads"],
                "flops": 5 * st}
    if c["kind"] in ("border", "heads"):
        el = c["rows"] * c["dim"]
        if c["kind"] == "heads":
            moved = 3 + (5 if c["grad"] else 0)       # x, gate -> out; x, gate, dout -> dx, dgate
        else:                                         # x, residual (, gate) -> out, s; the same and two gradients -> dx, dresidual (, dgate)
            moved = 4 + c["gate"] + ((6 + 2 * c["gate"]) if c["grad"] else 0)
        return {"bytes": moved * el * e + 8 * c["dim"] * e, "flops": (30 if c["grad"] else 12) * el}
    el = sum(math.prod(sh) for sh in _shapes(c))
    return {"bytes": 3 * el * e, "flops": 3 * el}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ------------------------------------------------------ 64-bit recurrence --
def _exact_attn(s, grad):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    B, L, G, K = q.shape
    H, V = v.shape[2:]
    scale, r = K ** -0.5, H // G
    per_head = s["g"].dim() == 1
    a = torch.exp(s["g"].detach().double().expand(B, L, H).clone())
    lens = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=q.device)
    live = torch.arange(L, device=q.device)[None] < lens[:, None]
    a[~live] = 1.0
    for t in (q, k, v):
        t[~live] = 0.0
    q, k = q.repeat_interleave(r, 2) * scale, k.repeat_interleave(r, 2)
    S = torch.zeros(B, H, K, V, dtype=torch.float64, device=q.device)
    if s["initial"] is not None:
        S = S + s["initial"].detach().double()
    kept = torch.empty((L + 1, B, H, K, V), dtype=torch.float64, device=q.device) if grad else None
    out = torch.empty_like(v)
    for t in range(L):
        if grad:
            kept[t] = S
        S = S * a[:, t, :, None, None]
        S.addcmul_(k[:, t, :, :, None], v[:, t, :, None, :])
        out[:, t] = (q[:, t, :, :, None] * S).sum(-2)
    if not grad:
        return [out, S]
    kept[L] = S
    do = s["dout"].detach().double().clone()
    do[~live] = 0.0
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg = torch.empty((B, L, H), dtype=torch.float64, device=q.device)
    dS = torch.zeros_like(S) if s["dlast"] is None else s["dlast"].double().clone()
    for t in range(L - 1, -1, -1):
        dS.addcmul_(q[:, t, :, :, None], do[:, t, :, None, :])
        dq[:, t] = (kept[t + 1] * do[:, t, :, None, :]).sum(-1) * scale
        dk[:, t] = (dS * v[:, t, :, None, :]).sum(-1)
        dv[:, t] = (dS * k[:, t, :, :, None]).sum(-2)
        dS = dS * a[:, t, :, None, None]
        dg[:, t] = (dS * kept[t]).sum((-1, -2))
    for t in (dq, dk, dv, dg):
        t[~live] = 0.0
    dq, dk = (t.view(B, L, G, r, K).sum(3) for t in (dq, dk))
    dg = dg.sum((0, 1)) if per_head else dg
    if s["dlast"] is None:
        return [out, dq, dk, dv, dg]
    return [out, S, dq, dk, dv, dg, dS]


def _exact_rms(x, w, eps):
    n = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
    return x / torch.sqrt(n * n / x.shape[-1] + eps) * (w + 1)


def exact(case, seed):
    c = case
    if c["kind"] == "train":
        kept = 8.0 * c["batch"] * (c["len"] + 1) * c["heads"] * c["dk"] * c["dv"]
        if kept > 100e9 or c["len"] > 8192:
            return None
    s = prepare(case, seed)
    if c["kind"] in ("train", "prompt"):
        return _exact_attn(s, c["kind"] == "train")
    if c["kind"] == "step":
        r = c["heads"] // c["groups"]
        q, k = (s[n].double().unsqueeze(2).expand(-1, -1, r, -1).reshape(c["batch"], c["heads"], c["dk"]) for n in ("q", "k"))
        S = s["state"].double() * s["g"].double().exp().view(c["batch"], c["heads"], 1, 1)
        S = S + k.unsqueeze(-1) * s["v"].double().unsqueeze(-2)
        return [torch.matmul(q.unsqueeze(-2), S).squeeze(-2) / math.sqrt(c["dk"]), S]
    if c["kind"] == "clip":
        n = math.sqrt(sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
        return [torch.tensor(n, dtype=torch.float64), torch.cat([g.double().flatten() for g in s["grads"]]) * min(1.0, 1.0 / (n + EPS))]
    names = [n for n in ("x", "residual", "post", "pre", "gate", "scale", "weight") if isinstance(s.get(n), torch.Tensor)]
    d = {n: s[n].detach().double().requires_grad_(c["grad"]) for n in names}
    if c["kind"] == "border":
        t = _exact_rms(d["x"], d["post"], EPS)
        if "gate" in d:
            t = t * (d["gate"] / (1 + torch.exp(-d["gate"])))
        r = d["residual"] + t * d.get("scale", s["scale"])
        outs, ups = [_exact_rms(r, d["pre"], EPS), r], ("dout", "ds")
    else:
        R, D, G = c["rows"], c["dim"], c["groups"]
        t = _exact_rms(d["x"].reshape(R * G, D // G), d["weight"].reshape(1, G, D // G).expand(R, -1, -1).reshape(R * G, -1), EPS)
        outs, ups = [t.reshape(R, D) * d["gate"] / (1 + torch.exp(-d["gate"]))], ("dout",)
    if not c["grad"]:
        return [o.detach() for o in outs] if c["kind"] == "border" else outs[0].detach()
    grads = torch.autograd.grad(outs, [d[n] for n in names if n != "weight"] + ([d["weight"]] if "weight" in d else []),
                                [s[n].double() for n in ups])
    return [o.detach() for o in outs] + list(grads)
