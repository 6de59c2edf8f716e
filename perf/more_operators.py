"""The gated delta rule, the unit norm of its queries and keys, and layer norm, case by case.

A case is a dict of plain values.  Its "kind" names the call:

* train    delta_rule_fn, forward and backward: one layer of a training step;
* prompt   delta_rule_fn without autograd: a prompt that fills the decode state;
* step     delta_rule_update: one token per sequence, the state advancing in place;
* unit     unit_norm_fn: the queries and keys of a layer, one row per head, scaled to length one;
* layer    layer_norm_fn: the residual add and the norm in front of a block.

With ``own`` false the plain forms below run, elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
CHUNK = 64          # tokens per chunk of the plain delta rule


# ---------------------------------------------------------------- cases --
def listed():
    return [
        # one token of one conversation in a 768-wide model: launches and latency
        {"name": "step_single", "kind": "step", "batch": 1, "heads": 24, "groups": 24, "dk": 64, "dv": 64, "dtype": "bf16"},
        # one token of a full serving batch of a 1024-wide model
        {"name": "step_batch", "kind": "step", "batch": 64, "heads": 16, "groups": 16, "dk": 128, "dv": 128, "dtype": "bf16"},
        # one long document read by a single user: few rows, a long axis
        {"name": "prompt_long", "kind": "prompt", "batch": 1, "len": 32768, "heads": 24, "groups": 24, "dk": 64, "dv": 64,
         "dtype": "bf16", "ragged": False, "initial": False},
        # prompts of different lengths continued from earlier turns, keys shared by several heads, fp32
        {"name": "prompt_ragged", "kind": "prompt", "batch": 5, "len": 1021, "heads": 24, "groups": 4, "dk": 64, "dv": 64,
         "dtype": "f32", "ragged": True, "initial": True},
        # one layer of a 768-wide model's training step
        {"name": "train_layer", "kind": "train", "batch": 8, "len": 2048, "heads": 24, "groups": 24, "dk": 64, "dv": 64,
         "dtype": "bf16", "ragged": False, "initial": False},
        # one layer of a model with wide heads, fp16, longer sequences
        {"name": "train_wide", "kind": "train", "batch": 2, "len": 4096, "heads": 16, "groups": 16, "dk": 128, "dv": 128,
         "dtype": "f16", "ragged": False, "initial": False},
        # a small fp32 model, odd head sizes and lengths, keys shared by several heads, states carried between segments
        {"name": "train_odd", "kind": "train", "batch": 2, "len": 515, "heads": 6, "groups": 2, "dk": 96, "dv": 80,
         "dtype": "f32", "ragged": False, "initial": True},
        # queries and keys of a decode step's batch
        {"name": "unit_step", "kind": "unit", "rows": 64, "heads": 32, "dim": 128, "dtype": "bf16", "grad": False},
        # queries and keys of a training step, as they lie beside the values in the input projection's output
        {"name": "unit_train", "kind": "unit", "rows": 16384, "heads": 48, "dim": 64, "dtype": "bf16", "grad": True},
        # the norm in front of a block in a decode step
        {"name": "layer_step", "kind": "layer", "rows": 16, "dim": 768, "dtype": "bf16", "bias": True, "residual": True, "grad": False},
        # the same in a training step
        {"name": "layer_train", "kind": "layer", "rows": 16384, "dim": 768, "dtype": "bf16", "bias": True, "residual": True, "grad": True},
        # rows of an odd width in fp16, without a bias
        {"name": "layer_odd", "kind": "layer", "rows": 2047, "dim": 1001, "dtype": "f16", "bias": False, "residual": True, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _near(rng, v, unit):
    """v itself, or v rounded to the unit (half of the draws each)."""
    return v if rng.random() < 0.5 else max(unit, unit * round(v / unit))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["train", "train", "train", "prompt", "prompt", "step", "unit", "layer", "layer"])
        c = {"kind": kind, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
        if kind in ("train", "prompt", "step"):
            c["groups"] = _log(rng, 1, 24)
            c["heads"] = c["groups"] * rng.choice([1, 1, 1, 2, 3])
            c["dk"], c["dv"] = _near(rng, _log(rng, 16, 128), 16), _near(rng, _log(rng, 16, 128), 16)
            c["batch"] = _log(rng, 1, 64 if kind == "step" else 8)
        if kind in ("train", "prompt"):
            c["len"] = _near(rng, _log(rng, 2, 4096 if kind == "train" else 32768), 64)
            c["ragged"], c["initial"] = rng.random() < 0.3, rng.random() < 0.3
        if kind == "unit":
            c.update(rows=_log(rng, 1, 16384), heads=_log(rng, 1, 48), dim=_near(rng, _log(rng, 16, 256), 16), grad=rng.random() < 0.7)
        if kind == "layer":
            c.update(rows=_log(rng, 1, 16384), dim=_near(rng, _log(rng, 64, 5120), 64), bias=rng.random() < 0.7,
                     residual=rng.random() < 0.7, grad=rng.random() < 0.7)
        if _cost(c) <= top:
            return c


# --------------------------------------------------------------- inputs --
def prepare(case, seed):
    dev = torch.device("cuda")
    c, dt = case, DT[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, dtype=dt, mul=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * mul).to(dtype)

    def unit(*shape):                 # rows of length one: what the unit norm hands on
        x = torch.randn(shape, generator=gen, device=dev)
        return (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS)).to(dt)

    def gates(*shape):                # log decays -dt * A, dt over [1e-3, 0.1] and A over [1, 16]; rates in (0, 1)
        A = 1 + 15 * torch.rand(c["heads"], generator=gen, device=dev)
        dt_ = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(shape, generator=gen, device=dev))
        return -dt_ * A, torch.sigmoid(torch.randn(shape, generator=gen, device=dev))

    if c["kind"] in ("train", "prompt"):
        B, L, H, G, K, V = (c[n] for n in ("batch", "len", "heads", "groups", "dk", "dv"))
        g, beta = gates(B, L, H)
        s = {"q": unit(B, L, G, K), "k": unit(B, L, G, K), "v": rand(B, L, H, V), "g": g, "beta": beta,
             "initial": rand(B, H, K, V, dtype=torch.float32) if c["initial"] else None, "lengths": None}
        if c["ragged"]:       # one row of a ragged batch has nothing to read
            n = torch.randint(1, L + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            n[B // 2] = 0 if B > 1 else max(1, L // 2)
            s["lengths"] = n
        if c["kind"] == "train":
            s["dout"] = rand(B, L, H, V)
            s["dlast"] = rand(B, H, K, V, dtype=torch.float32) if c["initial"] else None
            s["leaves"] = [s[n].requires_grad_() for n in ("q", "k", "v", "g", "beta")]
            if c["initial"]:
                s["leaves"].append(s["initial"].requires_grad_())
    elif c["kind"] == "step":
        B, H, G, K, V = (c[n] for n in ("batch", "heads", "groups", "dk", "dv"))
        g, beta = gates(B, H)
        s = {"q": unit(B, G, K), "k": unit(B, G, K), "v": rand(B, H, V), "g": g, "beta": beta,
             "state": rand(B, H, K, V, dtype=torch.float32)}
    elif c["kind"] == "unit":
        R, H, D = c["rows"], c["heads"], c["dim"]
        wide = rand(R, (H + 1) * D)               # a projection's row: the heads, then columns of other use
        s = {"x": wide[:, :H * D].view(R, H, D)}
        if c["grad"]:
            s["dout"] = rand(R, H, D)
            s["leaves"] = [s["x"].requires_grad_()]
    else:
        R, D = c["rows"], c["dim"]
        s = {"x": rand(R, D, mul=2.0) + 0.5, "residual": rand(R, D) if c["residual"] else None, "weight": rand(D, mul=0.1) + 1.0,
             "bias": rand(D, mul=0.1) if c["bias"] else None}
        if c["grad"]:
            s["dout"], s["ds"] = rand(R, D), rand(R, D)
            s["leaves"] = [s[n].requires_grad_() for n in ("x", "weight", "bias", "residual") if s[n] is not None]
    s["case"] = c
    return s


# --------------------------------------------------------- plain forms --
def _inverse(n):
    """(I + n)^-1 of strictly lower triangular n (..., CHUNK, CHUNK), from blocks of one row on by halves."""
    t = torch.ones(n.shape[:-2] + (CHUNK, 1, 1), dtype=n.dtype, device=n.device)     # diagonal blocks
    size = 1
    while size < CHUNK:
        pairs = CHUNK // (2 * size)
        low = torch.stack([n[..., 2 * size * p + size:2 * size * (p + 1), 2 * size * p:2 * size * p + size] for p in range(pairs)], -3)
        a, b = t[..., 0::2, :, :], t[..., 1::2, :, :]
        top = torch.cat([a, torch.zeros_like(a)], -1)
        t = torch.cat([top, torch.cat([-(b @ low @ a), b], -1)], -2)
        size *= 2
    return t[..., 0, :, :]


def _plain_rule(s):
    """Chunks of CHUNK tokens: a triangular inverse in each, then the states from chunk to chunk."""
    q, k, v, g, beta = s["q"].float(), s["k"].float(), s["v"].float(), s["g"].double(), s["beta"].float()
    B, L, G, K = q.shape
    H, V = v.shape[2:]
    if s["lengths"] is not None:
        live = (torch.arange(L, device=q.device) < s["lengths"][:, None])[:, :, None]
        g, beta = torch.where(live, g, 0.0), torch.where(live, beta, 0.0)
        q, k, v = (torch.where(live[..., None], t, 0.0) for t in (q, k, v))
    n = -(-L // CHUNK)
    pad = n * CHUNK - L

    def cut(t):                                   # (B, L, heads, X) -> (B, H, n, CHUNK, X)
        t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pad)).view(B, n, CHUNK, t.shape[2], t.shape[3])
        return t.permute(0, 3, 1, 2, 4).repeat_interleave(H // t.shape[3], dim=1)

    q, k, v, beta = cut(q) * K ** -0.5, cut(k), cut(v), cut(beta[..., None])
    G1 = cut(g[..., None])[..., 0].cumsum(-1)     # within the chunk, 64 bits
    ones = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    w = torch.exp(torch.where(ones, G1[..., :, None] - G1[..., None, :], -math.inf).float())
    kt = k.transpose(-1, -2).contiguous()
    t = _inverse((k @ kt * w * beta.transpose(-1, -2)).tril(-1))        # of w_ij k_i.k_j beta_j
    u_v = beta * (t @ v)
    w_k = beta * (t @ (k * torch.exp(G1).float()[..., None]))
    p = q @ kt * w
    qd = q * torch.exp(G1).float()[..., None]
    kd = (k * torch.exp(G1[..., -1:] - G1).float()[..., None]).transpose(-1, -2).contiguous()
    total = torch.exp(G1[..., -1]).float()[..., None, None]
    S = s["initial"] if s["initial"] is not None else torch.zeros(B, H, K, V, device=q.device)
    out = []
    for i in range(n):
        u = u_v[:, :, i] - w_k[:, :, i] @ S
        out.append(qd[:, :, i] @ S + p[:, :, i] @ u)
        S = total[:, :, i] * S + kd[:, :, i] @ u
    o = torch.stack(out, 2).permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, V)[:, :L]
    return o.to(s["v"].dtype), S


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    r = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(r, 1) * q.shape[-1] ** -0.5, k.repeat_interleave(r, 1)
    s["state"].mul_(torch.exp(s["g"])[..., None, None])
    e = s["beta"][..., None] * (v - (k[..., :, None] * s["state"]).sum(-2))
    s["state"].add_(k[..., :, None] * e[..., None, :])
    o = (q[..., :, None] * s["state"]).sum(-2)
    return o.to(s["v"].dtype)


def _plain_unit(s):
    x = s["x"].float()
    return (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS)).to(s["x"].dtype)


def _plain_layer(s):
    """The residual stream is rounded to its type first; the norm is of what it then holds."""
    r = s["x"]
    if s["residual"] is not None:
        r = (r.float() + s["residual"].float()).to(r.dtype)
    f = r.float()
    c = f - f.mean(-1, keepdim=True)
    out = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(s["x"].dtype), r


# ------------------------------------------------------------- one pass --
def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        from mamba_amd.ops.delta_rule import delta_rule_fn, delta_rule_update
        from mamba_amd.ops.layer_norm import layer_norm_fn
        from mamba_amd.ops.unit_norm import unit_norm_fn
    if kind == "prompt":
        if not own:
            return _plain_rule(s)
        return delta_rule_fn(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["initial"], lengths=s["lengths"],
                             return_last_state=True)
    if kind == "train":
        if own:
            o, last = delta_rule_fn(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["initial"], lengths=s["lengths"],
                                    return_last_state=True)
        else:
            o, last = _plain_rule(s)
        if s["dlast"] is None:
            return [o.detach()] + list(torch.autograd.grad(o, s["leaves"], s["dout"]))
        return [o.detach(), last.detach()] + list(torch.autograd.grad([o, last], s["leaves"], [s["dout"], s["dlast"]]))
    if kind == "step":
        o = delta_rule_update(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"]) if own else _plain_step(s)
        return [o, s["state"]]
    if kind == "unit":
        o = unit_norm_fn(s["x"], eps=EPS) if own else _plain_unit(s)
        if not s["case"]["grad"]:
            return o
        return [o.detach()] + list(torch.autograd.grad(o, s["leaves"], s["dout"]))
    if own:
        o, r = layer_norm_fn(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS, prenorm=True)
    else:
        o, r = _plain_layer(s)
    if not s["case"]["grad"]:
        return [o, r]
    return [o.detach(), r.detach()] + list(torch.autograd.grad([o, r], s["leaves"], [s["dout"], s["ds"]]))


# ----------------------------------------------------------------- work --
def work(case):
    """Bytes: every input read once, every output written once.  FLOPs of the delta rule: its recurrence, 6 dk dv a token
    forward (the state's product with the key, its update, its product with the query) and 14 dk dv backward."""
    c, e = case, SIZE[case["dtype"]]
    if c["kind"] in ("train", "prompt"):
        n = c["batch"] * c["len"]
        qk, v, st = n * c["groups"] * c["dk"] * e, n * c["heads"] * c["dv"] * e, c["batch"] * c["heads"] * c["dk"] * c["dv"] * 4
        gb = 8 * n * c["heads"]
        mac = n * c["heads"] * c["dk"] * c["dv"]
        b = 2 * qk + 2 * v + gb + st * (1 + c["initial"])
        if c["kind"] == "prompt":
            return {"bytes": b, "flops": 6 * mac}
        b -= 0 if c["initial"] else st
        # backward: q, k, v, dout, g, beta in, their gradients out, and the states' where they are carried
        return {"bytes": b + 4 * qk + 3 * v + 2 * gb + 3 * st * c["initial"], "flops": 20 * mac}
    if c["kind"] == "step":
        n = c["batch"]
        st = n * c["heads"] * c["dk"] * c["dv"]
        return {"bytes": 8 * st + n * (2 * c["groups"] * c["dk"] + 2 * c["heads"] * c["dv"]) * e + 8 * n * c["heads"],
                "flops": 7 * st}
    if c["kind"] == "unit":
        el = c["rows"] * c["heads"] * c["dim"]                    # x -> out; x, dout -> dx
        return {"bytes": (5 if c["grad"] else 2) * el * e, "flops": (10 if c["grad"] else 3) * el}
    el = c["rows"] * c["dim"]
    moved = 3 + c["residual"] - (not c["residual"])               # x (, residual) -> out (, s); s, dout, ds -> dx
    return {"bytes": (moved + (4 if c["grad"] else 0)) * el * e + 4 * c["dim"] * e, "flops": (22 if c["grad"] else 9) * el}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ------------------------------------------------------ 64-bit recurrence --
def _exact_rule(s, grad):
    q, k, v, beta = (s[n].detach().double() for n in ("q", "k", "v", "beta"))
    B, L, G, K = q.shape
    H, V = v.shape[2:]
    scale, r = K ** -0.5, H // G
    a = torch.exp(s["g"].detach().double())
    beta = beta.clone()
    lens = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=q.device)
    live = torch.arange(L, device=q.device)[None] < lens[:, None]
    a[~live], beta[~live] = 1.0, 0.0
    q[~live] = 0.0
    q, k = q.repeat_interleave(r, 2) * scale, k.repeat_interleave(r, 2)
    S = torch.zeros(B, H, K, V, dtype=torch.float64, device=q.device)
    if s["initial"] is not None:
        S = S + s["initial"].detach().double()
    kept = torch.empty((L + 1, B, H, K, V), dtype=torch.float64, device=q.device) if grad else None
    err = torch.empty_like(v)
    out = torch.empty_like(v)
    for t in range(L):
        if grad:
            kept[t] = S
        S = S * a[:, t, :, None, None]
        err[:, t] = v[:, t] - torch.matmul(k[:, t, :, None, :], S)[:, :, 0]
        S.addcmul_(k[:, t, :, :, None], (beta[:, t, :, None] * err[:, t])[:, :, None, :])
        out[:, t] = torch.matmul(q[:, t, :, None, :], S)[:, :, 0]
    if not grad:
        return [out, S]
    kept[L] = S
    do = s["dout"].detach().double().clone()
    do[~live] = 0.0
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg, db = (torch.empty((B, L, H), dtype=torch.float64, device=q.device) for _ in range(2))
    dS = torch.zeros_like(S) if s["dlast"] is None else s["dlast"].double().clone()
    for t in range(L - 1, -1, -1):
        dS.addcmul_(q[:, t, :, :, None], do[:, t, :, None, :])
        dq[:, t] = (kept[t + 1] * do[:, t, :, None, :]).sum(-1) * scale
        du = (dS * k[:, t, :, :, None]).sum(-2)                   # of u = beta e
        db[:, t] = (du * err[:, t]).sum(-1)
        de = beta[:, t, :, None] * du
        dv[:, t] = de
        was = kept[t] * a[:, t, :, None, None]                    # the state that e saw
        dk[:, t] = (dS * (beta[:, t, :, None] * err[:, t])[:, :, None, :]).sum(-1) - (was * de[:, :, None, :]).sum(-1)
        dS.addcmul_(k[:, t, :, :, None], de[:, :, None, :], value=-1.0)
        dg[:, t] = (dS * was).sum((-1, -2))
        dS = dS * a[:, t, :, None, None]
    for x in (dq, dk, dv, dg, db):
        x[~live] = 0.0
    dq, dk = (x.view(B, L, G, r, K).sum(3) for x in (dq, dk))
    if s["dlast"] is None:
        return [out, dq, dk, dv, dg, db]
    return [out, S, dq, dk, dv, dg, db, dS]


def exact(case, seed):
    c = case
    if c["kind"] == "train" and (8.0 * c["batch"] * (c["len"] + 1) * c["heads"] * c["dk"] * c["dv"] > 100e9 or c["len"] > 8192):
        return None
    s = prepare(case, seed)
    if c["kind"] in ("train", "prompt"):
        return _exact_rule(s, c["kind"] == "train")
    if c["kind"] == "step":
        r = c["heads"] // c["groups"]
        q, k = (s[n].double().unsqueeze(2).expand(-1, -1, r, -1).reshape(c["batch"], c["heads"], c["dk"], 1) for n in ("q", "k"))
        S = s["state"].double() * s["g"].double().exp()[:, :, None, None]
        old = torch.matmul(S.transpose(-1, -2), k).squeeze(-1)
        S = S + k * (s["beta"].double()[:, :, None] * (s["v"].double() - old)).unsqueeze(-2)
        return [torch.matmul(S.transpose(-1, -2), q).squeeze(-1) / math.sqrt(c["dk"]), S]
    d = {n: s[n].detach().double().requires_grad_(c["grad"]) for n in ("x", "weight", "bias", "residual")
         if isinstance(s.get(n), torch.Tensor)}
    if c["kind"] == "unit":
        length = torch.linalg.vector_norm(d["x"], dim=-1, keepdim=True)
        o = d["x"] / torch.sqrt(length * length + EPS)
        if not c["grad"]:
            return o.detach()
        return [o.detach()] + list(torch.autograd.grad(o, [d["x"]], s["dout"].double()))
    # (the stream's rounding to its type is part of the definition; its gradient passes through)
    r = d["x"] + d["residual"] if c["residual"] else d["x"]
    r = r + (r.detach().to(DT[c["dtype"]]).double() - r.detach())
    var, mean = torch.var_mean(r, dim=-1, keepdim=True, correction=0)
    o = (r - mean) / torch.sqrt(var + EPS) * d["weight"] + d.get("bias", 0.0)
    if not c["grad"]:
        return [o.detach(), r.detach()]
    return [o.detach(), r.detach()] + list(torch.autograd.grad([o, r], list(d.values()), [s["dout"].double(), s["ds"].double()]))
