"""The gated delta rule's recurrence in float64, token by token, with its
gradients, and bounds on what fp32 arithmetic may make of it.

Value columns do not meet on the way through the states, and a token's transition
a (I - beta k k^T) does not lengthen a column where beta |k|^2 <= 2 and a <= 1.  So with s_c
the longest column c of a state or of a value, an error made in one chunk stays
as it is, and
    column c of a state is off by at most  chunks * n * 2^-24 * T * s_c
where n counts the summands of a chunk's products and T is the largest row sum of
|(I + N)^-1| over the chunks, by which a triangular solve may enlarge what enters it (the same for
the states' gradients, with column sums).  Outputs and gradients are sums of products of
these columns with rows of the inputs.
"""
import torch

CHUNK = 64


def recurrence(q, k, v, g, beta, scale, initial=None, lengths=None, dout=None, dlast=None):
    """dict of out, last and, with dout, dq, dk, dv, dg, dbeta, dinitial, in float64 on the CPU, and of what bounds() needs."""
    q, k, v, g, beta = (t.detach().double().cpu() for t in (q, k, v, g, beta))
    B, L, G, K = q.shape
    H, V = v.shape[2:]
    r = H // G
    n = torch.full((B,), L) if lengths is None else lengths.cpu().clamp(0, L)
    live = torch.arange(L)[None] < n[:, None]
    q, k, v = (torch.where(live[..., None, None], t, 0.0) for t in (q, k, v))
    a, beta = torch.where(live[..., None], torch.exp(g), 1.0), torch.where(live[..., None], beta, 0.0)
    q, k = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if initial is None else initial.detach().double().cpu().clone()
    states, err = [S], torch.zeros_like(v)
    out = torch.zeros(B, L, H, V, dtype=torch.float64)
    longest = torch.linalg.vector_norm(S, dim=2)
    for t in range(L):
        S = S * a[:, t, :, None, None]
        err[:, t] = v[:, t] - (k[:, t, :, :, None] * S).sum(2)
        S = S + k[:, t, :, :, None] * (beta[:, t, :, None] * err[:, t])[:, :, None, :]
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(2)
        states.append(S)
        longest = torch.maximum(longest, torch.linalg.vector_norm(S, dim=2))
    res = {"out": torch.where(live[..., None, None], out, 0.0), "last": S}
    res["s"] = torch.maximum(longest, v.abs().amax(1) if L else longest)          # (B, H, V)
    res.update(_solves(k, torch.where(live[..., None], g, 0.0), beta), q=q, k=k, beta=beta)
    if dout is None:
        return res
    do = torch.where(live[..., None, None], dout.detach().double().cpu(), 0.0)
    dS = torch.zeros_like(S) if dlast is None else dlast.detach().double().cpu().clone()
    dq, dk, dv, dg, db = (torch.zeros_like(t) for t in (q, k, v, a, a))
    longest = torch.linalg.vector_norm(dS, dim=2)
    for t in range(L - 1, -1, -1):
        dS = dS + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dq[:, t] = scale * (states[t + 1] * do[:, t, :, None, :]).sum(3)
        longest = torch.maximum(longest, torch.linalg.vector_norm(dS, dim=2))
        du = (dS * k[:, t, :, :, None]).sum(2)
        db[:, t] = (du * err[:, t]).sum(-1)
        dv[:, t] = beta[:, t, :, None] * du
        seen = states[t] * a[:, t, :, None, None]
        dk[:, t] = (dS * (beta[:, t, :, None] * err[:, t])[:, :, None, :]).sum(3) - (seen * dv[:, t][:, :, None, :]).sum(3)
        dS = dS - k[:, t, :, :, None] * dv[:, t][:, :, None, :]
        dg[:, t] = (dS * seen).sum((2, 3))
        dS = dS * a[:, t, :, None, None]
    for t in (dq, dk, dv, dg, db):
        t[~live] = 0.0
    res.update(dq=dq.view(B, L, G, r, K).sum(3), dk=dk.view(B, L, G, r, K).sum(3), dv=dv, dg=dg, dbeta=db, dinitial=dS,
               d=torch.maximum(longest, scale * (torch.linalg.vector_norm(q, dim=3)[..., None] * do.abs()).amax(1) if L else longest))
    return res


def _solves(k, g, beta):
    """Largest row and column sum of |(I + N)^-1| over the chunks of each (batch, head): (B, H)."""
    B, L, H, K = k.shape
    rows, cols = torch.ones(B, H, dtype=torch.float64), torch.ones(B, H, dtype=torch.float64)
    g = g.clamp(min=-1e5)
    for t in range(0, L, CHUNK):
        kc, gc, bc = (x[:, t:t + CHUNK].transpose(1, 2) for x in (k, g, beta))
        Gc = gc.cumsum(-1)
        n = (kc @ kc.transpose(-1, -2) * bc[..., None, :] * torch.exp((Gc[..., :, None] - Gc[..., None, :]).clamp(max=0.0))).tril(-1)
        inv = torch.linalg.inv(torch.eye(n.shape[-1], dtype=torch.float64) + n).abs()
        rows, cols = torch.maximum(rows, inv.sum(-1).amax(-1)), torch.maximum(cols, inv.sum(-2).amax(-1))
    return {"rows": rows, "cols": cols}


def bounds(ref, dtype, scale):
    """How far each result of ``recurrence`` may be off, elementwise: n = d_key + d_value + 2 * 64 + 32
    summands and factors of a chunk's sums at 2^-24 each.  16-bit results may be formed from two 16-bit terms (2^-16
    each, three such products on the way).  Heads of a group add up."""
    q, k = ref["q"], ref["k"]
    B, L, H, K = q.shape
    V, s = ref["last"].shape[3], ref["s"]
    chunks = -(-L // 32) + 1
    n = (K + V + 160) * 2.0 ** -24
    rows = n + (0 if dtype == torch.float32 else 3 * 2.0 ** -16)
    ds = chunks * n * ref["rows"][..., None] * s                                   # (B, H, V): a state's column
    qn, kn = (torch.linalg.vector_norm(x, dim=3) for x in (q, k))                  # (B, L, H)
    kmax = kn.amax(1)[..., None].clamp(min=1.0) if L else torch.ones(B, H, 1, dtype=torch.float64)
    b = {"out": scale * qn[..., None] * (ds + rows * ref["rows"][..., None] * s)[:, None], "last": ds[:, :, None, :].expand_as(ref["last"])}
    if "d" not in ref:
        return b
    d = ref["d"]
    dd = chunks * n * ref["cols"][..., None] * d * kmax
    G = ref["dq"].shape[2]
    both = (ds * d + dd * s).sum(-1)                                               # (B, H): inner products of columns
    near = rows * (ref["rows"] * ref["cols"])[..., None] * s * d
    keys = (2 * both + 4 * near.sum(-1)) * kmax[..., 0]
    per_key = keys[:, None, :, None].expand(B, L, H, K).reshape(B, L, G, H // G, K).sum(3)
    b.update(dq=per_key, dk=per_key, dv=(dd + rows * ref["cols"][..., None] * d * kmax)[:, None].expand(B, L, H, V),
             dbeta=keys[:, None].expand(B, L, H), dg=CHUNK * keys[:, None].expand(B, L, H), dinitial=dd[:, :, None, :].expand_as(ref["last"]))
    return b


def check(got, want, bound, what):
    """|got - want| <= bound + half a step of got's type, elementwise."""
    step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} vs {tuple(want.shape)}"
    over = (got - want).abs() - (bound * (1 + step) + step * want.abs() + tiny)
    assert not torch.isnan(over).any() and (over.numel() == 0 or float(over.max()) <= 0), \
        f"{what}: off by {float((got - want).abs().max())}, {float(over.max())} too much"
