"""The linear attention's recurrence in float64, token by token, with its
gradients, and bounds on what fp32 arithmetic may make of it.

The bounds come from the same recurrence on absolute values: a sum whose terms
have the absolute sum A, each rounded a few times, is off by at most a multiple
of 2^-24 A.
"""
import torch


def recurrence(q, k, v, g, scale, initial=None, lengths=None, dout=None, dlast=None):
    """dict of out, last and, with dout, dq, dk, dv, dg (per token), dinitial; float64, on the CPU."""
    q, k, v, g = (t.detach().double().cpu() for t in (q, k, v, g))
    B, L, G, K = q.shape
    H, V = v.shape[2:]
    r = H // G
    a = torch.exp(g.expand(B, L, H)).clone()
    n = torch.full((B,), L) if lengths is None else lengths.cpu().clamp(0, L)
    live = torch.arange(L)[None] < n[:, None]
    q, k, v = (torch.where(live[..., None, None], t, 0.0) for t in (q, k, v))
    a[~live] = 1.0
    q, k = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if initial is None else initial.detach().double().cpu().clone()
    states = [S]
    out = torch.zeros(B, L, H, V, dtype=torch.float64)
    for t in range(L):
        S = S * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(2)
        states.append(S)
    res = {"out": torch.where(live[..., None, None], out, 0.0), "last": S}
    if dout is None:
        return res
    do = torch.where(live[..., None, None], dout.detach().double().cpu(), 0.0)
    dS = torch.zeros_like(S) if dlast is None else dlast.detach().double().cpu().clone()
    dq, dk, dv, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(a)
    for t in range(L - 1, -1, -1):
        dS = dS + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dq[:, t] = scale * (states[t + 1] * do[:, t, :, None, :]).sum(3)
        dk[:, t] = (dS * v[:, t, :, None, :]).sum(3)
        dv[:, t] = (dS * k[:, t, :, :, None]).sum(2)
        dS = dS * a[:, t, :, None, None]
        dg[:, t] = (dS * states[t]).sum((2, 3))
    for t in (dq, dk, dv, dg):
        t[~live] = 0.0
    # (what dg is summed from: the products of q and k with their gradients, and the states')
    res.update(dq=dq.view(B, L, G, r, K).sum(3), dk=dk.view(B, L, G, r, K).sum(3), dv=dv, dg=dg, dinitial=dS,
               terms=((q * dq).sum(-1) + (k * dk).sum(-1)).flip(1).cumsum(1).flip(1) + dg.abs().amax(1, keepdim=True))
    return res


def bounds(q, k, v, g, scale, initial=None, lengths=None, dout=None, dlast=None):
    """How far each result of ``recurrence`` may be off, elementwise.

    Sums run over at most d_key + d_value + 64 terms at a time, 64-token chunks
    follow one another, and a decay's exponential and the factors beside it are
    rounded about 32 times: (d_key + d_value + 64 + L / 64 + 32) 2^-24 of the
    absolute sum.  16-bit rows may keep what they multiply with in two 16-bit
    terms (2^-16 each; three such products a result); states keep three terms
    (2^-24).  A 16-bit result is rounded once more, by eps / 2 of itself.
    """
    mag = {k_: None if t is None else t.detach().double().cpu().abs() for k_, t in
           (("q", q), ("k", k), ("v", v), ("i", initial), ("do", dout), ("dl", dlast))}
    m = recurrence(mag["q"], mag["k"], mag["v"], g, abs(scale), mag["i"], lengths, mag["do"], mag["dl"])
    K, V, L = q.shape[3], v.shape[3], q.shape[1]
    f32 = (K + V + 64 + L / 64 + 32) * 2.0 ** -24
    rows = f32 + (0 if v.dtype == torch.float32 else 3 * 2.0 ** -16)
    b = {n: rows * m[n] for n in ("out", "dq", "dk", "dv") if n in m}
    b.update({n: f32 * m[n] for n in ("last", "dinitial") if n in m})
    if "dg" in m:
        b["dg"] = rows * (m["terms"] + m["dg"])
    return b


def check(got, want, bound, what):
    """|got - want| <= bound + half a step of got's type, elementwise."""
    step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} vs {tuple(want.shape)}"
    room = bound * (1 + step) + step * want.abs() + tiny
    bad = ~((got - want).abs() <= room)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, (got - want).abs() / room, 0.0).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds; at {i}: got {got.flatten()[i]:.6g}, "
                             f"want {want.flatten()[i]:.6g}, room {room.flatten()[i]:.3g}")
