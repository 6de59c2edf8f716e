"""The norms around a block and the gated norm of heads in float64, with their
gradients in closed form, and bounds on what fp32 arithmetic may make of them.

Bounds count roundings of u = 2^-24.  A row's sums take at most 16 terms a
lane, 10 steps across lanes and waves and 6 roundings a term; a reciprocal
root, a sigmoid and the products of one term at most 32 more: C = 64 a level.
Where s = residual + scale t cancels, its error stands beside its terms' sizes:
by kappa = |(|residual| + |scale t|)| / |s| (row norms) in what is divided by
its norm.  Gradients pass through two such levels.  A 16-bit result is rounded
once more, by half a step.
"""
import torch

U = 2.0 ** -24
C = 64


def rms(v, eps):
    return torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)


def border(x, res, post, pre, gate, scale, eps, dout=None, ds=None):
    """(results, bounds): out, s and, with dout / ds, dx, dres, dgate, dpost, dpre, dscale; float64 on the CPU."""
    d = [None if t is None else torch.as_tensor(t).detach().double().cpu() for t in (x, res, post, pre, gate, scale, dout, ds)]
    x, res, post, pre, z, sc, do, ds = d
    n1 = rms(x, eps)
    sig = torch.ones_like(x) if z is None else torch.sigmoid(z)
    sil = torch.ones_like(x) if z is None else z * sig
    t = x * n1 * (1 + post) * sil
    s = res + sc * t
    n2 = rms(s, eps)
    out = s * n2 * (1 + pre)
    ms = res.abs() + (sc * t).abs()
    kap = 1 + (ms.square().sum(-1, keepdim=True) / s.square().sum(-1, keepdim=True).clamp_min(1e-300)).sqrt()
    r = {"out": out, "s": s}
    b = {"s": C * U * ms, "out": C * U * n2 * (1 + pre).abs() * (ms + kap * s.abs())}
    if do is None and ds is None:
        return r, b
    do, ds = (torch.zeros_like(x) if v is None else v for v in (do, ds))
    ow, c = do * (1 + pre), sc * sil * (1 + post) * x
    dr = ds + n2 * ow - s * n2 ** 3 * (ow * s).mean(-1, keepdim=True)
    mr = ds.abs() + n2 * ow.abs() + ms * n2 ** 3 * (ow * ms).abs().mean(-1, keepdim=True)
    dt = dr * sc
    r["dx"] = n1 * dt * sil * (1 + post) - x * n1 ** 3 * (dr * c).mean(-1, keepdim=True)
    mx = n1 * (mr * sc * sil * (1 + post)).abs() + x.abs() * n1 ** 3 * (mr * c).abs().mean(-1, keepdim=True)
    r["dres"] = dr
    b["dx"], b["dres"] = 2 * C * U * kap * mx, 2 * C * U * kap * mr
    if z is not None:
        f = sc * x * n1 * (1 + post) * sig * (1 + z * (1 - sig))
        r["dgate"] = dr * f
        b["dgate"] = 2 * C * U * kap * (mr * (sc * x * n1 * (1 + post)).abs() * sig * (1 + z.abs()))
    # sums over rows: a workgroup's rows one after another, workgroups 16 at a time, 4 teams
    rows = (2 * C * kap + x.shape[0] / 4 + 64) * U
    for n, f, m in (("dpost", dt * sil * x * n1, mr * (sc * sil * x * n1).abs()),
                    ("dpre", do * s * n2, (do * ms * n2).abs()), ("dscale", dr * t, mr * t.abs())):
        r[n], b[n] = f.sum(0), (rows * m).sum(0)
    return r, b


def heads(x, gate, w, groups, eps, dout=None):
    """(results, bounds): out and, with dout, dx, dgate, dweight; float64 on the CPU."""
    x, z, w, do = (None if t is None else t.detach().double().cpu() for t in (x, gate, w, dout))
    R, D = x.shape
    cut = lambda v: v.reshape(R, groups, D // groups)        # noqa: E731
    n = rms(cut(x), eps).expand(R, groups, D // groups).reshape(R, D)
    sig = torch.sigmoid(z)
    out = x * n * (1 + w) * z * sig
    r, b = {"out": out}, {"out": C * U * out.abs()}
    if do is None:
        return r, b
    g = do * z * sig

    def mean(v):
        return cut(v).mean(-1, keepdim=True).expand(R, groups, D // groups).reshape(R, D)

    r["dx"] = n * g * (1 + w) - x * n ** 3 * mean(g * (1 + w) * x)
    b["dx"] = 2 * C * U * (n * (g * (1 + w)).abs() + x.abs() * n ** 3 * mean((g * (1 + w) * x).abs()))
    r["dgate"] = do * x * n * (1 + w) * sig * (1 + z * (1 - sig))
    b["dgate"] = 2 * C * U * (do * x * n * (1 + w)).abs() * sig * (1 + z.abs())
    r["dweight"] = (g * x * n).sum(0)
    b["dweight"] = (2 * C + R / 4 + 128) * U * (g * x * n).abs().sum(0)
    return r, b


def check(got, want, bound, what):
    """|got - want| <= bound + half a step of got's type, elementwise."""
    step = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    got_d = got.detach().double().cpu()
    assert got_d.shape == want.shape, f"{what}: shape {tuple(got_d.shape)} vs {tuple(want.shape)}"
    # (below the type's normal range a step has a fixed size)
    room = bound * (1 + step) + step * want.abs() + torch.finfo(got.dtype).tiny * (1 if step == 0 else 2 * step)
    bad = ~((got_d - want).abs() <= room)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, (got_d - want).abs() / room, 0.0).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds; at {i}: got {got_d.flatten()[i]:.8g}, "
                             f"want {want.flatten()[i]:.8g}, room {room.flatten()[i]:.3g}")
