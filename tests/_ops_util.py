"""Float64 forms of layer norm and linear cross entropy with their first and
second gradients (from the formulas, on the CPU), and the bounds that the
kernels' outputs are held to.

Bounds.  A value rounded to type t is off by at most u |value|, u =
finfo(t).eps / 2.  The kernels round each output once; G and H of the linear
cross entropy once more before their products (16-bit types), so dX = G W may
be off by u |G| |W| on top, and so on.  Sums in fp32: a sum of n terms is off
by about sqrt(n) 2^-24 times the sum of their magnitudes, with a factor of 4
for the tail of that distribution; a difference of the logits of delta moves a
probability by the relative 2 delta.
"""
import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def within(name, got, ref, bound):
    """|got - ref| <= bound element by element, and finite where ref is."""
    g = got.detach().double().cpu()
    assert g.shape == ref.shape, f"{name}: shape {tuple(g.shape)}, expected {tuple(ref.shape)}"
    if not g.numel():
        return
    err = (g - ref).abs()
    bad = ~(err <= bound)
    worst = (err / bound.clamp_min(1e-300)).max()
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {g.numel()} values past their bound, worst {float(worst):.2f} "
                           f"times it (largest error {float(err.max()):.3e})")


# ---------------------------------------------------------------------------
def norm_ref(x, w, b, eps, dy=None, a=None, cw=None, cb=None):
    """(outputs, magnitudes) by name; float64 [N, D] and [D] operands."""
    n, d = x.shape
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mu) * r

    def away(t):
        return t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)

    def size(t):  # of a row's terms: each value, and what the row's means add to all
        return t.abs() + t.abs().mean(1, keepdim=True) + xh.abs() * (t * xh).abs().mean(1, keepdim=True)

    # of xh: x - mu loses digits of the row's own offset
    sx = xh.abs() + 1 + (x.abs() + mu.abs()) * r
    out, mag = {"y": xh * w + b}, {"y": sx * w.abs() + b.abs()}
    if dy is None:
        return out, mag
    g = dy * w
    sg = size(g) + g.abs() * sx + sx * (g.abs() * sx).mean(1, keepdim=True)
    out.update(dx=r * away(g), dw=(dy * xh).sum(0), db=dy.sum(0))
    mag.update(dx=r * sg, dw=(dy.abs() * sx).sum(0) * (n ** 0.5 + 8) / 8, db=dy.abs().sum(0) * (n ** 0.5 + 8) / 8)
    if a is None and cw is None and cb is None:
        return out, mag
    z = torch.zeros_like
    a = z(x) if a is None else a
    cw = z(w) if cw is None else cw
    cb = z(w) if cb is None else cb
    pa, pg = away(a), away(g)  # away(a) . away(g) is not a . away(g): eps keeps mean(xh^2) below 1
    mgx, max_ = (g * xh).mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    t = cw * dy - r * (a * mgx + g * max_)
    out.update(gx=r * away(t) - r * r * xh * (a * pg).mean(1, keepdim=True), gw=(dy * r * pa).sum(0),
               gdy=w * r * pa + cw * xh + cb)
    sa = size(a) + a.abs() * sx + sx * (a.abs() * sx).mean(1, keepdim=True)
    st = (cw * dy).abs() + r * (a.abs() * (g.abs() * sx).mean(1, keepdim=True) +
                                g.abs() * (a.abs() * sx).mean(1, keepdim=True))
    st = size(st) + st * sx + sx * (st * sx).mean(1, keepdim=True)
    mag.update(gx=r * st + r * r * sx * (sa * sg).mean(1, keepdim=True),
               gw=(dy.abs() * r * sa).sum(0) * (n ** 0.5 + 8) / 8,
               gdy=w.abs() * r * sa + cw.abs() * sx + cb.abs())
    return out, mag


def norm_bound(ref, mag, dtype):
    """One rounding to the output's type, and the fp32 arithmetic: some tens
    of operations deep, each off by 2^-24 of the magnitudes that meet in it."""
    return unit(dtype) * ref.abs() + 32 * F32 * mag + (1e-7 if dtype == torch.float16 else 1e-30)


# ---------------------------------------------------------------------------
def lce_ref(x, w, t, wt, up, inv, dtype, a=None, b=None):
    """(outputs, bounds) by name.  x [N, d], w [V, d] float64, t [N] with every
    row that counts in range, wt [N] row weights, up: the upstream gradient
    ([N] or a number), inv: 1 / the mean's denominator.  dtype: the operands'
    and the gradients' type."""
    n, d = x.shape
    v = w.shape[0]
    u = unit(dtype)
    live = wt != 0
    x = torch.where(live[:, None], x, 0.0)
    z = x @ w.t()
    # fp32 sums of the logits; three bf16 parts leave out products below 2^-24 of each
    dz = F32 * (4 * d ** 0.5 * torch.sqrt((x * x) @ (w * w).t()) + 8) + (4 * F32 * x.abs() @ w.abs().t() / d ** 0.5)
    lse = torch.logsumexp(z, 1)
    ts = torch.where(live, t, 0)
    nll = lse - z.gather(1, ts[:, None])[:, 0]
    p = torch.exp(z - lse[:, None])
    dl = dz.max(1).values
    out = {"rows": torch.where(live, nll * wt, 0.0)}
    bound = {"rows": wt.abs() * (4 * dl + 4 * F32 * (1 + nll.abs()))}
    out["loss"] = (out["rows"].sum() * inv).reshape(())
    bound["loss"] = (bound["rows"].sum() * inv + 4 * n ** 0.5 * F32 * out["rows"].abs().sum() * inv).reshape(())
    c = torch.where(live, torch.as_tensor(up, dtype=torch.float64) * wt * inv, 0.0)[:, None]
    onehot = torch.zeros_like(p).scatter_(1, ts[:, None], 1.0)
    gh = p - onehot
    g = c * gh
    two = dtype != torch.float32  # G and H are rounded to the operands' type
    rp = 2 * dl[:, None] + dz + 8 * F32 * (1 + (z - lse[:, None]).abs())  # relative, of p
    eg = c.abs() * p * rp + F32 * g.abs() + (u if two else 4 * F32) * g.abs()
    if dtype == torch.float16:  # G's smallest steps, at its scales: 2^-25 of 2^14 times the row's (the largest) bound
        eg = eg + 2.0 ** -38 * (c.abs() + c.abs().max())
    acc = lambda k: 4 * k ** 0.5 * F32  # noqa: E731
    # one more rounding to the gradient's type, and fp16's smallest step there
    step = lambda r: u * r.abs() + (3e-8 if dtype == torch.float16 else 1e-30)  # noqa: E731
    out.update(dx=g @ w, dw=g.t() @ x)
    bound.update(dx=eg @ w.abs() + acc(v) * (g.abs() @ w.abs()) + step(out["dx"]),
                 dw=eg.t() @ x.abs() + acc(n) * (g.abs().t() @ x.abs()) + step(out["dw"]))
    if a is None and b is None:
        return out, bound
    a = torch.zeros_like(x) if a is None else torch.where(live[:, None], a, 0.0)
    b = torch.zeros_like(w) if b is None else b
    uu = a @ w.t() + x @ b.t()
    du = F32 * (4 * (2 * d) ** 0.5 * torch.sqrt((a * a) @ (w * w).t() + (x * x) @ (b * b).t())) + \
        4 * F32 * (a.abs() @ w.abs().t() + x.abs() @ b.abs().t()) / d ** 0.5
    hs = (p * uu).sum(1, keepdim=True)
    dh = (p * (du + rp * uu.abs())).sum(1, keepdim=True) + acc(v) * (p * uu.abs()).sum(1, keepdim=True)
    # h may come from dX and G B, sums over the rounded G: u of each term of A . (|G| |W|) / c
    ra = (a.abs() * (eg @ w.abs() + acc(v) * (g.abs() @ w.abs()))).sum(1, keepdim=True)
    rb = (x.abs() * (eg @ b.abs() + acc(v) * (g.abs() @ b.abs()))).sum(1, keepdim=True)
    dh = dh + torch.where(c != 0, (ra + rb) / c.abs().clamp_min(1e-300), 0.0)
    h = c * p * (uu - hs)
    eh = c.abs() * p * (rp * (uu - hs).abs() + du + dh) + 2 * F32 * h.abs() + (u if two else 4 * F32) * h.abs()
    if dtype == torch.float16:
        top = torch.clamp(2 * uu.abs().max(1, keepdim=True).values, min=1.0)
        eh = eh + 2.0 ** -37 * (c.abs() * top + (c.abs() * top).max())
        eg = eg + 2.0 ** -37 * (c.abs() * top + (c.abs() * top).max())
    out.update(gx=h @ w + g @ b, gw=h.t() @ x + g.t() @ a,
               gup=torch.where(live, wt * inv * (hs[:, 0] - uu.gather(1, ts[:, None])[:, 0]), 0.0))
    bound.update(gx=eh @ w.abs() + eg @ b.abs() + acc(2 * v) * (h.abs() @ w.abs() + g.abs() @ b.abs()) + step(out["gx"]),
                 gw=eh.t() @ x.abs() + eg.t() @ a.abs() + acc(2 * n) * (h.abs().t() @ x.abs() + g.abs().t() @ a.abs()) +
                 step(out["gw"]),
                 gup=wt.abs() * inv * (dh[:, 0] + du.max(1).values + 8 * F32 * (hs.abs()[:, 0] + uu.abs().max(1).values)))
    out["gloss"], bound["gloss"] = out["gup"].sum().reshape(()), bound["gup"].sum().reshape(()) + \
        acc(n) * out["gup"].abs().sum()
    return out, bound
