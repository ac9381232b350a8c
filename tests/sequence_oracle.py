"""The token-sequence operators from their formulas in 64 bits on the CPU, gradients included.

Each function returns (results, magnitudes): `magnitudes` is the same sum with every term's absolute value in place of
the term.  A result computed in fp32 with at most n roundings on any path from an input is off by at most about
n 2^-24 times its magnitude, whatever cancels; that is what the tests allow, plus half a step of the output's type."""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def within(got, want, mag, n, name):
    """|got - want| <= half a step of the type + n fp32 roundings of the magnitude, everywhere."""
    g, w, m = got.detach().double().cpu(), want.double(), mag.double()
    assert g.shape == w.shape, (name, g.shape, w.shape)
    assert torch.isfinite(g).all(), name
    allowed = HALF[got.dtype] * w.abs() + n * 2.0 ** -24 * m * (1 + HALF[got.dtype]) + 1e-37
    over = (g - w).abs() / allowed
    assert float(over.max() if over.numel() else 0) <= 1.0, (name, float(over.max()), int(over.argmax()))


def silu(v):
    return v * torch.sigmoid(v)


def silu_slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def norm(x, w, b, eps, dy=None):
    x, w = x.double(), w.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    wide = (x.abs() + x.abs().mean(-1, keepdim=True)) * r           # |x - mu| r with nothing cancelled
    top = xh if b is not None else x * r
    out = {"y": top * w + (b.double() if b is not None else 0)}
    mag = {"y": wide * w.abs() + (b.double().abs() if b is not None else 0)}
    if dy is None:
        return out, mag
    dy = dy.double()
    g = dy * w
    mean = lambda t: t.mean(-1, keepdim=True)
    if b is not None:
        out["dx"] = r * (g - mean(g) - xh * mean(g * xh))
        mag["dx"] = r * (g.abs() + mean(g.abs()) + wide * mean(g.abs() * wide))
        out["db"], mag["db"] = dy.flatten(0, -2).sum(0), dy.abs().flatten(0, -2).sum(0)
    else:
        out["dx"] = r * g - r * r * xh * mean(g * x)
        mag["dx"] = r * g.abs() + r * wide * mean(g.abs() * (wide + mu.abs() * r)) + r * wide * r * mu.abs() * mean(g.abs())
    out["dw"], mag["dw"] = (dy * top).flatten(0, -2).sum(0), (dy.abs() * wide).flatten(0, -2).sum(0)
    return out, mag


def conv(x, w, b, state, act, dy=None, dend=None):
    """w (D, W); the state and the row as one sequence of W - 1 + L inputs."""
    x, w = x.double(), w.double()
    B, D, L = x.shape
    W = w.shape[1]
    h0 = state.double() if state is not None else torch.zeros(B, D, W - 1, dtype=torch.float64)
    full = torch.cat([h0, x], 2)
    bias = b.double()[:, None] if b is not None else torch.zeros(D, 1, dtype=torch.float64)
    win = full.unfold(2, W, 1)[:, :, :L] if L else full.new_zeros(B, D, 0, W)
    v = (win * w[:, None]).sum(-1) + bias
    vm = (win * w[:, None]).abs().sum(-1) + bias.abs()
    out = {"y": silu(v) if act else v, "end": full[:, :, L:]}
    mag = {"y": vm * (1 + v.abs()) if act else vm, "end": torch.zeros(B, D, W - 1)}     # (a state is copied: no rounding)
    if dy is None:
        return out, mag
    dy = dy.double()
    slope = silu_slope(v) if act else torch.ones_like(v)
    dv = dy * slope
    dm = dy.abs() * ((1.1 + vm) if act else 1)                       # |silu'| <= 1.1, |silu''| <= 1
    dfull, dfm = torch.zeros_like(full), torch.zeros_like(full)
    for k in range(W):
        dfull[:, :, k:k + L] += w[:, k, None] * dv
        dfm[:, :, k:k + L] += w[:, k, None].abs() * dm
    if dend is not None:
        dfull[:, :, L:] += dend.double()
        dfm[:, :, L:] += dend.double().abs()
    out.update(dx=dfull[:, :, W - 1:], dstate=dfull[:, :, :W - 1], db=dv.sum((0, 2)), dw=(win * dv[..., None]).sum((0, 2)))
    mag.update(dx=dfm[:, :, W - 1:], dstate=dfm[:, :, :W - 1], db=dm.sum((0, 2)), dw=(win.abs() * dm[..., None]).sum((0, 2)))
    return out, mag


def scan(x, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, h0=None, dy=None, dlast=None):
    x, A, B, C = x.double(), A.double(), B.double(), C.double()
    batch, chan, L = x.shape
    N = A.shape[1]
    raw = delta.double() + (delta_bias.double()[:, None] if delta_bias is not None else 0)
    dt = torch.nn.functional.softplus(raw, threshold=60.0) if softplus else raw
    group = torch.arange(chan) // (chan // B.shape[1])
    Bd, Cd = B[:, group], C[:, group]                                # (batch, chan, N, L)
    skip = D.double()[:, None] if D is not None else torch.zeros(chan, 1, dtype=torch.float64)
    a = torch.exp(dt[:, :, None] * A[:, :, None])
    start = h0.double() if h0 is not None else torch.zeros(batch, chan, N, dtype=torch.float64)
    gate = silu(z.double()) if z is not None else torch.ones_like(x)
    slope = silu_slope(z.double()) if z is not None else torch.zeros_like(x)
    results = []
    for sign in (lambda t: t, torch.abs):
        xs, Bs, Cs, ss, ga, sl, As = sign(x), sign(Bd), sign(Cd), sign(skip), sign(gate), slope, sign(A)
        if sign is torch.abs and z is not None:
            # silu' = q + q z (1 - q) has a zero at z = -1.28 where its two terms cancel: their magnitudes are what rounds
            q = torch.sigmoid(z.double())
            sl = q + q * z.double().abs() * (1 - q)
        us = sign(dt) * xs
        h = torch.zeros(batch, chan, N, L + 1, dtype=torch.float64)
        h[..., 0] = sign(start)
        for t in range(L):
            h[..., t + 1] = a[..., t] * h[..., t] + us[:, :, None, t] * Bs[..., t]
        s = (Cs * h[..., 1:]).sum(2) + ss * xs
        out = {"y": s * ga, "last": h[..., L]}
        if dy is not None:
            e = sign(dy.double()) * ga
            g = torch.zeros(batch, chan, N, L + 1, dtype=torch.float64)
            ahead = sign(dlast.double()) if dlast is not None else torch.zeros(batch, chan, N, dtype=torch.float64)
            for t in reversed(range(L)):
                g[..., t] = Cs[..., t] * e[:, :, None, t] + ahead
                ahead = a[..., t] * g[..., t]
            g = g[..., :L]
            p = g * a * h[..., :L]
            gB = (g * Bs).sum(2)
            back = lambda m: torch.zeros(batch, B.shape[1], N, L, dtype=torch.float64).index_add_(1, group, m)
            ddt = gB * xs + (p * As[:, :, None]).sum(2)
            ddelta = ddt * torch.sigmoid(raw) if softplus else ddt
            out.update(dx=gB * sign(dt) + ss * e, ddelta=ddelta, dA=(p * sign(dt)[:, :, None]).sum((0, 3)),
                       dB=back(g * us[:, :, None]), dC=back(h[..., 1:] * e[:, :, None]), dD=(e * xs).sum((0, 2)),
                       ddelta_bias=ddelta.sum((0, 2)), dz=sign(dy.double()) * s * sl, dh0=ahead)
        results.append(out)
    return tuple(results)
