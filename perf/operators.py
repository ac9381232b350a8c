"""What the token-sequence operators are measured on: the norm over token rows, the short causal convolution and the
selective state space scan, each for inference and for training, and the pair of convolution and scan for one token.

Shapes follow the package's own: channel widths of 48 to 384 (the four levels of the network, and twice a width where a
block expands its channels), images of 64 x 64 to 256 x 256 pixels read as sequences of tokens, 16 states a channel.
Tensors are (batch, channel, token), pixel-contiguous as everywhere in the package; the norm's rows are (token, channel).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the latent level of one small crop at inference: 8 x 8 tokens, latency only
        {"name": "norm_few_rows", "op": "norm", "rows": 64, "C": 384, "dtype": "f32", "bias": True, "grad": False},
        # first-level tokens of a training batch of eight 128 x 128 patches, bf16 activations
        {"name": "norm_train_patches", "op": "norm", "rows": 131072, "C": 96, "dtype": "bf16", "bias": True, "grad": True},
        # the full inference batch of sixteen 256 x 256 images, trained in fp32 with the bias-free norm
        {"name": "norm_train_images", "op": "norm", "rows": 1048576, "C": 96, "dtype": "f32", "bias": False, "grad": True},
        # an odd width and an odd number of rows: a cropped border batch of a net whose width is no power of two
        {"name": "norm_train_odd", "op": "norm", "rows": 12289, "C": 181, "dtype": "bf16", "bias": True, "grad": True},
        # the convolution in front of the scan, training on 64 x 64 patches
        {"name": "conv_train_patches", "op": "conv", "B": 8, "D": 384, "L": 4096, "W": 4, "dtype": "bf16", "silu": True, "state": False, "grad": True},
        # the next piece of a prompt that is fed in pieces: odd channels, odd length, state carried over
        {"name": "conv_piece_odd", "op": "conv", "B": 3, "D": 193, "L": 1021, "W": 3, "dtype": "f32", "silu": True, "state": True, "grad": False},
        # one 128 x 128 image as a prompt, gated, its last state kept for the tokens that follow
        {"name": "scan_prompt", "op": "scan", "B": 1, "D": 192, "G": 1, "N": 16, "L": 16384, "dtype": "bf16", "z": True, "state": True, "grad": False},
        # a training step on 64 x 64 patches scanned in four directions (four groups of B and C), fp32
        {"name": "scan_train_directions", "op": "scan", "B": 4, "D": 768, "G": 4, "N": 16, "L": 4096, "dtype": "f32", "z": False, "state": False, "grad": True},
        # odd everything: a short ragged crop, 12 states, two groups, states in and out with their gradients
        {"name": "scan_train_odd", "op": "scan", "B": 3, "D": 102, "G": 2, "N": 12, "L": 777, "dtype": "bf16", "z": True, "state": True, "grad": True},
        # the largest: a bf16 training step on eight 128 x 128 patches at the widest level, gated
        {"name": "scan_train_large", "op": "scan", "B": 8, "D": 384, "G": 1, "N": 16, "L": 16384, "dtype": "bf16", "z": True, "state": False, "grad": True},
        # one token of one sequence: latency
        {"name": "token_one", "op": "step", "B": 1, "D": 384, "G": 1, "N": 16, "W": 4, "dtype": "f32"},
        # one token of each of 256 sequences
        {"name": "token_batch", "op": "step", "B": 256, "D": 768, "G": 1, "N": 16, "W": 4, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "conv", "conv", "scan", "scan", "scan", "step"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "norm":
        C = _log_int(rng, 8, 2048)
        rows = _log_int(rng, 1, min(1048576, 60_000_000 // C))
        return {"op": op, "rows": rows, "C": C, "dtype": dtype, "bias": rng.random() < 0.7, "grad": rng.random() < 0.7}
    if op == "step":
        G = rng.choice([1, 1, 2, 4])
        return {"op": op, "B": _log_int(rng, 1, 256), "D": G * _log_int(rng, 8, 768 // G), "G": G,
                "N": rng.choice([4, 8, 12, 16, 16, 32]), "W": rng.randint(2, 4), "dtype": dtype}
    B = rng.randint(1, 8)
    if op == "conv":
        D = _log_int(rng, 8, 768)
        return {"op": op, "B": B, "D": D, "L": _log_int(rng, 1, min(65536, 30_000_000 // (B * D))), "W": rng.randint(2, 4),
                "dtype": dtype, "silu": rng.random() < 0.7, "state": rng.random() < 0.5, "grad": rng.random() < 0.6}
    G = rng.choice([1, 1, 2, 4])
    D = G * _log_int(rng, 8, 768 // G)
    N = rng.choice([4, 8, 12, 16, 16, 16, 32])
    return {"op": op, "B": B, "D": D, "G": G, "N": N, "L": _log_int(rng, 1, min(65536, 300_000_000 // (B * D * N))),
            "dtype": dtype, "z": rng.random() < 0.5, "state": rng.random() < 0.5, "grad": rng.random() < 0.6}


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape, dtype=t, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    s = {"case": case}
    f32 = torch.float32
    if op == "norm":
        rows, C = case["rows"], case["C"]
        s["x"] = normal(rows, C, shift=0.3)
        s["w"] = uniform(0.5, 1.5, C)
        s["b"] = normal(C, dtype=f32, scale=0.1) if case["bias"] else None
        if case["grad"]:
            s["dy"] = normal(rows, C)
        leaves = ["x", "w", "b"]
    elif op == "conv":
        B, D, L, W = case["B"], case["D"], case["L"], case["W"]
        s["x"] = normal(B, D, L)
        s["w"] = uniform(-1.0, 1.0, D, W) / math.sqrt(W)
        s["b"] = uniform(-1.0, 1.0, D) / math.sqrt(W)
        s["h0"] = normal(B, D, W - 1) if case["state"] else None
        if case["grad"]:
            s["dy"] = normal(B, D, L)
        leaves = ["x", "w", "b", "h0"]
    else:
        B, D, G, N = case["B"], case["D"], case["G"], case["N"]
        # step sizes between 0.001 and 0.1 before the tokens' own part, rates of 1 .. N with some spread: what training starts from
        dt = torch.exp(uniform(math.log(1e-3), math.log(1e-1), D))
        s["dbias"] = dt + torch.log(-torch.expm1(-dt))
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=f32) * uniform(0.8, 1.25, D, N)
        s["Dskip"] = uniform(0.5, 1.5, D)
        if op == "scan":
            L = case["L"]
            s["x"], s["delta"] = normal(B, D, L), normal(B, D, L, scale=0.5)
            s["B"], s["C"] = normal(B, G, N, L), normal(B, G, N, L)
            s["z"] = normal(B, D, L) if case["z"] else None
            s["h0"] = normal(B, D, N, dtype=f32) if case["state"] else None
            if case["grad"]:
                s["dy"] = normal(B, D, L)
                s["dlast"] = normal(B, D, N, dtype=f32) if case["state"] else None
            leaves = ["x", "delta", "A", "B", "C", "Dskip", "z", "dbias", "h0"]
        else:
            W = case["W"]
            s["x"], s["delta"], s["z"] = normal(B, D), normal(B, D, scale=0.5), normal(B, D)
            s["B"], s["C"] = normal(B, G, N), normal(B, G, N)
            s["w"] = uniform(-1.0, 1.0, D, W) / math.sqrt(W)
            s["b"] = uniform(-1.0, 1.0, D) / math.sqrt(W)
            s["conv_state"] = normal(B, D, W - 1)
            s["h0"] = normal(B, D, N, dtype=f32)
            # the next states go to a second pair of buffers, as a program does that may have to take a token back
            s["conv_next"], s["h_next"] = torch.empty_like(s["conv_state"]), torch.empty_like(s["h0"])
            leaves = []
    if case.get("grad"):
        s["leaves"] = [k for k in leaves if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "conv": _own_conv, "scan": _own_scan, "step": _own_step}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan, "step": _plain_step}[op](state)


def _grads(s, outputs, weights):
    g = torch.autograd.grad(outputs, [s[k] for k in s["leaves"]], weights)
    return {"d" + k: v for k, v in zip(s["leaves"], g)}


def _own_norm(s):
    from superresolution_amd import sequence
    y = sequence.layernorm(s["x"], s["w"], s["b"], EPS)
    return {"y": y.detach(), **_grads(s, [y], [s["dy"]])} if s["case"]["grad"] else {"y": y}


def _own_conv(s):
    from superresolution_amd import sequence
    c = s["case"]
    y = sequence.causal_conv1d(s["x"], s["w"], s["b"], initial_state=s["h0"], activation="silu" if c["silu"] else None,
                               return_final_state=c["state"])
    last = {}
    if c["state"]:
        y, end = y
        last = {"end": end.detach()}
    return {"y": y.detach(), **last, **(_grads(s, [y], [s["dy"]]) if c["grad"] else {})}


def _own_scan(s):
    from superresolution_amd import sequence
    c = s["case"]
    y = sequence.selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], s["Dskip"], z=s["z"], delta_bias=s["dbias"],
                                delta_softplus=True, initial_state=s["h0"], return_last_state=c["state"])
    outs, last = [y], {}
    if c["state"]:
        y, end = y
        outs, last = [y, end], {"end": end.detach()}
    return {"y": y.detach(), **last, **(_grads(s, outs, [s["dy"], s["dlast"]][:len(outs)]) if c["grad"] else {})}


def _own_step(s):
    from superresolution_amd import sequence
    xc = sequence.causal_conv1d_update(s["x"], s["conv_state"], s["w"], s["b"], activation="silu", state_out=s["conv_next"])
    y = sequence.selective_scan_update(s["h0"], xc, s["delta"], s["A"], s["B"], s["C"], s["Dskip"], z=s["z"],
                                       delta_bias=s["dbias"], delta_softplus=True, state_out=s["h_next"])
    return {"y": y, "conv_end": s["conv_next"], "end": s["h_next"]}


# ----------------------------------------------------------------------------------------------------------------
# plain forms: elementary operations in fp32, rounded once at the end
# ----------------------------------------------------------------------------------------------------------------
def _plain_norm(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"]
    mu = x.mean(1, keepdim=True)
    xc = x - mu
    r = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * r
    out = {"y": (xh * w + s["b"] if s["b"] is not None else x * r * w).to(t)}
    if not s["case"]["grad"]:
        return out
    dy = s["dy"].float()
    g = dy * w
    if s["b"] is not None:
        out["dx"] = (r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))).to(t)
        out["dw"], out["db"] = (dy * xh).sum(0), dy.sum(0)
    else:
        out["dx"] = (r * g - r * r * xh * (g * x).mean(1, keepdim=True)).to(t)
        out["dw"] = (dy * x * r).sum(0)
    return out


def _silu_slope(v):
    q = 1.0 / (1.0 + torch.exp(-v))
    return q * (1.0 + v * (1.0 - q))


def _taps(x, W):
    """(..., L + W - 1) -> (..., L, W): the W inputs under each output."""
    return x.unfold(-1, W, 1)


def _plain_conv(s):
    c, t = s["case"], s["x"].dtype
    B, D, L, W = c["B"], c["D"], c["L"], c["W"]
    x, w, b = s["x"].float(), s["w"], s["b"]
    h0 = s["h0"].float() if c["state"] else torch.zeros(B, D, W - 1, device=x.device)
    full = torch.cat([h0, x], 2)
    v = (_taps(full, W) * w[:, None, :]).sum(-1) + b[:, None]
    out = {"y": (v / (1.0 + torch.exp(-v)) if c["silu"] else v).to(t)}
    if c["state"]:
        out["end"] = full[:, :, L:].to(t)
    if not c["grad"]:
        return out
    dv = s["dy"].float() * (_silu_slope(v) if c["silu"] else 1.0)
    pad = torch.zeros(B, D, W - 1, device=x.device)
    dfull = (_taps(torch.cat([pad, dv, pad], 2), W) * w.flip(1)[:, None, :]).sum(-1)
    out["dx"] = dfull[:, :, W - 1:].to(t)
    out["dw"] = (_taps(full, W) * dv[..., None]).sum((0, 2))
    out["db"] = dv.sum((0, 2))
    if c["state"]:
        out["dh0"] = dfull[:, :, :W - 1].to(t)
    return out


def _running(a, b):
    """h_t = a_t h_{t-1} + b_t along the last axis, by doubling."""
    step, L = 1, a.shape[-1]
    while step < L:
        b = torch.cat([b[..., :step], b[..., step:] + a[..., step:] * b[..., :-step]], -1)
        a = torch.cat([a[..., :step], a[..., step:] * a[..., :-step]], -1)
        step *= 2
    return b


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _plain_scan(s):
    c, t = s["case"], s["x"].dtype
    B, D, G, N, L = c["B"], c["D"], c["G"], c["N"], c["L"]
    x = s["x"].float().view(B, G, D // G, L)
    raw = s["delta"].float().view(B, G, D // G, L) + s["dbias"].view(G, D // G, 1)
    dt = _softplus(raw)
    A = s["A"].view(G, D // G, N, 1)
    Bm, Cm = s["B"].float()[:, :, None], s["C"].float()[:, :, None]          # (B, G, 1, N, L)
    skip = s["Dskip"].view(G, D // G, 1)
    a = torch.exp(dt[..., None, :] * A)                                     # (B, G, Dg, N, L)
    u = (dt * x)[..., None, :]
    b = u * Bm
    h0 = s["h0"].view(B, G, D // G, N) if c["state"] else torch.zeros(B, G, D // G, N, device=x.device)
    b[..., 0] += a[..., 0] * h0
    h = _running(a, b)
    y = (h * Cm).sum(3) + skip * x
    out = {}
    if c["state"]:
        out["end"] = h[..., -1].reshape(B, D, N).clone()
    if c["z"]:
        z = s["z"].float().view(B, G, D // G, L)
        out["y"] = (y * z / (1.0 + torch.exp(-z))).view(B, D, L).to(t)
    else:
        out["y"] = y.view(B, D, L).to(t)
    if not c["grad"]:
        return out
    dy = s["dy"].float().view(B, G, D // G, L)
    if c["z"]:
        out["dz"] = (dy * y * _silu_slope(z)).view(B, D, L).to(t)
        dy = dy * z / (1.0 + torch.exp(-z))
    g = dy[..., None, :] * Cm
    if c["state"]:
        g[..., -1] += s["dlast"].view(B, G, D // G, N)
    ahead = torch.cat([a[..., 1:], torch.zeros_like(a[..., :1])], -1)
    g = _running(ahead.flip(-1), g.flip(-1)).flip(-1)
    out["dC"] = (h * dy[..., None, :]).sum(2).to(t)
    out["dB"] = (g * u).sum(2).to(t)
    gB = (g * Bm).sum(3)
    ga = g * a
    if c["state"]:
        out["dh0"] = ga[..., 0].reshape(B, D, N).clone()
    p = ga * torch.cat([h0[..., None], h[..., :-1]], -1)
    out["dA"] = (p * dt[..., None, :]).sum(-1).sum(0).view(D, N)
    ddt = (gB * x + (p * A).sum(3)) / (1.0 + torch.exp(-raw))
    out["dx"] = (gB * dt + skip * dy).view(B, D, L).to(t)
    out["ddelta"] = ddt.view(B, D, L).to(t)
    out["ddbias"] = ddt.sum(-1).sum(0).view(D)
    out["dDskip"] = (dy * x).sum(-1).sum(0).view(D)
    return out


def _plain_step(s):
    c, t = s["case"], s["x"].dtype
    B, D, G, N = c["B"], c["D"], c["G"], c["N"]
    full = torch.cat([s["conv_state"], s["x"][..., None]], 2)
    v = (full.float() * s["w"]).sum(-1) + s["b"]
    xc = (v / (1.0 + torch.exp(-v))).to(t).float()                          # the convolution's output has the input's type
    dt = _softplus(s["delta"].float() + s["dbias"])
    rep = lambda m: m.float().repeat_interleave(D // G, 1)                  # (B, G, N) -> (B, D, N)
    h = torch.exp(dt[..., None] * s["A"]) * s["h0"] + (dt * xc)[..., None] * rep(s["B"])
    z = s["z"].float()
    y = ((h * rep(s["C"])).sum(-1) + s["Dskip"] * xc) * z / (1.0 + torch.exp(-z))
    return {"y": y.to(t), "conv_end": full[:, :, 1:].contiguous(), "end": h}


# ----------------------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (v.detach().double() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
    with torch.no_grad() if case["op"] in ("scan", "step") else torch.enable_grad():
        return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan, "step": _exact_step}[case["op"]](case, d)


def _exact_grads(out, y, d):
    if "leaves" in d:
        out.update(zip(["d" + k for k in d["leaves"]], torch.autograd.grad(y, [d[k] for k in d["leaves"]], d["dy"])))
    out["y"] = y.detach()
    return out


def _exact_norm(c, d):
    for k in d.get("leaves", ()):
        d[k].requires_grad_(True)
    var, mean = torch.var_mean(d["x"], 1, unbiased=False, keepdim=True)
    top = d["x"] - mean if c["bias"] else d["x"]
    y = top / torch.sqrt(var + EPS) * d["w"]
    return _exact_grads({}, y + d["b"] if c["bias"] else y, d)


def _exact_conv(c, d):
    for k in d.get("leaves", ()):
        d[k].requires_grad_(True)
    D, W, L = c["D"], c["W"], c["L"]
    full = torch.cat([d["h0"], d["x"]], 2) if c["state"] else torch.nn.functional.pad(d["x"], (W - 1, 0))
    v = sum(full[:, :, k:k + L] * d["w"][:, k, None] for k in range(W)) + d["b"][:, None]
    out = {"end": full[:, :, L:].detach()} if c["state"] else {}
    return _exact_grads(out, torch.nn.functional.silu(v) if c["silu"] else v, d)


def _exact_scan(c, d):
    B, D, G, N, L = c["B"], c["D"], c["G"], c["N"], c["L"]
    if B * D * N * L > 1 << 30:
        return None
    first = lambda m: m.permute(2, 0, 1).contiguous()                       # token first: (L, B, D)
    wide = lambda m: m.permute(3, 0, 1, 2).contiguous()                     # (L, B, G, N)
    x, z = first(d["x"]), (first(d["z"]) if c["z"] else None)
    raw = first(d["delta"]) + d["dbias"]
    dt = torch.nn.functional.softplus(raw, threshold=40.0)
    Bm, Cm = wide(d["B"]), wide(d["C"])
    groups = lambda m: m.view(L, B, G, D // G, -1)
    a = torch.exp(dt[..., None] * d["A"])                                   # (L, B, D, N)
    h = (groups(dt * x) * Bm[:, :, :, None]).view(L, B, D, N)
    h0 = d["h0"] if c["state"] else torch.zeros(B, D, N, dtype=torch.float64, device=x.device)
    prev = h0
    for t in range(L):
        prev = h[t].addcmul_(a[t], prev)
    y = (groups(h) * Cm[:, :, :, None]).sum(-1).view(L, B, D) + d["Dskip"] * x
    back = lambda m: m.permute(1, 2, 0)
    out = {"end": h[-1].clone()} if c["state"] else {}
    gate = torch.nn.functional.silu(z) if c["z"] else 1.0
    out["y"] = back(y * gate)
    if not c["grad"]:
        return out
    dy = first(d["dy"])
    if c["z"]:
        q = torch.sigmoid(z)
        out["dz"] = back(dy * y * (q + z * q * (1 - q)))
        dy = dy * gate
    out["dC"] = (groups(h) * groups(dy)).sum(3).permute(1, 2, 3, 0)
    g = (groups(dy) * Cm[:, :, :, None]).view(L, B, D, N)
    if c["state"]:
        g[-1] += d["dlast"]
    for t in range(L - 2, -1, -1):
        g[t].addcmul_(a[t + 1], g[t + 1])
    out["dB"] = (groups(g) * groups(dt * x)).sum(3).permute(1, 2, 3, 0)
    gB = (groups(g) * Bm[:, :, :, None]).sum(-1).view(L, B, D)
    g *= a
    if c["state"]:
        out["dh0"] = g[0].clone()
    g[1:] *= h[:-1]
    g[0] *= h0
    out["dA"] = (g * dt[..., None]).sum((0, 1))
    ddelta = (gB * x + (g * d["A"]).sum(-1)) * torch.sigmoid(raw)
    out.update({"dx": back(gB * dt + d["Dskip"] * dy), "ddelta": back(ddelta), "ddbias": ddelta.sum((0, 1)), "dDskip": (dy * x).sum((0, 1))})
    return out


def _exact_step(c, d):
    F = torch.nn.functional
    full = torch.cat([d["conv_state"], d["x"][..., None]], 2)
    xc = F.silu(torch.einsum("bdw,dw->bd", full, d["w"]) + d["b"])
    xc = xc.to(TYPES[c["dtype"]]).double()                                  # the convolution hands over the input's type
    dt = F.softplus(d["delta"] + d["dbias"], threshold=40.0)
    group = torch.arange(c["D"], device=xc.device) // (c["D"] // c["G"])
    h = d["h0"] * torch.exp(dt[..., None] * d["A"]) + (dt * xc)[..., None] * d["B"][:, group]
    y = (torch.einsum("bdn,bdn->bd", h, d["C"][:, group]) + d["Dskip"] * xc) * F.silu(d["z"])
    return {"y": y, "conv_end": full[:, :, 1:], "end": h}


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    op, grad = case["op"], case.get("grad", False)
    if op == "norm":
        n, C = case["rows"] * case["C"], case["C"]
        return {"bytes": n * size * (5 if grad else 2) + C * 4 * (4 if grad else 2), "flops": n * (22 if grad else 8)}
    if op == "conv":
        n, D, W = case["B"] * case["D"] * case["L"], case["D"], case["W"]
        ends = case["B"] * D * (W - 1) * size if case["state"] else 0
        return {"bytes": n * size * (5 if grad else 2) + D * (W + 1) * 4 * (2 if grad else 1) + ends * (3 if grad else 2),
                "flops": n * ((8 * W + 14) if grad else (2 * W + 5))}
    B, D, G, N = case["B"], case["D"], case["G"], case["N"]
    if op == "step":
        W = case["W"]
        return {"bytes": B * D * (4 * size + 2 * 4 * N + 2 * (W - 1) * size) + 2 * B * G * N * size + D * (N + W + 3) * 4,
                "flops": B * D * (7 * N + 2 * W + 20)}
    L = case["L"]
    n, bc, st = B * D * L, 2 * B * G * N * L, (B * D * N * 4 if case["state"] else 0)
    if not grad:
        return {"bytes": n * size * (4 if case["z"] else 3) + bc * size + 2 * st + D * (N + 2) * 4, "flops": n * (7 * N + 12)}
    return {"bytes": n * size * (8 if case["z"] else 6) + bc * size * 2 + 4 * st + D * (N + 2) * 8, "flops": n * (23 * N + 40)}
