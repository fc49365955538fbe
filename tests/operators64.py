"""The operator kernels' formulas in 64 bits, each value with a bound on how far a 32-bit evaluation may be from it.

u = 2^-24 is the half step of f32.  A sum of n terms that are added 32 in a row per thread and then in a tree is off by
at most SUM*u*sum|terms| with SUM = 32 + log2(512) + a few; a column sum over the rows by COLUMN*u*sum|terms|, COLUMN
the longest run of rows of one team plus the final adds at the tested sizes.  What is stored in a 16-bit type adds
half a step of that type relative to the value, and half its smallest subnormal."""
import torch

U = 2.0 ** -24
SUM = 48
COLUMN = 96
BLOCK = 128


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stored(value, error, dtype):
    """(value, bound) of a value with a 32-bit error that is stored in dtype."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return value, error + half_step(dtype) * (value.abs() + error) + tiny


def statistics(v, kind, eps):
    mean = v.mean(1) if kind == "layer" else torch.zeros_like(v[:, 0])
    rstd = 1.0 / torch.sqrt((v - mean[:, None]).square().mean(1) + eps)
    return mean, rstd


def normed(v, kind, eps, w, b):
    """normed rows times weight plus bias, statistics, and their bounds."""
    mean, rstd = statistics(v, kind, eps)
    d_mean = (SUM + 2) * U * v.abs().mean(1) if kind == "layer" else torch.zeros_like(mean)
    # the variance: (SUM + 4)*u of itself, and d_mean^2 (its first-order part drops out with the sum of v - mean)
    d_rstd = rstd * ((SUM / 2 + 8) * U + 0.5 * (d_mean * rstd) ** 2 + d_mean * rstd * SUM * U)
    n = (v - mean[:, None]) * rstd[:, None]
    r = n * w + (b if b is not None else 0.0)
    err = w.abs() * (rstd * d_mean)[:, None] + (n * w).abs() * (d_rstd / rstd)[:, None] + 6 * U * ((n * w).abs() + r.abs())
    return r, err, (mean, d_mean + U * mean.abs()), (rstd, d_rstd)


def act(g, name):
    """(value, slope, bound of the value's relative error, bound of the slope's absolute error)"""
    if name == "sigmoid":
        a = torch.sigmoid(g)
        rel = 6 * U * (1 + g.abs())  # exp's argument error is nothing, its result 2 ulp; 1 + e and the division one each
        return a, a * (1 - a), rel, 2 * a * rel + 2 * U * a
    if name == "tanh":
        a = torch.tanh(g)
        return a, 1 - a * a, 4 * U + 0 * a, 10 * U + 0 * a
    return g, torch.ones_like(g), 0 * g, 0 * g


def gate_rows(t, c):
    if c["gate"] == "none":
        one = torch.ones(1, c["D"], dtype=torch.float64, device=t["weight"].device)
        return one, one, 0 * one, 0 * one
    g = t["gate"]
    if c["gate"] == "group":
        g = g[torch.arange(c["T"], device=g.device) // c["G"]]
    return act(g, c["act"])


def forward(t, c):
    """t: the inputs in 64 bits by name; c: T, D, dtype (torch), kind, eps, alpha, gate, act, G, next, op."""
    dt, kind = c["dtype"], c["kind"]
    out = {}
    layer = kind == "layer"
    if c["op"] == "norm":
        h, err, mean, rstd = normed(t["x"], kind, c["eps"], t["weight"], t.get("bias") if layer else None)
        out["h"] = stored(h, err, dt)
        out["rstd"] = rstd
        if layer:
            out["mean"] = mean
        return out
    u, err, mean, rstd = normed(t["y"], kind, c["eps"], t["weight"], t.get("bias") if layer else None)
    out["rstd"] = rstd
    if layer:
        out["mean"] = mean
    a, _, rel, _ = gate_rows(t, c)
    f = a * t["scale"] if "scale" in t else a
    z = c["alpha"] * t["x"] + f * u
    err = f.abs() * err + (rel + 4 * U) * (f * u).abs() + 2 * U * z.abs() + U * (c["alpha"] * t["x"]).abs()
    out["out"] = stored(z, err, dt)
    return out


def next_norm(z, t, c):
    """normB of the stream as it was stored (z: the kernel's own `out`)."""
    layer = c["kind"] == "layer"
    h, err, mean, rstd = normed(z, c["kind"], c["eps"], t["next_weight"], t.get("next_bias") if layer else None)
    out = {"h": stored(h, err, c["dtype"]), "next_rstd": rstd}
    if layer:
        out["next_mean"] = mean
    return out


def through(dn, e_dn, n, rstd, kind):
    """dv = rstd*(dn - n*avg(dn*n) - avg(dn)) with its bound; n is off by 3u of itself (the statistics are given), and where
    the mean does not vanish, by u of rstd*|v|: counted by the callers in e_n."""
    e_n = 4 * U * n.abs()
    along = (dn * n).mean(1, keepdim=True)
    e_along = (SUM * U * (dn * n).abs() + e_dn * n.abs() + dn.abs() * e_n).mean(1, keepdim=True)
    d = dn - n * along
    err = e_dn + n.abs() * e_along + e_n * along.abs() + 4 * U * (dn.abs() + (n * along).abs())
    if kind == "layer":
        const = dn.mean(1, keepdim=True)
        d = d - const
        err = err + (SUM * U * dn.abs() + e_dn).mean(1, keepdim=True) + U * const.abs()
    return d * rstd[:, None], (err + 2 * U * d.abs()) * rstd[:, None]


def column(terms, errors):
    return terms.sum(0), (errors + COLUMN * U * terms.abs()).sum(0) + 2.0 ** -149


def gradient(t, c):
    """t: dh, x / out (normB's source, already restored from a checkpoint), y, ..., the statistics as the kernel got them."""
    dt, kind, layer = c["dtype"], c["kind"], c["kind"] == "layer"
    out = {}
    pre, post = c["op"] == "norm" or c["next"], c["op"] != "norm"
    prefix = "next_" if post else ""
    zero = torch.zeros(c["T"], c["D"], dtype=torch.float64, device=t["weight"].device)
    dz, e_dz = t.get("dout", zero), zero
    if pre:
        src = t["out"] if post else t["x"]
        mean = t[prefix + "mean"] if layer else torch.zeros_like(t[prefix + "rstd"])
        rstd = t[prefix + "rstd"]
        n = (src - mean[:, None]) * rstd[:, None]
        dn = t["dh"] * t[prefix + "weight"]
        d, err = through(dn, 2 * U * dn.abs(), n, rstd, kind)
        dz = dz + d
        e_dz = err + 2 * U * dz.abs()
        out["d" + prefix + "weight"] = column(t["dh"] * n, 6 * U * (t["dh"] * n).abs())
        if layer:
            out["d" + prefix + "bias"] = column(t["dh"], 0 * t["dh"])
    if not post:
        out["dx"] = stored(dz, e_dz, dt)
        return out
    al = c["alpha"]
    out["dx"] = stored(al * dz, abs(al) * e_dz + 2 * U * (al * dz).abs(), dt)
    mean = t["mean"] if layer else torch.zeros_like(t["rstd"])
    n = (t["y"] - mean[:, None]) * t["rstd"][:, None]
    a, slope, rel, e_slope = gate_rows(t, c)
    s = t["scale"] if "scale" in t else torch.ones_like(t["weight"])
    w = t["weight"]
    b = t["bias"] if layer else torch.zeros_like(w)
    u = n * w + b
    e_u = 6 * U * ((n * w).abs() + b.abs())
    dn = dz * s * a * w
    e_dn = (s * a * w).abs() * e_dz + (rel + 6 * U) * dn.abs()
    d, err = through(dn, e_dn, n, t["rstd"], kind)
    out["dy"] = stored(d, err, dt)
    az, e_az = a * dz, a.abs() * e_dz + (rel + 3 * U) * (a * dz).abs()
    p, e_p = column(az * n, e_az * n.abs() + 8 * U * (az * n).abs())
    q, e_q = column(az, e_az)
    out["dweight"] = s * p, s.abs() * e_p + 4 * U * (s * p).abs()
    if layer:
        out["dbias"] = s * q, s.abs() * e_q + 4 * U * (s * q).abs()
    if "scale" in t:
        ds = w * p + b * q
        out["dscale"] = ds, w.abs() * e_p + b.abs() * e_q + 6 * U * ((w * p).abs() + (b * q).abs())
    if c["gate"] == "token":
        g = dz * s * u * slope
        e_g = (s * u * slope).abs() * e_dz + (dz * s * slope).abs() * e_u + (dz * s * u).abs() * e_slope + 8 * U * g.abs()
        out["dgate"] = stored(g, e_g, dt)
    elif c["gate"] == "group":
        groups = t["gate"].shape[0]
        row = torch.arange(c["T"], device=w.device) // c["G"]
        add = lambda v: torch.zeros(groups, c["D"], dtype=torch.float64, device=w.device).index_add_(0, row, v.expand(c["T"], -1))  # noqa: E731
        P, Q = add(dz * n), add(dz)
        e_P = add(e_dz * n.abs() + (COLUMN + 8) * U * (dz * n).abs())
        e_Q = add(e_dz + COLUMN * U * dz.abs())
        _, slope, _, e_slope = act(t["gate"], c["act"])
        inner, e_inner = w * P + b * Q, w.abs() * e_P + b.abs() * e_Q + 4 * U * ((w * P).abs() + (b * Q).abs())
        out["dgate"] = s * inner * slope, (s * slope).abs() * e_inner + (s * inner).abs() * e_slope + 8 * U * (s * inner * slope).abs()
    return out


def restore(codes, exps):
    """Values of a checkpoint from the bits of its codes."""
    k = codes.long()
    expo, mant = (k >> 3) & 15, (k & 7).double()
    mag = torch.where(expo == 0, mant * 2.0 ** -9, (8 + mant) * torch.exp2((expo - 10).double()))
    mag = torch.where((k & 127) == 127, torch.full_like(mag, float("nan")), mag)
    power = torch.exp2(exps.double() - 127)[:, torch.arange(codes.shape[1], device=codes.device) // BLOCK]
    return torch.where(k >= 128, -mag, mag) * power


def pack(x):
    """(values on the grid over the power, exponents) of a checkpoint of x, by search and rounding in 64 bits."""
    lo, hi = (-15, 8) if x.dtype == torch.float16 else (-124, 120)
    v = x.double()
    q = torch.empty_like(v)
    exps = torch.empty(x.shape[0], -(-x.shape[1] // BLOCK), dtype=torch.int64, device=x.device)
    for b in range(exps.shape[1]):
        w = v[:, b * BLOCK:(b + 1) * BLOCK]
        top = torch.where(torch.isfinite(w), w.abs(), torch.zeros_like(w)).amax(1)
        e = torch.full_like(exps[:, 0], lo)
        for k in range(lo, hi):  # one power up wherever the block does not fit yet
            e += (e == k) & (448.0 * 2.0 ** k < top)
        most = torch.where(e == hi, 240.0, 448.0).double()[:, None]
        r = w / torch.exp2(e.double())[:, None]
        step = torch.exp2(torch.floor(torch.log2(r.abs().clamp_min(2.0 ** -6))) - 3)
        r = torch.minimum(torch.maximum(torch.round(r / step) * step, -most), most)  # round: ties to even
        q[:, b * BLOCK:(b + 1) * BLOCK] = torch.where(torch.isfinite(w), r, torch.full_like(r, float("nan")))
        exps[:, b] = e + 127
    return q, exps
