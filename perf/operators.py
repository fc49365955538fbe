"""The norm, gate and checkpoint operators at work: what is timed, on which inputs, and what the results have to be.

A residual block of a model is  h = norm(x),  y = block(h),  out = alpha*x + scale*act(gate)*norm(y).  The cases below
are the row passes around such a block (both directions), the 8-bit checkpoint of an activation and the weight gradient
that reads it.  `run` computes them in elementary torch operations, or, with `own`, by the calls a user makes of
this package; `exact` is the same in 64 bits, written from the formulas.
"""
import functools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
ALPHA = 0.75
BLOCK = 128  # columns that share one scale in a checkpoint


# ---- the cases ----------------------------------------------------------------------------------------------
def _norm(name, T, D, dtype, kind, checkpoint, residual=False):
    return {"name": name, "op": name.split(":")[0], "T": T, "D": D, "dtype": dtype, "kind": kind, "checkpoint": checkpoint,
            "residual": residual}


def _gated(name, T, D, dtype, kind, gate, act, G, next_norm):
    return {"name": name, "op": name.split(":")[0], "T": T, "D": D, "dtype": dtype, "kind": kind, "gate": gate, "act": act, "G": G,
            "next": next_norm}


def listed():
    return [
        # one new token of a decoder: nothing but latency
        _norm("norm_fwd:token", 1, 4096, "bf16", "rms", False),
        # the norm before a block in a training step, its input kept in 8 bits for the backward pass
        _norm("norm_fwd:train", 8192, 4096, "bf16", "rms", True),
        # its backward pass from that checkpoint, the residual path's gradient added on the way
        _norm("norm_bwd:train", 8192, 4096, "bf16", "rms", True, residual=True),
        # a layer norm in full precision at ragged sizes (a small model, a packed batch)
        _norm("norm_bwd:ragged", 1023, 1000, "f32", "layer", False),
        # a few decoding streams: norm, gate and residual after one block and the norm before the next
        _gated("gated_fwd:decode", 16, 8192, "bf16", "rms", "token", "sigmoid", 1, True),
        # the same in training, 16 sequences of 1024 tokens, one gate row per sequence
        _gated("gated_fwd:train", 16384, 4096, "f16", "layer", "group", "none", 1024, True),
        # the backward pass of the widest rows, a gate value for every element
        _gated("gated_bwd:train", 8192, 8192, "bf16", "rms", "token", "sigmoid", 1, True),
        # the backward pass where one gate row serves a sequence: its gradient is a sum over the sequence
        _gated("gated_bwd:sequences", 4096, 1024, "f16", "layer", "group", "tanh", 512, True),
        # a short sequence's activations into 8 bits, at a width that ends inside a block
        {"name": "pack:ragged", "op": "pack", "T": 257, "D": 1000, "dtype": "f16"},
        # a training step's
        {"name": "pack:train", "op": "pack", "T": 16384, "D": 8192, "dtype": "bf16"},
        # the weight gradient of a small layer over a short ragged batch
        {"name": "weight_grad:small", "op": "weight_grad", "T": 300, "D": 1024, "N": 1024, "dtype": "f16"},
        # of the largest layer
        {"name": "weight_grad:train", "op": "weight_grad", "T": 8192, "D": 8192, "N": 8192, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "gated_fwd", "gated_bwd", "pack", "weight_grad"])
    if op == "weight_grad":
        while True:
            c = {"op": op, "T": _log(rng, 1, 16384), "D": 16 * _log(rng, 4, 512), "N": 8 * _log(rng, 8, 1024),
                 "dtype": rng.choice(["f16", "bf16"])}
            if c["T"] * c["D"] * c["N"] <= 1 << 38:
                return c
    while True:
        T, D = _log(rng, 1, 16384), _log(rng, 64, 8192)
        if T * D <= 1 << 25:
            break
    if rng.random() < 0.6:
        D = max(64, D // 64 * 64)  # most models' widths are round
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "pack":
        return {"op": op, "T": T, "D": D, "dtype": dtype}
    kind = rng.choice(["rms", "layer"])
    if op.startswith("norm"):
        return {"op": op, "T": T, "D": D, "dtype": dtype, "kind": kind, "checkpoint": rng.random() < 0.5,
                "residual": op == "norm_bwd" and rng.random() < 0.5}
    gate = rng.choice(["none", "token", "group"])
    G = _log(rng, 2, max(2, T)) if gate == "group" else 1
    return {"op": op, "T": T, "D": D, "dtype": dtype, "kind": kind, "gate": gate, "act": rng.choice(["none", "sigmoid", "tanh"]),
            "G": G, "next": rng.random() < 0.6}


# ---- the inputs ---------------------------------------------------------------------------------------------
def _codes(x, dtype):
    """The checkpoint of x (32 bits): e4m3 codes, and the biased exponent of the power of two that each block of 128
    columns is divided by.  The smallest power that brings the block's largest finite magnitude to 448 or less, kept
    inside the type's range; what is not finite becomes NaN."""
    T, D = x.shape
    pad = -D % BLOCK
    v = torch.nn.functional.pad(x, (0, pad)).view(T, -1, BLOCK)
    finite = torch.isfinite(v)
    top = torch.where(finite, v.abs(), torch.zeros((), device=x.device)).amax(2).view(torch.int32)
    e = (top >> 23) - 8 + ((top & 0x7FFFFF) > 0x600000).to(torch.int32)
    lo, hi = (112, 135) if dtype == "f16" else (3, 247)
    e = e.clamp(lo, hi)
    inverse = ((254 - e) << 23).view(torch.float32)[..., None]
    most = torch.where(e == hi, 240.0, 448.0)[..., None]
    q = (v * inverse).clamp(-most, most)
    q = torch.where(finite, q, torch.full((), float("nan"), device=x.device))
    q = q.to(torch.float8_e4m3fn).view(torch.uint8).view(T, -1)[:, :D].contiguous()
    return q, e.to(torch.uint8)


def _values(codes, exps):
    """What a checkpoint stands for, in 32 bits (exact: a power of two times four bits)."""
    scale = (exps.to(torch.int32) << 23).view(torch.float32).repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.view(torch.float8_e4m3fn).float() * scale


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    T, D = c["T"], c["D"]

    def randn(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device=dev) * std + mean

    def stream(std=1.0):
        """A residual stream or a block's output: some channels far larger than the others, a little offset."""
        x = randn(T, D, std=std)
        x *= torch.exp(randn(D, std=0.5))
        return x.add_(0.1 * std).to(dt)

    s = {"case": dict(c)}
    if c["op"] == "pack":
        s["x"] = stream()
    elif c["op"] == "weight_grad":
        s["codes"], s["exps"] = _codes(stream().float(), c["dtype"])
        s["dy"] = randn(T, c["N"], std=0.02).to(dt)
    elif c["op"].startswith("norm"):
        s["weight"] = randn(D, std=0.1, mean=1.0).to(dt)
        s["bias"] = randn(D, std=0.1).to(dt)
        x = stream()
        if c["op"] == "norm_bwd":
            if c["checkpoint"]:
                s["codes"], s["exps"] = _codes(x.float(), c["dtype"])
            else:
                s["x"] = x
            s["mean"], s["rstd"] = _statistics(x.float(), c["kind"])
            s["dh"] = randn(T, D, std=0.1).to(dt)
            if c["residual"]:
                s["dres"] = randn(T, D, std=0.1).to(dt)
        else:
            s["x"] = x
    else:
        B = -(-T // c["G"])
        s["x"], s["y"] = stream(), stream(0.5)
        s["weight"], s["bias"] = randn(D, std=0.1, mean=1.0).to(dt), randn(D, std=0.1).to(dt)
        s["scale"] = randn(D, std=0.1, mean=0.5).to(dt)
        if c["gate"] != "none":
            s["gate"] = randn(T if c["gate"] == "token" else B, D).to(dt)
        s["next_weight"], s["next_bias"] = randn(D, std=0.1, mean=1.0).to(dt), randn(D, std=0.1).to(dt)
        if c["op"] == "gated_bwd":
            s["mean"], s["rstd"] = _statistics(s["y"].float(), c["kind"])
            s["dout"] = randn(T, D, std=0.1).to(dt)
            if c["next"]:
                s["out"] = s.pop("x")  # the stream after the block, kept by the forward pass
                s["next_mean"], s["next_rstd"] = _statistics(s["out"].float(), c["kind"])
                s["dh"] = randn(T, D, std=0.1).to(dt)
            else:
                s.pop("x")
    if own:
        s["call"] = _bind(s)
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------
def _statistics(x, kind):
    mean = x.mean(1) if kind == "layer" else torch.zeros_like(x[:, 0])
    rstd = 1.0 / torch.sqrt((x - mean[:, None]).square().mean(1) + EPS)
    return mean, rstd


def _act(g, act):
    """The gate's activation and its derivative."""
    if act == "sigmoid":
        a = 1.0 / (1.0 + torch.exp(-g))
        return a, a * (1.0 - a)
    if act == "tanh":
        a = torch.tanh(g)
        return a, 1.0 - a * a
    return g, torch.ones_like(g)


def _norm_backward(dn, n, rstd, kind):
    """Through n = (x - mean) * rstd to x."""
    d = dn - n * (dn * n).mean(1, keepdim=True)
    if kind == "layer":
        d = d - dn.mean(1, keepdim=True)
    return d * rstd[:, None]


def _affine(n, s, kind, prefix=""):
    u = n * s[prefix + "weight"].float()
    return u + s[prefix + "bias"].float() if kind == "layer" else u


def _plain_norm_fwd(s, c, dt):
    x = s["x"].float()
    mean, rstd = _statistics(x, c["kind"])
    out = {"h": _affine((x - mean[:, None]) * rstd[:, None], s, c["kind"]).to(dt), "rstd": rstd}
    if c["kind"] == "layer":
        out["mean"] = mean
    if c["checkpoint"]:
        codes, out["exps"] = _codes(x, c["dtype"])
        out["codes"] = codes.view(torch.float8_e4m3fn)
    return out


def _plain_norm_bwd(s, c, dt):
    x = _values(s["codes"], s["exps"]) if c["checkpoint"] else s["x"].float()
    n = (x - s["mean"][:, None]) * s["rstd"][:, None]
    dh = s["dh"].float()
    dx = _norm_backward(dh * s["weight"].float(), n, s["rstd"], c["kind"])
    if c["residual"]:
        dx = dx + s["dres"].float()
    out = {"dx": dx.to(dt), "dweight": (dh * n).sum(0)}
    if c["kind"] == "layer":
        out["dbias"] = dh.sum(0)
    return out


def _gate_rows(s, c):
    """The gate of every row, its derivative, both [T, D] (or [1, D] of ones)."""
    if c["gate"] == "none":
        one = torch.ones(1, c["D"], device=s["weight"].device)
        return one, one
    a, da = _act(s["gate"].float(), c["act"])
    if c["gate"] == "group":
        a, da = (v.repeat_interleave(c["G"], 0)[:c["T"]] for v in (a, da))
    return a, da


def _plain_gated_fwd(s, c, dt):
    mean, rstd = _statistics(s["y"].float(), c["kind"])
    u = _affine((s["y"].float() - mean[:, None]) * rstd[:, None], s, c["kind"])
    a, _ = _gate_rows(s, c)
    z = (ALPHA * s["x"].float() + s["scale"].float() * a * u).to(dt)
    out = {"out": z, "rstd": rstd}
    if c["kind"] == "layer":
        out["mean"] = mean
    if c["next"]:  # reads the stream as it was stored
        mean, rstd = _statistics(z.float(), c["kind"])
        out["h"] = _affine((z.float() - mean[:, None]) * rstd[:, None], s, c["kind"], "next_").to(dt)
        out["next_rstd"] = rstd
        if c["kind"] == "layer":
            out["next_mean"] = mean
    return out


def _plain_gated_bwd(s, c, dt):
    out = {}
    dz = s["dout"].float()
    if c["next"]:
        n2 = (s["out"].float() - s["next_mean"][:, None]) * s["next_rstd"][:, None]
        dh = s["dh"].float()
        dz = dz + _norm_backward(dh * s["next_weight"].float(), n2, s["next_rstd"], c["kind"])
        out["dnext_weight"] = (dh * n2).sum(0)
        if c["kind"] == "layer":
            out["dnext_bias"] = dh.sum(0)
    out["dx"] = (ALPHA * dz).to(dt)
    n = (s["y"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    w, scale = s["weight"].float(), s["scale"].float()
    u = _affine(n, s, c["kind"])
    a, da = _gate_rows(s, c)
    du = dz * scale * a
    out["dy"] = _norm_backward(du * w, n, s["rstd"], c["kind"]).to(dt)
    out["dweight"] = (du * n).sum(0)
    if c["kind"] == "layer":
        out["dbias"] = du.sum(0)
    out["dscale"] = (dz * a * u).sum(0)
    if c["gate"] != "none":
        dg = dz * scale * u * da
        if c["gate"] == "group":
            dg = torch.nn.functional.pad(dg, (0, 0, 0, -c["T"] % c["G"])).view(-1, c["G"], c["D"]).sum(1)
            out["dgate"] = dg
        else:
            out["dgate"] = dg.to(dt)
    return out


def _plain_pack(s, c, dt):
    codes, exps = _codes(s["x"].float(), c["dtype"])
    return {"codes": codes.view(torch.float8_e4m3fn), "exps": exps}


def _plain_weight_grad(s, c, dt):
    return {"dweight": (_values(s["codes"], s["exps"]).t() @ s["dy"].float()).to(dt)}


_PLAIN = {"norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd, "gated_fwd": _plain_gated_fwd, "gated_bwd": _plain_gated_bwd,
          "pack": _plain_pack, "weight_grad": _plain_weight_grad}


# ---- the package's own --------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _runtime():
    from ascend_mlir_b200.runtime import CudaRuntime
    rt = CudaRuntime()
    rt.set_device(torch.cuda.current_device())
    return rt


@functools.lru_cache(maxsize=None)
def _plan(items):
    """The kernel of a case and its packed sizes, kept as a program keeps them."""
    from ascend_mlir_b200 import descriptors
    c = dict(items)
    op, dtype = c["op"], c["dtype"]
    sizes = {"T": c["T"], "D": c["D"]}
    if op == "norm_fwd":
        spec = descriptors.block_norm(dtype, kind=c["kind"], eps=EPS, checkpoint=c["checkpoint"])
    elif op == "norm_bwd":
        spec = descriptors.block_norm_grad(dtype, kind=c["kind"], checkpoint=c["checkpoint"], residual_grad=c["residual"])
    elif op == "gated_fwd":
        spec = descriptors.gated_residual(dtype, kind=c["kind"], eps=EPS, alpha=ALPHA, gate=c["gate"], gate_act=c["act"], next_norm=c["next"])
    elif op == "gated_bwd":
        spec = descriptors.gated_residual_grad(dtype, kind=c["kind"], alpha=ALPHA, gate=c["gate"], gate_act=c["act"], next_norm=c["next"])
    elif op == "pack":
        spec = descriptors.checkpoint_pack(dtype)
    else:
        spec = descriptors.checkpoint_weight_grad(dtype)
        sizes["N"] = c["N"]
    if c.get("gate") == "group":
        sizes["G"], sizes["B"] = c["G"], -(-c["T"] // c["G"])
    tiling = spec.pack(sizes)
    return spec, tiling, _runtime().workspace_bytes(spec.binary, tiling)


def _bind(s):
    """The arguments of a case's launch, in the kernel's order, with buffers for what it returns."""
    c = s["case"]
    op, T, D, dt = c["op"], c["T"], c["D"], DTYPES[c["dtype"]]
    dev = torch.device("cuda")
    layer = c.get("kind") == "layer"
    f32, u8 = torch.float32, torch.uint8

    def new(shape, dtype):
        return torch.empty(shape, dtype=dtype, device=dev)

    packed = [("codes", new((T, D), u8)), ("exps", new((T, -(-D // BLOCK)), u8))]
    if op == "norm_fwd":
        ins = ["x", "weight"] + ["bias"] * layer
        outs = [("h", new((T, D), dt)), ("rstd", new(T, f32))] + [("mean", new(T, f32))] * layer + packed * c["checkpoint"]
    elif op == "norm_bwd":
        ins = ["dh"] + (["codes", "exps"] if c["checkpoint"] else ["x"]) + ["weight", "rstd"] + ["mean"] * layer + ["dres"] * c["residual"]
        outs = [("dx", new((T, D), dt)), ("dweight", new(D, f32))] + [("dbias", new(D, f32))] * layer
    elif op == "gated_fwd":
        ins = (["x", "y", "weight"] + ["bias"] * layer + ["gate"] * (c["gate"] != "none") + ["scale"] +
               (["next_weight"] + ["next_bias"] * layer) * c["next"])
        outs = [("out", new((T, D), dt)), ("rstd", new(T, f32))] + [("mean", new(T, f32))] * layer
        if c["next"]:
            outs += [("h", new((T, D), dt)), ("next_rstd", new(T, f32))] + [("next_mean", new(T, f32))] * layer
    elif op == "gated_bwd":
        ins = (["dout", "y", "weight"] + ["bias"] * layer + ["gate"] * (c["gate"] != "none") + ["scale", "rstd"] + ["mean"] * layer +
               (["dh", "out", "next_weight", "next_rstd"] + ["next_mean"] * layer) * c["next"])
        outs = [("dx", new((T, D), dt)), ("dy", new((T, D), dt)), ("dweight", new(D, f32))] + [("dbias", new(D, f32))] * layer
        if c["gate"] != "none":
            outs += [("dgate", new((T, D), dt) if c["gate"] == "token" else new((-(-T // c["G"]), D), f32))]
        outs += [("dscale", new(D, f32))]
        if c["next"]:
            outs += [("dnext_weight", new(D, f32))] + [("dnext_bias", new(D, f32))] * layer
    elif op == "pack":
        ins, outs = ["x"], packed
    else:
        ins, outs = ["codes", "exps", "dy"], [("dweight", new((D, c["N"]), dt))]
    spec, tiling, ws_bytes = _plan(tuple(sorted((k, v) for k, v in c.items() if k != "name")))
    ws = new(ws_bytes, u8)
    results = {k: t.view(torch.float8_e4m3fn) if k == "codes" else t for k, t in outs}
    return {"spec": spec, "tiling": tiling, "workspace": ws, "results": results,
            "inputs": [(s[k].data_ptr(), s[k].nbytes) for k in ins], "outputs": [(t.data_ptr(), t.nbytes) for _, t in outs]}


def _own_run(s):
    b = s["call"]
    spec, ws = b["spec"], b["workspace"]
    _runtime().launch_device(spec.binary, spec.name, b["inputs"], b["outputs"], b["tiling"], 0, spec.magic, (ws.data_ptr(), ws.numel()),
                             torch.cuda.current_stream().cuda_stream)
    return b["results"]


def run(state):
    if own:
        return _own_run(state)
    c = state["case"]
    return _PLAIN[c["op"]](state, c, DTYPES[c["dtype"]])


# ---- work ---------------------------------------------------------------------------------------------------
def work(case):
    """Each input read once and each output written once."""
    c = case
    T, D = c["T"], c["D"]
    e = 4 if c["dtype"] == "f32" else 2
    full, packed, row = T * D * e, T * D + T * -(-D // BLOCK), T * 4
    layer = c.get("kind") == "layer"
    if c["op"] == "pack":
        return {"bytes": full + packed, "flops": 3 * T * D}
    if c["op"] == "weight_grad":
        return {"bytes": packed + T * c["N"] * e + D * c["N"] * e, "flops": 2 * T * D * c["N"]}
    affine, stats = D * e * (1 + layer), row * (1 + layer)
    if c["op"] == "norm_fwd":
        return {"bytes": 2 * full + affine + stats + packed * c["checkpoint"], "flops": 6 * T * D}
    sums = 4 * D * (1 + layer)
    if c["op"] == "norm_bwd":
        source = packed if c["checkpoint"] else full
        return {"bytes": 2 * full + source + full * c["residual"] + D * e + stats + sums, "flops": 12 * T * D}
    gate = {"none": 0, "token": full, "group": -(-T // c["G"]) * D * e}[c["gate"]]
    if c["op"] == "gated_fwd":
        return {"bytes": 3 * full + affine + gate + D * e + stats + (full + affine + stats) * c["next"], "flops": (12 + 6 * c["next"]) * T * D}
    dgate = {"none": 0, "token": full, "group": -(-T // c["G"]) * D * 4}[c["gate"]]
    return {"bytes": 4 * full + affine + gate + dgate + D * e + stats + sums + 4 * D + (2 * full + D * e + stats + sums) * c["next"],
            "flops": (24 + 12 * c["next"]) * T * D}


# ---- 64 bits ------------------------------------------------------------------------------------------------
def _moments64(v, kind):
    m = v.sum(1) / v.shape[1] if kind == "layer" else v.new_zeros(v.shape[0])
    var = ((v - m.unsqueeze(1)) ** 2).sum(1) / v.shape[1]
    return m, (var + EPS) ** -0.5


def _restore64(codes, exps):
    """Codes to values from the bits: sign, four exponent bits (bias 7), three mantissa bits."""
    k = codes.long()
    sign, expo, mant = 1.0 - 2.0 * (k >> 7).double(), (k >> 3) & 15, (k & 7).double()
    mag = torch.where(expo == 0, mant * 2.0 ** -9, (8.0 + mant) * torch.exp2((expo - 10).double()))
    mag = torch.where((k & 127) == 127, torch.full_like(mag, float("nan")), mag)
    power = torch.exp2(exps.double() - 127.0)
    col = torch.arange(codes.shape[1], device=codes.device) // BLOCK
    return sign * mag * power[:, col]


def _grid64(x, dtype):
    """Checkpoint values and exponents by a search over the powers of two and rounding to the grid, ties to even."""
    T, D = x.shape
    lo, hi = (112, 135) if dtype == "f16" else (3, 247)
    nb = -(-D // BLOCK)
    v = x.double()
    exps = torch.empty(T, nb, dtype=torch.uint8, device=x.device)
    q = torch.empty(T, D, dtype=torch.float64, device=x.device)
    for b in range(nb):
        w = v[:, b * BLOCK:(b + 1) * BLOCK]
        top = torch.where(torch.isfinite(w), w.abs(), torch.zeros_like(w)).amax(1)
        e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0))
        e = torch.where(448.0 * torch.exp2(e - 1) >= top, e - 1, e)  # the logarithm may land one off
        e = torch.where(448.0 * torch.exp2(e) < top, e + 1, e).clamp(lo - 127, hi - 127)
        most = torch.where(e == hi - 127, 240.0, 448.0).double().unsqueeze(1)
        r = w / torch.exp2(e).unsqueeze(1)
        step = torch.exp2(torch.floor(torch.log2(r.abs().clamp_min(2.0 ** -6))) - 3)
        r = torch.minimum(torch.maximum(torch.round(r / step) * step, -most), most)
        q[:, b * BLOCK:(b + 1) * BLOCK] = torch.where(torch.isfinite(w), r, torch.full_like(r, float("nan")))
        exps[:, b] = (e + 127).to(torch.uint8)
    return q, exps


def exact(case, seed):
    c = case
    global own
    mine, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = mine
    kind, T, D = c.get("kind"), c["T"], c["D"]
    layer = kind == "layer"
    if c["op"] == "pack":
        q, exps = _grid64(s["x"], c["dtype"])
        return {"codes": q, "exps": exps}
    if c["op"] == "weight_grad":
        return {"dweight": _restore64(s["codes"], s["exps"]).T @ s["dy"].double()}
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v) and v.dtype != torch.uint8}
    col = lambda v: v.unsqueeze(1)  # noqa: E731

    def through_norm(g, n, r):
        """Gradient of sum(g * n) by the rows' entries: the part along n (and the constant part) drops out."""
        back = g - n * col((g * n).sum(1) / D)
        return col(r) * (back - col(g.sum(1) / D) if layer else back)

    if c["op"] == "norm_fwd":
        m, r = _moments64(d["x"], kind)
        h = (d["x"] - col(m)) * col(r) * d["weight"] + (d["bias"] if layer else 0.0)
        out = {"h": h, "rstd": r}
        if layer:
            out["mean"] = m
        if c["checkpoint"]:
            out["codes"], out["exps"] = _grid64(s["x"], c["dtype"])
        return out
    if c["op"] == "norm_bwd":
        x = _restore64(s["codes"], s["exps"]) if c["checkpoint"] else d["x"]
        n = (x - col(d["mean"])) * col(d["rstd"])
        dx = through_norm(d["dh"] * d["weight"], n, d["rstd"]) + (d["dres"] if c["residual"] else 0.0)
        out = {"dx": dx, "dweight": torch.einsum("td,td->d", d["dh"], n)}
        if layer:
            out["dbias"] = d["dh"].sum(0)
        return out
    row = torch.arange(T, device=s["y"].device) // c["G"]
    if c["gate"] == "none":
        a = slope = torch.ones(1, D, dtype=torch.float64, device=s["y"].device)
    else:
        g = d["gate"][row]
        a = {"none": lambda: g, "sigmoid": lambda: torch.sigmoid(g), "tanh": lambda: torch.tanh(g)}[c["act"]]()
        slope = {"none": lambda: torch.ones_like(g), "sigmoid": lambda: a - a ** 2, "tanh": lambda: 1 - a ** 2}[c["act"]]()
    bias = d["bias"] if layer else 0.0
    if c["op"] == "gated_fwd":
        m, r = _moments64(d["y"], kind)
        z = ALPHA * d["x"] + d["scale"] * a * ((d["y"] - col(m)) * col(r) * d["weight"] + bias)
        out = {"out": z, "rstd": r}
        if layer:
            out["mean"] = m
        if c["next"]:
            z = z.to(DTYPES[c["dtype"]]).double()  # the next norm reads the stream as stored
            m, r = _moments64(z, kind)
            out["h"] = (z - col(m)) * col(r) * d["next_weight"] + (d["next_bias"] if layer else 0.0)
            out["next_rstd"] = r
            if layer:
                out["next_mean"] = m
        return out
    out, dz = {}, d["dout"]
    if c["next"]:
        n2 = (d["out"] - col(d["next_mean"])) * col(d["next_rstd"])
        dz = dz + through_norm(d["dh"] * d["next_weight"], n2, d["next_rstd"])
        out["dnext_weight"] = torch.einsum("td,td->d", d["dh"], n2)
        if layer:
            out["dnext_bias"] = d["dh"].sum(0)
    out["dx"] = ALPHA * dz
    n = (d["y"] - col(d["mean"])) * col(d["rstd"])
    out["dy"] = through_norm(dz * d["scale"] * a * d["weight"], n, d["rstd"])
    out["dweight"] = (dz * a * n).sum(0) * d["scale"]
    if layer:
        out["dbias"] = (dz * a).sum(0) * d["scale"]
    u = n * d["weight"] + bias
    out["dscale"] = (dz * a * u).sum(0)
    if c["gate"] == "token":
        out["dgate"] = dz * d["scale"] * u * slope
    elif c["gate"] == "group":
        out["dgate"] = torch.zeros_like(d["gate"]).index_add_(0, row, dz * d["scale"] * u * slope)
    return out
