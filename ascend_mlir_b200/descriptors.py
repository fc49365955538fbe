"""Launch descriptors and tiling spaces for the fused-group classes.

A launch descriptor is what the translate step emits for one fused kernel (the counterpart of the
reference's generated step8_kernel.cpp) and `tiling_space.json` keeps the reference's schema
(lib/Target/CannKernel/CannTranslation.cpp:1987-2042): {kernel, kernel_file, soc, block_dim_expr,
tiling_params:[{name, type, fixed, shape_key | values | min/max/step | value}]}.  TilingData is the
reference's all-int64 struct: tile parameters first, then dim_arg<N>_<D> for every dynamic dim
(lib/Conversion/AscendCPrepareForEmit/AscendCPrepareForEmitPass.cpp:200-216).

The builders below write the descriptors of the groups this repository benchmarks and of the
reference's six examples; any other fused elementwise / reduce / gather group is expressed with the
same vocabulary (domain, loads, store, body).
"""
from __future__ import annotations

import json
import struct
from dataclasses import dataclass, field
from typing import Dict, List, Optional

from .runtime.tiling_schema import TilingSchema

FORMAT = "afir-cuda-launch"
SOC = "sm_100a"


def op(name: str, a, b) -> dict:
    return {"op": name, "a": a, "b": b}


def container(descriptor: dict) -> bytes:
    """Seal a descriptor into the .bin container (what afirt_compiler_compile writes)."""
    text = json.dumps(descriptor, separators=(",", ":")).encode()
    return b"AFCU" + struct.pack("<II", 1, len(text)) + text


@dataclass
class KernelSpec:
    name: str
    descriptor: dict
    tiling_space: dict
    shape_keys: Dict[str, str] = field(default_factory=dict)  # tiling field -> shape key
    defaults: Dict[str, int] = field(default_factory=dict)    # tile-parameter defaults
    magic: int = 0x41415246
    derived: Dict[str, object] = field(default_factory=dict)  # shape key -> its value from the other keys

    def __post_init__(self):
        self.binary = container(self.descriptor)
        self.schema = TilingSchema.from_dict(self.tiling_space, self.name)

    def pack(self, shape: Dict[str, int], **tile_params: int) -> bytes:
        values = dict(self.defaults)
        values.update(tile_params)
        for fname, key in self.shape_keys.items():
            values[fname] = self.derived[key](shape) if key in self.derived and key not in shape else shape[key]
        return self.schema.pack(**values)

    def descriptor_json(self) -> str:
        return json.dumps(self.descriptor, indent=2)

    def tiling_space_json(self) -> str:
        return json.dumps(self.tiling_space, indent=2)


def _spec(name, kernel_class, dtype, num_inputs, num_outputs, tile_params, dims, body_fields, launch,
          block_dim_expr="0", magic=0x41415246) -> KernelSpec:
    """tile_params: [(name, default, values)], dims: [(field, shape_key)]."""
    tiling_names = [p[0] for p in tile_params] + [d[0] for d in dims]
    desc = {"format": FORMAT, "version": 1, "kernel": name, "kernel_class": kernel_class, "arch": SOC, "dtype": dtype,
            "num_inputs": num_inputs, "num_outputs": num_outputs,
            "tiling": [{"name": n, "type": "int64"} for n in tiling_names], "launch": launch}
    desc.update(body_fields)
    params = []
    for pname, default, values in tile_params:
        params.append({"name": pname, "type": "int64", "values": list(values), "default": default})
    for fname, key in dims:
        params.append({"name": fname, "type": "int64", "fixed": True, "shape_key": key})
    space = {"kernel": name, "kernel_file": f"{name}.cuda.json", "soc": SOC, "block_dim_expr": block_dim_expr,
             "tiling_params": params}
    return KernelSpec(name=name, descriptor=desc, tiling_space=space, shape_keys=dict(dims),
                      defaults={p[0]: p[1] for p in tile_params}, magic=magic)


_EW_TILE = [("CTA_THREADS", 128, (128, 256, 512)), ("UNROLL", 2, (1, 2, 4))]
_GATHER_TILE = [("CTA_THREADS", 128, (128, 256, 512)), ("UNROLL", 1, (1, 2, 4)), ("BULK_COPY", 0, (0, 1)),
                ("STREAM_STAGES", 0, (0, 2, 3, 4, 6)), ("STREAM_ROWS", 0, (0, 2, 4, 8, 16)),
                ("STREAM_WARPS", 0, (0, 4, 8, 16))]
_GATHER_LAUNCH = {"cta_threads": "CTA_THREADS", "unroll": "UNROLL", "bulk_copy": "BULK_COPY",
                  "stream_stages": "STREAM_STAGES", "stream_rows": "STREAM_ROWS",
                  "stream_warps": "STREAM_WARPS"}
_EW_LAUNCH = {"cta_threads": "CTA_THREADS", "unroll": "UNROLL"}


# ---- elementwise / broadcast / split / concat ------------------------------------------------------
def add_mul(dtype: str = "f32", name: str = "add_mul") -> KernelSpec:
    """out = (a + b) * b on [M, N] (afir.add then afir.mul)."""
    dims = [("dim_arg0_0", "M"), ("dim_arg0_1", "N")]
    shp = ["dim_arg0_0", "dim_arg0_1"]
    view = lambda arg: {"arg": arg, "shape": shp, "map": [0, 1]}  # noqa: E731
    body = {"domain": shp, "loads": [view(0), view(1)], "store": view(2),
            "body": [op("addf", "v0", "v1"), op("mulf", "%0", "v1")]}
    return _spec(name, "elementwise", dtype, 2, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def split_relu_bias_mul(bias_axis: int = 1, dtype: str = "f16", name: str = "split_relu_broadcast_add_mul") -> KernelSpec:
    """x[B,R,2C] split on the last axis into h0,h1; out[B,R,C] = (relu(h0) + bias) * h1.

    bias_axis 1: bias[R] follows the row (the reference example's row map); 2: bias[C] follows the column.
    """
    dims = [("dim_arg0_0", "B"), ("dim_arg0_1", "R"), ("dim_arg0_2", "C2"), ("dim_arg2_2", "C"), ("dim_arg1_0", "BIAS")]
    xshape = ["dim_arg0_0", "dim_arg0_1", "dim_arg0_2"]
    oshape = ["dim_arg0_0", "dim_arg0_1", "dim_arg2_2"]
    body = {"domain": oshape,
            "loads": [{"arg": 0, "shape": xshape, "map": [0, 1, 2], "offset": [0, 0, 0]},
                      {"arg": 1, "shape": ["dim_arg1_0"], "map": [bias_axis]},
                      {"arg": 0, "shape": xshape, "map": [0, 1, 2], "offset": [0, 0, "dim_arg2_2"]}],
            "store": {"arg": 2, "shape": oshape, "map": [0, 1, 2]},
            "body": [op("maximumf", "v0", 0.0), op("addf", "%0", "v1"), op("mulf", "%1", "v2")]}
    return _spec(name, "elementwise", dtype, 2, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def split_rows_relu_bias_scale(dtype: str = "f16", name: str = "ewop_broadcast_split") -> KernelSpec:
    """The reference example: rows of a[M,N] split in halves, out_h = (relu(a_h) + bias_h[m]) * scale_h[n],
    halves concatenated on axis 0 (two groups writing the two halves of one output, no copy)."""
    dims = [("dim_arg0_0", "M"), ("dim_arg0_1", "N"), ("dim_arg1_0", "HM"), ("dim_arg2_0", "HM"),
            ("dim_arg3_0", "N"), ("dim_arg4_0", "N")]
    ashape = ["dim_arg0_0", "dim_arg0_1"]
    dom = ["dim_arg1_0", "dim_arg0_1"]
    body_ops = [op("maximumf", "v0", 0.0), op("addf", "%0", "v1"), op("mulf", "%1", "v2")]

    def group(off, bias_arg, scale_arg, hm):
        return {"domain": dom,
                "loads": [{"arg": 0, "shape": ashape, "map": [0, 1], "offset": [off, 0]},
                          {"arg": bias_arg, "shape": [hm], "map": [0]},
                          {"arg": scale_arg, "shape": ["dim_arg0_1"], "map": [1]}],
                "store": {"arg": 5, "shape": ashape, "map": [0, 1], "offset": [off, 0]},
                "body": body_ops}

    body = {"groups": [group(0, 1, 3, "dim_arg1_0"), group("dim_arg1_0", 2, 4, "dim_arg2_0")]}
    return _spec(name, "elementwise", dtype, 5, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def add_mul_concat(dtype: str = "f16", name: str = "ewop_broadcast_concat") -> KernelSpec:
    """The reference example: out[2M,N] = concat(a[m] + b[m,n], c[m] * d[m,n], axis 0)."""
    dims = [("dim_arg0_0", "M"), ("dim_arg1_1", "N"), ("dim_arg4_0", "M2")]
    dom = ["dim_arg0_0", "dim_arg1_1"]
    oshape = ["dim_arg4_0", "dim_arg1_1"]

    def group(vec_arg, mat_arg, opname, off):
        return {"domain": dom,
                "loads": [{"arg": vec_arg, "shape": ["dim_arg0_0"], "map": [0]},
                          {"arg": mat_arg, "shape": dom, "map": [0, 1]}],
                "store": {"arg": 4, "shape": oshape, "map": [0, 1], "offset": [off, 0]},
                "body": [op(opname, "v0", "v1")]}

    body = {"groups": [group(0, 1, "addf", 0), group(2, 3, "mulf", "dim_arg0_0")]}
    return _spec(name, "elementwise", dtype, 4, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def relu_bcast_transpose_add(dtype: str = "f16", name: str = "relu_transpose_broadcast_add") -> KernelSpec:
    """The reference example: out[n,m] = relu(d0[m,0]) + d1[n,m]; d0 is read through the map (d0,d1)->(d1,0)."""
    dims = [("dim_arg0_0", "M"), ("dim_arg1_0", "N")]
    dom = ["dim_arg1_0", "dim_arg0_0"]
    body = {"domain": dom,
            "loads": [{"arg": 0, "shape": ["dim_arg0_0", 1], "map": [1, -1]},
                      {"arg": 1, "shape": dom, "map": [0, 1]}],
            "store": {"arg": 2, "shape": dom, "map": [0, 1]},
            "body": [op("maximumf", "v0", 0.0), op("addf", "%0", "v1")]}
    return _spec(name, "elementwise", dtype, 2, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def transposed_add_mul(dtype: str = "f16", name: str = "transposed_add_mul") -> KernelSpec:
    """out[n, m] = (a[m, n] + b[n, m]) * c[n]: `a` is read through a transposed view, `c` is constant along the
    inner dim.  Arguments: a [M, N], b [N, M], c [N] -> out [N, M]."""
    dims = [("dim_arg0_0", "M"), ("dim_arg0_1", "N")]
    dom = ["dim_arg0_1", "dim_arg0_0"]
    body = {"domain": dom,
            "loads": [{"arg": 0, "shape": ["dim_arg0_0", "dim_arg0_1"], "map": [1, 0]},
                      {"arg": 1, "shape": dom, "map": [0, 1]},
                      {"arg": 2, "shape": ["dim_arg0_1"], "map": [0]}],
            "store": {"arg": 3, "shape": dom, "map": [0, 1]},
            "body": [op("addf", "v0", "v1"), op("mulf", "%0", "v2")]}
    return _spec(name, "elementwise", dtype, 3, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def batched_transposed_relu_sub(dtype: str = "f32", name: str = "batched_transposed_relu_sub") -> KernelSpec:
    """out[b, n, m] = max(a[b, m, n], 0) - bias[m]: a batch of transposed reads with a row-vector operand.
    Arguments: a [B, M, N], bias [M] -> out [B, N, M]."""
    dims = [("dim_arg0_0", "B"), ("dim_arg0_1", "M"), ("dim_arg0_2", "N")]
    dom = ["dim_arg0_0", "dim_arg0_2", "dim_arg0_1"]
    body = {"domain": dom,
            "loads": [{"arg": 0, "shape": ["dim_arg0_0", "dim_arg0_1", "dim_arg0_2"], "map": [0, 2, 1]},
                      {"arg": 1, "shape": ["dim_arg0_1"], "map": [2]}],
            "store": {"arg": 2, "shape": dom, "map": [0, 1, 2]},
            "body": [op("maximumf", "v0", 0.0), op("subf", "%0", "v1")]}
    return _spec(name, "elementwise", dtype, 2, 1, _EW_TILE, dims, body, _EW_LAUNCH)


def transpose_2d(dtype: str = "f16", name: str = "transpose_2d") -> KernelSpec:
    """out[c, r] = in[r, c]."""
    dims = [("dim_arg0_0", "R"), ("dim_arg0_1", "C")]
    body = {"domain": ["dim_arg0_1", "dim_arg0_0"],
            "loads": [{"arg": 0, "shape": ["dim_arg0_0", "dim_arg0_1"], "map": [1, 0]}],
            "store": {"arg": 1, "shape": ["dim_arg0_1", "dim_arg0_0"], "map": [0, 1]}, "body": []}
    tile = [("WARP_ROWS", 0, (0, 1, 2, 4, 8)), ("CTAS_PER_SM", 0, (0, 4, 8, 16)), ("TILE_KERNEL", 0, (0, 1)),
            ("TILE_ORDER", 0, (0, 1, 2)), ("VARIANT", 0, (0, 1, 2, 3, 4))]
    return _spec(name, "transpose", dtype, 1, 1, tile, dims, body,
                 {"warp_rows": "WARP_ROWS", "ctas_per_sm": "CTAS_PER_SM", "tile_kernel": "TILE_KERNEL",
                  "tile_order": "TILE_ORDER", "variant": "VARIANT"})


# ---- broadcast + add + row reduction -----------------------------------------------------------------
def bcast_add_rowsum(dtype: str = "f32", name: str = "broadcast_add_reducesum") -> KernelSpec:
    """out[m] = sum_n (a[m] + b[m,n]) with f32 accumulation."""
    tile = [("CTA_THREADS", 0, (0, 128, 256, 512)), ("TEAM_LANES", 0, (0, 32, 64, 128, 256)), ("SPLIT_N", 0, (0,)),
            ("BULK_COPY", 1, (1, 0)), ("STREAM_STAGES", 0, (0, 4, 6, 8)), ("STREAM_CHUNK", 0, (0, 2048, 4096, 8192))]
    dims = [("dim_arg0_0", "M"), ("dim_arg1_1", "N")]
    dom = ["dim_arg0_0", "dim_arg1_1"]
    body = {"domain": dom,
            "loads": [{"arg": 0, "shape": ["dim_arg0_0"], "map": [0]}, {"arg": 1, "shape": dom, "map": [0, 1]}],
            "store": {"arg": 2, "shape": ["dim_arg0_0"], "map": [0]},
            "body": [op("addf", "v0", "v1")]}
    return _spec(name, "row_reduce", dtype, 2, 1, tile, dims, body, {"cta_threads": "CTA_THREADS", "team_lanes": "TEAM_LANES", "split_cols": "SPLIT_N", "bulk_copy": "BULK_COPY", "stream_stages": "STREAM_STAGES",
                  "stream_chunk_bytes": "STREAM_CHUNK"})


# ---- gather + elementwise --------------------------------------------------------------------------------
def gather_rows_scale_resid(dtype: str = "bf16", index_dtype: str = "i32", name: str = "gather_scale_resid") -> KernelSpec:
    """out[i,:] = table[idx[i],:] * scale + resid[i,:]."""
    dims = [("dim_arg0_0", "T"), ("dim_arg0_1", "W"), ("dim_arg1_0", "R")]
    dom = ["dim_arg1_0", "dim_arg0_1"]
    body = {"domain": dom,
            "loads": [{"arg": 0, "shape": ["dim_arg0_0", "dim_arg0_1"]},
                      {"arg": 2, "shape": ["dim_arg0_1"], "map": [1]},
                      {"arg": 3, "shape": dom, "map": [0, 1]}],
            "gather": {"axis": 0, "indices": {"arg": 1, "dtype": index_dtype, "shape": ["dim_arg1_0"]}},
            "store": {"arg": 4, "shape": dom, "map": [0, 1]},
            "body": [op("mulf", "v0", "v1"), op("addf", "%0", "v2")]}
    return _spec(name, "gather", dtype, 4, 1, _GATHER_TILE, dims, body, _GATHER_LAUNCH)


def relu_gather_cols_bias(dtype: str = "f16", index_dtype: str = "i64", name: str = "relu_index_select_add") -> KernelSpec:
    """The reference example: out[i,j] = relu(data[i, idx[j]]) + bias[j]."""
    dims = [("dim_arg0_0", "M"), ("dim_arg0_1", "N"), ("dim_arg1_0", "K")]
    dom = ["dim_arg0_0", "dim_arg1_0"]
    body = {"domain": dom,
            "loads": [{"arg": 0, "shape": ["dim_arg0_0", "dim_arg0_1"]}, {"arg": 2, "shape": ["dim_arg1_0"], "map": [1]}],
            "gather": {"axis": 1, "indices": {"arg": 1, "dtype": index_dtype, "shape": ["dim_arg1_0"]}},
            "store": {"arg": 3, "shape": dom, "map": [0, 1]},
            "body": [op("maximumf", "v0", 0.0), op("addf", "%0", "v1")]}
    return _spec(name, "gather", dtype, 3, 1, _GATHER_TILE, dims, body, _GATHER_LAUNCH)


# ---- matmul + bias + LeakyReLU -----------------------------------------------------------------------------
def matmul_bias_leakyrelu(in_dtype: str = "bf16", out_dtype: str = "bf16", bias_dtype: str = "bf16", alpha: float = 0.01,
                          epilogue: str = "BiasAddLeakyRelu", name: str = "matmul_add_leakyrelu",
                          transpose_b: bool = False) -> KernelSpec:
    """E = max(x, alpha*x), x = A[M,K].B[K,N] + bias[N].  Arguments (a, b, bias, out): `out` is the
    reference's init/result tensor (its initial contents are not read).  transpose_b: B is given as [N,K]
    (x = A.B^T, a torch Linear weight); the reference's ABI names the attribute (abi_matmul_trans_b) and always
    sets it false."""
    tile = [("STAGES", 0, (0,))]
    dims = [("dim_arg3_0", "M"), ("dim_arg3_1", "N"), ("dim_arg0_1", "K")]
    body = {"matmul": {"a": 0, "b": 1, "bias": 2, "out": 3, "in_dtype": in_dtype, "out_dtype": out_dtype,
                       "bias_dtype": bias_dtype, "epilogue": epilogue, "alpha": alpha,
                       "m": "dim_arg3_0", "n": "dim_arg3_1", "k": "dim_arg0_1"}}
    if transpose_b:
        body["matmul"]["transpose_b"] = True
    return _spec(name, "matmul", in_dtype, 3, 1, tile, dims, body, {"stages": "STAGES"})


# ---- row passes of a residual block, activation checkpoints --------------------------------------------------------
# No counterpart in the reference (it compiles inference groups).  Sizes: T rows (tokens), D columns, N output columns,
# G rows per gate row and B = ceil(T / G) gate rows.  A tensor named in `strided` is a slice of a wider one: its size
# keys are LD_<name> (row length) and OFF_<name> (first column), and its argument is the whole wide tensor.
CHECKPOINT_BLOCK = 128  # columns that share one power of two


class _Roles:
    """Collects the arguments of an operator kernel in order: inputs, then outputs."""

    def __init__(self, dtype: str, strided):
        self.dtype, self.strided = dtype, tuple(strided)
        self.inputs: List[tuple] = []
        self.outputs: List[tuple] = []
        self.dims: List[tuple] = []

    def _add(self, side, role, dtype, shape):
        side.append((role, {"dtype": dtype, "shape": list(shape)}))

    def _row_shape(self, role, view):
        if role in self.strided:
            self.dims += [(f"ld_{role}", f"LD_{role}"), (f"off_{role}", f"OFF_{role}")]
            view["shape"][1] = f"ld_{role}"
            view["offset"] = [0, f"off_{role}"]

    def rows(self, role, out=False, dtype=None, shape=("rows", "cols")):
        side = self.outputs if out else self.inputs
        self._add(side, role, dtype or self.dtype, shape)
        self._row_shape(role, side[-1][1])
        return self

    def vector(self, role, dtype, out=False, n="cols"):
        self._add(self.outputs if out else self.inputs, role, dtype, (n,))
        return self

    def checkpoint(self, out=False):
        self.rows("codes", out, "u8")
        return self.rows("exps", out, "u8", ("rows", "exp_cols"))

    def spec(self, name, kernel_class, operator, dims) -> KernelSpec:
        unknown = [s for s in self.strided if f"ld_{s}" not in [d[0] for d in self.dims]]
        if unknown:
            raise ValueError(f"{name}: no row tensor named {', '.join(unknown)}")
        roles = {}
        for i, (role, view) in enumerate(self.inputs + self.outputs):
            roles[role] = dict(view, arg=i)
        operator = dict(operator, rows="rows", cols="cols", roles=roles)
        spec = _spec(name, kernel_class, self.dtype, len(self.inputs), len(self.outputs), [], list(dims) + self.dims,
                     {"operator": operator}, {})
        if "exp_cols" in spec.shape_keys:
            spec.derived = {"EXP_COLS": lambda shape: -(-shape["D"] // CHECKPOINT_BLOCK)}
        return spec


def _one_of(what, value, words):
    if value not in words:
        raise ValueError(f"{what} is one of {', '.join(words)}: got {value!r}")


_ROW_DIMS = [("rows", "T"), ("cols", "D")]
_EXP_DIMS = [("exp_cols", "EXP_COLS")]
_FLOATS = ("f32", "f16", "bf16")


def _block_operator(dtype, kind, param_dtype, direction, pass_, **more):
    _one_of("dtype", dtype, _FLOATS)
    _one_of("kind", kind, ("rms", "layer"))
    _one_of("param_dtype", param_dtype or dtype, (dtype, "f32"))
    return dict({"direction": direction, "pass": pass_, "kind": kind, "param_dtype": param_dtype or dtype}, **more)


def block_norm(dtype: str = "bf16", kind: str = "rms", eps: float = 1e-6, checkpoint: bool = False, save_stats: bool = True,
               param_dtype: Optional[str] = None, strided=(), name: str = "block_norm") -> KernelSpec:
    """h = (x - mean) * rstd * weight [+ bias] over each row: rms (mean = 0, no bias) or layer norm.

    Inputs: x [T, D], weight [D] (, bias [D]).  Outputs: h [T, D] (, rstd [T] f32 (, mean [T] f32)) (, codes [T, D] u8,
    exps [T, ceil(D/128)] u8).  With `checkpoint` x is also kept in 8 bits, in the same pass; `save_stats` leaves the
    statistics for block_norm_grad.  Statistics are f32.  D up to 16384."""
    op_ = _block_operator(dtype, kind, param_dtype, "forward", "pre", eps=eps)
    layer, pt = kind == "layer", param_dtype or dtype
    r = _Roles(dtype, strided).rows("x").vector("weight", pt)
    if layer:
        r.vector("bias", pt)
    r.rows("h", out=True)
    if save_stats:
        r.vector("rstd", "f32", True, "rows")
        if layer:
            r.vector("mean", "f32", True, "rows")
    if checkpoint:
        r.checkpoint(out=True)
    return r.spec(name, "block_norm", op_, _ROW_DIMS + (_EXP_DIMS if checkpoint else []))


def block_norm_grad(dtype: str = "bf16", kind: str = "rms", checkpoint: bool = False, residual_grad: bool = False,
                    param_dtype: Optional[str] = None, strided=(), name: str = "block_norm_grad") -> KernelSpec:
    """Gradients of block_norm from dh: dx = rstd*(dn - n*avg(dn*n) [- avg(dn)]) (+ dout), dn = dh*weight.

    Inputs: dh [T, D], x [T, D] (with `checkpoint`: codes, exps instead), weight, rstd (, mean) (, dout [T, D]: with
    `residual_grad`, the gradient of x's other uses, added to dx).  Outputs: dx [T, D], dweight [D] f32 (, dbias [D] f32).
    Needs a workspace (workspace_bytes).  The sums over the rows are added in a fixed order."""
    op_ = _block_operator(dtype, kind, param_dtype, "gradient", "pre")
    layer, pt = kind == "layer", param_dtype or dtype
    r = _Roles(dtype, strided).rows("dh")
    r.checkpoint() if checkpoint else r.rows("x")
    r.vector("weight", pt).vector("rstd", "f32", n="rows")
    if layer:
        r.vector("mean", "f32", n="rows")
    if residual_grad:
        r.rows("dout")
    r.rows("dx", out=True).vector("dweight", "f32", True)
    if layer:
        r.vector("dbias", "f32", True)
    return r.spec(name, "block_norm", op_, _ROW_DIMS + (_EXP_DIMS if checkpoint else []))


_GATE_DIMS = [("group_rows", "G"), ("gate_rows", "B")]


def _gate_fields(gate, gate_act, alpha):
    _one_of("gate", gate, ("none", "token", "group"))
    _one_of("gate_act", gate_act, ("none", "sigmoid", "tanh"))
    fields = {"gate": gate, "gate_act": gate_act, "alpha": alpha}
    if gate == "group":
        fields["group_rows"] = "group_rows"
    return fields, (_GATE_DIMS if gate == "group" else [])


def gated_residual(dtype: str = "bf16", kind: str = "rms", eps: float = 1e-6, alpha: float = 1.0, gate: str = "none",
                   gate_act: str = "none", scale: bool = True, next_norm: bool = False, next_eps: Optional[float] = None,
                   checkpoint: bool = False, save_stats: bool = True, param_dtype: Optional[str] = None, strided=(),
                   name: str = "gated_residual") -> KernelSpec:
    """out = alpha*x + scale * act(gate) * (norm(y)*weight [+ bias]); with `next_norm` also h = norm(out)*next_weight [+ next_bias].

    x is the residual stream, y a block's output.  gate: "token" a value per element [T, D]; "group" one row [B, D] for
    every G rows (a sequence, say; the last group may be short).  Inputs: x, y, weight (, bias) (, gate) (, scale [D])
    (, next_weight (, next_bias)).  Outputs: out (, rstd (, mean)) (, h (, next_rstd (, next_mean))) (, codes, exps of y).
    The next norm reads `out` as it is stored.  `out` or `h` may take the place of x, y or a token gate."""
    fields, gate_dims = _gate_fields(gate, gate_act, alpha)
    op_ = _block_operator(dtype, kind, param_dtype, "forward", "post_pre" if next_norm else "post", eps=eps,
                          next_eps=eps if next_eps is None else next_eps, **fields)
    layer, pt = kind == "layer", param_dtype or dtype
    r = _Roles(dtype, strided).rows("x").rows("y").vector("weight", pt)
    if layer:
        r.vector("bias", pt)
    if gate != "none":
        r.rows("gate", shape=("rows", "cols") if gate == "token" else ("gate_rows", "cols"))
    if scale:
        r.vector("scale", pt)
    if next_norm:
        r.vector("next_weight", pt)
        if layer:
            r.vector("next_bias", pt)
    r.rows("out", out=True)
    if save_stats:
        r.vector("rstd", "f32", True, "rows")
        if layer:
            r.vector("mean", "f32", True, "rows")
    if next_norm:
        r.rows("h", out=True)
        if save_stats:
            r.vector("next_rstd", "f32", True, "rows")
            if layer:
                r.vector("next_mean", "f32", True, "rows")
    if checkpoint:
        r.checkpoint(out=True)
    return r.spec(name, "block_norm", op_, _ROW_DIMS + gate_dims + (_EXP_DIMS if checkpoint else []))


def gated_residual_grad(dtype: str = "bf16", kind: str = "rms", alpha: float = 1.0, gate: str = "none", gate_act: str = "none",
                        scale: bool = True, next_norm: bool = False, checkpoint: bool = False, param_dtype: Optional[str] = None,
                        strided=(), name: str = "gated_residual_grad") -> KernelSpec:
    """Gradients of gated_residual from dout (the stream's later uses) and, with `next_norm`, dh.

    Inputs: dout, y (with `checkpoint`: codes, exps), weight (, bias) (, gate) (, scale), rstd (, mean) (, dh, out,
    next_weight, next_rstd (, next_mean)).  Outputs: dx, dy, dweight [D] f32 (, dbias f32) (, dgate: "token" [T, D], "group"
    [B, D] f32) (, dscale f32) (, dnext_weight f32 (, dnext_bias f32)).  Needs a workspace (workspace_bytes)."""
    fields, gate_dims = _gate_fields(gate, gate_act, alpha)
    op_ = _block_operator(dtype, kind, param_dtype, "gradient", "post_pre" if next_norm else "post", **fields)
    layer, pt = kind == "layer", param_dtype or dtype
    gate_shape = ("rows", "cols") if gate == "token" else ("gate_rows", "cols")
    r = _Roles(dtype, strided).rows("dout")
    r.checkpoint() if checkpoint else r.rows("y")
    r.vector("weight", pt)
    if layer:
        r.vector("bias", pt)
    if gate != "none":
        r.rows("gate", shape=gate_shape)
    if scale:
        r.vector("scale", pt)
    r.vector("rstd", "f32", n="rows")
    if layer:
        r.vector("mean", "f32", n="rows")
    if next_norm:
        r.rows("dh").rows("out").vector("next_weight", pt).vector("next_rstd", "f32", n="rows")
        if layer:
            r.vector("next_mean", "f32", n="rows")
    r.rows("dx", out=True).rows("dy", out=True).vector("dweight", "f32", True)
    if layer:
        r.vector("dbias", "f32", True)
    if gate != "none":
        r.rows("dgate", out=True, dtype=dtype if gate == "token" else "f32", shape=gate_shape)
    if scale:
        r.vector("dscale", "f32", True)
    if next_norm:
        r.vector("dnext_weight", "f32", True)
        if layer:
            r.vector("dnext_bias", "f32", True)
    return r.spec(name, "block_norm", op_, _ROW_DIMS + gate_dims + (_EXP_DIMS if checkpoint else []))


def checkpoint_pack(dtype: str = "bf16", strided=(), name: str = "checkpoint_pack") -> KernelSpec:
    """An activation in 8 bits: value = e4m3(code) * 2^(exp - 127), one exponent per row and 128 columns.

    Inputs: x [T, D].  Outputs: codes [T, D] u8, exps [T, ceil(D/128)] u8.  The power is the smallest that brings the
    block's largest finite magnitude to 448 or less, kept where the restored value is exact in `dtype`; infinities and NaN
    become NaN."""
    _one_of("dtype", dtype, _FLOATS)
    r = _Roles(dtype, strided).rows("x").checkpoint(out=True)
    return r.spec(name, "checkpoint", {"direction": "forward"}, _ROW_DIMS + _EXP_DIMS)


def checkpoint_restore(dtype: str = "bf16", strided=(), name: str = "checkpoint_restore") -> KernelSpec:
    """The values of a checkpoint made from `dtype`.  Inputs: codes, exps.  Outputs: x [T, D]."""
    _one_of("dtype", dtype, _FLOATS)
    r = _Roles(dtype, strided).checkpoint().rows("x", out=True)
    return r.spec(name, "checkpoint", {"direction": "gradient"}, _ROW_DIMS + _EXP_DIMS)


def checkpoint_weight_grad(dtype: str = "bf16", out_dtype: Optional[str] = None, accumulate: bool = False, strided=(),
                           name: str = "checkpoint_weight_grad") -> KernelSpec:
    """dweight [D, N] = x^T dy of a linear layer y = x weight whose input x [T, D] was kept as a checkpoint.

    Inputs: codes, exps (made from `dtype`), dy [T, N] in `dtype` (f16 or bf16).  Outputs: dweight in `out_dtype` (f32 or
    `dtype`); with `accumulate` the product is added to what dweight holds.  The restored x is exact in `dtype`, products
    are summed in f32 by the tensor cores.  Needs a workspace where workspace_bytes says more than 256.  D a multiple of 16,
    N of 8, as are strided row lengths and offsets."""
    _one_of("dtype", dtype, ("f16", "bf16"))
    _one_of("out_dtype", out_dtype or dtype, (dtype, "f32"))
    r = _Roles(dtype, strided).checkpoint().rows("dy", shape=("rows", "out_cols"))
    r.rows("dweight", out=True, dtype=out_dtype or dtype, shape=("cols", "out_cols"))
    return r.spec(name, "checkpoint_grad", {"out_cols": "out_cols", "out_dtype": out_dtype or dtype, "accumulate": accumulate},
                  _ROW_DIMS + [("out_cols", "N")] + _EXP_DIMS)
