"""Calls of the operator kernels on torch tensors, through CudaRuntime.launch_device."""
import torch

from ascend_mlir_b200 import descriptors

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}



def outputs_for(spec, sizes, device, fill=None):
    """New output tensors in the kernel's order, by role."""
    dims = dict(sizes)
    if "D" in dims:
        dims["EXP_COLS"] = -(-dims["D"] // descriptors.CHECKPOINT_BLOCK)
    keys = {f: k for f, k in spec.shape_keys.items()}
    outs = {}
    roles = spec.descriptor["operator"]["roles"]
    for role, view in sorted(roles.items(), key=lambda kv: kv[1]["arg"]):
        if view["arg"] < spec.descriptor["num_inputs"]:
            continue
        shape = [dims[keys[d]] if isinstance(d, str) else d for d in view["shape"]]
        t = torch.empty(shape, dtype=TORCH[view["dtype"]], device=device)
        if fill is not None:
            t.fill_(fill)
        outs[role] = t
    return outs


def arguments(spec, inputs, outs):
    roles = sorted(spec.descriptor["operator"]["roles"].items(), key=lambda kv: kv[1]["arg"])
    n = spec.descriptor["num_inputs"]
    addr = lambda t: (t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
    return [addr(inputs[r]) for r, v in roles if v["arg"] < n], [addr(outs[r]) for r, v in roles if v["arg"] >= n]


def call(rt, spec, sizes, inputs, outs=None, stream=None, workspace=None):
    """Enqueues the kernel on `stream` (the current one) and returns its outputs by role."""
    device = next(iter(inputs.values())).device
    outs = outputs_for(spec, sizes, device) if outs is None else outs
    tiling = spec.pack(sizes)
    if workspace is None:
        workspace = torch.empty(rt.workspace_bytes(spec.binary, tiling), dtype=torch.uint8, device=device)
    a, b = arguments(spec, inputs, outs)
    stream = torch.cuda.current_stream().cuda_stream if stream is None else stream
    rt.launch_device(spec.binary, spec.name, a, b, tiling, 0, spec.magic, (workspace.data_ptr(), workspace.numel()), stream)
    outs["_workspace"] = workspace
    return outs
