"""One training step of a residual block on the GPU through the package's kernels, as they are used together:

    h = norm(x);  y = h W (the tensor-core matmul);  out = alpha*x + scale*sigmoid(g)*norm'(y);  h2 = norm''(out)

and back, with h kept in 8 bits for W's gradient, on one stream and as one captured graph.  Against autograd in 64 bits.

Every tensor between the kernels is stored in bf16 (half step 2^-8).  A gradient passes at most eight such stores, each of
which adds at most 2^-8 of its size in the 2-norm; the norms in between pass errors on with a factor of about one (they
remove two directions and scale): 8 * 2^-8 bounds the relative error.  W's gradient reads h in e4m3 (half step 2^-4 of each
element, at random signs): elementwise at most 2^-4 * |h|^T |dy| on top."""
import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime.executor import CudaRuntime

from operator_calls import call, outputs_for

pytestmark = pytest.mark.gpu
EPS, ALPHA = 1e-6, 0.8


def norm64(v, w, eps=EPS):
    return v / torch.sqrt(v.square().mean(1, keepdim=True) + eps) * w


class Step:
    def __init__(self, T, D, seed):
        gen = torch.Generator("cuda").manual_seed(seed)
        r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=gen, device="cuda") * std + mean).bfloat16()  # noqa: E731
        self.T, self.D = T, D
        self.rt = CudaRuntime()
        self.rt.set_device(0)
        self.t = {"x": r(T, D), "w1": r(D, std=0.1, mean=1.0), "W": r(D, D, std=D ** -0.5), "gate": r(T, D), "scale": r(D, std=0.1, mean=0.5),
                  "w2": r(D, std=0.1, mean=1.0), "w3": r(D, std=0.1, mean=1.0), "r1": r(T, D, std=0.1), "r2": r(T, D, std=0.1)}
        self.zero_bias = torch.zeros(D, device="cuda").bfloat16()
        self.kernels = {
            "pre": descriptors.block_norm("bf16", eps=EPS, name="pre"),
            "pack": descriptors.checkpoint_pack("bf16", name="pack"),
            "post": descriptors.gated_residual("bf16", eps=EPS, alpha=ALPHA, gate="token", gate_act="sigmoid", next_norm=True, name="post"),
            "post_grad": descriptors.gated_residual_grad("bf16", alpha=ALPHA, gate="token", gate_act="sigmoid", next_norm=True, name="post_grad"),
            "w_grad": descriptors.checkpoint_weight_grad("bf16", out_dtype="f32", name="w_grad"),
            "pre_grad": descriptors.block_norm_grad("bf16", residual_grad=True, name="pre_grad")}
        self.mm = {False: descriptors.matmul_bias_leakyrelu("bf16", epilogue="None", name="mm"),
                   True: descriptors.matmul_bias_leakyrelu("bf16", epilogue="None", transpose_b=True, name="mm_t")}
        # a workspace for each kernel and outputs that stay, as a program with a captured step keeps them
        s = {"T": T, "D": D, "N": D}
        self.ws = {k: torch.zeros(self.rt.workspace_bytes(v.binary, v.pack(self.sizes(v))), dtype=torch.uint8, device="cuda") for k, v in self.kernels.items()}
        self.outs = {k: outputs_for(v, s, torch.device("cuda")) for k, v in self.kernels.items()}
        self.products = [torch.empty(T, D, device="cuda").bfloat16() for _ in range(2)]
        self.mm_ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")

    def sizes(self, spec):
        return {k: {"T": self.T, "D": self.D, "N": self.D}[k] for k in spec.shape_keys.values() if k in "TDN"}

    def kernel(self, name, **inputs):
        spec = self.kernels[name]
        return call(self.rt, spec, self.sizes(spec), inputs, self.outs[name], workspace=self.ws[name])

    def matmul(self, a, b, out, transpose_b=False):
        spec = self.mm[transpose_b]
        addr = lambda t: (t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
        self.rt.launch_device(spec.binary, spec.name, [addr(a), addr(b), addr(self.zero_bias)], [addr(out)],
                              spec.pack({"M": self.T, "N": self.D, "K": self.D}), 0, spec.magic, (self.mm_ws.data_ptr(), 4096),
                              torch.cuda.current_stream().cuda_stream)
        return out

    def run(self):
        t = self.t
        pre = self.kernel("pre", x=t["x"], weight=t["w1"])
        kept = self.kernel("pack", x=pre["h"])
        y = self.matmul(pre["h"], t["W"], self.products[0])
        post = self.kernel("post", x=t["x"], y=y, weight=t["w2"], gate=t["gate"], scale=t["scale"], next_weight=t["w3"])
        g = self.kernel("post_grad", dout=t["r1"], y=y, weight=t["w2"], gate=t["gate"], scale=t["scale"], rstd=post["rstd"], dh=t["r2"],
                        out=post["out"], next_weight=t["w3"], next_rstd=post["next_rstd"])
        dW = self.kernel("w_grad", codes=kept["codes"], exps=kept["exps"], dy=g["dy"])
        dh = self.matmul(g["dy"], t["W"], self.products[1], transpose_b=True)
        p = self.kernel("pre_grad", dh=dh, x=t["x"], weight=t["w1"], rstd=pre["rstd"], dout=g["dx"])
        return {"out": post["out"], "h2": post["h"], "W": dW["dweight"], "x": p["dx"], "w1": p["dweight"], "w2": g["dweight"], "gate": g["dgate"],
                "scale": g["dscale"], "w3": g["dnext_weight"]}

    def exact(self):
        v = {k: t.double().requires_grad_(k not in ("r1", "r2")) for k, t in self.t.items()}
        h = norm64(v["x"], v["w1"])
        h.retain_grad()
        y = h @ v["W"]
        y.retain_grad()
        out = ALPHA * v["x"] + v["scale"] * torch.sigmoid(v["gate"]) * norm64(y, v["w2"])
        h2 = norm64(out, v["w3"])
        ((out * v["r1"]).sum() + (h2 * v["r2"]).sum()).backward()
        grads = {k: v[k].grad for k in ("W", "x", "w1", "w2", "gate", "scale", "w3")}
        return dict(grads, out=out.detach(), h2=h2.detach()), h.detach().abs().T @ y.grad.abs()


@pytest.mark.parametrize("T,D", [(200, 256), (1, 512), (777, 1024)])
def test_step_against_autograd(T, D):
    step = Step(T, D, T)
    got = step.run()
    step.rt.synchronize(torch.cuda.current_stream().cuda_stream)
    want, w_bound = step.exact()
    for name, value in want.items():
        off = got[name].double() - value
        if name == "W":
            size = value.norm() / value.numel() ** 0.5
            assert (off.abs() <= 2.0 ** -4 * w_bound + 8 * 2.0 ** -8 * (w_bound + size)).all()
        else:
            assert off.norm() <= 8 * 2.0 ** -8 * value.norm(), (name, float(off.norm() / value.norm()))


def test_two_captured_steps_at_once():
    """Two steps, each with its own workspaces, captured and replayed on two streams at the same time: the eager results."""
    steps = [Step(300, 512, k) for k in range(2)]
    want = []
    for s in steps:
        want.append({k: v.clone() for k, v in s.run().items()})
    torch.cuda.synchronize()
    graphs, results = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(s.run())
        graphs.append(g)
    for r in results:
        for v in r.values():
            v.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for r, w in zip(results, want):
        for k in w:
            assert torch.equal(r[k], w[k]), k
