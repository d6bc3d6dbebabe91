"""What is measured of the dense 16-bit operators: the gated feed-forward block, the linear layer with its epilogue and the
8-bit activation checkpoints, each in its plain form (elementary torch operations in fp32) and as this package's calls.

Layouts are those of the operators: activations row-major [rows, features], weights [in, out] (a transposed view of an
[out, in] parameter is as good), the gate half of the first projection before its up half.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_CODES = {"bf16": 15, "fp16": 5}          # the dtype numbers that the operators take
_BLOCK = 64                               # values that share one scale in an 8-bit checkpoint
_MOST_FLOPS = 3 * 2 * 8192 * 3 * 4096 * 2048


def listed():
    return [
        # the shared expert of a decode step that serves a single user: latency, the weights are read once
        dict(name="ffn_one_token", op="ffn", mode="serve", rows=1, hidden=7168, inner=2048, dtype="bf16", act="silu",
             bias=False, residual=False, transposed=False),
        # a small decode batch through a block with biases, GELU and the residual stream added at the end
        dict(name="ffn_decode_batch", op="ffn", mode="serve", rows=37, hidden=4096, inner=1408, dtype="fp16", act="gelu_tanh",
             bias=True, residual=True, transposed=True),
        # a chunk of prompts through the shared expert
        dict(name="ffn_prompt", op="ffn", mode="serve", rows=4096, hidden=7168, inner=2048, dtype="bf16", act="silu",
             bias=False, residual=True, transposed=True),
        # a training step of a dense block: the result and every gradient
        dict(name="ffn_train", op="ffn", mode="train", rows=8192, hidden=4096, inner=2048, dtype="bf16", act="silu",
             bias=False, residual=False, transposed=False, int8=False),
        # packed sequences of no round length, in a training step that keeps its activations in 8 bits
        dict(name="ffn_train_int8", op="ffn", mode="train", rows=3001, hidden=2048, inner=1408, dtype="fp16", act="gelu",
             bias=True, residual=False, transposed=True, int8=True),
        # an output projection of a decode step, added to the residual stream
        dict(name="linear_decode", op="linear", mode="serve", rows=8, inputs=2048, outputs=7168, dtype="bf16", act="none",
             bias=False, residual=True, transposed=False),
        # features that are multiples of nothing
        dict(name="linear_ragged", op="linear", mode="serve", rows=777, inputs=1003, outputs=1501, dtype="fp16", act="relu",
             bias=True, residual=False, transposed=False),
        # the widening projection of a classic feed-forward block over a prompt
        dict(name="linear_prompt", op="linear", mode="serve", rows=4096, inputs=1024, outputs=4096, dtype="bf16", act="gelu_tanh",
             bias=True, residual=False, transposed=True),
        # a training step of a projection with bias, activation and residual
        dict(name="linear_train", op="linear", mode="train", rows=8192, inputs=2048, outputs=7168, dtype="bf16", act="gelu",
             bias=True, residual=True, transposed=False, int8=False),
        # a layer's input put away in 8 bits and taken out again
        dict(name="checkpoint_layer", op="checkpoint", mode="keep", rows=8192, inputs=7168, dtype="bf16"),
        # the same of a short ragged batch
        dict(name="checkpoint_short", op="checkpoint", mode="keep", rows=37, inputs=1003, dtype="fp16"),
        # the weight gradient of a projection whose input was kept in 8 bits
        dict(name="checkpoint_weight_grad", op="checkpoint", mode="weight_grad", rows=8192, inputs=4096, outputs=2048, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _feature(rng, low, high):
    """A number of features: usually a multiple of 64 or 8, now and then of nothing."""
    v = _log_int(rng, low, high)
    step = rng.choice((64, 64, 64, 8, 1))
    return max(low, v // step * step)


def draw(rng):
    op = rng.choice(("ffn", "ffn", "linear", "linear", "checkpoint"))
    case = dict(op=op, rows=_log_int(rng, 1, 8192), dtype=rng.choice(("bf16", "fp16")))
    if op == "checkpoint":
        case.update(mode=rng.choice(("keep", "weight_grad")), inputs=_feature(rng, 64, 7168))
        if case["mode"] == "weight_grad":
            case.update(outputs=_feature(rng, 64, 7168))
    else:
        case.update(mode=rng.choice(("serve", "train")), bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                    transposed=rng.random() < 0.5)
        if op == "ffn":
            case.update(hidden=_feature(rng, 128, 7168), inner=_feature(rng, 128, 2048), act=rng.choice(("silu", "gelu", "gelu_tanh", "relu")))
        else:
            case.update(inputs=_feature(rng, 64, 7168), outputs=_feature(rng, 64, 7168),
                        act=rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")))
        if case["mode"] == "train":
            case.update(int8=rng.random() < 0.5)
    while work(case)["flops"] > _MOST_FLOPS:
        case["rows"] //= 2
    return case


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * scale).to(dtype)

    def weight(n_in, n_out):
        # as a parameter [out, in] seen through its transpose, or as the operator's own [in, out]
        return normal(n_out, n_in, scale=n_in ** -0.5).t() if case["transposed"] else normal(n_in, n_out, scale=n_in ** -0.5)

    rows = case["rows"]
    s = {"case": case}
    if case["op"] == "checkpoint":
        # activations behind a norm have features of different sizes
        s["x"] = normal(rows, case["inputs"]) * (0.25 + 2.0 * torch.rand(case["inputs"], generator=g, device=dev)).to(dtype)
        if case["mode"] == "weight_grad":
            s["grad"] = normal(rows, case["outputs"], scale=0.1)
            s["q"], s["scale"] = _quantise(s["x"].float())
        return s
    if case["op"] == "ffn":
        n_in, inner = case["hidden"], case["inner"]
        s["weight1"], s["weight2"] = weight(n_in, 2 * inner), weight(inner, n_in)
        n_out = n_in
        s["bias1"] = normal(2 * inner, scale=0.5) if case["bias"] else None
        s["bias2"] = normal(n_in, scale=0.5) if case["bias"] else None
    else:
        n_in, n_out = case["inputs"], case["outputs"]
        s["weight"] = weight(n_in, n_out)
        s["bias"] = normal(n_out, scale=0.5) if case["bias"] else None
    s["x"] = normal(rows, n_in)
    s["residual"] = normal(rows, n_out) if case["residual"] else None
    if case["mode"] == "train":
        s["grad"] = normal(rows, n_out, scale=0.1)
        for name in ("x", "weight1", "weight2", "weight", "bias1", "bias2", "bias", "residual"):
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------------

def _quantise(x):
    """fp32 [rows, n] -> int8 [rows, n] and one fp32 scale per row and block of 64 values."""
    rows, n = x.shape
    blocks = -(-n // _BLOCK)
    padded = torch.zeros(rows, blocks * _BLOCK, dtype=torch.float32, device=x.device)
    padded[:, :n] = x
    b = padded.view(rows, blocks, _BLOCK)
    scale = b.abs().amax(-1) / 127.0
    q = torch.where(scale[..., None] > 0, torch.round(b / scale[..., None]), torch.zeros_like(b))
    return q.view(rows, -1)[:, :n].to(torch.int8).contiguous(), scale


def _dequantise(q, scale):
    return q.float() * scale.repeat_interleave(_BLOCK, 1)[:, :q.shape[1]]


def _kept(x):
    """A value as the backward pass finds it after an 8-bit checkpoint."""
    return _dequantise(*_quantise(x))


def _act(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).float()
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    t = torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * (2.0 / math.pi) ** 0.5 * (1.0 + 3 * 0.044715 * z * z)


def _plain_ffn(s):
    case, dtype = s["case"], s["x"].dtype
    inner, act = case["inner"], case["act"]
    x, w1, w2 = s["x"].float(), s["weight1"].float(), s["weight2"].float()
    z = x @ w1
    if s["bias1"] is not None:
        z = z + s["bias1"].float()
    gate, up = z[:, :inner], z[:, inner:]
    y = (_act(gate, act)[0] * up) @ w2
    if s["bias2"] is not None:
        y = y + s["bias2"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["mode"] == "serve":
        return out
    if case["int8"]:
        x, gate, up = _kept(x), _kept(gate), _kept(up)
    dy = s["grad"].float()
    a, da = _act(gate, act)
    dh = dy @ w2.t()
    dz = torch.cat((dh * up * da, dh * a), 1)
    out.update(x=(dz @ w1.t()).to(dtype), weight1=(x.t() @ dz).to(dtype), weight2=((a * up).t() @ dy).to(dtype))
    if s["bias1"] is not None:
        out.update(bias1=dz.sum(0).to(dtype), bias2=dy.sum(0).to(dtype))
    if s["residual"] is not None:
        out.update(residual=dy.to(dtype))
    return out


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["act"])[0]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["mode"] == "serve":
        return out
    if case["int8"]:
        x, z = _kept(x), _kept(z)
    dy = s["grad"].float()
    dz = dy * _act(z, case["act"])[1]
    out.update(x=(dz @ w.t()).to(dtype), weight=(x.t() @ dz).to(dtype))
    if s["bias"] is not None:
        out.update(bias=dz.sum(0).to(dtype))
    if s["residual"] is not None:
        out.update(residual=dy.to(dtype))
    return out


def _plain_checkpoint(s):
    dtype = s["x"].dtype
    if s["case"]["mode"] == "keep":
        return {"x": _kept(s["x"].float()).to(dtype)}
    return {"weight": (_dequantise(s["q"], s["scale"]).t() @ s["grad"].float()).to(dtype)}


# ---- the package's calls -------------------------------------------------------------------------------------------------

def _own(s):
    import torchair_b200  # noqa: F401  (registers torch.ops.npu.*)
    npu = torch.ops.npu
    case = s["case"]
    if case["op"] == "checkpoint":
        if case["mode"] == "keep":
            q, scale = npu.npu_checkpoint_quant(s["x"])
            return {"x": npu.npu_checkpoint_dequant(q, scale, output_dtype=_CODES[case["dtype"]])}
        return {"weight": npu.npu_checkpoint_weight_grad(s["q"], s["scale"], s["grad"])}
    if case["op"] == "ffn":
        names = ("x", "weight1", "weight2", "bias1", "bias2", "residual")
        y = npu.npu_gated_ffn(s["x"], s["weight1"], s["weight2"], bias1=s["bias1"], bias2=s["bias2"], residual=s["residual"],
                              activation=case["act"], checkpoint_int8=case.get("int8", False))
    else:
        names = ("x", "weight", "bias", "residual")
        y = npu.npu_linear_act(s["x"], s["weight"], bias=s["bias"], residual=s["residual"], activation=case["act"],
                               checkpoint_int8=case.get("int8", False))
    if case["mode"] == "serve":
        return {"y": y}
    names = [n for n in names if s[n] is not None]
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [s[n] for n in names], s["grad"])))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"ffn": _plain_ffn, "linear": _plain_linear, "checkpoint": _plain_checkpoint}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    m = case["rows"]
    if case["op"] == "checkpoint":
        n = case["inputs"]
        kept = m * n + 4 * m * -(-n // _BLOCK)
        if case["mode"] == "keep":                 # read, put away, taken out, written
            return {"bytes": 2 * (2 * m * n) + 2 * kept, "flops": 4 * m * n}
        return {"bytes": kept + 2 * case["outputs"] * (m + n), "flops": 2 * m * n * case["outputs"]}
    if case["op"] == "ffn":
        n_in = n_out = case["hidden"]
        weights, biases = 3 * n_in * case["inner"], 2 * case["inner"] + n_in
    else:
        n_in, n_out = case["inputs"], case["outputs"]
        weights, biases = n_in * n_out, n_out
    values = m * n_in + m * n_out + weights + (biases if case["bias"] else 0) + (m * n_out if case["residual"] else 0)
    flops = 2 * m * weights
    if case["mode"] == "train":                    # the result's gradient comes in, one for every input goes out
        values += m * n_out + m * n_in + weights + (biases if case["bias"] else 0) + (m * n_out if case["residual"] else 0)
        flops *= 3
    return {"bytes": 2 * values, "flops": flops}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def _round_trip64(v):
    """v [rows, n] through the 8-bit form: per row and block of 64 values, amax / 127 steps, to the nearest (ties to even)."""
    pad = -v.shape[1] % _BLOCK
    b = torch.cat((v, v.new_zeros(v.shape[0], pad)), 1).reshape(v.shape[0], -1, _BLOCK)
    step = b.abs().max(-1, keepdim=True).values / 127
    b = torch.round(b / torch.where(step == 0, torch.ones_like(step), step)) * step
    return b.reshape(v.shape[0], -1)[:, :v.shape[1]]


def _phi64(z, act):
    """Activation and derivative by autograd of its definition."""
    with torch.enable_grad():
        z = z.detach().clone().requires_grad_()
        if act == "none":
            y = z * 1
        elif act == "relu":
            y = z * (z.detach() > 0)
        elif act == "silu":
            y = z / (1 + (-z).exp())
        elif act == "gelu":
            y = z * (1 + (z / math.sqrt(2)).erf()) / 2
        else:
            y = z * (1 + (math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)).tanh()) / 2
        d, = torch.autograd.grad(y, z, torch.ones_like(y))
    return y.detach(), d


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        v = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor)}
        keep = _round_trip64 if case.get("int8") else (lambda t: t)
        if case["op"] == "checkpoint":
            if case["mode"] == "keep":
                return {"x": _round_trip64(v["x"])}
            blocks = v["scale"].shape[1]
            x = torch.cat([v["q"][:, _BLOCK * b:_BLOCK * (b + 1)] * v["scale"][:, b:b + 1] for b in range(blocks)], 1)
            return {"weight": torch.einsum("mk,mn->kn", x, v["grad"])}
        if case["op"] == "linear":
            z = v["x"] @ v["weight"] + v.get("bias", 0)
            out = {"y": _phi64(z, case["act"])[0] + v.get("residual", 0)}
            if case["mode"] == "train":
                dz = v["grad"] * _phi64(keep(z), case["act"])[1]
                out.update(x=torch.einsum("mn,kn->mk", dz, v["weight"]), weight=torch.einsum("mk,mn->kn", keep(v["x"]), dz))
                if "bias" in v:
                    out.update(bias=dz.sum(0))
                if "residual" in v:
                    out.update(residual=v["grad"])
            return out
        z = v["x"] @ v["weight1"] + v.get("bias1", 0)
        gate, up = z.chunk(2, 1)
        out = {"y": (_phi64(gate, case["act"])[0] * up) @ v["weight2"] + v.get("bias2", 0) + v.get("residual", 0)}
        if case["mode"] == "train":
            gate, up = keep(gate), keep(up)
            phi, slope = _phi64(gate, case["act"])
            dh = torch.einsum("mn,kn->mk", v["grad"], v["weight2"])
            dgate, dup = dh * up * slope, dh * phi
            w_gate, w_up = v["weight1"].chunk(2, 1)
            x = keep(v["x"])
            out.update(x=dgate @ w_gate.t() + dup @ w_up.t(), weight1=torch.cat((x.t() @ dgate, x.t() @ dup), 1),
                       weight2=(phi * up).t() @ v["grad"])
            if "bias1" in v:
                out.update(bias1=torch.cat((dgate.sum(0), dup.sum(0))), bias2=v["grad"].sum(0))
            if "residual" in v:
                out.update(residual=v["grad"])
        return out
