"""The dense 16-bit operators (npu_gated_ffn, npu_linear_act and their gradients, the 8-bit checkpoints) against their formulas in
64 bits.

Bounds are computed element by element next to each reference.  u = eps / 2 is the relative error of one rounding to the
16-bit type; a product over K terms is accumulated in fp32, each addition off by at most 2^-23 (the tensor core may truncate)
of the sum of magnitudes: G(K) = (K + 16) 2^-23 times |x| @ |w|.  Activations and their derivatives are evaluated in fp32 with
the hardware exponential and division: within S |z| = 2^-18 |z| of the formula (the exponential's argument z log2(e) is
rounded to 24 bits, which for |z| <= 64 is a relative error of 2^-17 in exp and at most half of that in the sigmoid).
"""
import math

import pytest
import torch

import torchair_b200
from torchair_b200 import _lib

npu = torch.ops.npu
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
DTYPES = [torch.bfloat16, torch.float16]
SLOPE = 1.13          # no activation here is steeper


@pytest.fixture(scope="module")
def dev():
    torchair_b200.clear_weight_cache()
    yield torch.device("cuda:0")
    assert torchair_b200.dense_status("cuda:0") == 0


# ---- references ----------------------------------------------------------------------------------------------------------
def act64(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    v = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(2 * v)
    return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)


def U(dtype):
    return torch.finfo(dtype).eps / 2


def G(k):
    return (k + 16) * 2.0 ** -23


S = 2.0 ** -18


def tiny(dtype):
    """half the step between the type's subnormal values"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def mm(a, b):
    """product, bound of its fp32 accumulation"""
    return a @ b, G(a.shape[1]) * (a.abs() @ b.abs())


def check(got, want, bound, what):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    err = (got.double() - want).abs() - (bound + U(got.dtype) * (want.abs() + bound) + tiny(got.dtype))
    assert not torch.isnan(got).any(), f"{what}: NaN"
    assert err.numel() == 0 or err.max() <= 0, f"{what}: over the bound by {err.max():.3e}, at {int((err > 0).sum())} of {err.numel()} places"


def quant64(v):
    """(q, scale) as defined, on exactly representable fp32 input"""
    rows, n = v.shape
    pad = -n % 64
    b = torch.cat((v.float(), torch.zeros(rows, pad, device=v.device)), 1).view(rows, -1, 64)
    scale = b.abs().amax(-1)
    scale = scale / torch.full_like(scale, 127.0)        # by a tensor: by a number, torch multiplies by its rounded reciprocal
    q = torch.where(scale[..., None] > 0, torch.round(b / scale[..., None]), torch.zeros_like(b))
    return q.view(rows, -1)[:, :n].to(torch.int8), scale


def deq64(q, scale):
    return q.double() * scale.double().repeat_interleave(64, 1)[:, :q.shape[1]]


def make(g, *shape, scale=1.0, dtype=torch.bfloat16, dev="cuda"):
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(g, k, n, transposed, dtype):
    return make(g, n, k, scale=k ** -0.5, dtype=dtype).t() if transposed else make(g, k, n, scale=k ** -0.5, dtype=dtype)


def ref_linear(x, w, b, r, act):
    z, e = mm(x.double(), w.double())
    if b is not None:
        z, e = z + b.double(), e + 2.0 ** -23 * b.double().abs()
    y = act64(z, act)[0]
    e = SLOPE * e + (S * z.abs() if act != "none" else 0)
    if r is not None:
        y, e = y + r.double(), e + 2.0 ** -23 * r.double().abs()
    return y, e


def ref_ffn(x, w1, w2, b1, b2, r, act):
    z, e = mm(x.double(), w1.double())
    if b1 is not None:
        z, e = z + b1.double(), e + 2.0 ** -23 * b1.double().abs()
    inner = w2.shape[0]
    a = act64(z[:, :inner], act)[0]
    ea = SLOPE * e[:, :inner] + S * z[:, :inner].abs()
    up, eu = z[:, inner:], e[:, inner:]
    h = a * up
    eh = ea * up.abs() + (a.abs() + ea) * eu + 2.0 ** -23 * h.abs()
    eh = eh + U(x.dtype) * (h.abs() + eh) + tiny(x.dtype)           # h is rounded to the 16-bit type
    y, e = mm(h, w2.double())
    e = e + eh @ w2.double().abs() * (1 + G(inner))
    for t in (b2, r):
        if t is not None:
            y, e = y + t.double(), e + 2.0 ** -23 * t.double().abs()
    return y, e


# ---- npu_linear_act ------------------------------------------------------------------------------------------------------
LINEAR = [  # rows, in, out, transposed weight, act, bias, residual
    (1, 8, 8, False, "none", False, False),
    (1, 512, 256, True, "silu", True, True),
    (2, 72, 136, False, "gelu", True, False),
    (16, 2048, 7168, False, "none", False, True),
    (17, 1000, 264, True, "relu", False, True),
    (33, 640, 120, False, "gelu_tanh", True, True),
    (64, 64, 1024, True, "none", True, False),
    (65, 4096, 520, False, "silu", False, False),
    (128, 1536, 640, True, "gelu", True, True),
    (129, 8, 16, False, "none", False, False),
    (129, 200, 264, True, "relu", True, True),
    (256, 64, 256, False, "gelu_tanh", True, False),
    (257, 2048, 520, True, "silu", False, True),
    (300, 1024, 2056, False, "gelu", True, True),
    (1000, 72, 3000, True, "none", False, False),
    (2049, 512, 4096, False, "silu", True, True),
    (5000, 4096, 1032, True, "relu", False, False),
    # a few tiles in a last turn that share their contraction (81 = 74 + 7 and 100 = 74 + 26 tiles of 256 x 256)
    (2300, 4160, 2104, False, "gelu", True, True),
    (2560, 4096, 2560, True, "none", False, False),
    # clusters that share narrow tiles, up to eight to one
    (128, 8192, 1000, True, "silu", True, False),
    (70, 2048, 136, False, "none", False, True),
    (20, 8192, 128, True, "gelu_tanh", True, True),
    # sizes that are multiples of nothing
    (2301, 4161, 2101, True, "relu", True, True),
    (1, 1, 1, False, "none", True, True),
    (3, 7, 13, True, "silu", True, False),
    (777, 1003, 1501, False, "relu", True, False),
    (130, 65, 129, True, "gelu", True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LINEAR, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_linear_act(dev, case, dtype):
    m, k, n, transposed, act, bias, residual = case
    g = gen(m * 7 + k)
    x, w = make(g, m, k, dtype=dtype), weight(g, k, n, transposed, dtype)
    b = make(g, n, dtype=dtype) if bias else None
    r = make(g, m, n, dtype=dtype) if residual else None
    y = npu.npu_linear_act(x, w, bias=b, residual=r, activation=act)
    assert y.dtype == dtype and y.is_contiguous()
    check(y, *ref_linear(x, w, b, r, act), f"linear {case}")
    assert torch.equal(y, npu.npu_linear_act(x, w, bias=b, residual=r, activation=act)), "the same call gives the same bits"


# ---- npu_gated_ffn -------------------------------------------------------------------------------------------------------
FFN = [  # rows, hidden, inner, transposed weights, act, biases, residual
    (1, 7168, 2048, False, "silu", False, False),
    (1, 64, 8, True, "gelu", True, True),
    (8, 1024, 1000, True, "silu", False, True),
    (37, 4096, 1408, True, "gelu_tanh", True, True),
    (100, 512, 72, False, "relu", True, False),
    (128, 256, 640, False, "none", False, True),
    (129, 264, 136, True, "silu", True, True),
    (300, 1024, 520, False, "gelu", False, False),
    (2500, 768, 1024, True, "silu", True, True),
    (2300, 4160, 1104, False, "silu", True, True),       # 81 tiles of gate and up: the last 7 share their contraction
    (90, 4096, 200, True, "gelu", False, True),
    (5, 33, 17, False, "silu", True, True),
    (200, 100, 129, True, "gelu_tanh", True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", FFN, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gated_ffn(dev, case, dtype):
    m, h, inner, transposed, act, bias, residual = case
    g = gen(m + h)
    x = make(g, m, h, dtype=dtype)
    w1, w2 = weight(g, h, 2 * inner, transposed, dtype), weight(g, inner, h, transposed, dtype)
    b1, b2 = (make(g, 2 * inner, dtype=dtype), make(g, h, dtype=dtype)) if bias else (None, None)
    r = make(g, m, h, dtype=dtype) if residual else None
    y = npu.npu_gated_ffn(x, w1, w2, bias1=b1, bias2=b2, residual=r, activation=act)
    check(y, *ref_ffn(x, w1, w2, b1, b2, r, act), f"ffn {case}")
    kept = npu.npu_gated_ffn_keep(x, w1, w2, bias1=b1, bias2=b2, residual=r, activation=act)
    assert torch.equal(y, kept[0])
    kept8 = npu.npu_gated_ffn_keep(x, w1, w2, bias1=b1, bias2=b2, residual=r, activation=act, checkpoint_int8=True)
    assert torch.equal(y, kept8[0])
    # what is kept: the values before the activation, rounded once; in 8 bits within half a step
    z, e = mm(x.double(), w1.double())
    if b1 is not None:
        z, e = z + b1.double(), e + 2.0 ** -23 * b1.double().abs()
    i8, i64 = -(-inner // 8) * 8, -(-inner // 64) * 64
    for half in range(2):
        zh, eh = z[:, half * inner:(half + 1) * inner], e[:, half * inner:(half + 1) * inner]
        check(kept[1][:, half * i8:half * i8 + inner], zh, eh, "kept")
        q = kept8[1][:, half * i64:(half + 1) * i64]
        s = kept8[2][:, half * i64 // 64:(half + 1) * i64 // 64]
        step = s.double().repeat_interleave(64, 1)[:, :inner]
        off = (deq64(q[:, :inner], s) - zh).abs()
        assert (off <= 0.5 * step * (1 + 2.0 ** -20) + eh).all(), "8-bit kept values"
        assert (q[:, :inner].abs().max() == 127) and (q[:, inner:] == 0).all()
    want_q, want_s = quant64(x)
    assert torch.equal(kept8[3], want_q) and torch.equal(kept8[4], want_s)


# ---- gradients -----------------------------------------------------------------------------------------------------------
def ref_ffn_grads(x64, kept_g, kept_u, w1, w2, dy, act, dtype):
    """Gradients at the kept values, with bounds; dz and h are rounded to the 16-bit type on the way."""
    u = U(dtype)
    inner = w2.shape[0]
    a, d = act64(kept_g, act)
    dh, edh = mm(dy, w2.double().t())
    h = a * kept_u
    eh = S * (1 + kept_g.abs()) * kept_u.abs()
    eh = eh + u * (h.abs() + eh) + tiny(dtype)
    dg, du = dh * kept_u * d, dh * a
    edg = edh * (kept_u * d).abs() + (dh.abs() + edh) * kept_u.abs() * 2 * S * (1 + kept_g.abs())
    edu = edh * a.abs() + (dh.abs() + edh) * S * (1 + kept_g.abs())
    dz, edz = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    edz = edz + (u + 2.0 ** -22) * (dz.abs() + edz) + tiny(dtype)
    dx, edx = mm(dz, w1.double().t())
    dw1, ew1 = mm(x64.t(), dz)
    dw2, ew2 = mm(h.t(), dy)
    m = x64.shape[0]
    return {"x": (dx, edx + edz @ w1.double().abs().t() * (1 + G(2 * inner))),
            "weight1": (dw1, ew1 + x64.abs().t() @ edz * (1 + G(m))),
            "weight2": (dw2, ew2 + eh.t() @ dy.abs() * (1 + G(m))),
            "bias1": (dz.sum(0), edz.sum(0) * (1 + G(m)) + G(m) * dz.abs().sum(0)),
            "bias2": (dy.sum(0), G(m) * dy.abs().sum(0))}


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
@pytest.mark.parametrize("case", FFN, ids=str)
def test_gated_ffn_gradients(dev, case, int8):
    m, h, inner, transposed, act, bias, residual = case
    dtype = DTYPES[m % 2]
    g = gen(m + 3 * h)
    x = make(g, m, h, dtype=dtype)
    w1, w2 = weight(g, h, 2 * inner, transposed, dtype), weight(g, inner, h, transposed, dtype)
    b1, b2 = (make(g, 2 * inner, dtype=dtype), make(g, h, dtype=dtype)) if bias else (None, None)
    r = make(g, m, h, dtype=dtype) if residual else None
    dy = make(g, m, h, dtype=dtype, scale=0.25)
    leaves = {"x": x, "weight1": w1, "weight2": w2, "bias1": b1, "bias2": b2, "residual": r}
    leaves = {k: v.detach().requires_grad_() for k, v in leaves.items() if v is not None}
    args = [leaves[k] for k in ("x", "weight1", "weight2")]
    kw = {k: leaves[k] for k in ("bias1", "bias2", "residual") if k in leaves}
    y = npu.npu_gated_ffn(*args, **kw, activation=act, checkpoint_int8=int8)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    kept = npu.npu_gated_ffn_keep(x, w1, w2, bias1=b1, bias2=b2, residual=r, activation=act, checkpoint_int8=int8)
    assert torch.equal(kept[0], y)
    if int8:
        i64 = -(-inner // 64) * 64
        kg, ku = (deq64(kept[1][:, o:o + inner], kept[2][:, o // 64:]) for o in (0, i64))
        x64 = deq64(kept[3], kept[4])
        # x goes into its product rounded to the 16-bit type
        x64 = x64.to(dtype).double()
    else:
        i8 = -(-inner // 8) * 8
        kg, ku = kept[1][:, :inner].double(), kept[1][:, i8:i8 + inner].double()
        x64 = x.double()
    want = ref_ffn_grads(x64, kg, ku, w1, w2, dy.double(), act, dtype)
    for name in leaves:
        if name == "residual":
            assert torch.equal(got[name], dy)
        else:
            check(got[name], *want[name], f"d{name} {case}")
    if transposed:
        assert got["weight1"].stride(0) == 1 and got["weight2"].stride(0) == 1, "the gradient lies in memory as its weight does"


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
@pytest.mark.parametrize("case", LINEAR, ids=str)
def test_linear_act_gradients(dev, case, int8):
    m, k, n, transposed, act, bias, residual = case
    dtype = DTYPES[(m + 1) % 2]
    g = gen(m + 5 * k)
    x, w = make(g, m, k, dtype=dtype), weight(g, k, n, transposed, dtype)
    b = make(g, n, dtype=dtype) if bias else None
    r = make(g, m, n, dtype=dtype) if residual else None
    dy = make(g, m, n, dtype=dtype, scale=0.25)
    leaves = {k_: v.detach().requires_grad_() for k_, v in {"x": x, "weight": w, "bias": b, "residual": r}.items() if v is not None}
    kw = {k_: leaves[k_] for k_ in ("bias", "residual") if k_ in leaves}
    y = npu.npu_linear_act(leaves["x"], leaves["weight"], **kw, activation=act, checkpoint_int8=int8)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    kept = npu.npu_linear_act_keep(x, w, bias=b, residual=r, activation=act, checkpoint_int8=int8)
    assert torch.equal(kept[0], y)
    x64 = x.double()
    if int8:
        x64 = deq64(kept[3], kept[4]).to(dtype).double()
    dz, edz = dy.double(), torch.zeros(m, n, dtype=torch.float64, device="cuda")
    if act != "none":
        z = deq64(kept[1][:, :n], kept[2]) if int8 else kept[1][:, :n].double()
        zref, ez = mm(x.double(), w.double())
        if b is not None:
            zref, ez = zref + b.double(), ez + 2.0 ** -23 * b.double().abs()
        if int8:
            step = kept[2].double().repeat_interleave(64, 1)[:, :n]
            assert ((z - zref).abs() <= 0.5 * step * (1 + 2.0 ** -20) + ez).all()
        else:
            check(kept[1][:, :n], zref, ez, "kept")
        d = act64(z, act)[1]
        dz = dy.double() * d
        edz = dy.double().abs() * 2 * S * (1 + z.abs())
        edz = edz + (U(dtype) + 2.0 ** -22) * (dz.abs() + edz) + tiny(dtype)
    dx, edx = mm(dz, w.double().t())
    dw, edw = mm(x64.t(), dz)
    check(got["x"], dx, edx + edz @ w.double().abs().t() * (1 + G(n)), f"dx {case}")
    check(got["weight"], dw, edw + x64.abs().t() @ edz * (1 + G(m)), f"dw {case}")
    if b is not None:
        check(got["bias"], dz.sum(0), edz.sum(0) * (1 + G(m)) + G(m) * dz.abs().sum(0), f"db {case}")
    if r is not None:
        assert torch.equal(got["residual"], dy)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(dev, act):
    """Directional derivatives: fp16 operands, a step that is exact in fp16, differences of the 64-bit reference's own formula
    around the same point (so the bound is the reference's: curvature times the step squared)."""
    g = gen(11)
    dtype, m, h, inner = torch.float16, 40, 64, 48
    x, w1, w2 = make(g, m, h, dtype=dtype), weight(g, h, 2 * inner, False, dtype), weight(g, inner, h, True, dtype)
    dy = make(g, m, h, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w1, w2)]
    grads = torch.autograd.grad(npu.npu_gated_ffn(*leaves, activation=act), leaves, dy)

    def loss(x_, w1_, w2_):
        z = x_ @ w1_
        return (((act64(z[:, :inner], act)[0] * z[:, inner:]) @ w2_) * dy.double()).sum()

    point = [t.double() for t in (x, w1, w2)]
    for i in range(3):
        v = torch.randn(point[i].shape, generator=g, device="cuda", dtype=torch.float64)
        eps = 1e-4
        hi, lo = list(point), list(point)
        hi[i], lo[i] = point[i] + eps * v, point[i] - eps * v
        slope = (loss(*hi) - loss(*lo)) / (2 * eps)
        got = (grads[i].double() * v).sum()
        # every gradient value carries a few roundings of 2^-11; their errors are independent of v: 8 u |grad| |v| in the 2-norm
        bound = 8 * U(dtype) * grads[i].double().norm() * v.norm()
        assert (got - slope).abs() <= bound, f"{i}: {got} {slope} {bound}"


# ---- the forms that the choice of kernel leads to ------------------------------------------------------------------------
# together with the lists above, every kernel, tile height and kind of split that the three products of a block can take
FFN_FORMS = [
    (1024, 2048, 1024, False, "silu", False, True),
    (2001, 1024, 1024, True, "gelu", True, False),
    (701, 4096, 2048, False, "silu", True, False),
    (1000, 4096, 1024, True, "gelu_tanh", True, True),
    (3000, 4096, 2048, False, "silu", False, False),
    (2000, 64, 264, True, "silu", True, False),
    (3001, 4096, 8, False, "relu", True, True),
    (4095, 64, 520, False, "silu", True, True),
    (33, 64, 8, True, "none", True, False),
    (2999, 4096, 136, True, "gelu_tanh", True, False),
    (1023, 1024, 1001, False, "silu", True, False),
]
LINEAR_FORMS = [
    (3001, 3000, 8, False, "gelu", True, True),
    (4097, 2000, 520, False, "silu", True, False),
    (4100, 520, 2000, True, "none", False, True),
    # results whose rows are not whole 16-byte pieces
    (3000, 4096, 5, False, "silu", True, True),
    (9, 1000, 517, True, "gelu", True, True),
    (17, 1500, 261, False, "relu", True, False),
    (40, 2001, 263, True, "gelu_tanh", False, True),
    (129, 4096, 7165, False, "silu", True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", FFN_FORMS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gated_ffn_in_every_form(dev, case, dtype):
    test_gated_ffn(dev, case, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
@pytest.mark.parametrize("case", FFN_FORMS, ids=str)
def test_gated_ffn_gradients_in_every_form(dev, case, int8):
    test_gated_ffn_gradients(dev, case, int8)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
@pytest.mark.parametrize("case", LINEAR_FORMS, ids=str)
def test_linear_act_gradients_in_every_form(dev, case, int8):
    test_linear_act(dev, case, DTYPES[int8])
    test_linear_act_gradients(dev, case, int8)


def _forms(gated, m, n, k, a_mn=0):
    """The kernel forms of one product: (product, kernel, rows of a tile or share, ...)."""
    import ctypes
    plan = (ctypes.c_int64 * 4)()
    _lib.call("tab_dense_plan", gated, m, n, k, a_mn, plan)
    rows, tiles, share, rest = plan
    name = ("linear", "linear mn")[a_mn] if gated == 0 else ("glu", "glu grad")[gated - 1]
    if gated == 0 and n % 8:
        name = "linear any"
    if rows:
        assert rows in (16, 32, 64, 128, 256) and tiles >= -(-m // rows) and 1 <= share <= 8 and share <= -(-k // 64)
        return {(name, "narrow", rows, share > 1)}
    assert rest <= tiles and share in (1, 2, 4) and (share > 1) == (rest > 0)
    return ({(name, "pair", 1)} if rest < tiles else set()) | ({(name, "pair", share)} if rest else set())


def test_every_form_that_the_choice_of_kernel_leads_to_is_tested(built_library):
    """The plans over a grid of sizes, and those of the cases above: a change of the estimates that leads to a form without a case fails
    here."""
    tested = set()
    for m, h, inner, *_ in FFN + FFN_FORMS:
        i8 = -(-inner // 8) * 8
        tested |= _forms(1, m, i8, h) | _forms(0, m, h, inner) | _forms(2, m, i8, h) | _forms(0, m, h, 2 * i8)
        tested |= _forms(0, h, 2 * i8, m, 1) | _forms(0, inner, h, m, 1)
    for m, k, n, transposed, *_ in LINEAR + LINEAR_FORMS:
        tested |= _forms(0, m, n, k) | _forms(0, m, k, n) | (_forms(0, n, k, m, 1) if transposed else _forms(0, k, n, m, 1))
    reached = set()
    for m in (1, 16, 17, 32, 33, 64, 65, 80, 100, 128, 129, 160, 200, 256, 257, 300, 384, 400, 512, 600, 700, 1000, 1024, 1500, 2000, 2048, 4096):
        for n in (5, 8, 64, 72, 128, 136, 200, 256, 261, 264, 517, 520, 640, 768, 1000, 1024, 1408, 2048, 2056, 2816, 4096, 7165, 7168, 8192):
            for k in (8, 64, 128, 200, 256, 512, 768, 1024, 1536, 2048, 4096, 7168, 8192, 16384):
                for gated, a_mn in ((0, 0), (0, 1), (1, 0), (2, 0)) if n % 8 == 0 else ((0, 0),):
                    reached |= _forms(gated, m, n, k, a_mn)
    assert reached <= tested, sorted(reached - tested)
    assert len(reached) > 30


def test_few_rows_share_tiles_as_far_as_all_ctas_are_resident(built_library):
    """The rule for up to 64 rows, at every number of tiles: the largest cluster of which the GPU holds enough at a time."""
    import ctypes
    room = {1: 148, 2: 148, 3: 135, 4: 132, 5: 130, 6: 132, 7: 105, 8: 120}        # CTAs in clusters of that size, one to an SM
    plan = (ctypes.c_int64 * 4)()
    for m, per_sm in ((1, 2), (8, 2), (32, 2), (33, 1), (64, 1)):
        for k in (64, 640, 1408, 8192):
            for tiles in range(1, 400):
                for gated, features in ((0, 128), (1, 64), (2, 128)):
                    _lib.call("tab_dense_plan", gated, m, tiles * features, k, 0, plan)
                    fit = [s for s in room if s == 1 or tiles * s <= per_sm * room[s] and s * 5 <= -(-k // 64)]
                    assert list(plan)[1:3] == [tiles, max(fit)], (m, k, tiles, gated)


# ---- 8-bit checkpoints ---------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 64), (3, 63), (5, 65), (7, 8), (4, 1024), (37, 1003), (2, 3, 200), (1000, 192), (300, 7168), (0, 64), (4, 0)], ids=str)
def test_checkpoint_round_trip(dev, shape, dtype):
    g = gen(sum(shape))
    x = make(g, *shape, dtype=dtype) * 3
    if x.numel() > 64:
        x.view(-1)[:64] = 0                                   # a block (at least part of one) of zeros
        x[-1] *= 1e-3
    q, scale = npu.npu_checkpoint_quant(x)
    flat = x.reshape(math.prod(shape[:-1]), shape[-1])
    if x.numel():
        want_q, want_s = quant64(flat)
        assert torch.equal(scale.view(flat.shape[0], -1), want_s)
        assert torch.equal(q.view(flat.shape), want_q)
    for code, out in ((5, torch.float16), (6, torch.float32), (15, torch.bfloat16)):
        y = npu.npu_checkpoint_dequant(q, scale, output_dtype=code)
        assert y.dtype == out and y.shape == x.shape
        if x.numel():
            want = (q.view(flat.shape).float() * scale.view(flat.shape[0], -1).repeat_interleave(64, 1)[:, :shape[-1]]).to(out)
            assert torch.equal(y.view(flat.shape), want)


@pytest.mark.gpu
def test_checkpoint_of_strided_and_shifted_inputs(dev):
    g = gen(5)
    base = make(g, 50, 400)
    for x in (base[:, :128], base[:, 8:136], base[:, 3:131], base[::2, 1:66], base.t(), base.t()[:, 1:], base[:, :64].unsqueeze(1)):
        q, s = npu.npu_checkpoint_quant(x)
        qc, sc = npu.npu_checkpoint_quant(x.contiguous())
        assert torch.equal(q, qc) and torch.equal(s, sc)
        assert torch.equal(npu.npu_checkpoint_dequant(q.transpose(0, 1).contiguous().transpose(0, 1), s), npu.npu_checkpoint_dequant(qc, sc))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32], ids=str)
def test_checkpoint_keeps_what_is_not_finite_visible(dev, dtype):
    x = torch.ones(4, 256, dtype=dtype, device=dev)
    x[0, 70], x[1, 0], x[2, 255] = float("inf"), float("nan"), float("-inf")
    q, s = npu.npu_checkpoint_quant(x)
    y = npu.npu_checkpoint_dequant(q, s, output_dtype=6)
    bad = torch.zeros(4, 4, dtype=torch.bool, device=dev)
    bad[0, 1] = bad[1, 0] = bad[2, 3] = True
    assert torch.equal(torch.isnan(y.view(4, 4, 64)).all(-1), bad) and torch.equal(torch.isnan(y.view(4, 4, 64)).any(-1), bad)
    assert (y[~torch.isnan(y)] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(1, 8, 8), (37, 200, 136), (300, 65, 33), (2000, 512, 1024), (4096, 1024, 72)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_checkpoint_weight_grad(dev, case, dtype):
    m, k, n = case
    g = gen(m)
    q, s = npu.npu_checkpoint_quant(make(g, m, k, dtype=dtype))
    dy = make(g, m, n, dtype=dtype)
    x64 = deq64(q, s).to(dtype).double()
    dw, e = mm(x64.t(), dy.double())
    check(npu.npu_checkpoint_weight_grad(q, s, dy), dw, e, f"weight grad {case}")
    assert torch.equal(npu.npu_checkpoint_weight_grad(q.view(1, m, k), s.view(1, m, -1), dy.view(1, m, n)), npu.npu_checkpoint_weight_grad(q, s, dy))


@pytest.mark.gpu
def test_checkpoint_weight_grad_beyond_the_range_of_fp16(dev):
    """The input goes into the product in the gradient's type: what does not fit becomes infinite or zero there, as a cast makes it, and
    stays in its own rows of the result; bf16 has the range."""
    g = gen(20)
    size = torch.cat((torch.ones(64), torch.full((64,), 1e6), torch.full((2,), 1e-9))).to(dev)
    x = (1 + torch.rand(48, 130, generator=g, device=dev)) * size
    q, s = npu.npu_checkpoint_quant(x)
    for dtype in DTYPES:
        dy = make(g, 48, 72, dtype=dtype)
        got = npu.npu_checkpoint_weight_grad(q, s, dy)
        x64 = deq64(q, s).to(dtype).double()
        ok = slice(0, 64) if dtype == torch.float16 else slice(0, 130)
        want, e = mm(x64[:, ok].t(), dy.double())
        check(got[ok], want, e, "in range")
        if dtype == torch.float16:
            assert not torch.isfinite(got[64:128]).any() and (got[128:] == 0).all()


# ---- layouts, sizes, values ----------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_operands_of_other_strides(dev):
    """Column slices, row gaps, shifted starts, broadcast rows: the same bits as their contiguous copies."""
    g = gen(3)
    big = make(g, 300, 700)
    wbig = make(g, 700, 900, scale=0.05)
    for m in (40, 200):
        for x, w in ((big[:m, :256], wbig[:256, :512]), (big[:m, 8:264], wbig[:256, 8:520]), (big[:m, 3:259], wbig[1:257, 5:517]),
                     (big[:2 * m:2, :256] if m == 40 else big[:m, :256], wbig.t()[:256, :512]), (big.t()[:m, :256], wbig[::2, ::1][:256, :512]),
                     (big[:1, :256].expand(m, 256), wbig.t()[3:259, 5:517]), (big[:m, :512:2], wbig[:256, 1::2][:, :440])):
            want = npu.npu_linear_act(x.contiguous(), w.contiguous(), activation="silu")
            assert torch.equal(npu.npu_linear_act(x, w, activation="silu"), want)
            w2 = wbig[:w.shape[1] // 2, :256].contiguous()
            assert torch.equal(npu.npu_gated_ffn(x, w, w2), npu.npu_gated_ffn(x.contiguous(), w.contiguous(), w2))
        r = big[:m, 1:513:2][:, :256]
        x, w = big[:m, :64], wbig[:64, :256]
        b = wbig[0, 1:513:2]
        want = npu.npu_linear_act(x.contiguous(), w.contiguous(), residual=r.contiguous(), bias=b.contiguous())
        assert torch.equal(npu.npu_linear_act(x, w, residual=r, bias=b), want)
    # gradients that arrive as a broadcast scalar
    x = make(g, 20, 64).requires_grad_()
    w = make(g, 64, 72).requires_grad_()
    npu.npu_linear_act(x, w, activation="gelu").sum().backward()
    dx, dw = torch.autograd.grad(npu.npu_linear_act(x, w, activation="gelu"), (x, w), torch.ones(20, 72, device=dev, dtype=x.dtype))
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)


@pytest.mark.gpu
def test_leading_dimensions_and_empty_batches(dev):
    g = gen(4)
    x, w1, w2 = make(g, 2, 3, 5, 64), make(g, 64, 96, scale=0.1), make(g, 48, 64, scale=0.1)
    y = npu.npu_gated_ffn(x, w1, w2, residual=x)
    assert y.shape == x.shape and torch.equal(y.view(30, 64), npu.npu_gated_ffn(x.view(30, 64), w1, w2, residual=x.view(30, 64)))
    assert torch.equal(npu.npu_linear_act(x[0, 0, 0], w1), npu.npu_linear_act(x[0, 0, :1], w1)[0])
    for int8 in (False, True):
        e = torch.empty(0, 64, dtype=x.dtype, device=dev, requires_grad=True)
        p1, p2 = w1.detach().requires_grad_(), w2.detach().requires_grad_()
        for y, ps in ((npu.npu_gated_ffn(e, p1, p2, checkpoint_int8=int8), (p1, p2)),
                      (npu.npu_linear_act(e, p1, activation="silu", checkpoint_int8=int8), (p1,))):
            assert y.shape[0] == 0
            grads = torch.autograd.grad(y, (e,) + ps, torch.empty_like(y))
            assert grads[0].shape == e.shape and all((t == 0).all() and t.shape == p.shape for t, p in zip(grads[1:], ps))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 150])
def test_nan_and_infinity_stay_in_their_rows(dev, m):
    g = gen(6)
    x, w1, w2 = make(g, m, 128), make(g, 128, 256, scale=0.1), make(g, 128, 128, scale=0.1)
    want = npu.npu_gated_ffn(x, w1, w2)
    bad = x.clone()
    bad[1, 3], bad[m - 1, 100] = float("nan"), float("inf")
    got = npu.npu_gated_ffn(bad, w1, w2)
    rows = torch.ones(m, dtype=torch.bool, device=dev)
    rows[1] = rows[m - 1] = False
    assert torch.equal(got[rows], want[rows]) and torch.isnan(got[1]).all() and not torch.isfinite(got[m - 1]).any()
    # an fp16 result over the type's range becomes infinite, as a conversion does
    big = torch.full((m, 64), 200.0, dtype=torch.float16, device=dev)
    assert torch.isinf(npu.npu_linear_act(big, big[:1].expand(64, 64).contiguous())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("inner", [33, 40])
@pytest.mark.parametrize("m", [5, 300])
def test_padding_of_the_inner_features_adds_nothing_to_infinities(dev, m, inner):
    """Weights and values are positive, so a row that holds an infinity has infinities and no NaN in its results and gradients,
    whether or not the inner features are padded to a multiple of 8.  (The gradient of up * relu(gate) at gate = up = inf is
    dh * up * 1 and dh * gate.)"""
    g = gen(inner + m)
    x, dy = make(g, m, 48).abs() + 0.125, make(g, m, 48).abs() + 0.125
    w1, w2 = make(g, 48, 2 * inner).abs() + 0.125, make(g, inner, 48).abs() + 0.125
    x[2, 3] = math.inf
    dy[3, 5] = math.inf
    leaf = x.clone().requires_grad_()
    y = npu.npu_gated_ffn(leaf, w1, w2, activation="relu")
    dx, = torch.autograd.grad(y, leaf, dy)
    inf = torch.zeros(m, dtype=torch.bool, device=dev)
    inf[2] = True
    assert torch.equal(torch.isposinf(y), inf[:, None].expand_as(y)) and not torch.isnan(y).any()
    inf[3] = True
    assert torch.equal(torch.isposinf(dx), inf[:, None].expand_as(dx)) and not torch.isnan(dx).any()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_gradient_at_nan_is_nan(dev, act):
    """as in the formulas: also of relu, where neither branch holds at NaN"""
    x = torch.ones(4, 8, dtype=torch.bfloat16, device=dev)
    x[1, 0] = math.nan
    w = torch.ones(8, 16, dtype=torch.bfloat16, device=dev)
    leaf = x.requires_grad_()
    dx, = torch.autograd.grad(npu.npu_linear_act(leaf, w, activation=act), leaf, torch.ones(4, 16, dtype=torch.bfloat16, device=dev))
    nan = torch.tensor([False, act != "none", False, False], device=dev)
    assert torch.equal(torch.isnan(dx), nan[:, None].expand_as(dx))


@pytest.mark.gpu
def test_gradients_have_the_strides_that_the_meta_implementation_gives(dev):
    meta = lambda t: t if not isinstance(t, torch.Tensor) else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="meta")
    g = gen(16)
    for m in (0, 3):
        for transposed in (False, True):
            for h, inner in ((16, 24), (9, 5), (1, 1)):
                w1, w2 = weight(g, h, 2 * inner, transposed, torch.float16), weight(g, inner, h, transposed, torch.float16)
                x = make(g, m, h, dtype=torch.float16)
                y, kept, ks, xq, xs = npu.npu_gated_ffn_keep(x, w1, w2)
                for op, args in ((npu.npu_gated_ffn_backward, (y, x, xs, w1, w2, kept, ks, "silu", [True] * 5)),
                                 (npu.npu_linear_act_backward, (make(g, m, 2 * inner, dtype=torch.float16), x, xs, w1, kept, ks, "none", [True] * 3))):
                    for real, want in zip(op(*args), op(*[meta(a) for a in args])):
                        assert real.shape == want.shape and real.stride() == want.stride() and real.dtype == want.dtype


@pytest.mark.gpu
def test_rows_of_a_batch_do_not_depend_on_each_other(dev):
    """The same row at another place of a batch of the same size gives the same bits; other rows do not touch it."""
    g = gen(8)
    w = make(g, 512, 1000, scale=0.05)
    for m in (16, 100, 700):
        x = make(g, m, 512)
        y = npu.npu_linear_act(x, w, activation="gelu_tanh")
        perm = torch.randperm(m, generator=torch.Generator().manual_seed(m)).to(dev)
        assert torch.equal(npu.npu_linear_act(x[perm], w, activation="gelu_tanh"), y[perm])


@pytest.mark.gpu
def test_large_offsets(dev):
    """More than 2^31 elements in one operand: rows behind that offset are computed from their own values."""
    g = gen(9)
    m, k, n = 2 ** 31 // 4096 + 300, 4096, 64
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=dev)
    tail = make(g, 280, k)
    x[-280:] = tail
    w = make(g, k, n, scale=0.02)
    y = npu.npu_linear_act(x, w, activation="silu")
    check(y[-280:], *ref_linear(tail, w, None, None, "silu"), "tail")
    assert (y[:1000] == 0).all()
    q, s = npu.npu_checkpoint_quant(x)
    want_q, want_s = quant64(tail)
    assert torch.equal(q[-280:], want_q) and torch.equal(s[-280:], want_s)
    del y, s
    dy = torch.zeros(m, n, dtype=torch.bfloat16, device=dev)
    dy[-280:] = make(g, 280, n)
    xl, wl = x.requires_grad_(), w.detach().requires_grad_()
    dw, = torch.autograd.grad(npu.npu_linear_act(xl, wl), (wl,), dy)
    want, e = mm(tail.double().t(), dy[-280:].double())
    check(dw, want, e, "dw")


# ---- streams, graphs, compile --------------------------------------------------------------------------------------------
def _train_step(x, w1, w2, w, dy, int8):
    h = npu.npu_gated_ffn(x, w1, w2, residual=x, checkpoint_int8=int8)
    y = npu.npu_linear_act(h, w, activation="gelu", checkpoint_int8=int8)
    # detached: a live eager graph of the same leaves would tie a later capture to the stream that it ran on
    return (y.detach(),) + torch.autograd.grad(y, (x, w1, w2, w), dy)


def _step_inputs(m, seed=0, h=256, inner=200, n=520):
    g = gen(seed)
    x, dy = make(g, m, h), make(g, m, n)
    ws = (weight(g, h, 2 * inner, False, torch.bfloat16), weight(g, inner, h, True, torch.bfloat16), weight(g, h, n, True, torch.bfloat16))
    return [x.requires_grad_()] + [w.detach().requires_grad_() for w in ws] + [dy]


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
@pytest.mark.parametrize("m", [3, 100, 700])
def test_a_run_of_them_on_other_streams_and_in_graphs(dev, m, int8):
    """A feed-forward block, a projection behind it and their backward pass: the current stream, a side stream, two captured
    graphs replayed in turn, all with the same bits."""
    ins = _step_inputs(m)
    want = _train_step(*ins, int8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _train_step(*ins, int8)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    # inference parts captured twice, replayed in turn, each with its own workspaces
    x, w1, w2, w, _ = [t.detach() for t in ins]
    static = x.clone()
    graphs, outs = [], []
    for _ in range(2):
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            outs.append(npu.npu_linear_act(npu.npu_gated_ffn(static, w1, w2, residual=static), w, activation="gelu"))
        graphs.append(gph)
    for i in range(4):
        nx = make(gen(50 + i), *x.shape)
        static.copy_(nx)
        graphs[i % 2].replay()
        graphs[(i + 1) % 2].replay()
        y = npu.npu_linear_act(npu.npu_gated_ffn(nx, w1, w2, residual=nx), w, activation="gelu")
        assert torch.equal(outs[0], y) and torch.equal(outs[1], y)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 200, 2000])
def test_every_operand_written_by_the_call_before(dev, m):
    """Launches overlap the end of the one before; what that one writes (x, weight, bias, residual, an 8-bit checkpoint, a gradient)
    or still reads must be waited for.  The same calls with the GPU idle before each give the same bits."""
    g = gen(m)
    h = 512
    x, w, v = make(g, m, h), make(g, h, h, scale=h ** -0.5), make(g, h, h, scale=h ** -0.5)

    def chain(wait):
        def call(f, *args, **kwargs):
            if wait:
                torch.cuda.synchronize()
            return f(*args, **kwargs)

        out = []
        for _ in range(4):
            weight2 = call(npu.npu_linear_act, w, v)                                   # written here, used as a weight
            y = call(npu.npu_linear_act, x, weight2, activation="relu")
            y = call(npu.npu_linear_act, x, w, residual=y)                             # as the residual
            weight1 = call(npu.npu_linear_act, v, torch.cat((w, v), 1))
            y = call(npu.npu_gated_ffn, y, weight1, weight2)
            b = call(npu.npu_linear_act, y[:1], w)[0]
            y = call(npu.npu_linear_act, y, w.t(), bias=b)                             # as the bias
            q, s = call(npu.npu_checkpoint_quant, y)
            d = call(npu.npu_checkpoint_weight_grad, q, s, x)
            y = call(npu.npu_checkpoint_dequant, *call(npu.npu_checkpoint_quant, call(npu.npu_linear_act, y, d)))
            leaf = y.detach().requires_grad_()
            z = call(npu.npu_gated_ffn, leaf, weight1, weight2, checkpoint_int8=True)
            dx, = torch.autograd.grad(z, leaf, call(npu.npu_linear_act, x, weight2))
            out += [y, d, z.detach(), dx]
            del weight1, weight2, b, q, s, z, leaf                                     # their memory goes to the next calls
        torch.cuda.synchronize()
        return out

    want = chain(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))


@pytest.mark.gpu
def test_a_graph_whose_branches_meet(dev):
    """Captured calls after a fork and a join: launches with several predecessors."""
    g = gen(17)
    x, w = make(g, 24, 256), make(g, 256, 256, scale=1 / 16)

    def work(side):
        a = npu.npu_linear_act(x, w, activation="silu")
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b = npu.npu_linear_act(a, w, activation="gelu")
        c = npu.npu_gated_ffn(a, torch.cat((w, w), 1), w)
        here.wait_stream(side)
        return npu.npu_linear_act(c, w, residual=b)

    side = torch.cuda.Stream()
    want = work(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(side)
    for _ in range(20):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls that overlap on two streams share nothing."""
    a, b = _step_inputs(700, seed=1), _step_inputs(90, seed=2)
    want_a, want_b = _train_step(*a, True), _train_step(*b, False)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            outs.append((_train_step(*a, True), want_a))
        with torch.cuda.stream(s2):
            outs.append((_train_step(*b, False), want_b))
    torch.cuda.synchronize()
    for got, want in outs:
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
def test_first_cuda_call_of_a_thread(dev):
    import threading
    ins = [t.detach() for t in _step_inputs(20)]
    x, w1, w2, w, _ = ins
    want = npu.npu_linear_act(npu.npu_gated_ffn(x, w1, w2), w)
    got = []
    thread = threading.Thread(target=lambda: got.append(npu.npu_linear_act(npu.npu_gated_ffn(x, w1, w2), w)))
    thread.start()
    thread.join()
    assert torch.equal(got[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [300, 2000])
def test_two_threads_on_one_stream(dev, m):
    """One host thread runs backward passes, another forward passes on the same stream: memory that either frees goes to the other while
    launches of both are in flight, and every result has the bits of the same calls alone."""
    import threading
    g = gen(m + 18)
    h = inner = 512                      # hidden rows, gradients and results of one size: they fit each other's memory
    x, dy, nx = make(g, m, h), make(g, m, h), make(g, m, h)
    w1, w2 = weight(g, h, 2 * inner, False, x.dtype), weight(g, inner, h, False, x.dtype)
    _, kept, ks, xq, xs = npu.npu_gated_ffn_keep(x, w1, w2, checkpoint_int8=True)
    _, lkept, lks, _, lxs = npu.npu_linear_act_keep(x, w1, activation="gelu")
    dyl = make(g, m, 2 * inner)

    def train():
        return npu.npu_gated_ffn_backward(dy, xq, xs, w1, w2, kept, ks, "silu", [True] * 5) + \
            npu.npu_linear_act_backward(dyl, x, lxs, w1, lkept, lks, "gelu", [True, True, False])[:2]

    def infer():
        return npu.npu_gated_ffn(nx, w1, w2), npu.npu_linear_act(nx, w1, activation="silu")

    want = train(), infer()
    torch.cuda.synchronize()
    start, failed = threading.Barrier(2), []

    def loop(call, want):
        try:
            start.wait()
            for _ in range(40):
                outs = [call() for _ in range(5)]
                if not all(torch.equal(a, b) for out in outs for a, b in zip(out, want)):
                    failed.append(call.__name__)
        except BaseException as e:       # seen by the test, not only by the thread
            failed.append(repr(e))

    threads = [threading.Thread(target=loop, args=a) for a in ((train, want[0]), (infer, want[1]))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.gpu
def test_training_step_in_a_graph(dev):
    ins = _step_inputs(300)
    want = [t.clone() for t in _train_step(*ins, True)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            _train_step(*ins, True)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _train_step(*ins, True)
    for t in outs:
        t.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
def test_only_the_wanted_gradients_and_no_second_order(dev):
    ins = _step_inputs(40)
    x, w1, w2, w, dy = ins
    y = npu.npu_linear_act(x.detach(), w, activation="silu")
    dw, = torch.autograd.grad(y, w, dy)
    full = npu.npu_linear_act(x, w, activation="silu")
    dx2, dw2 = torch.autograd.grad(full, (x, w), dy, create_graph=True)
    assert torch.equal(dw, dw2.detach())
    with pytest.raises(RuntimeError):
        dx2.sum().backward()
    with torch.no_grad():
        assert not npu.npu_gated_ffn(x, w1, w2).requires_grad
    assert not npu.npu_gated_ffn(x.detach(), w1.detach(), w2.detach()).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
@pytest.mark.parametrize("frozen", ["weights", "input", "nothing"])
def test_a_second_differentiation_raises_and_loses_nothing(dev, frozen, int8):
    """Gradients made with create_graph depend on what they were made from: a term that differentiates one again raises, whichever
    inputs require gradients, instead of adding nothing to the other terms' gradients."""
    g = gen(19)
    t = {"x": make(g, 20, 64), "weight1": make(g, 64, 64, scale=0.1), "weight2": make(g, 32, 64, scale=0.1), "bias1": make(g, 64), "bias2": make(g, 64),
         "residual": make(g, 20, 64)}
    names = {"weights": ["x"], "input": ["bias1", "bias2"], "nothing": list(t)}[frozen]
    leaves = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
    wanted = [leaves[k] for k in names]

    def ffn():
        return npu.npu_gated_ffn(leaves["x"], leaves["weight1"], leaves["weight2"], bias1=leaves["bias1"], bias2=leaves["bias2"],
                                 residual=leaves["residual"], checkpoint_int8=int8)

    def linear():
        return npu.npu_linear_act(leaves["x"], leaves["weight1"], bias=leaves["bias1"], residual=leaves["residual"], activation="silu",
                                  checkpoint_int8=int8)

    for call in (ffn, linear):
        some = [p for k, p in zip(names, wanted) if call is ffn or k in ("x", "weight1", "bias1", "residual")]
        y = call()
        plain = torch.autograd.grad(y, some, torch.ones_like(y), retain_graph=True)
        for i, p in enumerate(some):
            grads = torch.autograd.grad(call().sum(), some, create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(grads, plain))
            if p is leaves["residual"]:
                continue                                     # the incoming gradient itself
            assert grads[i].requires_grad
            with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
                ((p * 2).sum() + grads[i].float().pow(2).sum()).backward()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(700, 256, 200), (3001, 512, 352), (77, 100, 33), (5, 64, 48)], ids=str)
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
def test_each_gradient_alone_equals_all_at_once(dev, case, int8):
    """The products of a backward pass overlap on the GPU; asked for one by one they cannot."""
    m, h, inner = case
    g = gen(m)
    x, dy = make(g, m, h), make(g, m, h)
    w1, w2 = weight(g, h, 2 * inner, False, x.dtype), weight(g, inner, h, True, x.dtype)
    b1, b2 = make(g, 2 * inner), make(g, h)
    _, kept, ks, xq, xs = npu.npu_gated_ffn_keep(x, w1, w2, bias1=b1, bias2=b2, checkpoint_int8=int8)
    src = xq if int8 else x
    for _ in range(3):
        both = npu.npu_gated_ffn_backward(dy, src, xs, w1, w2, kept, ks, "silu", [True] * 5)
        for i in range(5):
            one = npu.npu_gated_ffn_backward(dy, src, xs, w1, w2, kept, ks, "silu", [i == j for j in range(5)])
            assert torch.equal(one[i], both[i]) and all(t.numel() == 0 for j, t in enumerate(one) if j != i)
    w = weight(g, h, inner, True, x.dtype)
    _, kept, ks, xq, xs = npu.npu_linear_act_keep(x, w, activation="gelu", checkpoint_int8=int8)
    src, dyl = (xq if int8 else x), make(g, m, inner)
    both = npu.npu_linear_act_backward(dyl, src, xs, w, kept, ks, "gelu", [True] * 3)
    for i in range(3):
        one = npu.npu_linear_act_backward(dyl, src, xs, w, kept, ks, "gelu", [i == j for j in range(3)])
        assert torch.equal(one[i], both[i])


@pytest.mark.gpu
def test_gradients_of_some_inputs_only(dev):
    g = gen(14)
    t = {"x": make(g, 30, 64), "weight1": make(g, 64, 96, scale=0.1), "weight2": make(g, 48, 64, scale=0.1), "bias1": make(g, 96),
         "bias2": make(g, 64), "residual": make(g, 30, 64)}
    dy = make(g, 30, 64)

    def grads(names):
        leaves = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        y = npu.npu_gated_ffn(leaves["x"], leaves["weight1"], leaves["weight2"], **{k: leaves[k] for k in ("bias1", "bias2", "residual")})
        return dict(zip(names, torch.autograd.grad(y, [leaves[k] for k in names], dy)))

    full = grads(list(t))
    for names in (["bias1"], ["bias2"], ["residual"], ["x", "bias2"], ["weight2", "residual"], ["weight1"]):
        for k, v in grads(names).items():
            assert torch.equal(v, full[k]), (names, k)
    # a tensor that is an input twice gets both gradients
    x = t["x"].detach().requires_grad_()
    y = npu.npu_gated_ffn(x, t["weight1"], t["weight2"], bias1=t["bias1"], bias2=t["bias2"], residual=x)
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, (full["x"] + full["residual"]))


@pytest.mark.gpu
def test_outputs_that_lie_anywhere(dev):
    """The C entry with out, residual and bias one element past a 16-byte boundary, and what lies around out left alone."""
    import ctypes
    g = gen(15)
    for m in (20, 300):
        x, w = make(g, m, 64), make(g, 64, 136, scale=0.1)
        b, r = make(g, 137)[1:], make(g, m * 136 + 1)[1:]
        flat = torch.full((m * 136 + 9,), 7.0, dtype=x.dtype, device=dev)
        out = flat[1:1 + m * 136]
        none = ctypes.c_void_p(None)
        _lib.call("tab_dense_matmul", x.data_ptr(), 64, 0, w.data_ptr(), 136, 1, 15, m, 136, 64, b.data_ptr(), r.data_ptr(), 4, none, none, none, 0,
                  out.data_ptr(), 0, torch.cuda.current_stream(dev).cuda_stream)
        want = npu.npu_linear_act(x, w, bias=b, residual=r.view(m, 136), activation="silu")
        assert torch.equal(out.view(m, 136), want) and flat[0] == 7 and (flat[1 + m * 136:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
def test_traced_forward_and_backward(dev, int8):
    """The operators under AOT autograd: the same bits as eager, forward and gradients."""
    ins = _step_inputs(30)
    want = _train_step(*ins, int8)

    def model(x, w1, w2, w):
        h = npu.npu_gated_ffn(x, w1, w2, residual=x, checkpoint_int8=int8)
        return npu.npu_linear_act(h, w, activation="gelu", checkpoint_int8=int8)

    compiled = torch.compile(model, backend="aot_eager", fullgraph=True, dynamic=False)
    y = compiled(*ins[:4])
    got = (y.detach(),) + torch.autograd.grad(y, ins[:4], ins[4])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        assert torch.equal(model(*[t.detach() for t in ins[:4]]), want[0])


@pytest.mark.gpu
def test_compiled_by_the_backend(dev):
    ins = [t.detach() for t in _step_inputs(50)]
    x, w1, w2, w, _ = ins

    def model(x):
        return npu.npu_linear_act(npu.npu_gated_ffn(x, w1, w2, residual=x), w, activation="gelu")

    config = torchair_b200.CompilerConfig()
    config.mode = "reduce-overhead"
    compiled = torch.compile(model, backend=torchair_b200.get_npu_backend(compiler_config=config), dynamic=False)
    for i in range(3):
        nx = make(gen(70 + i), *x.shape)
        assert torch.equal(compiled(nx), model(nx))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["max-autotune", "reduce-overhead"])
@pytest.mark.parametrize("int8", [False, True], ids=["keep16", "keep8"])
def test_training_compiled_by_the_backend(dev, mode, int8):
    """What one forward pass keeps survives the next one, gradients survive the next backward pass, and weights that an optimiser changed
    are seen: eager bits throughout."""
    from torchair_b200 import backend

    class Block(torch.nn.Module):
        def __init__(self, *weights):
            super().__init__()
            self.w1, self.w2, self.w = (torch.nn.Parameter(t.detach().clone()) for t in weights)

        def forward(self, x):
            h = npu.npu_gated_ffn(x, self.w1, self.w2, residual=x, checkpoint_int8=int8)
            return npu.npu_linear_act(h, self.w, activation="gelu", checkpoint_int8=int8)

    ins = _step_inputs(50)
    eager, model = Block(*ins[1:4]), Block(*ins[1:4])
    config = torchair_b200.CompilerConfig()
    config.mode = mode
    compiled = torch.compile(model, backend=torchair_b200.get_npu_backend(compiler_config=config), dynamic=False)
    xs = [make(gen(80 + i), *ins[0].shape) for i in range(2)]
    before = backend.counters["captures"]
    for step in range(4):
        results = []
        for f, module in ((eager, eager), (compiled, model)):
            leaves = [x.clone().requires_grad_() for x in xs]
            params = list(module.parameters())
            ys = [f(x) for x in leaves]                                                   # both forward passes first
            results.append([y.detach() for y in ys] + [t for x, y in zip(leaves, ys) for t in torch.autograd.grad(y, [x] + params, ins[4])])
            with torch.no_grad():
                for p, d in zip(params, results[-1][-3:]):
                    p.sub_(d, alpha=2.0 ** -14)
        for i, (want, got) in enumerate(zip(*results)):
            assert torch.equal(got, want), (step, i)
    assert backend.counters["captures"] - before <= 4, "an optimiser's steps do not capture anew each time"
    with torch.no_grad():
        assert torch.equal(compiled(xs[0]), eager(xs[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [True, False])
def test_moe_layer_with_a_shared_expert(dev, fused):
    """The layer's shared expert is npu_gated_ffn handed to the combine; without one nothing changes."""
    from oracle import moe_oracle as O
    from torchair_b200.layer import moe_layer
    cfg = O.CONFIGS["cfg0"]
    w = O.make_weights(cfg, seed=3)
    x, ids, wt = (t.to(dev) for t in O.make_tokens(cfg, seed=3))
    args = (x, ids, wt, w.w1.to(dev), w.s1.to(dev), w.w2.to(dev), w.s2.to(dev))
    g = gen(2)
    h = x.shape[1]
    s1, s2 = weight(g, h, 512, True, x.dtype), weight(g, 256, h, True, x.dtype)
    plain = moe_layer(*args, fused=fused)
    got = moe_layer(*args, fused=fused, shared_w1=s1, shared_w2=s2)
    shared = npu.npu_gated_ffn(x, s1, s2)
    check(shared, *ref_ffn(x, s1, s2, None, None, None, "silu"), "shared expert")
    # the routed sum was rounded once in `plain`, and is not in `got`: both roundings apart
    off = (got.double() - plain.double() - shared.double()).abs()
    assert (off <= U(x.dtype) * (plain.double().abs() + got.double().abs()) + 2.0 ** -20).all()
    with pytest.raises(RuntimeError, match="both shared_w1 and shared_w2"):
        moe_layer(*args, fused=fused, shared_w1=s1)
    assert torch.equal(plain.cpu(), O.moe_layer([x.cpu()], [ids.cpu()], [wt.cpu()], w, [])[0])


@pytest.mark.gpu
@pytest.mark.parametrize("leaf", ["x", "shared_w1", "shared_w2"])
def test_a_gradient_through_moe_layer_raises(dev, leaf):
    """The routed half has no gradients, so a gradient of the shared expert through the layer is refused instead of lost; the forward
    result with parameters as weights is the same."""
    from oracle import moe_oracle as O
    from torchair_b200.layer import moe_layer
    cfg = O.CONFIGS["cfg0"]
    w = O.make_weights(cfg, seed=3)
    x, ids, wt = (t.to(dev) for t in O.make_tokens(cfg, seed=3))
    g = gen(2)
    t = {"x": x, "shared_w1": weight(g, x.shape[1], 512, True, x.dtype), "shared_w2": weight(g, 256, x.shape[1], True, x.dtype)}

    modes = []

    def call():
        return moe_layer(t["x"], ids, wt, w.w1.to(dev), w.s1.to(dev), w.w2.to(dev), w.s2.to(dev), shared_w1=t["shared_w1"], shared_w2=t["shared_w2"],
                         after_dispatch=lambda: modes.append(torch.is_grad_enabled()))

    want = call()
    t[leaf] = t[leaf].detach().requires_grad_()
    got = call()
    assert torch.equal(got.detach(), want)
    with pytest.raises(NotImplementedError, match="no backward pass"):
        (got.float().sum() + t[leaf].float().sum()).backward()
    with torch.no_grad():
        assert torch.equal(call(), want)
    assert modes == [True, True, False], "the caller's own work runs in the caller's mode"


@pytest.mark.gpu
def test_moe_layer_with_a_shared_expert_compiled(dev):
    """One graph, shared weights that require gradients included."""
    from oracle import moe_oracle as O
    from torchair_b200.layer import moe_layer
    cfg = O.CONFIGS["cfg0"]
    w = O.make_weights(cfg, seed=3)
    x, ids, wt = (t.to(dev) for t in O.make_tokens(cfg, seed=3))
    routed = [t.to(dev) for t in (w.w1, w.s1, w.w2, w.s2)]
    g = gen(2)
    shared = [weight(g, x.shape[1], 512, True, x.dtype).detach().requires_grad_(), weight(g, 256, x.shape[1], True, x.dtype).detach().requires_grad_()]

    def fn(x, ids, wt, w1, s1, w2, s2, a, b):
        return moe_layer(x, ids, wt, w1, s1, w2, s2, shared_w1=a, shared_w2=b)

    config = torchair_b200.CompilerConfig()
    config.mode = "reduce-overhead"
    compiled = torch.compile(fn, backend=torchair_b200.get_npu_backend(compiler_config=config), fullgraph=True, dynamic=False)
    with torch.no_grad():
        want = fn(x, ids, wt, *routed, *shared)
        for _ in range(3):
            assert torch.equal(compiled(x, ids, wt, *routed, *shared), want)


# ---- refusals (CPU) ------------------------------------------------------------------------------------------------------
def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("kwargs,error,match", [
    (dict(x=_meta(4, 64, dtype=torch.float32)), NotImplementedError, "bf16 or fp16"),
    (dict(weight1=_meta(64, 95)), RuntimeError, "do not fit"),
    (dict(weight1=_meta(63, 96)), RuntimeError, "do not fit"),
    (dict(weight2=_meta(48, 65)), RuntimeError, "do not fit"),
    (dict(weight2=_meta(48, 64, dtype=torch.float16)), RuntimeError, "one dtype"),
    (dict(bias1=_meta(48)), RuntimeError, "bias1"),
    (dict(bias2=_meta(63)), RuntimeError, "bias2"),
    (dict(residual=_meta(1, 64)), RuntimeError, "residual"),
    (dict(activation="swish"), RuntimeError, "activation"),
    (dict(x=_meta(4, 0), weight1=_meta(0, 96), weight2=_meta(48, 0)), RuntimeError, "do not fit"),
], ids=lambda v: str(v)[:40] if isinstance(v, dict) else None)
def test_gated_ffn_refusals(kwargs, error, match):
    a = dict(x=_meta(4, 64), weight1=_meta(64, 96), weight2=_meta(48, 64))
    a.update(kwargs)
    with pytest.raises(error, match=match):
        npu.npu_gated_ffn(a.pop("x"), a.pop("weight1"), a.pop("weight2"), **a)


@pytest.mark.parametrize("kwargs,error,match", [
    (dict(x=_meta(4, 64, dtype=torch.int8)), NotImplementedError, "bf16 or fp16"),
    (dict(weight=_meta(65, 96)), RuntimeError, "do not fit"),
    (dict(weight=_meta(1, 64, 96)), RuntimeError, "do not fit"),
    (dict(bias=_meta(4, 96)), RuntimeError, "bias"),
    (dict(bias=_meta(96, dtype=torch.float32)), RuntimeError, "one dtype"),
    (dict(residual=_meta(96)), RuntimeError, "residual"),
    (dict(activation="tanh"), RuntimeError, "activation"),
], ids=lambda v: str(v)[:40] if isinstance(v, dict) else None)
def test_linear_act_refusals(kwargs, error, match):
    a = dict(x=_meta(4, 64), weight=_meta(64, 96))
    a.update(kwargs)
    with pytest.raises(error, match=match):
        npu.npu_linear_act(a.pop("x"), a.pop("weight"), **a)


def test_checkpoint_refusals():
    q, s = npu.npu_checkpoint_quant(_meta(3, 130))
    assert q.shape == (3, 130) and q.dtype == torch.int8 and s.shape == (3, 3) and s.dtype == torch.float32
    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        npu.npu_checkpoint_quant(_meta(3, 64, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="one value per row"):
        npu.npu_checkpoint_dequant(q, _meta(3, 2, dtype=torch.float32))
    with pytest.raises(RuntimeError, match="int8"):
        npu.npu_checkpoint_dequant(_meta(3, 130), s)
    with pytest.raises(NotImplementedError, match="output_dtype"):
        npu.npu_checkpoint_dequant(q, s, output_dtype=3)
    with pytest.raises(RuntimeError, match="same rows"):
        npu.npu_checkpoint_weight_grad(q, s, _meta(4, 64))
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        npu.npu_checkpoint_weight_grad(q, s, _meta(3, 64, dtype=torch.float32))
    assert npu.npu_checkpoint_weight_grad(q, s, _meta(3, 64)).shape == (130, 64)


def test_no_cpu_implementation():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: npu.npu_gated_ffn(x, torch.zeros(64, 96, dtype=x.dtype), torch.zeros(48, 64, dtype=x.dtype)),
                 lambda: npu.npu_linear_act(x, torch.zeros(64, 96, dtype=x.dtype)), lambda: npu.npu_checkpoint_quant(x)):
        with pytest.raises(NotImplementedError):
            call()


def test_shapes_of_the_meta_implementations():
    y, kept, ks, xq, xs = npu.npu_gated_ffn_keep(_meta(2, 3, 64), _meta(64, 200), _meta(100, 64), checkpoint_int8=True)
    assert y.shape == (2, 3, 64) and kept.shape == (6, 256) and ks.shape == (6, 4) and xq.shape == (6, 64) and xs.shape == (6, 1)
    y, kept, ks, xq, xs = npu.npu_gated_ffn_keep(_meta(6, 64), _meta(64, 200), _meta(100, 64))
    assert kept.shape == (6, 208) and kept.dtype == torch.bfloat16 and ks.numel() == xq.numel() == xs.numel() == 0
    outs = npu.npu_gated_ffn_backward(_meta(6, 64), _meta(6, 64), xs, _meta(64, 200), _meta(100, 64), kept, ks, "silu", [True, True, False, True, True])
    assert [tuple(t.shape) for t in outs] == [(6, 64), (64, 200), (0,), (200,), (64,)]
    y, kept, ks, xq, xs = npu.npu_linear_act_keep(_meta(6, 64), _meta(64, 30), activation="none")
    assert y.shape == (6, 30) and kept.shape == (6, 0)


def test_c_entries_refuse_bad_arguments_before_any_cuda_call(built_library):
    import ctypes
    one, n, odd = ctypes.c_void_p(256), ctypes.c_void_p(None), ctypes.c_void_p(260)
    mat = lambda **kw: [kw.get("a", one), kw.get("lda", 64), 0, kw.get("b", one), kw.get("ldb", 64), 0, kw.get("dtype", 15), kw.get("M", 4),  # noqa: E731
                        kw.get("N", 64), kw.get("K", 64), kw.get("bias", n), n, kw.get("act", 0), kw.get("keep", n), kw.get("keep_q", n),
                        kw.get("keep_scale", n), kw.get("keep_ld", 0), kw.get("out", one), 0, n]
    for kw, match in ((dict(a=n), "null"), (dict(dtype=6), "dtype"), (dict(lda=63), "multiple of 8"),
                      (dict(lda=56), "shorter"), (dict(ldb=32), "shorter"), (dict(act=9), "activation"), (dict(K=0), "K=0"),
                      (dict(M=-1), "M=-1"), (dict(out=n), "null output"), (dict(a=odd), "aligned"), (dict(bias=ctypes.c_void_p(261)), "aligned"),
                      (dict(keep=one, keep_ld=32), "kept rows"), (dict(keep_q=one, keep_ld=64), "scales"),
                      (dict(keep=one, keep_q=one, keep_scale=one, keep_ld=64), "either"), (dict(keep_q=one, keep_scale=one, keep_ld=72), "multiple of 8"),
                      (dict(M=2 ** 40), "too large")):
        with pytest.raises(RuntimeError, match=match):
            _lib.call("tab_dense_matmul", *mat(**kw))
    _lib.call("tab_dense_matmul", *mat(M=0))
    with pytest.raises(RuntimeError, match="too short"):
        _lib.call("tab_checkpoint_quant", one, 15, 32, 4, 64, one, 64, one, 1, n)
    with pytest.raises(RuntimeError, match="too short"):
        _lib.call("tab_checkpoint_dequant", one, 64, one, 0, 4, 64, one, 15, 64, 64, 0, n)
    with pytest.raises(RuntimeError, match="dtype"):
        _lib.call("tab_checkpoint_quant", one, 1, 64, 4, 64, one, 64, one, 1, n)
    with pytest.raises(RuntimeError, match="nothing to compute"):
        _lib.call("tab_act_grad", one, 64, 15, 4, 64, 0, n, n, n, 0, n, n, n)
    with pytest.raises(RuntimeError, match="null"):
        _lib.call("tab_act_grad", one, 64, 15, 4, 64, 4, n, n, n, 64, one, n, n)
    sums = lambda **kw: [one, kw.get("lda", 64), kw.get("Na", 64), kw.get("b", one), 64, kw.get("Nb", 64), kw.get("dtype", 5), 4, one,  # noqa: E731
                         kw.get("splits", 1), one, kw.get("out_b", one), 0, n]
    for kw, match in ((dict(b=n), "null"), (dict(out_b=n), "null"), (dict(lda=56), "shorter"), (dict(Na=60), "multiples of 8"), (dict(Na=0), "Na=0"),
                      (dict(dtype=6), "dtype"), (dict(splits=0), "splits=0"), (dict(splits=1 << 16), "splits=65536")):
        with pytest.raises(RuntimeError, match=match):
            _lib.call("tab_two_column_sums", *sums(**kw))
    with pytest.raises(RuntimeError, match="256-byte"):
        _lib.call("tab_gated_ffn", one, 64, one, 128, 1, one, 64, 1, 64, 15, 4, 64, 64, n, n, n, 4, n, n, n, 0, one, n, 0, n)
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("tab_gated_ffn", one, 64, one, 128, 1, one, 64, 1, 64, 15, 4, 64, 64, n, n, n, 4, n, n, n, 0, one, one, 16, n)
    assert _lib.workspace_bytes("tab_gated_ffn_workspace_bytes", 4, 64, 64) >= 4 * 64 * 2


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_forward_mode_raises(which):
    """A tangent is refused, whether or not something requires a gradient; it used to be dropped where nothing did."""
    import torch.autograd.forward_ad as fw
    from torch._subclasses.fake_tensor import FakeTensorMode
    fake = lambda *shape: torch.empty(*shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    with FakeTensorMode(), fw.dual_level():
        t = {"x": fake(4, 64), "weight": fake(64, 64), "bias": fake(64), "residual": fake(4, 64)}
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        for grad in (False, True):
            v = fake(32, 64).requires_grad_(grad)
            with pytest.raises(NotImplementedError, match="npu_linear_act: forward-mode"):
                npu.npu_linear_act(t["x"], t["weight"].requires_grad_(grad) if which == "bias" else t["weight"], bias=t["bias"], residual=t["residual"])
            with pytest.raises(NotImplementedError, match="npu_gated_ffn: forward-mode"):
                npu.npu_gated_ffn(t["x"], t["weight"], v, bias1=t["bias"], residual=t["residual"])
        for call in (lambda: npu.npu_checkpoint_quant(t["x"]), lambda: npu.npu_linear_act_keep(t["x"], t["weight"], bias=t["bias"], residual=t["residual"])):
            if which == "x":
                with pytest.raises(NotImplementedError, match="forward AD"):
                    call()


def test_jvp_raises():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(64, 32, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda v: npu.npu_linear_act(v, w), (x,), (torch.ones_like(x),))


def test_another_torch_rebuilds_the_library(tmp_path, monkeypatch):
    """The PyTorch side is compiled again when the installed torch is not the one it was compiled against, and only then."""
    import subprocess
    from torchair_b200 import _build
    lib, calls = tmp_path / "lib.so", []

    def compiler(cmd, **kwargs):
        calls.append(cmd)
        lib.write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build, "TORCH_LIB_PATH", str(lib))
    monkeypatch.setattr(_build, "TORCH_STAMP_PATH", str(lib) + ".torch", raising=False)
    monkeypatch.setattr(_build.subprocess, "run", compiler)
    for built_against, compiles in ((None, 1), (None, 1), ("another", 2), (None, 2)):
        if built_against:
            (tmp_path / "lib.so.torch").write_text(built_against)
        _build.build_torch_library()
        assert len(calls) == compiles
