"""Performance cases of the normalisation and inner-product operators around transformer and diffusion blocks.

* ``group_norm``: statistics per image and group of channels, affine, activation, on channels-last tensors (``groups`` = 1 on a
  [tokens, channels] tensor is layer norm): ``y = act((x - mean) / sqrt(var + eps) * gamma + beta)``;
* ``linear``: an inner product whose epilogue adds the bias, applies an activation and adds a residual:
  ``y = act(x w^T + b) + r``.

The framework runs them as ops of a module: the inputs lie in the module's tensors, where the op before would have left them,
``launch()`` enqueues the module, and the result stays in the device tensor. Weights are loaded with the module.
"""
import math

import torch

own = False

EPS = 1e-5
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
MOST_VALUES = 1 << 26            # of a normalised tensor: the largest listed
MOST_MACS = 8192 * 4096 * 4096   # of a product: the largest listed
MOST_WEIGHTS = 1 << 26
MOST_MACS_FP32 = 1 << 32         # fp32 products are those of a calibration pass over a few hundred rows


def listed():
    return [
        # decoding: the layer norm of one token
        {"name": "norm_t1_c1024", "kind": "group_norm", "n": 1, "c": 1024, "h": 1, "w": 1, "groups": 1, "act": "none", "dtype": "bf16"},
        # prefill: the layer norm of an odd number of tokens
        {"name": "norm_t4099_c4096", "kind": "group_norm", "n": 4099, "c": 4096, "h": 1, "w": 1, "groups": 1, "act": "none",
         "dtype": "bf16"},
        # the innermost level of an image network: little data, many channels
        {"name": "norm_n2_c1280_8x8_silu", "kind": "group_norm", "n": 2, "c": 1280, "h": 8, "w": 8, "groups": 32, "act": "silu",
         "dtype": "bf16"},
        # its outermost level: groups of ten channels, which are no whole number of 16-byte vectors
        {"name": "norm_n8_c320_64x64_silu", "kind": "group_norm", "n": 8, "c": 320, "h": 64, "w": 64, "groups": 32, "act": "silu",
         "dtype": "bf16"},
        # a calibration forward in fp32 over odd extents and groups of 25 channels
        {"name": "norm_fp32_n3_c200_31x57_gelu", "kind": "group_norm", "n": 3, "c": 200, "h": 31, "w": 57, "groups": 8, "act": "gelu",
         "dtype": "fp32"},
        # an image decoder at full resolution: one image larger than the L2
        {"name": "norm_n1_c256_512x512_silu", "kind": "group_norm", "n": 1, "c": 256, "h": 512, "w": 512, "groups": 32, "act": "silu",
         "dtype": "bf16"},
        # decoding: one token, the weights are read once
        {"name": "linear_m1_k4096_n4096_res", "kind": "linear", "m": 1, "k": 4096, "n": 4096, "act": "none", "residual": True,
         "dtype": "bf16"},
        # a small ragged batch on odd widths
        {"name": "linear_m17_k1000_n2050_silu_res", "kind": "linear", "m": 17, "k": 1000, "n": 2050, "act": "silu", "residual": True,
         "dtype": "bf16"},
        # a decoding batch through the widening product of a feed-forward block
        {"name": "linear_m256_k4096_n16384_gelut", "kind": "linear", "m": 256, "k": 4096, "n": 16384, "act": "gelu_tanh",
         "residual": False, "dtype": "bf16"},
        # a classifier's product in a calibration forward
        {"name": "linear_fp32_m200_k1024_n1000", "kind": "linear", "m": 200, "k": 1024, "n": 1000, "act": "relu", "residual": False,
         "dtype": "fp32"},
        # prefill of an odd number of tokens, exact GELU
        {"name": "linear_m4100_k2048_n8192_gelu", "kind": "linear", "m": 4100, "k": 2048, "n": 8192, "act": "gelu", "residual": False,
         "dtype": "bf16"},
        # the largest prefill
        {"name": "linear_m8192_k4096_n4096_res", "kind": "linear", "m": 8192, "k": 4096, "n": 4096, "act": "none", "residual": True,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    act, dtype = rng.choice(ACTS), rng.choice(["bf16", "bf16", "bf16", "fp32"])
    kind = rng.choice(["rows", "images", "linear", "linear"])
    if kind == "rows":
        return {"kind": "group_norm", "n": _log_int(rng, 1, 8192), "c": _log_int(rng, 32, 8192), "h": 1, "w": 1, "groups": 1, "act": act,
                "dtype": dtype}
    while kind == "images":
        n, h, w = _log_int(rng, 1, 16), _log_int(rng, 4, 512), _log_int(rng, 4, 512)
        groups = rng.choice([1, 2, 8, 16, 32, 32])
        c = groups * _log_int(rng, 1, 64)
        if c >= 16 and n * c * h * w * (2 if dtype == "fp32" else 1) <= MOST_VALUES:
            return {"kind": "group_norm", "n": n, "c": c, "h": h, "w": w, "groups": groups, "act": act, "dtype": dtype}
    while True:
        m, k, n = _log_int(rng, 1, 8192), _log_int(rng, 16, 8192), _log_int(rng, 16, 16384)
        if m * k * n <= (MOST_MACS_FP32 if dtype == "fp32" else MOST_MACS) and n * k <= MOST_WEIGHTS:
            return {"kind": "linear", "m": m, "k": k, "n": n, "act": act, "residual": rng.random() < 0.5, "dtype": dtype}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """Activations with a mean and a spread of their own per channel, as a network's have; products scaled to unit variance."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["kind"] == "group_norm":
        c = case["c"]
        x = normal(case["n"], case["h"], case["w"], c).mul_(normal(c).mul_(0.5).exp_()).add_(normal(c))
        return {"x": x.to(dt), "gamma": normal(c).mul_(0.2).add_(1.0), "beta": normal(c).mul_(0.2)}
    m, k, n = case["m"], case["k"], case["n"]
    d = {"x": normal(m, k).to(dt), "w": normal(n, k).mul_(k ** -0.5).to(dt), "b": normal(n).mul_(0.2)}
    if case["residual"]:
        d["r"] = normal(m, n).to(dt)
    return d


class _DeviceArray:
    def __init__(self, m, ptr, shape, typestr):
        self.module = m  # the storage is the module's: it lives as long as a view of it does
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": typestr, "version": 2}


def _view(m, name, shape):
    """The module's tensor where it lies on the device, with the channels last, in the shape of the torch tensors here."""
    t = m.tensor_device(name)
    rows = math.prod(shape[:-1])
    v = torch.as_tensor(_DeviceArray(m, t["ptr"], (rows, t["pitch"]), {1: "<i2", 2: "<f4"}[t["dtype"]]), device="cuda")
    v = v.view(torch.bfloat16) if t["dtype"] == 1 else v
    return v.view(*shape[:-1], t["pitch"])[..., :shape[-1]]


def _load(case, d):
    """The module of one op, its weights loaded and its inputs in place, and a view of its result."""
    from tpu_compiler_b200 import module
    dt = "BF16" if case["dtype"] == "bf16" else "FP32"
    if case["kind"] == "group_norm":
        dims = (case["n"], case["c"]) if case["h"] * case["w"] == 1 else (case["n"], case["c"], case["h"], case["w"])
        shape = ",".join(map(str, dims))
        text = "input name=x shape=%s dtype=%s\ngroup_norm name=y in=x,gamma,beta shape=%s dtype=%s groups=%d variance_epsilon=%g activation=%s\n" % (
            shape, dt, shape, dt, case["groups"], EPS, case["act"])
        fixed, out = ("gamma", "beta"), tuple(d["x"].shape)
    else:
        m, k, n = case["m"], case["k"], case["n"]
        text = "input name=x shape=%d,%d dtype=%s\n" % (m, k, dt)
        if case["residual"]:
            text += "input name=r shape=%d,%d dtype=%s\n" % (m, n, dt)
        text += "fully_connected name=y in=x,w,b,-,-,-,-,%s shape=%d,%d dtype=%s activation=%s\n" % (
            "r" if case["residual"] else "-", m, n, dt, case["act"])
        fixed, out = ("w", "b"), (m, n)
    mod = module(0)
    mod.load_text(text, {name: d[name].float().cpu().numpy() for name in fixed})
    for name in d:
        if name not in fixed:
            _view(mod, name, tuple(d[name].shape)).copy_(d[name])
    torch.cuda.synchronize()
    return mod, _view(mod, "y", out)


def prepare(case, seed):
    state = {"case": case, "data": _inputs(case, seed)}
    if own:
        state["module"], state["y"] = _load(case, state.pop("data"))
    return state


# ------------------------------------------------------------------------------------------------------------------- run
def _activation(act, v):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def run(state):
    if own:
        state["module"].launch()
        return state["y"]
    case, d = state["case"], state["data"]
    x = d["x"].float()
    if case["kind"] == "group_norm":
        n, h, w, c = x.shape
        x = x.view(n, h * w, case["groups"], c // case["groups"])
        x = x - x.mean((1, 3), keepdim=True)
        x = x / torch.sqrt((x * x).mean((1, 3), keepdim=True) + EPS)
        return _activation(case["act"], x.view(n, h, w, c) * d["gamma"] + d["beta"]).to(d["x"].dtype)
    y = _activation(case["act"], torch.matmul(x, d["w"].float().t()) + d["b"])
    if case["residual"]:
        y = y + d["r"].float()
    return y.to(d["x"].dtype)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "group_norm":
        values = case["n"] * case["c"] * case["h"] * case["w"]
        return {"bytes": 2.0 * es * values + 8.0 * case["c"], "flops": 8.0 * values}
    m, k, n = case["m"], case["k"], case["n"]
    return {"bytes": es * (m * k + n * k + m * n * (2.0 if case["residual"] else 1.0)) + 4.0 * n, "flops": 2.0 * m * k * n}


def exact(case, seed):
    """From the definitions, in 64 bits."""
    d = {name: t.double() for name, t in _inputs(case, seed).items()}
    if case["kind"] == "group_norm":
        g, cg = case["groups"], case["c"] // case["groups"]
        per_group = [d["x"][..., i * cg:(i + 1) * cg] for i in range(g)]
        normed = []
        for t in per_group:
            count = t[0].numel()
            mean = t.sum((1, 2, 3), keepdim=True) / count
            var = (t - mean).pow(2).sum((1, 2, 3), keepdim=True) / count
            normed.append((t - mean) * (var + EPS).pow(-0.5))
        y = torch.cat(normed, -1) * d["gamma"] + d["beta"]
    else:
        y = torch.einsum("mk,nk->mn", d["x"], d["w"]) + d["b"]
    if case["act"] == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    elif case["act"] == "gelu_tanh":
        u = 2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y.pow(3))
        y = y * torch.sigmoid(u)
    return y + d["r"] if "r" in d else y
