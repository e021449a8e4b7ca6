"""Cases of the token-block operators: matrix product with a fused epilogue, layer norm, counter-based dropout.

Tokens are the rows of a matrix [rows, features]: the positions of a latent grid, or the tokens of a sequence.

    linear        out = residual + dropout(act(x . W^T + bias)),  pre = x . W^T + bias (on request)
    linear_grad   dz = dropout(g_out) * act'(pre);  g_x = dz . W,  g_w = dz^T . x,  g_bias = sum of dz over rows
    norm          y = (x - mean) * rstd * weight + bias,  mean and rstd of each row (rstd = 1 / sqrt(var + eps))
    norm_grad     the gradients of it w.r.t. x (plus the gradient that arrives past the norm), weight and bias
    dropout       y = residual + (keep ? x / (1 - p) : 0)

keep of element i (of rows * cols, row by row): word i % 4 of Philox4x32-10 with the counter (i / 4 as 64 bits, offset as
64 bits) and the key seed as 64 bits, is at least round(p * 2^32).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _linear(name, dtype, rows, inn, out, act="none", bias=True, residual=False, p=0.0, pre=False, gap=0):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "inn": inn, "out": out, "act": act, "bias": bias,
            "residual": residual, "p": p, "pre": pre, "gap": gap}


def _linear_grad(name, dtype, rows, inn, out, act="none", p=0.0, gap=0):
    return {"name": name, "op": "linear_grad", "dtype": dtype, "rows": rows, "inn": inn, "out": out, "act": act, "p": p, "gap": gap}


def _norm(name, dtype, rows, cols, param="same", gap=0):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "param": param, "gap": gap}


def _norm_grad(name, dtype, rows, cols, param="same", add=True, gap=0):
    return {"name": name, "op": "norm_grad", "dtype": dtype, "rows": rows, "cols": cols, "param": param, "add": add, "gap": gap}


def _dropout(name, dtype, rows, cols, p=0.1, residual=False, gap=0):
    return {"name": name, "op": "dropout", "dtype": dtype, "rows": rows, "cols": cols, "p": p, "residual": residual, "gap": gap}


def listed():
    return [
        # one token through an output projection with its residual: latency, and the weight read once
        _linear("linear-token", "bf16", 1, 4096, 4096, residual=True),
        # a dozen sequences, one token each, through the widening product of a block
        _linear("linear-decode12", "f16", 12, 2560, 10240, act="gelu_tanh"),
        # the widening product of a block over a training batch, with what its backward pass needs
        _linear("linear-up-train", "bf16", 8192, 4096, 16384, act="gelu", pre=True),
        # the narrowing product of a block over a prompt, closing the residual branch with dropout
        _linear("linear-down-residual", "bf16", 2048, 8192, 2048, residual=True, p=0.1),
        # float32 and sizes that divide by nothing, rows cut out of a wider buffer
        _linear("linear-ragged-f32", "f32", 1537, 1001, 777, act="relu", residual=True, gap=3),
        # both gradients of the widening product over a training batch
        _linear_grad("linear-grad-up", "bf16", 8192, 2048, 8192, act="gelu"),
        # float32 gradients over the 32 x 48 latent positions of a 512 x 768 image at 192 channels
        _linear_grad("linear-grad-latents", "f32", 1536, 192, 768, act="silu", p=0.1),
        # the norm in front of one token's block: latency alone
        _norm("norm-token", "bf16", 1, 4096),
        # the norm over a long batch
        _norm("norm-batch", "bf16", 16384, 4096, param="f32"),
        # its gradients with the residual branch's added
        _norm_grad("norm-grad-batch", "bf16", 8192, 4096, param="f32"),
        # dropout of a small odd float32 matrix
        _dropout("dropout-odd-f32", "f32", 777, 1001, p=0.25),
        # dropout and the residual sum over a training batch
        _dropout("dropout-residual", "bf16", 8192, 8192, residual=True),
    ]


def _log(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = min(max(n, low), high)
    return n if rng.random() < 0.4 else max(low, n // 8 * 8)


def draw(rng):
    kind = rng.choices(["linear", "linear_grad", "norm", "norm_grad", "dropout"], [8, 4, 3, 3, 2])[0]
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    p = rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.6), 3)])
    gap = rng.choice([0, 0, 0, rng.randint(1, 40)])
    if kind in ("linear", "linear_grad"):
        inn, out = _log(rng, 32, 8192), _log(rng, 32, 16384)
        most = 2.0e11 if dtype == "f32" else 1.0e12
        rows = _log(rng, 1, max(1, min(16384, int(most / (2.0 * inn * out) / (2 if kind == "linear_grad" else 1)))))
        act = rng.choice(ACTS)
        if kind == "linear":
            c = _linear("", dtype, rows, inn, out, act, rng.random() < 0.8, rng.random() < 0.5, p, rng.random() < 0.3, gap)
        else:
            c = _linear_grad("", dtype, rows, inn, out, act, p, gap)
    else:
        cols = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(1, min(65536, 64 * 1024 * 1024 // cols)))
        param = rng.choice(["same", "f32"])
        if kind == "norm":
            c = _norm("", dtype, rows, cols, param, gap)
        elif kind == "norm_grad":
            c = _norm_grad("", dtype, rows, cols, param, rng.random() < 0.5, gap)
        else:
            c = _dropout("", dtype, rows, cols, p or 0.1, rng.random() < 0.5, gap)
    del c["name"]
    return c


def _make(case, seed):
    """The inputs as tensors: the same for every side that asks for this seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    t = TYPES[case["dtype"]]
    rows, gap = case["rows"], case["gap"]

    def rand(*shape, scale=1.0, shift=0.0, wide=False):
        v = torch.randn(*shape[:-1], shape[-1] + (gap if wide else 0), generator=g, device="cuda")
        v = v.mul_(scale).add_(shift).to(t)
        return v[..., :shape[-1]] if wide and gap else v

    s = {"case": case, "seed": int(seed) * 1000003 + 12345, "offset": int(seed) % 5 + (3 << 32)}
    if case["op"] in ("linear", "linear_grad"):
        inn, out = case["inn"], case["out"]
        s["x"] = rand(rows, inn, wide=True)
        s["w"] = rand(out, inn, scale=inn ** -0.5)
        if case["op"] == "linear":
            s["bias"] = rand(out, scale=0.1) if case["bias"] else None
            s["residual"] = rand(rows, out, scale=2.0) if case["residual"] else None
        else:
            s["g_out"] = rand(rows, out, scale=0.05)
            s["pre"] = rand(rows, out) if case["act"] != "none" else None
        return s
    cols = case["cols"]
    if case["op"] == "dropout":
        s["x"] = rand(rows, cols, wide=True)
        s["residual"] = rand(rows, cols, scale=2.0) if case["residual"] else None
        return s
    # activations of a deep residual stream: a spread of its own for each row and a few features that stand out
    x = torch.randn(rows, cols + gap, generator=g, device="cuda")
    x.mul_(torch.rand(rows, 1, generator=g, device="cuda").mul_(3.0).add_(0.5))
    x.add_(torch.randn(rows, 1, generator=g, device="cuda"))
    x[:, ::97] *= 8.0
    s["x"] = x.to(t)[:, :cols] if gap else x.to(t)
    tp = torch.float32 if case["param"] == "f32" else t
    s["w"] = torch.randn(cols, generator=g, device="cuda").mul_(0.2).add_(1.0).to(tp)
    if case["op"] == "norm":
        s["b"] = torch.randn(cols, generator=g, device="cuda").mul_(0.1).to(tp)
        return s
    s["g_out"] = rand(rows, cols, scale=0.05)
    s["g_add"] = rand(rows, cols, scale=0.05) if case["add"] else None
    xf = s["x"].double()
    mean = xf.mean(1)
    s["mean"], s["rstd"] = mean.float(), ((xf - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
    return s


def prepare(case, seed):
    return _make(case, seed)


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ------------------------------------------------

_LOW = 0xFFFFFFFF


def _words(n, seed, offset, device):
    """The n first random words of (seed, offset) in int64: ten Philox rounds over the counters."""
    i = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
    c0, c1 = i & _LOW, i >> 32
    c2, c3 = torch.full_like(i, offset & _LOW), torch.full_like(i, (offset >> 32) & _LOW)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57      # the low 64 bits are those of the unsigned product
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _dropped(v, p, seed, offset):
    """v / (1 - p) where the element is kept, 0 elsewhere (v: [rows, cols] in 32 bits)."""
    if p == 0.0:
        return v
    keep = _words(v.numel(), seed, offset, v.device).view(v.shape) >= round(p * 2.0 ** 32)
    return torch.where(keep, v * (1.0 / (1.0 - p)), torch.zeros((), device=v.device))


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    if act == "gelu_tanh":
        k = (2.0 / math.pi) ** 0.5
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * k * (1.0 + 3.0 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain(s):
    c = s["case"]
    t = TYPES[c["dtype"]]
    if c["op"] == "linear":
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        out = _dropped(_act(z, c["act"]), c["p"], s["seed"], s["offset"])
        if s["residual"] is not None:
            out = out + s["residual"].float()
        return (out.to(t), z.to(t)) if c["pre"] else (out.to(t),)
    if c["op"] == "linear_grad":
        dz = _dropped(s["g_out"].float(), c["p"], s["seed"], s["offset"])
        if c["act"] != "none":
            dz = dz * _act_slope(s["pre"].float(), c["act"])
        return (dz @ s["w"].float()).to(t), (dz.t() @ s["x"].float()).to(t), dz.sum(0).to(t)
    if c["op"] == "dropout":
        y = _dropped(s["x"].float(), c["p"], s["seed"], s["offset"])
        return ((y if s["residual"] is None else y + s["residual"].float()).to(t),)
    x, w = s["x"].float(), s["w"].float()
    if c["op"] == "norm":
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        return (d * rstd * w + s["b"].float()).to(t), mean[:, 0], rstd[:, 0]
    rstd = s["rstd"][:, None]
    h = (x - s["mean"][:, None]) * rstd
    dy = s["g_out"].float()
    g = dy * w
    gx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    if s["g_add"] is not None:
        gx = gx + s["g_add"].float()
    return gx.to(t), (dy * h).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)


def run(s):
    if not own:
        return _plain(s)
    from sga_amd import blocks
    c = s["case"]
    if c["op"] == "linear":
        drop = (c["p"], s["seed"], s["offset"]) if c["p"] else None
        out = blocks.linear(s["x"], s["w"], s["bias"], act=c["act"], residual=s["residual"], dropout=drop, want_pre=c["pre"])
        return out if c["pre"] else (out,)
    if c["op"] == "linear_grad":
        drop = (c["p"], s["seed"], s["offset"]) if c["p"] else None
        return blocks.linear_grad(s["g_out"], s["x"], s["w"], pre=s["pre"], act=c["act"], dropout=drop)
    if c["op"] == "dropout":
        return (blocks.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["residual"]),)
    if c["op"] == "norm":
        return blocks.layer_norm(s["x"], s["w"], s["b"], eps=EPS, want_stats=True)
    return blocks.layer_norm_grad(s["g_out"], s["x"], s["mean"], s["rstd"], s["w"], g_add=s["g_add"])


def work(case):
    e, rows = SIZE[case["dtype"]], case["rows"]
    if case["op"] in ("linear", "linear_grad"):
        inn, out = case["inn"], case["out"]
        act, wgt, wide = rows * inn, out * inn, rows * out
        if case["op"] == "linear":
            n = act + wgt + wide * (1 + case["residual"] + case["pre"]) + out * case["bias"]
            return {"bytes": n * e, "flops": 2.0 * rows * inn * out}
        return {"bytes": (2 * act + 2 * wgt + wide * (1 + (case["act"] != "none")) + out) * e, "flops": 4.0 * rows * inn * out}
    n, cols = rows * case["cols"], case["cols"]
    pe = 4 if case.get("param") == "f32" else e
    if case["op"] == "norm":
        return {"bytes": 2 * n * e + 2 * cols * pe + 8 * rows, "flops": 7.0 * n}
    if case["op"] == "norm_grad":
        return {"bytes": (3 + case["add"]) * n * e + 3 * cols * pe + 8 * rows, "flops": 13.0 * n}
    return {"bytes": (2 + case["residual"]) * n * e, "flops": 25.0 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _keep64(rows, cols, p, seed, offset):
    """The mask on the host, in unsigned 64-bit arithmetic."""
    n = rows * cols
    ctr = np.arange(-(-n // 4), dtype=np.uint64)
    m32, s32 = np.uint64(_LOW), np.uint64(32)
    w = [ctr & m32, ctr >> s32, np.full_like(ctr, offset & _LOW), np.full_like(ctr, offset >> 32 & _LOW)]
    key = [seed & _LOW, seed >> 32 & _LOW]
    for _ in range(10):
        even, odd = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(odd >> s32) ^ w[1] ^ np.uint64(key[0]), odd & m32, (even >> s32) ^ w[3] ^ np.uint64(key[1]), even & m32]
        key = [(key[0] + 0x9E3779B9) & _LOW, (key[1] + 0xBB67AE85) & _LOW]
    flat = np.empty((len(ctr), 4), np.bool_)
    for j in range(4):
        flat[:, j] = w[j] >= np.uint64(round(p * 2.0 ** 32))
    return torch.from_numpy(flat.reshape(-1)[:n].reshape(rows, cols)).cuda()


def exact(case, seed):
    s = _make(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    rows, op = case["rows"], case["op"]
    cols = case.get("out", case.get("cols"))
    p = case.get("p", 0.0)
    gain = _keep64(rows, cols, p, s["seed"], s["offset"]).double() / (1.0 - p) if p else None
    if op == "linear":
        z = torch.mm(d["x"], d["w"].t().contiguous())
        if "bias" in d:
            z += d["bias"]
        y = z.clone()
        if case["act"] == "relu":
            y = torch.relu(z)
        elif case["act"] == "gelu":
            y = z * torch.special.ndtr(z)
        elif case["act"] == "gelu_tanh":
            y = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
        elif case["act"] == "silu":
            y = z * torch.sigmoid(z)
        y = y if gain is None else y * gain
        y = y + d["residual"] if "residual" in d else y
        return (y, z) if case["pre"] else (y,)
    if op == "linear_grad":
        dz = d["g_out"] if gain is None else d["g_out"] * gain
        if "pre" in d:
            z = d["pre"].clone().requires_grad_(True)
            q = 2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
            y = {"relu": lambda: torch.relu(z), "gelu": lambda: z * torch.special.ndtr(z),
                 "gelu_tanh": lambda: z * torch.sigmoid(q), "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
            dz, = torch.autograd.grad(y, z, dz)
        return torch.mm(dz, d["w"]), torch.mm(dz.t().contiguous(), d["x"]), dz.sum(0)
    if op == "dropout":
        y = d["x"] * gain
        return (y + d["residual"] if "residual" in d else y,)
    if op == "norm":
        var, mean = torch.var_mean(d["x"], 1, unbiased=False)
        rstd = (var + EPS) ** -0.5
        return (d["x"] - mean[:, None]) * rstd[:, None] * d["w"] + d["b"], mean, rstd
    h = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None]
    g = d["g_out"] * d["w"]
    along = torch.einsum("rc,rc->r", g, h) / cols
    gx = (g - g.sum(1, keepdim=True) / cols - h * along[:, None]) * d["rstd"][:, None]
    return gx + d["g_add"] if "g_add" in d else gx, (d["g_out"] * h).sum(0), d["g_out"].sum(0)
