"""Cases for the operators of a trained and served residual block: group norm
with an activation (channels last, forward and backward), counter-based
dropout, the 8-bit quantiser and the 8-bit matrix product.

`run` computes them in plain torch operations, or, with `own` set, through
libnpl_b200's nplk_* entry points as a caller that keeps its buffers does.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
DTYPE_CODE = {"fp32": 0, "fp16": 1, "bf16": 2}  # NPLK_DTYPE_*
ACT_CODE = {"none": 0, "relu": 1, "gelu": 5, "swish": 6}  # npl_activation_t
EPS = 1e-5
GELU_C, GELU_A = 0.7978845608, 0.044715  # the library's tanh form of GELU
LARGEST_NORM = 262144 * 128
LARGEST_GEMM = 8192 * 16384 * 4096


# ---- cases -------------------------------------------------------------------

def listed():
    return [
        # the lowest level of a latent U-Net (8 x 8 pixels), one image: latency
        {"name": "norm_8x8_bf16", "op": "norm", "dtype": "bf16", "n": 1, "hw": 64, "groups": 32,
         "cg": 40, "act": "swish"},
        # its top level (64 x 64 latents), a small batch; 10 channels a group
        {"name": "norm_64x64_fp16", "op": "norm", "dtype": "fp16", "n": 4, "hw": 4096,
         "groups": 32, "cg": 10, "act": "swish"},
        # last block of an image decoder at 512 x 512, in 32 bits
        {"name": "norm_512x512_fp32", "op": "norm", "dtype": "fp32", "n": 1, "hw": 262144,
         "groups": 32, "cg": 4, "act": "swish"},
        # a training step's gradient at the top level of the U-Net
        {"name": "norm_grad_64x64_bf16", "op": "norm_grad", "dtype": "bf16", "n": 8, "hw": 4096,
         "groups": 32, "cg": 10, "act": "swish"},
        # odd plane (31 x 31) and an odd channel count per group, in 32 bits
        {"name": "norm_grad_31x31_fp32", "op": "norm_grad", "dtype": "fp32", "n": 3, "hw": 961,
         "groups": 30, "cg": 17, "act": "gelu"},
        # dropout on the activations of the framework's bandwidth chain (256 x 512 x 14 x 14)
        {"name": "dropout_chain_bf16", "op": "dropout", "dtype": "bf16", "count": 25690112,
         "p": 0.1, "offset": 0},
        # a short odd vector that starts inside the generator's block of eight
        {"name": "dropout_small_fp32", "op": "dropout", "dtype": "fp32", "count": 1001, "p": 0.5,
         "offset": 3},
        # a prompt's tokens ahead of an 8-bit projection
        {"name": "quantize_prompt_bf16", "op": "quantize", "dtype": "bf16", "axis": "rows",
         "rows": 8192, "cols": 4096},
        # a short odd batch of class scores (1000 classes), in 32 bits
        {"name": "quantize_small_fp32", "op": "quantize", "dtype": "fp32", "axis": "rows",
         "rows": 77, "cols": 1000},
        # one token through a 4096 x 4096 projection: the weights' bytes count
        {"name": "gemm_token_bf16", "op": "gemm", "dtype": "bf16", "m": 1, "n": 4096, "k": 4096,
         "act": "none"},
        # a short ragged prompt into 1000 classes, bias and ReLU, 32-bit result
        {"name": "gemm_ragged_fp32", "op": "gemm", "dtype": "fp32", "m": 333, "n": 1000,
         "k": 1280, "act": "relu"},
        # the framework's large product (8192 x 16384 x 4096) in 8 bits
        {"name": "gemm_large_bf16", "op": "gemm", "dtype": "bf16", "m": 8192, "n": 16384,
         "k": 4096, "act": "none"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "dropout", "quantize", "gemm", "gemm"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op in ("norm", "norm_grad"):
        groups, cg = rng.choice([1, 4, 8, 16, 30, 32]), _log_int(rng, 1, 80)
        n = rng.randint(1, 8)
        most = LARGEST_NORM // (1 if op == "norm" else 2) // (n * groups * cg)
        # a gradient of fewer than four values a group is mostly cancellation
        return {"op": op, "dtype": dtype, "n": n,
                "hw": _log_int(rng, 1 if op == "norm" else 4, min(262144, most)),
                "groups": groups, "cg": cg,
                "act": rng.choice(["none", "relu", "gelu", "swish"])}
    if op == "dropout":
        return {"op": op, "dtype": dtype, "count": _log_int(rng, 1, 33554432),
                "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "offset": rng.choice([0, 5, 1 << 35])}
    if op == "quantize":
        rows = _log_int(rng, 1, 16384)
        # by columns: a weight matrix, laid out once for the product
        return {"op": op, "dtype": dtype, "axis": rng.choice(["rows", "rows", "cols"]), "rows": rows,
                "cols": _log_int(rng, 16, min(16384, LARGEST_NORM // rows))}
    m, n = _log_int(rng, 1, 8192), _log_int(rng, 16, 16384)
    return {"op": op, "dtype": dtype, "m": m, "n": n,
            "k": _log_int(rng, 16, min(16384, LARGEST_GEMM // (m * n))),
            "act": rng.choice(["none", "relu", "gelu", "swish"])}


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op in ("norm", "norm_grad"):
        c = case["groups"] * case["cg"]
        e = case["n"] * case["hw"] * c
        small = 4 * (2 * c + 2 * case["n"] * case["groups"])
        if op == "norm":
            return {"bytes": 2 * e * size + small, "flops": 8 * e}
        return {"bytes": 3 * e * size + small + 8 * c, "flops": 20 * e}
    if op == "dropout":
        return {"bytes": 2 * case["count"] * size, "flops": 2 * case["count"]}
    if op == "quantize":
        e = case["rows"] * case["cols"]
        return {"bytes": e * (size + 1) + 4 * case[case["axis"]], "flops": 3 * e}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * k + n * k + m * n * size + 4 * m + 8 * n, "flops": 2 * m * n * k}


# ---- inputs --------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _pitched(rows, cols, low, high, g):
    """8-bit rows at a pitch of whole 16-byte pieces, as the quantiser's caller keeps them."""
    pitch = (cols + 15) // 16 * 16
    return torch.randint(low, high, (rows, pitch), generator=g, device=DEVICE,
                         dtype=torch.int8)[:, :cols]


def prepare(case, seed):
    g, op, t = _generator(seed), case["op"], TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    s = dict(case)
    if op in ("norm", "norm_grad"):
        n, hw, c = case["n"], case["hw"], case["groups"] * case["cg"]
        # features of a network under way: channels of their own means and spreads
        s["x"] = (randn(n, hw, c) * (0.5 + randn(c).abs()) + 0.5 * randn(c)).to(t)
        s["gamma"], s["beta"] = 1.0 + 0.2 * randn(c), 0.2 * randn(c)
        s["mean"] = torch.empty(n, case["groups"], device=DEVICE)
        s["rstd"] = torch.empty(n, case["groups"], device=DEVICE)
        s["y"] = torch.empty_like(s["x"])
        if op == "norm_grad":
            s["dy"] = randn(n, hw, c).to(t)
            # the statistics that the forward pass kept
            parts = s["x"].view(n, hw, case["groups"], case["cg"])
            for i in range(n):
                one = parts[i].double()
                mean = one.mean((0, 2))
                var = (one - mean.view(1, -1, 1)).square().mean((0, 2))
                s["mean"][i], s["rstd"][i] = mean, 1.0 / torch.sqrt(var + EPS)
            s["dgamma"], s["dbeta"] = torch.empty(c, device=DEVICE), torch.empty(c, device=DEVICE)
    elif op == "dropout":
        s["x"] = randn(case["count"]).to(t)
        s["y"] = torch.empty_like(s["x"])
        s["seed"] = seed * 0x9E3779B97F4A7C15 % (1 << 64)
    elif op == "quantize":
        # a few rows (columns) are much larger than the others
        rows, cols = case["rows"], case["cols"]
        spread = randn(rows, 1) if case["axis"] == "rows" else randn(1, cols)
        s["x"] = (randn(rows, cols) * torch.exp(spread)).to(t)
        lines, length = (rows, cols) if case["axis"] == "rows" else (cols, rows)
        s["q"] = torch.empty(lines, (length + 15) // 16 * 16, device=DEVICE, dtype=torch.int8)
        s["scale"] = torch.empty(lines, device=DEVICE)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["b"] = _pitched(m, k, -127, 128, g), _pitched(n, k, -127, 128, g)
        s["a_scale"] = (0.5 + torch.rand(m, generator=g, device=DEVICE)) / 127
        s["b_scale"] = (0.5 + torch.rand(n, generator=g, device=DEVICE)) / (127 * math.sqrt(k))
        s["bias"] = 0.1 * randn(n)
        s["c"] = torch.empty(m, n, device=DEVICE, dtype=t)
    return s


# ---- one pass ------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_C * (z + GELU_A * z * z * z)))
    if name == "swish":
        return z * (1.0 / (1.0 + torch.exp(-z)))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        t = torch.tanh(GELU_C * (z + GELU_A * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * GELU_A * z * z)
    if name == "swish":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    return torch.ones_like(z)


def _keep_threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _philox_bits(count, seed, offset):
    """16 random bits for each of `count` elements: Philox4x32-10 (Salmon et al., 2011) with the
    seed as its key, counted in blocks of eight elements, in 64-bit integer arithmetic."""
    low = 0xFFFFFFFF
    first, last = offset // 8, (offset + count - 1) // 8
    block = torch.arange(first, last + 1, device=DEVICE, dtype=torch.int64)
    c0, c1 = block & low, (block >> 32) & low
    c2, c3 = torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & low, seed >> 32

    def mul(a, b):  # high and low halves of a 32 x 32 bit product
        high = (b * (a >> 16) + ((b * (a & 0xFFFF)) >> 16)) >> 16
        return high & low, (b * a) & low

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)
    start = offset - 8 * first
    return bits[start:start + count]


def _plain(s):
    op = s["op"]
    if op in ("norm", "norm_grad"):
        n, hw, groups, cg = s["n"], s["hw"], s["groups"], s["cg"]
        shape, gc = (n, hw, groups, cg), (1, 1, groups, cg)
        x = s["x"].float().view(shape)
        gamma, beta = s["gamma"].view(gc), s["beta"].view(gc)
        if op == "norm":
            mean = x.mean((1, 3), keepdim=True)
            d = x - mean
            rstd = 1.0 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + EPS)
            y = _act(d * rstd * gamma + beta, s["act"])
            return {"y": y.view(n, hw, -1).to(s["x"].dtype), "mean": mean.view(n, groups),
                    "rstd": rstd.view(n, groups)}
        rstd = s["rstd"].view(n, 1, groups, 1)
        xh = (x - s["mean"].view(n, 1, groups, 1)) * rstd
        dz = s["dy"].float().view(shape) * _act_slope(xh * gamma + beta, s["act"])
        dh = dz * gamma
        a = dh.mean((1, 3), keepdim=True)
        b = (dh * xh).mean((1, 3), keepdim=True)
        dx = rstd * (dh - (a + xh * b))
        return {"dx": dx.view(n, hw, -1).to(s["x"].dtype), "dgamma": (dz * xh).sum((0, 1)).view(-1),
                "dbeta": dz.sum((0, 1)).view(-1)}
    if op == "dropout":
        t = _keep_threshold(s["p"])
        keep = _philox_bits(s["count"], s["seed"], s["offset"]) >= t
        y = torch.where(keep, s["x"].float() * (65536.0 / (65536 - t)), 0.0)
        return {"y": y.to(s["x"].dtype)}
    if op == "quantize":
        x = s["x"].float() if s["axis"] == "rows" else s["x"].float().t()
        # divided by a tensor: torch divides by a number as a product with its reciprocal
        top = x.abs().amax(1)
        scale = (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126)
        return {"q": torch.round(x / scale[:, None]).to(torch.int8).contiguous(),
                "scale": scale}
    total = s["a"].float() @ s["b"].float().t()
    z = total * s["a_scale"][:, None] * s["b_scale"][None, :] + s["bias"][None, :]
    return {"c": _act(z, s["act"]).to(s["c"].dtype)}


_lib = None


def _library():
    global _lib
    if _lib is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "project-jcore_b200"))
        import npl_b200
        _lib = npl_b200.load()
    return _lib


def _norm_workspace(lib, s, c):
    """The caller's scratch and its size, kept with the state like its other buffers."""
    if "work" not in s:
        size = lib.nplk_group_norm_workspace_size(s["n"], s["hw"], c, s["groups"])
        s["work"] = torch.empty(max(size, 1), device=DEVICE, dtype=torch.uint8)
    return s["work"].data_ptr(), s["work"].numel()


def _own(s):
    lib, op = _library(), s["op"]
    stream = torch.cuda.current_stream().cuda_stream
    code = DTYPE_CODE[s["dtype"]]
    if op in ("norm", "norm_grad"):
        n, hw, groups, c = s["n"], s["hw"], s["groups"], s["groups"] * s["cg"]
        work_ptr, size = _norm_workspace(lib, s, c)
        if op == "norm":
            rc = lib.nplk_group_norm_act(
                stream, n, hw, c, groups, code, s["x"].data_ptr(), c, s["gamma"].data_ptr(),
                s["beta"].data_ptr(), EPS, ACT_CODE[s["act"]], 0.0, s["y"].data_ptr(), c,
                s["mean"].data_ptr(), s["rstd"].data_ptr(), work_ptr, size)
            out = {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
        else:
            rc = lib.nplk_group_norm_act_backward(
                stream, n, hw, c, groups, code, s["dy"].data_ptr(), c, s["x"].data_ptr(), c,
                s["mean"].data_ptr(), s["rstd"].data_ptr(), s["gamma"].data_ptr(),
                s["beta"].data_ptr(), ACT_CODE[s["act"]], 0.0, s["y"].data_ptr(), c,
                s["dgamma"].data_ptr(), s["dbeta"].data_ptr(), work_ptr, size)
            out = {"dx": s["y"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    elif op == "dropout":
        rc = lib.nplk_dropout(stream, s["count"], code, s["x"].data_ptr(), s["y"].data_ptr(),
                              s["p"], s["seed"], s["offset"], None)
        out = {"y": s["y"]}
    elif op == "quantize":
        rows, cols = s["rows"], s["cols"]
        call = lib.nplk_quantize_rows if s["axis"] == "rows" else lib.nplk_quantize_cols
        rc = call(stream, rows, cols, code, s["x"].data_ptr(), cols, s["q"].data_ptr(),
                  s["q"].stride(0), s["scale"].data_ptr())
        out = {"q": s["q"][:, :cols if s["axis"] == "rows" else rows], "scale": s["scale"]}
    else:
        m, n, k = s["m"], s["n"], s["k"]
        rc = lib.nplk_gemm_i8(
            stream, m, n, k, s["a"].data_ptr(), s["a"].stride(0), s["a_scale"].data_ptr(),
            s["b"].data_ptr(), s["b"].stride(0), s["b_scale"].data_ptr(), s["bias"].data_ptr(),
            ACT_CODE[s["act"]], 0.0, code, s["c"].data_ptr(), n, None)
        out = {"c": s["c"]}
    if rc != 0:
        raise RuntimeError(f"{op}: the library returned {rc}")
    return out


# ---- the definition in 64 bits ---------------------------------------------------

def _exact_act(z, name):
    """act(z) and its derivative."""
    one = torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        u = GELU_C * (z + GELU_A * z ** 3)
        t = torch.tanh(u)
        return z * (1 + t) / 2, (1 + t + z * (1 - t ** 2) * GELU_C * (1 + 3 * GELU_A * z ** 2)) / 2
    if name == "swish":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, one


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("norm", "norm_grad"):
        n, hw, groups, cg = case["n"], case["hw"], case["groups"], case["cg"]
        rows = {"y": [], "mean": [], "rstd": [], "dx": [], "dgamma": [], "dbeta": []}
        for i in range(n):  # an image at a time: its groups as rows
            flat = s["x"][i].double().view(hw, groups, cg).permute(1, 0, 2).reshape(groups, -1)
            var, mean = torch.var_mean(flat, dim=1, correction=0, keepdim=True)
            rstd = (var + EPS).rsqrt()
            if op == "norm_grad":  # the saved statistics are inputs
                mean, rstd = s["mean"][i].double()[:, None], s["rstd"][i].double()[:, None]
            gamma = s["gamma"].double().view(groups, 1, cg).expand(groups, hw, cg).reshape(groups, -1)
            beta = s["beta"].double().view(groups, 1, cg).expand(groups, hw, cg).reshape(groups, -1)
            h = (flat - mean) * rstd
            value, slope = _exact_act(torch.addcmul(beta, h, gamma), case["act"])
            back = lambda v: v.view(groups, hw, cg).permute(1, 0, 2).reshape(hw, -1)  # noqa: E731
            if op == "norm":
                rows["y"].append(back(value))
                rows["mean"].append(mean[:, 0])
                rows["rstd"].append(rstd[:, 0])
                continue
            dz = s["dy"][i].double().view(hw, groups, cg).permute(1, 0, 2).reshape(groups, -1) * slope
            dh = dz * gamma
            dx = rstd * (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True))
            rows["dx"].append(back(dx))
            rows["dgamma"].append((dz * h).view(groups, hw, cg).sum(1).reshape(-1))
            rows["dbeta"].append(dz.view(groups, hw, cg).sum(1).reshape(-1))
        if op == "norm":
            return {k: torch.stack(rows[k]) for k in ("y", "mean", "rstd")}
        return {"dx": torch.stack(rows["dx"]), "dgamma": torch.stack(rows["dgamma"]).sum(0),
                "dbeta": torch.stack(rows["dbeta"]).sum(0)}
    if op == "dropout":
        index = np.arange(case["offset"], case["offset"] + case["count"], dtype=np.uint64)
        first = index[0] >> np.uint64(3)
        block = np.arange(first, (index[-1] >> np.uint64(3)) + np.uint64(1), dtype=np.uint64)
        mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
        c = [block & mask, block >> half, np.zeros_like(block), np.zeros_like(block)]
        key = [s["seed"] % (1 << 32), s["seed"] >> 32]
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> half) ^ c[1] ^ np.uint64(key[0]), b & mask,
                 (a >> half) ^ c[3] ^ np.uint64(key[1]), a & mask]
            key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
        words = np.stack(c, 1).astype(np.uint32).view(np.uint16).reshape(-1)  # low half first
        bits = words[(index - (first << np.uint64(3))).astype(np.int64)]
        t = _keep_threshold(case["p"])
        keep = torch.from_numpy((bits >= t).astype(np.float64)).to(DEVICE)
        return {"y": s["x"].double() * keep / (1 - t / 65536)}
    if op == "quantize":
        along = 1 if case["axis"] == "rows" else 0
        top = s["x"].double().abs().max(dim=along).values / 127
        return {"q": None, "scale": torch.maximum(top, torch.full_like(top, 2.0 ** -126))}
    a, b = s["a"].double(), s["b"].double()
    scaled = torch.addmm(s["bias"].double(), a * s["a_scale"].double()[:, None],
                         (b * s["b_scale"].double()[:, None]).t())
    return {"c": _exact_act(scaled, case["act"])[0]}
