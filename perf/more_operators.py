"""Cases for the operators of a language model's head, served and trained: the
quantiser of weights to 4 bits by groups, the product with such weights, the log
probabilities of given tokens with their entropy and alternatives, and their
gradient.

`run` computes them in plain torch operations, or, with `own` set, through
libnpl_b200's nplk_* entry points as a caller that keeps its buffers does.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
DTYPE_CODE = {"fp32": 0, "fp16": 1, "bf16": 2}  # NPLK_DTYPE_*
ACT_CODE = {"none": 0, "relu": 1, "gelu": 5, "swish": 6}  # npl_activation_t
GELU_C, GELU_A = 0.7978845608, 0.044715  # the library's tanh form of GELU
TINY = {"fp32": 2.0 ** -126, "fp16": 2.0 ** -14, "bf16": 2.0 ** -126}  # least scales
LARGEST_WEIGHTS = 128000 * 4096
LARGEST_PRODUCT = 512 * 4096 * 16384
LARGEST_LOGITS = 4096 * 32000


# ---- cases -------------------------------------------------------------------

def listed():
    return [
        # a projection of the framework's large product (16384 x 4096), laid out once
        {"name": "quantize_16384x4096_bf16", "op": "quantize", "dtype": "bf16", "n": 16384,
         "k": 4096, "group": 128, "scale": "bf16", "zeros": False},
        # a small layer of odd sizes in 32 bits, with zero points
        {"name": "quantize_small_fp32", "op": "quantize", "dtype": "fp32", "n": 333, "k": 1281,
         "group": 32, "scale": "fp32", "zeros": True},
        # one token through a 4096 x 4096 projection: latency and the weights' bytes
        {"name": "product_token_bf16", "op": "product", "dtype": "bf16", "out": "bf16", "m": 1,
         "n": 4096, "k": 4096, "group": 128, "scale": "bf16", "zeros": False, "act": "none"},
        # a few tokens into 1000 classes, odd depth, zero points, all in 32 bits
        {"name": "product_ragged_fp32", "op": "product", "dtype": "fp32", "out": "fp32", "m": 7,
         "n": 1000, "k": 1281, "group": 32, "scale": "fp32", "zeros": True, "act": "relu"},
        # the projection into a vocabulary for a few requests, logits in 32 bits
        {"name": "product_vocabulary_fp16", "op": "product", "dtype": "fp16", "out": "fp32",
         "m": 4, "n": 128000, "k": 4096, "group": 64, "scale": "fp16", "zeros": False,
         "act": "none"},
        # a serving batch through the wide projection of the framework's large product
        {"name": "product_batch_bf16", "op": "product", "dtype": "bf16", "out": "bf16", "m": 48,
         "n": 16384, "k": 4096, "group": 128, "scale": "bf16", "zeros": True, "act": "swish"},
        # a piece of a prompt
        {"name": "product_prompt_bf16", "op": "product", "dtype": "bf16", "out": "bf16", "m": 512,
         "n": 4096, "k": 4096, "group": 128, "scale": "bf16", "zeros": False, "act": "none"},
        # the token just sampled, with the alternatives that a client asks for
        {"name": "logprobs_token_bf16", "op": "logprobs", "dtype": "bf16", "rows": 1,
         "vocab": 128000, "top": 20, "temperature": 1.0},
        # a prompt scored, five alternatives for each of its tokens
        {"name": "logprobs_prompt_fp16", "op": "logprobs", "dtype": "fp16", "rows": 2048,
         "vocab": 50021, "top": 5, "temperature": 0.7},
        # a batch of class scores (1000 classes) in 32 bits, no alternatives
        {"name": "logprobs_classes_fp32", "op": "logprobs", "dtype": "fp32", "rows": 333,
         "vocab": 1000, "top": 0, "temperature": 1.0},
        # a training step's gradient into the logits
        {"name": "logprobs_grad_bf16", "op": "logprobs_grad", "dtype": "bf16", "rows": 4096,
         "vocab": 32000, "temperature": 1.0, "entropy": False},
        # a policy's step on a short odd batch: log probabilities and entropy
        {"name": "logprobs_grad_odd_fp32", "op": "logprobs_grad", "dtype": "fp32", "rows": 37,
         "vocab": 50021, "temperature": 0.7, "entropy": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "product", "logprobs", "logprobs",
                     "logprobs_grad"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op in ("quantize", "product"):
        case = {"op": op, "dtype": dtype, "group": rng.choice([32, 64, 128]),
                "scale": rng.choice(["fp32", dtype]), "zeros": rng.choice([False, True])}
        if op == "quantize":
            case["n"] = _log_int(rng, 1, 16384)
            case["k"] = _log_int(rng, 1, min(16384, 16384 * 4096 // (2 * case["n"])))
            return case
        case["m"] = rng.choice([1, _log_int(rng, 1, 16), _log_int(rng, 1, 512)])
        case["n"] = _log_int(rng, 16, 65536)
        most = min(LARGEST_WEIGHTS // (2 * case["n"]), LARGEST_PRODUCT // (4 * case["m"] * case["n"]))
        case["k"] = _log_int(rng, 16, max(16, min(16384, most)))
        case["out"] = rng.choice(["fp32", dtype])
        case["act"] = rng.choice(["none", "relu", "gelu", "swish"])
        return case
    rows = _log_int(rng, 1, 4096)
    case = {"op": op, "dtype": dtype, "rows": rows,
            "vocab": _log_int(rng, 2, min(262144, LARGEST_LOGITS // (2 * rows))),
            "temperature": rng.choice([0.6, 1.0, 1.3])}
    if op == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20, 32])
    else:
        case["entropy"] = rng.choice([False, True])
    return case


def _groups(case):
    return -(-case["k"] // case["group"])


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op in ("quantize", "product"):
        n, k = case["n"], case["k"]
        held = n * ((k + 1) // 2 + _groups(case) * (BYTES[case["scale"]] + case["zeros"]))
        if op == "quantize":
            return {"bytes": n * k * size + held, "flops": 5 * n * k}
        m = case["m"]
        return {"bytes": held + m * k * size + m * n * BYTES[case["out"]] + 4 * n,
                "flops": 2 * m * n * k}
    rows, e = case["rows"], case["rows"] * case["vocab"]
    if op == "logprobs":
        return {"bytes": e * size + rows * (8 + 16 + 12 * case["top"]), "flops": 6 * e}
    return {"bytes": 2 * e * size + rows * (8 + 12 + 8 * case["entropy"]), "flops": 6 * e}


# ---- inputs --------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _pitch(values):
    """Bytes of a row of 4-bit values, in whole 16-byte pieces as the product reads best."""
    return ((values + 1) // 2 + 15) // 16 * 16


def prepare(case, seed):
    g, op, t = _generator(seed), case["op"], TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    s = dict(case)
    if op in ("quantize", "product"):
        n, k, groups, st = case["n"], case["k"], _groups(case), TYPES[case["scale"]]
        if op == "quantize":
            # rows of their own spread, a few of them far larger
            s["w"] = (randn(n, k) * torch.exp(0.5 * randn(n, 1)) / math.sqrt(k)).to(t)
            s["q"] = torch.zeros(n, _pitch(k), device=DEVICE, dtype=torch.uint8)
            s["s"] = torch.empty(n, groups, device=DEVICE, dtype=st)
            s["z"] = torch.empty(n, groups, device=DEVICE, dtype=torch.uint8) if case["zeros"] else None
            return s
        m = case["m"]
        # normal weights in 4 bits, two a byte
        nibbles = torch.zeros(n, 2 * _pitch(k), device=DEVICE, dtype=torch.uint8)
        nibbles[:, :k] = (randn(n, k) * 2.5 + 8.0).round_().clamp_(0, 15).to(torch.uint8)
        s["q"] = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)
        del nibbles
        s["s"] = ((0.5 + torch.rand(n, groups, generator=g, device=DEVICE)) / (2.5 * math.sqrt(k))).to(st)
        s["z"] = (torch.randint(6, 11, (n, groups), generator=g, device=DEVICE, dtype=torch.uint8)
                  if case["zeros"] else None)
        s["x"] = (randn(m, k) * (0.5 + randn(k).abs())).to(t)
        s["bias"] = 0.1 * randn(n)
        s["c"] = torch.empty(m, n, device=DEVICE, dtype=TYPES[case["out"]])
        return s
    rows, vocab = case["rows"], case["vocab"]
    masked = vocab // 64
    logits = 2.5 * randn(rows, vocab)
    targets = torch.randint(0, vocab - masked, (rows,), generator=g, device=DEVICE)
    # most targets are likely ones, the vocabulary's padding is masked, a few
    # rows (a batch's padding) ask for no token
    likely = torch.rand(rows, generator=g, device=DEVICE) < 0.7
    logits[torch.arange(rows, device=DEVICE), targets] += 8.0 * likely
    logits[:, vocab - masked:] = -math.inf
    if rows > 1:
        targets[torch.rand(rows, generator=g, device=DEVICE) < 0.05] = -1
    s["logits"], s["targets"] = logits.to(t), targets
    s["factor"] = 1.0 / case["temperature"]
    f32 = lambda *shape: torch.empty(*shape, device=DEVICE)  # noqa: E731
    if op == "logprobs":
        s["logprob"], s["ent"], s["stats"] = f32(rows), f32(rows), f32(rows, 2)
        s["ids"] = torch.empty(rows, case["top"], device=DEVICE, dtype=torch.int64)
        s["top_logprob"] = f32(rows, case["top"])
        return s
    # what the forward pass kept
    s["stats"], s["ent"] = f32(rows, 2), f32(rows)
    factor = float(torch.tensor(s["factor"], dtype=torch.float32))
    for i in range(0, rows, 512):
        part = s["logits"][i:i + 512].double()
        top = part.amax(1)
        d = (part - top[:, None]) * factor
        log_sum = torch.log(torch.exp(d).sum(1))
        p = torch.exp(d - log_sum[:, None])
        s["stats"][i:i + 512, 0], s["stats"][i:i + 512, 1] = top, log_sum
        s["ent"][i:i + 512] = -(p * torch.where(p > 0, d - log_sum[:, None], 0.0)).sum(1)
    s["d_logprob"] = -1.0 / rows * (0.5 + torch.rand(rows, generator=g, device=DEVICE))
    s["d_entropy"] = -0.01 / rows * torch.ones(rows, device=DEVICE) if case["entropy"] else None
    s["dlogits"] = torch.empty_like(s["logits"])
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


def _plain_quantize(s):
    n, k, group, groups = s["n"], s["k"], s["group"], _groups(s)
    # the last group is filled up with zeros: they move neither a limit nor a scale
    w = torch.zeros(n, groups * group, device=DEVICE)
    w[:, :k] = s["w"].float()
    w = w.view(n, groups, group)
    # divided by tensors: torch divides by a number as a product with its reciprocal
    if s["z"] is None:
        top = w.abs().amax(2)
        scale = top / torch.full_like(top, 7.0)
    else:
        low, high = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
        scale = (high - low) / torch.full_like(low, 15.0)
    scale = scale.to(TYPES[s["scale"]]).clamp(min=TINY[s["scale"]])
    wide = scale.float()
    if s["z"] is None:
        zero = None
        nibble = torch.round(w / wide[:, :, None]).clamp(-8, 7) + 8
    else:
        zero = torch.round(-low / wide).clamp(0, 15)
        nibble = (torch.round(w / wide[:, :, None]) + zero[:, :, None]).clamp(0, 15)
        zero = zero.to(torch.uint8)
    nibble = nibble.view(n, -1)[:, :k]
    if k % 2:  # the half byte behind an odd row is 0
        nibble = torch.cat([nibble, nibble.new_zeros(n, 1)], 1)
    nibble = nibble.to(torch.uint8)
    out = {"q": nibble[:, 0::2] | (nibble[:, 1::2] << 4), "scale": scale}
    if zero is not None:
        out["zero"] = zero
    return out


def _plain_product(s):
    n, k, group = s["n"], s["k"], s["group"]
    nibble = torch.stack([s["q"] & 15, s["q"] >> 4], 2).view(n, -1)[:, :k].float()
    per_column = lambda t: t.float().repeat_interleave(group, 1)[:, :k]  # noqa: E731
    w = nibble - (per_column(s["z"]) if s["z"] is not None else 8.0)
    w = w * per_column(s["s"])
    return {"c": _act(s["x"].float() @ w.t() + s["bias"], s["act"]).to(s["c"].dtype)}


def _plain_logprobs(s):
    rows, x = torch.arange(s["rows"], device=DEVICE), s["logits"].float()
    top = x.amax(1, keepdim=True)
    d = (x - top) * s["factor"]
    e = torch.exp(d)
    total = e.sum(1)
    log_sum = torch.log(total)
    asked = s["targets"] >= 0
    given = d[rows, s["targets"].clamp(min=0)] - log_sum
    weighted = torch.where(e > 0, e * d, 0.0).sum(1)
    out = {"logprob": torch.where(asked, given, 0.0), "entropy": log_sum - weighted / total,
           "stats": torch.stack([top[:, 0], log_sum], 1)}
    ids, values, left = [], [], x
    column = torch.arange(s["vocab"], device=DEVICE)
    if s["top"]:
        left = x.clone()
    for _ in range(s["top"]):
        best = left.amax(1)
        # the first column that holds it
        at = torch.where(left == best[:, None], column, s["vocab"]).amin(1)
        none = best == -math.inf
        ids.append(torch.where(none, -1, at))
        values.append((best - top[:, 0]) * s["factor"] - log_sum)
        left[rows, at] = -math.inf
    out["ids"] = torch.stack(ids, 1) if ids else torch.empty_like(s["ids"])
    out["top_logprob"] = torch.stack(values, 1) if values else torch.empty_like(s["top_logprob"])
    return out


def _plain_logprobs_grad(s):
    rows, x = torch.arange(s["rows"], device=DEVICE), s["logits"].float()
    log_p = (x - s["stats"][:, :1]) * s["factor"] - s["stats"][:, 1:]
    p = torch.exp(log_p)
    asked = s["targets"] >= 0
    g = torch.where(asked, s["d_logprob"], 0.0)
    dx = -p * g[:, None]
    dx[rows, s["targets"].clamp(min=0)] += g
    if s["d_entropy"] is not None:
        moved = torch.where(p > 0, log_p + s["ent"][:, None], 0.0)
        dx = dx - s["d_entropy"][:, None] * p * moved
    return {"dlogits": (dx * s["factor"]).to(s["logits"].dtype)}


def _plain(s):
    return {"quantize": _plain_quantize, "product": _plain_product, "logprobs": _plain_logprobs,
            "logprobs_grad": _plain_logprobs_grad}[s["op"]](s)


_lib = None


def _library():
    global _lib
    if _lib is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "project-jcore_b200"))
        import npl_b200
        _lib = npl_b200.load()
    return _lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    lib, op = _library(), s["op"]
    stream = torch.cuda.current_stream().cuda_stream
    code = DTYPE_CODE[s["dtype"]]
    if op == "quantize":
        n, k, groups = s["n"], s["k"], _groups(s)
        rc = lib.nplk_quantize_w4(stream, n, k, s["group"], code, s["w"].data_ptr(), k,
                                  s["q"].data_ptr(), s["q"].stride(0), DTYPE_CODE[s["scale"]],
                                  s["s"].data_ptr(), groups, _ptr(s["z"]), groups)
        out = {"q": s["q"][:, :(k + 1) // 2], "scale": s["s"]}
        if s["z"] is not None:
            out["zero"] = s["z"]
    elif op == "product":
        m, n, k, groups = s["m"], s["n"], s["k"], _groups(s)
        rc = lib.nplk_gemm_w4(stream, m, n, k, s["group"], code, s["x"].data_ptr(), k,
                              s["q"].data_ptr(), s["q"].stride(0), DTYPE_CODE[s["scale"]],
                              s["s"].data_ptr(), groups, _ptr(s["z"]), groups,
                              s["bias"].data_ptr(), ACT_CODE[s["act"]], 0.0,
                              DTYPE_CODE[s["out"]], s["c"].data_ptr(), n, None)
        out = {"c": s["c"]}
    elif op == "logprobs":
        rc = lib.nplk_token_logprobs(stream, s["rows"], s["vocab"], code, s["logits"].data_ptr(),
                                     s["vocab"], s["factor"], s["targets"].data_ptr(),
                                     s["logprob"].data_ptr(), s["ent"].data_ptr(),
                                     s["stats"].data_ptr(), s["top"],
                                     s["ids"].data_ptr() if s["top"] else None,
                                     s["top_logprob"].data_ptr() if s["top"] else None)
        out = {"logprob": s["logprob"], "entropy": s["ent"], "stats": s["stats"],
               "ids": s["ids"], "top_logprob": s["top_logprob"]}
    else:
        rc = lib.nplk_token_logprobs_backward(
            stream, s["rows"], s["vocab"], code, s["logits"].data_ptr(), s["vocab"], s["factor"],
            s["targets"].data_ptr(), s["stats"].data_ptr(),
            s["ent"].data_ptr() if s["d_entropy"] is not None else None,
            s["d_logprob"].data_ptr(), _ptr(s["d_entropy"]), s["dlogits"].data_ptr(), s["vocab"])
        out = {"dlogits": s["dlogits"]}
    if rc != 0:
        raise RuntimeError(f"{op}: the library returned {rc}")
    return out


# ---- the definition in 64 bits ---------------------------------------------------

def _exact_act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * (1 + torch.tanh(GELU_C * (z + GELU_A * z ** 3))) / 2
    if name == "swish":
        return z * torch.sigmoid(z)
    return z


def _exact_limits(s):
    """Scales by the definition, a group of columns at a time, before their rounding."""
    scales = []
    for j in range(0, s["k"], s["group"]):
        part = s["w"][:, j:j + s["group"]].double()
        if s["z"] is None:
            scales.append(part.abs().max(dim=1).values / 7)
        else:
            high = part.max(dim=1).values.clamp(min=0)
            scales.append((high - part.min(dim=1).values.clamp(max=0)) / 15)
    return torch.stack(scales, 1).clamp(min=TINY[s["scale"]])


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantize":
        # the 4-bit numbers are roundings of quotients with the stored scale: no 64-bit value
        out = {"q": None, "scale": _exact_limits(s)}
        if case["zeros"]:
            out["zero"] = None
        return out
    if op == "product":
        k, group, rows = case["k"], case["group"], []
        x = s["x"].double()
        for i in range(0, case["n"], 16384):  # some output channels at a time
            q = s["q"][i:i + 16384].to(torch.int16)
            total = s["bias"][i:i + 16384].double().expand(case["m"], -1).clone()
            for j in range(0, k, group):  # a group at a time: its integers first, then its scale
                width = min(group, k - j)
                part = q[:, j // 2:(j + width + 1) // 2]
                value = torch.empty(part.shape[0], 2 * part.shape[1], device=DEVICE,
                                    dtype=torch.float64)
                value[:, 0::2], value[:, 1::2] = part % 16, part // 16
                zero = 8.0 if s["z"] is None else s["z"][i:i + 16384, j // group, None].double()
                inner = x[:, j:j + width] @ (value[:, :width] - zero).t()
                total += inner * s["s"][i:i + 16384, j // group].double()
            rows.append(_exact_act(total, case["act"]))
        return {"c": torch.cat(rows, 1)}
    factor = float(torch.tensor(s["factor"], dtype=torch.float32))  # as the call takes it
    parts = []
    for i in range(0, case["rows"], 256):
        z = s["logits"][i:i + 256].double()
        at = torch.arange(z.shape[0], device=DEVICE)
        target = s["targets"][i:i + 256]
        here = torch.where(target < 0, 0, target)
        if op == "logprobs":
            log_p = torch.log_softmax(z * factor, dim=1)
            top = z.max(dim=1).values
            order = torch.sort(z, dim=1, descending=True, stable=True)
            ids, best = order.indices[:, :case["top"]], order.values[:, :case["top"]]
            if ids.shape[1] < case["top"]:  # fewer tokens than alternatives
                more = case["top"] - ids.shape[1]
                ids = torch.nn.functional.pad(ids, (0, more), value=-1)
                best = torch.nn.functional.pad(best, (0, more), value=-math.inf)
            lse = torch.logsumexp(z * factor, dim=1)
            parts.append({
                "logprob": torch.where(target < 0, 0.0, log_p[at, here]),
                "entropy": torch.special.entr(torch.exp(log_p)).sum(1),
                "stats": torch.stack([top, lse - top * factor], 1),
                "ids": torch.where(best == -math.inf, -1, ids),
                "top_logprob": best * factor - lse[:, None]})
            continue
        # the statistics and the entropy are inputs of the call
        stats = s["stats"][i:i + 256].double()
        log_p = (z - stats[:, :1]) * factor - stats[:, 1:]
        p = torch.exp(log_p)
        hot = torch.zeros_like(z)
        hot[at, here] = 1.0
        g = torch.where(target < 0, 0.0, s["d_logprob"][i:i + 256].double())
        dz = (hot - p) * g[:, None]
        if case["entropy"]:
            h = s["d_entropy"][i:i + 256].double()
            dz += h[:, None] * (torch.special.entr(p) - p * s["ent"][i:i + 256].double()[:, None])
        parts.append({"dlogits": dz * factor})
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
