"""Weights in 4 bits for the tests: packing, what they stand for, and the calls."""
import torch

import support as S

TYPES = {"fp32": (torch.float32, 0), "fp16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
CODE = {v[0]: v[1] for v in TYPES.values()}


def ptr(t):
    return None if t is None else t.data_ptr()


def pack(nibbles, ldq=None, behind=0):
    """[N, K] numbers 0..15 as rows of ldq bytes; `behind` fills each byte past a row's end
    and the half byte behind an odd row."""
    n, k = nibbles.shape
    ldq = ldq or ((k + 1) // 2 + 15) // 16 * 16
    q = torch.full((n, ldq), behind, device=nibbles.device, dtype=torch.uint8)
    even = torch.full((n, (k + 1) // 2 * 2), behind & 15, device=nibbles.device, dtype=torch.uint8)
    even[:, :k] = nibbles.to(torch.uint8)
    q[:, :(k + 1) // 2] = even[:, 0::2] | (even[:, 1::2] << 4)
    return q


def unpack(q, k):
    return torch.stack([q & 15, q >> 4], 2).view(q.shape[0], -1)[:, :k]


def weights64(q, scale, zero, group, k):
    """What nibbles, scales and zeros stand for, in 64 bits: [N, K]."""
    wide = lambda t: t.double().repeat_interleave(group, 1)[:, :k]  # noqa: E731
    return wide(scale) * (unpack(q, k).double() - (8.0 if zero is None else wide(zero)))


def quantize(lib, w, group, scale_type, zeros, ldq=None, q=None):
    n, k = w.shape
    groups = -(-k // group)
    if q is None:
        q = torch.full((n, ldq or ((k + 1) // 2 + 15) // 16 * 16), 171, device=w.device,
                       dtype=torch.uint8)
    scale = torch.full((n, groups), 9.0, device=w.device, dtype=scale_type)
    zero = torch.full((n, groups), 99, device=w.device, dtype=torch.uint8) if zeros else None
    rc = lib.nplk_quantize_w4(S.cuda_stream(), n, k, group, CODE[w.dtype], w.data_ptr(),
                              w.stride(0), q.data_ptr(), q.stride(0), CODE[scale_type],
                              scale.data_ptr(), groups, ptr(zero), groups)
    assert rc == 0
    return q, scale, zero


def product(lib, x, q, scale, zero, group, n, k, bias=None, act=0, alpha=0.1,
            out=torch.float32, c=None, status=None, stream=None):
    m = x.shape[0]
    c = torch.full((m, n), 99.0, device=x.device, dtype=out) if c is None else c
    rc = lib.nplk_gemm_w4(stream or S.cuda_stream(), m, n, k, group, CODE[x.dtype], x.data_ptr(),
                          x.stride(0), q.data_ptr(), q.stride(0), CODE[scale.dtype],
                          scale.data_ptr(), scale.stride(0), ptr(zero),
                          zero.stride(0) if zero is not None else 0, ptr(bias), act, alpha,
                          CODE[c.dtype], c.data_ptr(), c.stride(0), ptr(status))
    assert rc == 0
    return c
