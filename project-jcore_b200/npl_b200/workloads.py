"""Device-resident compositions of the NPL benchmark workloads, as one caller
of the nplk_* ABI runs them back to back on one stream. The benchmark times
these functions and the parity tests check the same functions' outputs
against the reference's own CPU chain, so what is timed is what is checked.

All tensors are contiguous CUDA tensors on the current device, fp32 unless a
function says otherwise; `stream` is a cudaStream_t as c_void_p. Each function
returns 0 or the first non-zero library return code.
"""
from __future__ import annotations

import ctypes as C


def _p(t):
    return C.c_void_p(t.data_ptr())


def bandwidth_chain(lib, stream, x, w, mean, var, gamma, beta, dw_out, act_out, gap, probs,
                    eps: float = 1e-5) -> int:
    """depthwise 3x3 (stride 1, pad 1, no bias) -> inference batch norm ->
    ReLU in place -> global average pool -> softmax over the channels of each
    image: the reference's npl_depthwise_conv2d (npl_convolution.cpp:60-90),
    npl_batch_norm (npl_activation_norm.cpp:118-153), npl_relu (:51-54),
    npl_global_avg_pool (npl_pooling.cpp:63-87) and npl_softmax axis 1
    (npl_activation_norm.cpp:88-112).

    x, dw_out, act_out: [N, C, H, W]; w: [C, 1, 3, 3]; mean/var/gamma/beta:
    [C]; gap, probs: [N, C]. dw_out keeps the depthwise output, act_out the
    ReLU(BN(.)) output."""
    from . import conv_geom

    n, c, h, wd = x.shape
    g = conv_geom(n, c, h, wd, c, 3, 3, 1, 1)
    hw = h * wd
    rcs = (lib.nplk_depthwise_conv2d(stream, C.byref(g), _p(x), _p(w), None, _p(dw_out)),
           lib.nplk_batch_norm_infer(stream, n, c, hw, _p(dw_out), _p(act_out), _p(mean),
                                     _p(var), _p(gamma), _p(beta), eps),
           lib.nplk_activation(stream, n * c * hw, _p(act_out), _p(act_out), 1, 0.0, 0),
           lib.nplk_global_avg_pool(stream, n * c, hw, _p(act_out), _p(gap)),
           lib.nplk_softmax(stream, n, c, 1, _p(gap), _p(probs)))
    return next((r for r in rcs if r != 0), 0)


def bandwidth_chain_fused(lib, stream, x, w, mean, var, gamma, beta, gap, probs,
                          act_out=None, eps: float = 1e-5) -> int:
    """The same chain with its first four calls in one pass
    (nplk_depthwise_bn_act_gap: depthwise, BN, ReLU and the average pool
    without writing the intermediate maps; act_out, when given, receives the
    ReLU(BN(.)) map), then the softmax over the channels. gap and probs equal
    bandwidth_chain's bit for bit."""
    from . import conv_geom

    n, c, h, wd = x.shape
    g = conv_geom(n, c, h, wd, c, 3, 3, 1, 1)
    rc = lib.nplk_depthwise_bn_act_gap(stream, C.byref(g), _p(x), _p(w), None, _p(mean),
                                       _p(var), _p(gamma), _p(beta), eps, 1, 0.0,
                                       _p(act_out) if act_out is not None else None, _p(gap))
    if rc != 0:
        return rc
    return lib.nplk_softmax(stream, n, c, 1, _p(gap), _p(probs))


def gemm_bias_relu_layer_norm(lib, stream, A, B, Cm, Y, work, ws: int, eps: float = 1e-5,
                              flags: int = 0, between=None) -> int:
    """The large-GEMM workload after its bias fill: Cm = ReLU(A @ B + Cm) with
    Cm holding the per-column bias row in every row on entry (the reference's
    bias through beta = 1 on a pre-filled C, npl_tensor_ops.cpp:115-311, with
    npl_relu applied in the GEMM epilogue), then Y = layer norm of each row of
    Cm (gamma 1, beta 0; npl_activation_norm.cpp:470-522).

    A: [M, K]; B: [K, N]; Cm, Y: [M, N]; work: the GEMM's hi/lo workspace of
    `ws` bytes (nplk_gemm_workspace_size). `between`, if given, is called
    after the GEMM is launched and before the layer norm (a timing event)."""
    M, K = A.shape
    N = B.shape[1]
    rc = lib.nplk_gemm(stream, M, N, K, 1.0, _p(A), K, _p(B), N, 1.0, _p(Cm), N, None, 1, 0.0,
                       flags, _p(work), ws, None)
    if rc != 0:
        return rc
    if between is not None:
        between()
    return lib.nplk_layer_norm(stream, M, N, _p(Cm), _p(Y), None, None, eps)


def fill_bias_rows(Cm, bias) -> None:
    """Cm[i, :] = bias for every row (the pre-fill that carries the bias
    through beta = 1)."""
    Cm.copy_(bias.expand(Cm.shape[0], Cm.shape[1]))


def _dtype(t) -> int:
    """The NPLK_DTYPE_* code of a torch tensor."""
    from . import NPLK_DTYPE_BF16, NPLK_DTYPE_FP16, NPLK_DTYPE_FP32

    return {"torch.float32": NPLK_DTYPE_FP32, "torch.float16": NPLK_DTYPE_FP16,
            "torch.bfloat16": NPLK_DTYPE_BF16}[str(t.dtype)]


def norm_act_project_i8(lib, stream, x, groups, gamma, beta, act, y, q, q_scale, w, w_scale, bias,
                        out, work, ws: int, eps: float = 1e-5) -> int:
    """A served block's norm and projection: group norm with its activation over
    channels-last x, its rows (pixels) quantised to 8 bits, and their product
    with 8-bit weights.

    x, y: [N, HW, C] of one type; q: int8 [N * HW, ldq], ldq >= C (a multiple of
    16 for the tensor-core product); q_scale: [N * HW]; w: int8 [D, ldw] with
    w_scale [D] (nplk_quantize_rows of [D][C] weights or nplk_quantize_cols of
    [C][D] ones, once); bias: [D] or None; out: [N, HW, D] of any of the types;
    work: nplk_group_norm_workspace_size bytes."""
    n, hw, c = x.shape
    rows, d = n * hw, out.shape[2]
    rc = lib.nplk_group_norm_act(stream, n, hw, c, groups, _dtype(x), _p(x), c, _p(gamma),
                                 _p(beta), eps, act, 0.0, _p(y), c, None, None, _p(work), ws)
    if rc != 0:
        return rc
    rc = lib.nplk_quantize_rows(stream, rows, c, _dtype(y), _p(y), c, _p(q), q.stride(0),
                                _p(q_scale))
    if rc != 0:
        return rc
    return lib.nplk_gemm_i8(stream, rows, d, c, _p(q), q.stride(0), _p(q_scale), _p(w),
                            w.stride(0), _p(w_scale), _p(bias) if bias is not None else None, 0,
                            0.0, _dtype(out), _p(out), d, None)


def norm_act_dropout(lib, stream, x, groups, gamma, beta, act, p, seed, offset, y, mean, rstd,
                     work, ws: int, eps: float = 1e-5) -> int:
    """A trained block's norm, activation and dropout, y in place of both steps'
    results: y = dropout(act(group_norm(x))). x, y: [N, HW, C] of one type; mean,
    rstd: [N, groups], kept for the gradient."""
    n, hw, c = x.shape
    rc = lib.nplk_group_norm_act(stream, n, hw, c, groups, _dtype(x), _p(x), c, _p(gamma),
                                 _p(beta), eps, act, 0.0, _p(y), c, _p(mean), _p(rstd), _p(work),
                                 ws)
    if rc != 0:
        return rc
    return lib.nplk_dropout(stream, y.numel(), _dtype(y), _p(y), _p(y), p, seed, offset, None)


def norm_act_dropout_backward(lib, stream, dy, x, groups, mean, rstd, gamma, beta, act, p, seed,
                              offset, dx, dgamma, dbeta, work, ws: int) -> int:
    """The gradient of norm_act_dropout from the same seed and offset, in dx
    (which also holds the masked dy in between)."""
    n, hw, c = x.shape
    rc = lib.nplk_dropout(stream, dy.numel(), _dtype(dy), _p(dy), _p(dx), p, seed, offset, None)
    if rc != 0:
        return rc
    return lib.nplk_group_norm_act_backward(stream, n, hw, c, groups, _dtype(x), _p(dx), c, _p(x),
                                            c, _p(mean), _p(rstd), _p(gamma), _p(beta), act, 0.0,
                                            _p(dx), c, _p(dgamma), _p(dbeta), _p(work), ws)
