"""mlxr ops on the MoE path, over the gfx950 C ABI.

Same names, argument meaning and error behaviour as the reference's Rust
op wrappers; torch tensors on a ROCm device stand in for mlx arrays (torch
is plumbing here: device memory and the current stream).  Every array op
runs a kernel of libmlxr_moe.so; there is no fallback.

    quantize          crates/mlxr/src/ops/quantization.rs:47-70
    dequantize        crates/mlxr/src/ops/quantization.rs:118-146
    gather_qmm        crates/mlxr/src/ops/quantization.rs:171-221
    argpartition_axis crates/mlxr/src/ops/sort.rs:211-226
    softmax_axis      crates/mlxr/src/ops/arithmetic.rs:1298-1311

quantize, dequantize and gather_qmm take mode "mxfp4" (microscaled 4-bit
weights) beside "affine".  router_balance and router_balance_vjp, the router's
load-balance loss with its per-expert counts and the router's gradients, have no
counterpart there.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _capi as C
from ._capi import MlxrMoeError

DEFAULT_GROUP_SIZE = 64
DEFAULT_BITS = 4
# mode "mxfp4": e2m1 codes, a power-of-two scale byte per 32
MXFP4_GROUP_SIZE = 32
MODES = ("affine", "mxfp4")


def _check_mode(mode: str) -> bool:
    """True for mode "mxfp4"."""
    if mode not in MODES:
        raise MlxrMoeError(f"unsupported quantization mode {mode!r} (only {MODES})")
    return mode == "mxfp4"


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor):
    """The current stream of t's device, as a handle (a Stream object around it
    costs more than the launch)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


class _Here:
    """The device is the current one already."""

    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


_HERE = _Here()


def _on(t: torch.Tensor):
    """t's device as the current one (kernels are launched there)."""
    if torch._C._cuda_getDevice() == t.device.index:
        return _HERE
    return torch.cuda.device(t.device)


def _code(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return C.FLOAT32
    if t.dtype == torch.bfloat16:
        return C.BFLOAT16
    raise MlxrMoeError(f"unsupported dtype {t.dtype} (float32 or bfloat16)")


def _dev(*ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise MlxrMoeError("arrays must live on a ROCm device")
        d = t.device
        if dev is None:
            dev = d
        elif d != dev:
            raise MlxrMoeError("arrays live on different devices")
    return dev


def workspace(nbytes: int, device) -> torch.Tensor:
    """Device scratch for one call (torch's allocator aligns to 512 B)."""
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name: str, *sizes) -> int:
    """The library's workspace size for these sizes (a function of them alone)."""
    return getattr(C.lib(), f"mlxr_moe_{name}_workspace_size")(*sizes)


def _as_u32(idx: torch.Tensor) -> torch.Tensor:
    # mlx indices are uint32; int32 storage carries the same bits.
    if idx.dtype == torch.int32 and idx.is_contiguous():
        return idx
    if idx.dtype not in (torch.int32, torch.int64, torch.uint32):
        raise MlxrMoeError(f"indices must be integer, got {idx.dtype}")
    return _as_int32(idx)


def _as_int32(idx: torch.Tensor) -> torch.Tensor:
    """idx as contiguous int32.  64-bit values that do not fit go to the type's
    ends, which are out of every range here, not to their low bits."""
    if idx.dtype == torch.int64:
        idx = idx.clamp(-2 ** 31, 2 ** 31 - 1)
    return idx.to(torch.int32).contiguous()


def _check_x_batch(name: str, x_batch_shape, idx_shape):
    """Without lhs indices the kernels take x's batch b as b // (B // x_batch)
    (B = the index count): right for x's batch shape equal to the index
    shape's leading axes followed by singletons (x [.., T, 1, 1, K] against
    indices [.., T, top_k], or one x batch for all).  Other broadcasts (a
    leading singleton against a larger index axis) would pick wrong rows:
    they are rejected."""
    if (len(x_batch_shape) == len(idx_shape) and x_batch_shape[-1:] == (1,)
            and x_batch_shape[:-1] == idx_shape[:-1]):
        return  # x [.., T, 1, 1, K] against indices [.., T, top_k]
    xs = list(x_batch_shape)
    while len(xs) > len(idx_shape) and xs[0] == 1:
        xs.pop(0)
    ok = len(xs) <= len(idx_shape)
    if ok:
        pad = [1] * (len(idx_shape) - len(xs)) + xs
        j = 0
        while j < len(pad) and pad[j] == idx_shape[j]:
            j += 1
        ok = all(p == 1 for p in pad[j:])
    if not ok:
        raise MlxrMoeError(
            f"{name}: x batch shape {tuple(x_batch_shape)} must be the indices' leading axes "
            f"{tuple(idx_shape)} followed by singletons (or pass lhs_indices)")


def quantize(w: torch.Tensor, group_size=None, bits=None, mode="affine"):
    """(w_q, scales, biases) of MLX affine quantisation along the last axis.
    w_q is int32 storage of mlx's uint32 words.  Mode "mxfp4" (group_size 32,
    4 bits): e2m1 codes, scales uint8 (the exponent of a power of two plus
    127; 255 is NaN), biases None."""
    if _check_mode(mode):
        return _quantize_mxfp4(w, group_size, bits)
    _dev(w)
    w = w.contiguous()
    gs = DEFAULT_GROUP_SIZE if group_size is None else group_size
    b = DEFAULT_BITS if bits is None else bits
    cols = w.shape[-1]
    rows = w.numel() // cols if cols else 0
    lead = tuple(w.shape[:-1])
    if b in (2, 4, 8) and cols * b % 32 == 0 and gs and cols % gs == 0:
        wq = torch.empty(lead + (cols * b // 32,), dtype=torch.int32, device=w.device)
        sc = torch.empty(lead + (cols // gs,), dtype=w.dtype, device=w.device)
        bi = torch.empty_like(sc)
    else:  # let the library produce the error message
        wq = sc = bi = torch.empty(1, device=w.device)
    with _on(w):
        C.check(C.lib().mlxr_moe_quantize(
            _p(w), _code(w), rows, cols, C.OptionalInt.of(group_size), C.OptionalInt.of(bits),
            b"affine", _p(wq), _p(sc), _p(bi), _stream(w)))
    return wq, sc, bi


def _quantize_mxfp4(w, group_size, bits):
    _dev(w)
    w = w.contiguous()
    cols = w.shape[-1] if w.ndim else 0
    rows = w.numel() // cols if cols else 0
    lead = tuple(w.shape[:-1])
    ok = cols > 0 and cols % MXFP4_GROUP_SIZE == 0  # (else the library says what is wrong)
    wq = torch.empty(lead + (cols // 8,) if ok else 1, dtype=torch.int32, device=w.device)
    sc = torch.empty(lead + (cols // MXFP4_GROUP_SIZE,) if ok else 1, dtype=torch.uint8,
                     device=w.device)
    with _on(w):
        C.check(C.lib().mlxr_moe_quantize(
            _p(w), _code(w), rows, cols, C.OptionalInt.of(group_size), C.OptionalInt.of(bits),
            b"mxfp4", _p(wq), _p(sc), None, _stream(w)))
    return wq, sc, None


def _dense(*ts):
    """The tensors as contiguous ones, for the caller to hold until its call is made:
    the memory of a copy that nothing holds is the next copy's."""
    return [None if t is None else t.contiguous() for t in ts]


def _aligned(t, nbytes):
    """t, or a copy of it where its address is not a multiple of nbytes."""
    return t if t.data_ptr() % nbytes == 0 else t.clone()


def _check_mxfp4(name, w, scales, biases):
    """w [.., K/8] words and scales [.., K/32] bytes of the same rows: the C
    ABI reads that much of both."""
    if biases is not None:
        raise MlxrMoeError(f"{name}: mode mxfp4 has no biases")
    if w.dtype not in (torch.int32, torch.uint32) or scales.dtype != torch.uint8:
        raise MlxrMoeError(f"{name}: mode mxfp4 takes 32-bit words and uint8 scales, got "
                           f"{w.dtype} and {scales.dtype}")
    if (w.ndim < 1 or w.ndim != scales.ndim or w.shape[:-1] != scales.shape[:-1]
            or w.shape[-1] * 8 != scales.shape[-1] * MXFP4_GROUP_SIZE):
        raise MlxrMoeError(f"{name}: scales {tuple(scales.shape)} must hold one byte for each "
                           f"four words of w {tuple(w.shape)}")


def _dequantize_mxfp4(w, scales, biases, group_size, bits, out_dtype):
    _dev(w, scales)
    _check_mxfp4("dequantize", w, scales, biases)
    w, scales = w.contiguous(), scales.contiguous()
    cols = w.shape[-1] * 8
    rows = w.numel() // w.shape[-1] if cols else 0
    out = torch.empty(tuple(w.shape[:-1]) + (cols,), dtype=out_dtype or torch.bfloat16,
                      device=w.device)
    with _on(w):
        C.check(C.lib().mlxr_moe_dequantize(
            _p(w), _p(scales), None, C.UINT8, rows, cols, C.OptionalInt.of(group_size),
            C.OptionalInt.of(bits), b"mxfp4", _p(out), _code(out), _stream(w)))
    return out


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases=None, group_size=None,
               bits=None, out_dtype=None, mode="affine"):
    """code * scale + bias (one fused multiply-add, rounded once) in scales'
    dtype unless out_dtype is given.  Mode "mxfp4": code * scale, exact, in
    bf16 unless out_dtype is given."""
    if _check_mode(mode):
        return _dequantize_mxfp4(w, scales, biases, group_size, bits, out_dtype)
    _dev(w, scales, biases)
    w, scales, biases = _dense(w, scales, biases)
    b = DEFAULT_BITS if bits is None else bits
    cols = w.shape[-1] * 32 // b
    rows = w.numel() // w.shape[-1]
    out_dtype = out_dtype or scales.dtype
    out = torch.empty(tuple(w.shape[:-1]) + (cols,), dtype=out_dtype, device=w.device)
    with _on(w):
        C.check(C.lib().mlxr_moe_dequantize(
            _p(w), _p(scales), _p(biases), _code(scales), rows, cols,
            C.OptionalInt.of(group_size), C.OptionalInt.of(bits), b"affine", _p(out),
            _code(out), _stream(w)))
    return out


def gather_qmm(x, w, scales, biases=None, lhs_indices=None, rhs_indices=None,
               transpose=True, group_size=None, bits=None, sorted_indices=False,
               mode="affine"):
    """out[b] = x[xb(b)] @ dequant(w[rhs_indices[b]])^T.

    x [..., M, K] bf16; w [E, N, K*bits/32]; output rhs_indices.shape +
    [M, N].  Without lhs_indices, x's batch broadcasts over the trailing
    index axis (x [.., T, 1, 1, K] against indices [.., T, top_k]).  Mode
    "mxfp4": scales uint8 [E, N, K/32], no biases."""
    mx = _check_mode(mode)
    if rhs_indices is None:
        raise MlxrMoeError("gather_qmm: rhs_indices are required")
    if lhs_indices is None and rhs_indices.numel():
        _check_x_batch("gather_qmm", x.shape[:-2], tuple(rhs_indices.shape))
    _dev(x, w, scales, biases, lhs_indices, rhs_indices)
    b = DEFAULT_BITS if bits is None else bits
    x = x.contiguous()
    M, K = x.shape[-2], x.shape[-1]
    x_batch = math.prod(x.shape[:-2])
    E, N = w.shape[0], w.shape[1]
    if mx:
        _check_mxfp4("gather_qmm", w, scales, biases)
        if w.ndim != 3:
            raise MlxrMoeError("gather_qmm: w must be [E, N, K/8]")
        scales = _aligned(scales.contiguous(), 4)
    if w.shape[-1] * 32 != K * b and transpose:
        raise MlxrMoeError(
            f"gather_qmm: w last dim {w.shape[-1]} does not match K={K} at {b} bits")
    rhs = _as_u32(rhs_indices)
    lhs = None if lhs_indices is None else _as_u32(lhs_indices)
    B = rhs.numel()
    if lhs is not None and lhs.numel() != B:
        raise MlxrMoeError("gather_qmm: lhs and rhs indices must have the same size")
    out = torch.empty(tuple(rhs.shape) + (M, N), dtype=torch.bfloat16, device=x.device)
    lib = C.lib()
    ws = workspace(_workspace_bytes("gather_qmm", B, M, E), x.device)
    w, scales, biases = _dense(w, scales, biases)
    with _on(x):
        C.check(lib.mlxr_moe_gather_qmm(
            _p(x), _code(x), x_batch, M, K, _p(w), _p(scales), _p(biases),
            C.UINT8 if mx else _code(scales), E, N,
            _p(lhs), _p(rhs), B, int(bool(transpose)), C.OptionalInt.of(group_size),
            C.OptionalInt.of(bits), mode.encode(), int(bool(sorted_indices)), _p(out),
            C.BFLOAT16, _p(ws), ws.numel(), _stream(x)))
    out._mlxr_workspace = ws  # keep the status word alive with the result
    return out


def gather_mm(a, b, lhs_indices=None, rhs_indices=None, sorted_indices=False,
              b_transposed=True):
    """gather_mm (ops/arithmetic.rs:1577-1613) as SwitchLinear::apply calls
    it (nn/switch.rs:84-93): out[i] = a[ab(i)] @ b[rhs_indices[i]]^T with b
    the SwitchLinear weight as stored, bf16 [E, N, K] (the reference passes
    swap_axes(weight, -1, -2), the same memory).  a [..., M, K] bf16; output
    rhs_indices.shape + [M, N] bf16, f32 accumulation.  Without lhs_indices,
    a's batch broadcasts over the trailing index axis."""
    if rhs_indices is None:
        raise MlxrMoeError("gather_mm: rhs_indices are required")
    if lhs_indices is None and rhs_indices.numel():
        _check_x_batch("gather_mm", a.shape[:-2], tuple(rhs_indices.shape))
    _dev(a, b, lhs_indices, rhs_indices)
    if not b_transposed:
        raise MlxrMoeError("gather_mm: only b stored [E, N, K] (b_transposed) is supported")
    if b.ndim != 3:
        raise MlxrMoeError("gather_mm: b must be [E, N, K]")
    a = a.contiguous()
    M, K = a.shape[-2], a.shape[-1]
    a_batch = math.prod(a.shape[:-2])
    E, N = b.shape[0], b.shape[1]
    if b.shape[2] != K:
        raise MlxrMoeError(f"gather_mm: b last dim {b.shape[2]} does not match K={K}")
    rhs = _as_u32(rhs_indices)
    lhs = None if lhs_indices is None else _as_u32(lhs_indices)
    B = rhs.numel()
    if lhs is not None and lhs.numel() != B:
        raise MlxrMoeError("gather_mm: lhs and rhs indices must have the same size")
    out = torch.empty(tuple(rhs.shape) + (M, N), dtype=torch.bfloat16, device=a.device)
    lib = C.lib()
    ws = workspace(lib.mlxr_moe_gather_mm_workspace_size(B, M, E), a.device)
    bc = b.contiguous()
    with _on(a):
        C.check(lib.mlxr_moe_gather_mm(
            _p(a), _code(a), a_batch, M, K, _p(bc), _code(bc), E, N, 1, _p(lhs), _p(rhs), B,
            int(bool(sorted_indices)), _p(out), C.BFLOAT16, _p(ws), ws.numel(), _stream(a)))
    out._mlxr_workspace = ws  # keep the status word alive with the result
    return out


def _check_axis(a: torch.Tensor, axis: int, what: str) -> int:
    if not -a.ndim <= axis < a.ndim:
        raise MlxrMoeError(
            f"[{what}] Received invalid axis {axis} for array with {a.ndim} dimensions.")
    return axis % a.ndim


def argpartition_axis(a: torch.Tensor, kth: int, axis: int):
    """Indices partitioning `a` along `axis` around position kth (uint32
    semantics in int32 storage).  The full ascending order is returned,
    which satisfies every kth."""
    ax = _check_axis(a, axis, "argpartition")
    _dev(a)
    n = a.shape[ax]
    if not -n <= kth < n:
        raise MlxrMoeError(
            f"[argpartition] Received invalid kth {kth} along axis {axis} for array with "
            f"shape: {tuple(a.shape)}")
    if a.dtype != torch.float32:
        raise MlxrMoeError("argpartition: float32 input only")
    src = a.movedim(ax, -1).contiguous()
    out = torch.empty(src.shape, dtype=torch.int32, device=a.device)
    rows = src.numel() // n if n else 0
    with _on(a):
        C.check(C.lib().mlxr_moe_argpartition(_p(src), rows, n, kth, -1, _p(out), _stream(a)))
    return out.movedim(-1, ax)


def argpartition(a: torch.Tensor, kth: int):
    """argpartition over the flattened array (sort.rs:250-258)."""
    return argpartition_axis(a.reshape(-1), kth, 0)


def softmax_axis(a: torch.Tensor, axis: int, precise=None):
    ax = _check_axis(a, axis, "softmax")
    _dev(a)
    if a.dtype != torch.float32:
        raise MlxrMoeError("softmax: float32 input only")
    src = a.movedim(ax, -1).contiguous()
    n = src.shape[-1]
    out = torch.empty_like(src)
    with _on(a):
        C.check(C.lib().mlxr_moe_softmax(_p(src), src.numel() // max(n, 1), n, -1,
                                         int(bool(precise)), _p(out), _stream(a)))
    return out.movedim(-1, ax)


def _router_rows(name, x, d):
    """x bf16 [.., d] as rows: the C ABI reads T * d elements of that type."""
    if x.dtype != torch.bfloat16:
        raise MlxrMoeError(f"{name}: x must be bfloat16, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] != d:
        raise MlxrMoeError(f"{name}: x last dim must be {d}, got {tuple(x.shape)}")
    return x.reshape(-1, d).contiguous()


def router_topk(x: torch.Tensor, gate_w: torch.Tensor, k: int, return_logits=False):
    """softmax(x @ gate_w^T) -> top-k -> renormalise (moe.rs:122-138).
    Returns (indices int32 [T, k], weights f32 [T, k]), and with
    return_logits the f32 logits [T, E] too (what router_balance takes)."""
    if gate_w.ndim != 2 or gate_w.dtype != torch.float32:
        raise MlxrMoeError(f"router_topk: gate_w must be float32 [E, d], got {gate_w.dtype} "
                           f"{tuple(gate_w.shape)}")
    E, d = gate_w.shape
    gate_w, = _dense(gate_w)
    x2 = _router_rows("router_topk", x, d)
    _dev(x, gate_w)
    T = x2.shape[0]
    idx = torch.empty((T, k), dtype=torch.int32, device=x.device)
    wts = torch.empty((T, k), dtype=torch.float32, device=x.device)
    lib = C.lib()
    ws = workspace(lib.mlxr_moe_router_workspace_size(T, E), x.device)
    with _on(x):
        C.check(lib.mlxr_moe_router_topk(_p(x2), T, d, _p(gate_w), E, k, _p(idx),
                                         _p(wts), _p(ws), ws.numel(), _stream(x)))
    return _routing(x, k, E, idx, wts, ws, return_logits)


def _routing(x, k, E, idx, wts, ws, return_logits):
    lead = tuple(x.shape[:-1])
    out = idx.reshape(lead + (k,)), wts.reshape(lead + (k,))
    if not return_logits:
        return out
    T = idx.shape[0]  # the call's workspace is its logits [T, E] f32
    return out + (ws[:4 * T * E].view(torch.float32).reshape(lead + (E,)),)


def router_topk_quantized(x: torch.Tensor, gate, k: int, return_logits=False):
    """router_topk with the router as a QuantizedLinear (nn.QuantizedLinear,
    4 or 8 bits, group 64; layers/quantized.rs:356-373) or a bf16 Linear
    (nn.Linear): bf16 logits and probabilities, top-k on the probabilities.
    Returns (indices int32 [T, k], weights [T, k] -- bf16 values held in
    f32), and with return_logits the logits [T, E] (bf16 values in f32)."""
    x2 = _router_rows("router_topk_quantized", x, gate.input_dims)
    _dev(x, gate.weight)
    T = x2.shape[0]
    idx = torch.empty((T, k), dtype=torch.int32, device=x.device)
    wts = torch.empty((T, k), dtype=torch.float32, device=x.device)
    lib = C.lib()
    ws = workspace(lib.mlxr_moe_router_workspace_size(T, gate.output_dims), x.device)
    desc = gate.descriptor()
    with _on(x):
        C.check(lib.mlxr_moe_router_topk_quantized(_p(x2), T, ctypes.byref(desc), k, _p(idx),
                                                   _p(wts), _p(ws), ws.numel(), _stream(x)))
    return _routing(x, k, gate.output_dims, idx, wts, ws, return_logits)


def _balance_inputs(name, logits, indices, mask):
    """(logits rows, their stride, indices int32 [T, K], mask uint8 [T] or
    None) of router_balance and its gradient."""
    _dev(logits, indices, mask)
    E = logits.shape[-1] if logits.ndim else 0
    if logits.ndim < 1 or E < 1:
        raise MlxrMoeError(f"{name}: logits must be [.., T, E], got {tuple(logits.shape)}")
    if indices.ndim != logits.ndim or indices.shape[:-1] != logits.shape[:-1]:
        raise MlxrMoeError(f"{name}: indices {tuple(indices.shape)} must be [.., T, K] over "
                           f"logits {tuple(logits.shape)}")
    z = logits if logits.ndim == 2 else logits.reshape(-1, E)
    if z.stride(1) != 1 or z.stride(0) < E:
        z = z.contiguous()
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise MlxrMoeError(f"{name}: mask must be bool or uint8, got {mask.dtype}")
        if mask.shape != logits.shape[:-1]:
            raise MlxrMoeError(f"{name}: mask {tuple(mask.shape)} must be one value per token "
                               f"of logits {tuple(logits.shape)}")
        mask = mask.reshape(-1).contiguous()
    idx = _as_u32(indices)
    if idx.ndim != 2:  # (one token's [K] too)
        idx = idx.flatten(0, -2) if idx.ndim > 2 else idx[None]
    return z, max(z.stride(0), E), idx, mask


def router_balance(logits: torch.Tensor, indices: torch.Tensor, mask=None):
    """The load-balance loss of a router over its logits [.., T, E] (f32 or
    bf16) and its choices [.., T, K]: E * sum_e f_e P_e, f_e the share of the
    choices that fell on expert e and P_e its mean probability, over the
    tokens whose mask (bool or uint8, None: all) is not zero.  Returns (loss
    f32 [], counts int32 [E], probs f32 [E], tokens int32 []).  An index out
    of range is not counted and sets the workspace's status word.  The f_e sum
    to 1: a coefficient meant for shares of the tokens, which sum to K, is to
    be multiplied by K.  Not recorded by autograd: the gradient is
    router_balance_vjp's."""
    z, ld, idx, mask = _balance_inputs("router_balance", logits, indices, mask)
    (T, E), K = z.shape, idx.shape[1]
    dev = z.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    probs = torch.empty(E, dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    tokens = torch.empty((), dtype=torch.int32, device=dev)
    lib = C.lib()
    ws = workspace(_workspace_bytes("router_balance", T, E), dev)
    with _on(z):
        C.check(lib.mlxr_moe_router_balance(
            _p(z), _code(z), ld, T, E, _p(idx), K, _p(mask), _p(loss), _p(counts), _p(probs),
            _p(tokens), _p(ws), ws.numel(), _stream(z)))
    loss._mlxr_workspace = ws  # keep the status word alive with the result
    return loss, counts, probs, tokens


def router_balance_vjp(logits: torch.Tensor, indices: torch.Tensor, counts=None, tokens=None,
                       dloss=None, mask=None, dweights=None):
    """The gradient of router_balance's loss in the logits (their shape and
    dtype), for dloss f32 [] on the device, with counts and tokens as the
    forward call returned them; and, with dweights [.., T, K], plus that of
    router_topk's renormalised weights.  Masked tokens get zeros."""
    z, ld, idx, mask = _balance_inputs("router_balance_vjp", logits, indices, mask)
    (T, E), K = z.shape, idx.shape[1]
    _dev(z, counts, tokens, dloss, dweights)
    if dloss is not None:
        if dloss.dtype != torch.float32 or dloss.numel() != 1:
            raise MlxrMoeError("router_balance_vjp: dloss must be one float32")
        if counts is None or tokens is None:
            raise MlxrMoeError("router_balance_vjp: dloss takes the forward's counts and tokens")
        if (counts.dtype != torch.int32 or counts.shape != (E,)
                or tokens.dtype != torch.int32 or tokens.numel() != 1):
            raise MlxrMoeError(f"router_balance_vjp: counts must be int32 [{E}] and tokens one "
                               "int32")
        counts = counts.contiguous()
    if dweights is not None:
        if dweights.shape != indices.shape:
            raise MlxrMoeError(f"router_balance_vjp: dweights {tuple(dweights.shape)} must match "
                               f"indices {tuple(indices.shape)}")
        dweights = dweights.to(torch.float32).contiguous()
    dz = torch.empty((T, E), dtype=z.dtype, device=z.device)
    with _on(z):
        C.check(C.lib().mlxr_moe_router_balance_vjp(
            _p(z), _code(z), ld, T, E, _p(idx), K, _p(mask), _p(counts), _p(tokens), _p(dloss),
            _p(dweights), _p(dz), _stream(z)))
    return dz.reshape(logits.shape)


def dispatch(ids: torch.Tensor, num_experts: int):
    """Stable expert sort of flat ids (gather_sort, switch.rs:499-512).
    Returns (counts [E], offsets [E+1], order [n], inv_order [n])."""
    _dev(ids)
    flat = _as_u32(ids).reshape(-1)
    n = flat.numel()
    dev = ids.device
    counts = torch.empty(num_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    order = torch.empty(n, dtype=torch.int32, device=dev)
    inv = torch.empty(n, dtype=torch.int32, device=dev)
    lib = C.lib()
    ws = workspace(lib.mlxr_moe_dispatch_workspace_size(n, num_experts), dev)
    with _on(ids):
        C.check(lib.mlxr_moe_dispatch(_p(flat), n, num_experts, _p(counts), _p(offsets),
                                      _p(order), _p(inv), _p(ws), ws.numel(), _stream(ids)))
    order._mlxr_workspace = ws
    return counts, offsets, order, inv


def combine(y: torch.Tensor, weights: torch.Tensor, shared_y=None, shared_logit=None):
    """sum_k w * y over the top-k axis (combine_with_weights, switch.rs:
    223-234), plus shared_y * sigmoid(shared_logit) when given."""
    _dev(y, weights, shared_y, shared_logit)
    y, weights, shared_y, shared_logit = _dense(y, weights, shared_y, shared_logit)
    T, K, d = y.shape
    out = torch.empty((T, d), dtype=torch.float32, device=y.device)
    with _on(y):
        C.check(C.lib().mlxr_moe_combine(
            _p(y), _p(weights), T, K, d, _p(shared_y), _p(shared_logit), _p(out), _stream(y)))
    return out


def gather_qmm_tiled(rows: int, num_experts: int, mode="affine") -> bool:
    """True when a gather_qmm of `rows` flat rows over `num_experts` experts
    runs the M-tiled kernel (weights dequantised to bf16 tiles, the
    gather_mm(x, dequantize(w)) numerics), False for the streaming kernel
    (weights dequantised in f32).  Mode "mxfp4" has its own rule, and the same
    numerics in both."""
    _check_mode(mode)
    rc = C.lib().mlxr_moe_gather_qmm_tiled_mode(int(rows), int(num_experts), mode.encode())
    if rc < 0:
        raise MlxrMoeError("gather_qmm_tiled: negative size")
    return bool(rc)


def router_matrix_order(T: int, d: int, columns: int) -> bool:
    """True when a router's logits of T tokens over d inputs, `columns`
    logit columns (the experts, plus one for a shared-expert gate computed
    beside them), are summed in the matrix-core order (the oracle's
    router_logits(mfma=True)), False for the lane order."""
    rc = C.lib().mlxr_moe_router_matrix_order(int(T), int(d), int(columns))
    if rc < 0:
        raise MlxrMoeError("router_matrix_order: negative size")
    return bool(rc)


def workspace_status(ws: torch.Tensor) -> int:
    """Device status word of a call's workspace (1 = an index was out of
    range).  Synchronises the current stream."""
    with _on(ws):
        rc = C.lib().mlxr_moe_workspace_status(_p(ws), ws.numel(), _stream(ws))
    if rc < 0:
        raise MlxrMoeError(C.last_error())
    return rc
