"""torch-facing wrappers over the raw C ABI (include/fmxq.h).

Tensors are device buffers only: bf16 values travel as ``torch.bfloat16`` or
``torch.int16``/``torch.uint16`` bit patterns, packed weights as ``torch.int32``
or ``torch.uint32``, indices as ``torch.int32``/``torch.uint32``.  Every call
is enqueued on torch's current HIP stream.  Nothing here computes on the CPU.
"""
from __future__ import annotations

import torch

from ._lib import check, load

try:
    # The same calls checked and launched from C++ (ext/fmxq_fast.cpp): a function
    # returns None for anything out of the ordinary, and the Python path below takes it.
    from . import _fast
except ImportError:  # not built: every call takes the Python path
    _fast = None

_BF16_LIKE = (torch.bfloat16, torch.int16, torch.uint16)
_U32_LIKE = (torch.int32, torch.uint32)


def _dev(t: torch.Tensor, name: str, dtypes) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on the GPU (got {t.device})")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected one of {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def dequantize(w, scales, biases, group_size: int = 64, bits: int = 4, out=None):
    """MLX dequantize: [..., K*bits/32] packed -> [..., K] bf16."""
    if _fast is not None:
        y = _fast.dequantize(w, scales, biases, out, group_size, bits)
        if y is not None:
            return y
    K = w.shape[-1] * 32 // bits
    rows = w.numel() // max(w.shape[-1], 1)
    if out is None:
        out = torch.empty(*w.shape[:-1], K, dtype=torch.bfloat16, device=w.device)
    check(load().fmxq_dequantize(_dev(w, "w", _U32_LIKE), _dev(scales, "scales", _BF16_LIKE),
                                 _dev(biases, "biases", _BF16_LIKE), _dev(out, "out", _BF16_LIKE),
                                 rows, K, group_size, bits, _stream(w)))
    return out


def quantize(w, group_size: int = 64, bits: int = 4, out=None):
    """MLX affine quantize: bf16 [..., K] -> (packed [..., K*bits/32] int32 words,
    scales [..., K/group] bf16, biases [..., K/group] bf16); ``out`` may hold the
    three result tensors."""
    if _fast is not None and out is None:
        q = _fast.quantize(w, group_size, bits)
        if q is not None:
            return q
    K = w.shape[-1]
    rows = w.numel() // max(K, 1)
    if K % group_size:
        raise ValueError(f"K={K} is not a multiple of group_size={group_size}")
    if out is None:
        wq = torch.empty(*w.shape[:-1], K * bits // 32, dtype=torch.int32, device=w.device)
        scales = torch.empty(*w.shape[:-1], K // group_size, dtype=torch.bfloat16,
                             device=w.device)
        biases = torch.empty_like(scales)
    else:
        wq, scales, biases = out
    check(load().fmxq_quantize(_dev(w, "w", _BF16_LIKE), _dev(wq, "wq", _U32_LIKE),
                               _dev(scales, "scales", _BF16_LIKE),
                               _dev(biases, "biases", _BF16_LIKE), rows, K, group_size, bits,
                               _stream(w)))
    return wq, scales, biases


def quantized_matmul(x, w, scales, biases, transpose: bool = True, group_size: int = 64,
                     bits: int = 4, bias=None, out=None):
    """y = x @ deq(W)^T over x [..., K]; W [N, K*bits/32]; y [..., N] bf16."""
    if _fast is not None and transpose is True:
        y = _fast.quantized_matmul(x, w, scales, biases, bias, out, group_size, bits)
        if y is not None:
            return y
    K = x.shape[-1]
    N = w.shape[0]
    M = x.numel() // max(K, 1)
    if w.shape[-1] * 32 // bits != K:
        raise ValueError(f"x has K={K} but w packs {w.shape[-1] * 32 // bits} values per row")
    if out is None:
        out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    lib = load()
    args = (_dev(x, "x", _BF16_LIKE), _dev(w, "w", _U32_LIKE),
            _dev(scales, "scales", _BF16_LIKE), _dev(biases, "biases", _BF16_LIKE))
    if bias is None:
        check(lib.fmxq_quantized_matmul(*args, _dev(out, "out", _BF16_LIKE), M, N, K, transpose,
                                        group_size, bits, _stream(x)))
    else:
        check(lib.fmxq_quantized_matmul_bias(*args, _dev(bias, "bias", _BF16_LIKE),
                                             _dev(out, "out", _BF16_LIKE), M, N, K, transpose,
                                             group_size, bits, _stream(x)))
    return out


def quantized_matmul_group(x, mats, group_size: int = 64, bits: int = 4, outs=None):
    """Several products of the same x [..., K]: mats is a list of (w, scales, biases)
    triples (1 to 4), the result a list of y [..., N_i] bf16 (one launch where the
    shapes allow, fmxq_quantized_matmul_group)."""
    import ctypes

    K = x.shape[-1]
    M = x.numel() // max(K, 1)
    n = len(mats)
    for w, _, _ in mats:
        if w.shape[-1] * 32 // bits != K:
            raise ValueError(f"x has K={K} but w packs {w.shape[-1] * 32 // bits} values per row")
    if outs is None:
        outs = [torch.empty(*x.shape[:-1], w.shape[0], dtype=torch.bfloat16, device=x.device)
                for w, _, _ in mats]
    P = ctypes.c_void_p * n
    ws = P(*[_dev(w, "w", _U32_LIKE) for w, _, _ in mats])
    ss = P(*[_dev(s, "scales", _BF16_LIKE) for _, s, _ in mats])
    bs = P(*[_dev(b, "biases", _BF16_LIKE) for _, _, b in mats])
    ys = P(*[_dev(y, "out", _BF16_LIKE) for y in outs])
    Ns = (ctypes.c_int64 * n)(*[w.shape[0] for w, _, _ in mats])
    check(load().fmxq_quantized_matmul_group(_dev(x, "x", _BF16_LIKE), n, ws, ss, bs, ys, Ns, M, K,
                                             True, group_size, bits, _stream(x)))
    return outs


def gather_qmm(x, w, scales, biases, rhs_indices, lhs_indices=None, lhs_div: int = 1,
               transpose: bool = True, group_size: int = 64, bits: int = 4,
               sorted_indices: bool = False, out=None):
    """Flat-index gather_qmm (raw ABI form).

    x [x_batch, Mx, K]; w [E, N, K*bits/32]; rhs_indices [batch];
    lhs_indices [batch] or None (then item i reads x[i // lhs_div]).
    Returns y [batch, Mx, N]."""
    if x.dim() != 3:
        raise ValueError("x must be [x_batch, Mx, K] in the flat form")
    x_batch, Mx, K = x.shape
    E, N = w.shape[0], w.shape[1]
    batch = rhs_indices.numel()
    if out is None:
        out = torch.empty(batch, Mx, N, dtype=torch.bfloat16, device=x.device)
    lhs_ptr = None if lhs_indices is None else _dev(lhs_indices, "lhs_indices", _U32_LIKE)
    check(load().fmxq_gather_qmm(_dev(x, "x", _BF16_LIKE), _dev(w, "w", _U32_LIKE),
                                 _dev(scales, "scales", _BF16_LIKE),
                                 _dev(biases, "biases", _BF16_LIKE), lhs_ptr,
                                 _dev(rhs_indices, "rhs_indices", _U32_LIKE),
                                 _dev(out, "out", _BF16_LIKE), batch, x_batch, lhs_div, Mx, N, K,
                                 E, transpose, group_size, bits, sorted_indices, _stream(x)))
    return out


def switch_glu(x, inds, gate, up, down, group_size: int = 64, bits: int = 4, out=None):
    """SwitchGLU over stacked quantized experts (switchGLUCore).

    x [T, D] bf16; inds [T, top_k] int32/uint32; gate/up/down are (w, scales, biases)
    triples with w [E, I, D*bits/32] (gate, up) and [E, D, I*bits/32] (down).
    Returns [T, top_k, D] bf16."""
    T, D = x.shape
    topk = inds.shape[-1]
    E, I = gate[0].shape[0], gate[0].shape[1]
    if out is None:
        out = torch.empty(T, topk, D, dtype=torch.bfloat16, device=x.device)
    p = [_dev(x, "x", _BF16_LIKE), _dev(inds, "inds", _U32_LIKE)]
    for name, (w, s, b) in (("gate", gate), ("up", up), ("down", down)):
        p += [_dev(w, f"{name}.w", _U32_LIKE), _dev(s, f"{name}.scales", _BF16_LIKE),
              _dev(b, f"{name}.biases", _BF16_LIKE)]
    check(load().fmxq_switch_glu(*p, _dev(out, "out", _BF16_LIKE), T, topk, E, D, I, group_size,
                                 bits, _stream(x)))
    return out


def switch_glu_combine(x, inds, gate, up, down, weights, shared=None, shared_gate=None,
                       group_size: int = 64, bits: int = 4, out=None):
    """One MoE layer's routed part: switch_glu then moe_combine in one call.

    weights [T, top_k] bf16; shared [T, D] (optional) is added, sigmoid-gated by
    shared_gate [T] when given.  Returns [T, D] bf16."""
    if _fast is not None:
        y = _fast.moe_layer(x, inds, gate, up, down, weights, None, shared, shared_gate, out,
                            group_size, bits)
        if y is not None:
            return y
    T, D = x.shape
    topk = inds.shape[-1]
    E, I = gate[0].shape[0], gate[0].shape[1]
    if out is None:
        out = torch.empty(T, D, dtype=torch.bfloat16, device=x.device)
    p = [_dev(x, "x", _BF16_LIKE), _dev(inds, "inds", _U32_LIKE)]
    for name, (w, s, b) in (("gate", gate), ("up", up), ("down", down)):
        p += [_dev(w, f"{name}.w", _U32_LIKE), _dev(s, f"{name}.scales", _BF16_LIKE),
              _dev(b, f"{name}.biases", _BF16_LIKE)]
    sp = None if shared is None else _dev(shared, "shared", _BF16_LIKE)
    gp = None if shared_gate is None else _dev(shared_gate, "shared_gate", _BF16_LIKE)
    check(load().fmxq_switch_glu_combine(*p, _dev(weights, "weights", _BF16_LIKE), sp, gp,
                                         _dev(out, "out", _BF16_LIKE), T, topk, E, D, I,
                                         group_size, bits, _stream(x)))
    return out


def moe_layer(x, inds, gate, up, down, weights, shared_expert, shared_gate=None,
              group_size: int = 64, bits: int = 4, out=None):
    """switch_glu_combine with the shared expert computed in the same call.

    shared_expert = (gate, up, down) triples of a one-expert stack; shared_gate [T]
    (optional) sigmoid-gates its output.  Returns [T, D] bf16."""
    if _fast is not None and shared_expert is not None:
        y = _fast.moe_layer(x, inds, gate, up, down, weights, shared_expert, None, shared_gate, out,
                            group_size, bits)
        if y is not None:
            return y
    T, D = x.shape
    topk = inds.shape[-1]
    E, I = gate[0].shape[0], gate[0].shape[1]
    if out is None:
        out = torch.empty(T, D, dtype=torch.bfloat16, device=x.device)
    p = [_dev(x, "x", _BF16_LIKE), _dev(inds, "inds", _U32_LIKE)]
    for name, (w, s, b) in (("gate", gate), ("up", up), ("down", down)):
        p += [_dev(w, f"{name}.w", _U32_LIKE), _dev(s, f"{name}.scales", _BF16_LIKE),
              _dev(b, f"{name}.biases", _BF16_LIKE)]
    p.append(_dev(weights, "weights", _BF16_LIKE))
    for name, (w, s, b) in zip(("shared.gate", "shared.up", "shared.down"), shared_expert):
        p += [_dev(w, f"{name}.w", _U32_LIKE), _dev(s, f"{name}.scales", _BF16_LIKE),
              _dev(b, f"{name}.biases", _BF16_LIKE)]
    gp = None if shared_gate is None else _dev(shared_gate, "shared_gate", _BF16_LIKE)
    check(load().fmxq_moe_layer(*p, gp, _dev(out, "out", _BF16_LIKE), T, topk, E, D, I,
                                group_size, bits, _stream(x)))
    return out


def moe_combine(y, weights, shared=None, shared_gate=None, out=None):
    """sum_j y[:, j] * weights[:, j] (+ shared, optionally sigmoid-gated); y [T, k, D]."""
    T, topk, D = y.shape
    if out is None:
        out = torch.empty(T, D, dtype=torch.bfloat16, device=y.device)
    sp = None if shared is None else _dev(shared, "shared", _BF16_LIKE)
    gp = None if shared_gate is None else _dev(shared_gate, "shared_gate", _BF16_LIKE)
    check(load().fmxq_moe_combine(_dev(y, "y", _BF16_LIKE), _dev(weights, "weights", _BF16_LIKE),
                                  sp, gp, _dev(out, "out", _BF16_LIKE), T, topk, D, _stream(y)))
    return out


def _route_io(logits, T, k, weights_dtype):
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"router logits must be bfloat16 or float32, got {logits.dtype}")
    if weights_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"router weights must be bfloat16 or float32, got {weights_dtype}")
    inds = torch.empty(T, k, dtype=torch.int32, device=logits.device)
    weights = torch.empty(T, k, dtype=weights_dtype, device=logits.device)
    return inds, weights


def route_softmax_topk(logits, top_k, norm_topk_prob=True, weights_dtype=torch.bfloat16):
    """Softmax router (qwen3next_forward.go:513-518): logits [T, E] -> (inds [T, k] int32
    holding uint32 ids, weights [T, k]), largest gate first."""
    if _fast is not None and weights_dtype in (torch.bfloat16, torch.float32):
        r = _fast.route_softmax_topk(logits, top_k, bool(norm_topk_prob),
                                     weights_dtype is torch.bfloat16)
        if r is not None:
            return r
    T, E = logits.shape
    inds, weights = _route_io(logits, T, top_k, weights_dtype)
    ptr = _dev(logits, "logits", (torch.bfloat16, torch.float32))
    check(load().fmxq_route_softmax_topk(ptr, int(logits.dtype == torch.bfloat16), T, E, top_k,
                                         bool(norm_topk_prob), _dev(inds, "inds", _U32_LIKE),
                                         weights.data_ptr(),
                                         int(weights_dtype == torch.bfloat16), _stream(logits)))
    return inds, weights


def route_group_topk(gates, bias, top_k, n_group, topk_group, routed_scaling_factor=1.0,
                     norm_topk_prob=True, weights_dtype=torch.float32):
    """DeepSeek-V3 group-limited router (deepseekv3_forward.go:452-491): gates [T, E],
    bias [E] float32 or None -> (inds [T, k] int32 holding uint32 ids, weights [T, k])."""
    if _fast is not None and weights_dtype in (torch.bfloat16, torch.float32):
        r = _fast.route_group_topk(gates, bias, top_k, n_group, topk_group,
                                   float(routed_scaling_factor), bool(norm_topk_prob),
                                   weights_dtype is torch.bfloat16)
        if r is not None:
            return r
    T, E = gates.shape
    inds, weights = _route_io(gates, T, top_k, weights_dtype)
    bptr = None if bias is None else _dev(bias, "bias", (torch.float32,))
    ptr = _dev(gates, "gates", (torch.bfloat16, torch.float32))
    check(load().fmxq_route_group_topk(ptr, int(gates.dtype == torch.bfloat16), bptr, T, E, top_k,
                                       n_group, topk_group, float(routed_scaling_factor),
                                       bool(norm_topk_prob), _dev(inds, "inds", _U32_LIKE),
                                       weights.data_ptr(), int(weights_dtype == torch.bfloat16),
                                       _stream(gates)))
    return inds, weights


# ---- training and scoring over quantized weights --------------------------------
# Plain functions, forward and backward, without autograd: a gradient is a call of its own.


def _same_device(**tensors):
    """The tensors' device; ValueError where they are on several."""
    dev = None
    for name, t in tensors.items():
        if t is None and name == "grad_loss":
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if dev is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, other operands on {dev}")
        dev = t.device
    if dev is None or dev.type != "cuda":
        raise ValueError(f"operands must live on the GPU (got {dev})")
    return dev


def _shape(name, t, *shape):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _quant_shapes(w, scales, biases, lead, K, group_size, bits):
    if bits not in (4, 8) or group_size not in (32, 64, 128):
        return  # refused by the library, which names the supported ones
    if K % group_size:
        raise ValueError(f"K={K} is not a multiple of group_size={group_size}")
    _shape("w", w, *lead, K * bits // 32)
    _shape("scales", scales, *lead, K // group_size)
    _shape("biases", biases, *lead, K // group_size)


def _workspace(fn, dev, *sizes, more=0):
    """A workspace for a call with these sizes (and `more` bytes), from torch's allocator: its own
    in every call, stream and captured graph.  (pointer, bytes, the tensor that keeps it)"""
    import ctypes

    n = ctypes.c_size_t()
    check(fn(*sizes, ctypes.byref(n)))
    bytes_ = n.value + more
    t = torch.empty(bytes_, dtype=torch.uint8, device=dev)
    return (t.data_ptr() if bytes_ else None), bytes_, t


def _moved(dy):
    """The bytes that a gradient takes to move rows that do not begin at 16 bytes."""
    return 256 + dy.numel() * 2 if dy.data_ptr() % 16 and dy.shape[-1] % 8 == 0 else 0


def _head_operands(h, w, scales, biases, grad, grad_loss, group_size, bits):
    if h.dim() != 2 or w.dim() != 2:
        raise ValueError("h must be [M, K] and w [V, K*bits/32]")
    M, K = h.shape
    V = w.shape[0]
    _quant_shapes(w, scales, biases, (V,), K, group_size, bits)
    if grad_loss is not None:
        if not grad:
            raise ValueError("grad_loss without grad=True")
        _shape("grad_loss", grad_loss, M)
        _dev(grad_loss, "grad_loss", (torch.float32,))
    ptrs = (_dev(h, "h", _BF16_LIKE), _dev(w, "w", _U32_LIKE), _dev(scales, "scales", _BF16_LIKE),
            _dev(biases, "biases", _BF16_LIKE))
    return M, V, K, ptrs


def _head_results(M, K, dev, grad):
    loss = torch.empty(M, dtype=torch.float32, device=dev)
    lse = torch.empty(M, dtype=torch.float32, device=dev)
    dh = torch.empty(M, K, dtype=torch.bfloat16, device=dev) if grad else None
    return loss, lse, dh


def _ptr(t):
    return None if t is None else t.data_ptr()


def head_cross_entropy(h, w, scales, biases, targets, ignore_index: int = -100, grad: bool = False,
                       grad_loss=None, group_size: int = 64, bits: int = 4):
    """Cross entropy of a quantized vocabulary head, its logits never stored.

    h [M, K] bf16; w [V, K*bits/32] with scales and biases [V, K/group]; targets [M] int32.
    Returns (loss [M], lse [M]) float32 with lse the log of the row's sum of exponentials, and
    with ``grad`` also dh [M, K] bf16, the gradient of sum_t grad_loss[t] loss[t] (grad_loss
    [M] float32, ones without).  A target equal to ignore_index has loss and gradient 0; one
    outside the vocabulary too, which device_error reports."""
    if _fast is not None:
        r = _fast.head_loss(h, w, scales, biases, targets, None, 1.0, ignore_index, bool(grad),
                            grad_loss, group_size, bits)
        if r is not None:
            return r
    dev = _same_device(h=h, w=w, scales=scales, biases=biases, targets=targets,
                       grad_loss=grad_loss)
    M, V, K, ptrs = _head_operands(h, w, scales, biases, grad, grad_loss, group_size, bits)
    _shape("targets", targets, M)
    tp = _dev(targets, "targets", (torch.int32,))
    lib = load()
    with torch.cuda.device(dev):
        loss, lse, dh = _head_results(M, K, dev, grad)
        ws, n, keep = _workspace(lib.fmxq_head_workspace, dev, M, V, K, 1, bool(grad))
        check(lib.fmxq_head_cross_entropy(*ptrs, tp, _ptr(grad_loss), loss.data_ptr(),
                                          lse.data_ptr(), _ptr(dh), M, V, K, ignore_index,
                                          group_size, bits, ws, n, _stream(h)))
    return (loss, lse, dh) if grad else (loss, lse)


def head_distill(h, w, scales, biases, ids, teacher, temperature: float = 1.0, grad: bool = False,
                 grad_loss=None, group_size: int = 64, bits: int = 4):
    """Divergence of a quantized head's softmax from a teacher's top logits.

    ids [M, k] int32 and teacher [M, k] (bfloat16 or float32): the tokens and logits the
    teacher kept, k <= 64, an id below zero for an absent entry.  With q = softmax(teacher / T)
    over the entries and p = softmax(logits / T) over the vocabulary, returns (loss [M] =
    T^2 KL(q || p), lse [M] = log sum exp(logits / T)) float32, and with ``grad`` dh [M, K] as
    head_cross_entropy does."""
    if _fast is not None and teacher is not None:
        r = _fast.head_loss(h, w, scales, biases, ids, teacher, float(temperature), 0, bool(grad),
                            grad_loss, group_size, bits)
        if r is not None:
            return r
    dev = _same_device(h=h, w=w, scales=scales, biases=biases, ids=ids, teacher=teacher,
                       grad_loss=grad_loss)
    M, V, K, ptrs = _head_operands(h, w, scales, biases, grad, grad_loss, group_size, bits)
    if ids.dim() != 2:
        raise ValueError("ids must be [M, k]")
    k = min(ids.shape[1], 2**31 - 1)  # more than 64 are refused by the library
    _shape("ids", ids, M, k)
    _shape("teacher", teacher, M, k)
    ip = _dev(ids, "ids", (torch.int32,))
    tp = _dev(teacher, "teacher", (torch.bfloat16, torch.float32))
    lib = load()
    with torch.cuda.device(dev):
        loss, lse, dh = _head_results(M, K, dev, grad)
        ws, n, keep = _workspace(lib.fmxq_head_workspace, dev, M, V, K, k, bool(grad))
        check(lib.fmxq_head_distill(*ptrs, ip, tp, int(teacher.dtype == torch.bfloat16),
                                    _ptr(grad_loss), loss.data_ptr(), lse.data_ptr(), _ptr(dh), M,
                                    V, K, k, temperature, group_size, bits, ws, n, _stream(h)))
    return (loss, lse, dh) if grad else (loss, lse)


def _score_operands(h, w, scales, biases, ids, group_size, bits):
    M, V, K, ptrs = _head_operands(h, w, scales, biases, False, None, group_size, bits)
    if ids.dim() != 2:
        raise ValueError("ids must be [M, k]")
    k = min(ids.shape[1], 2**31 - 1)  # more than 64 are refused by the library
    _shape("ids", ids, M, k)
    return M, V, K, k, (*ptrs, _dev(ids, "ids", (torch.int32,)))


def head_logprobs(h, w, scales, biases, ids, top: int = 0, temperature: float = 1.0,
                  group_size: int = 64, bits: int = 4):
    """Log probabilities of given tokens through a quantized vocabulary head, its logits never
    returned, with the entropy and the likeliest tokens.

    h [M, K] bf16; w [V, K*bits/32] with scales and biases [V, K/group]; ids [M, k] int32, k <= 64,
    an id below zero for an absent entry (0 in logp).  With l = logits / temperature and p =
    softmax(l): (logp [M, k], entropy [M], lse [M]) float32, and with ``top`` (up to 64) also
    (top_ids [M, top] int32, top_logp [M, top]), likeliest first, equal ones to the lower token.
    The order is that of logits summed in 64 bits, at any temperature.  An id past the vocabulary counts
    as absent, and device_error reports it.  A row with a logit that is not finite gives NaN and
    top_ids -1."""
    if _fast is not None:
        r = _fast.head_logprobs(h, w, scales, biases, ids, top, float(temperature), group_size, bits)
        if r is not None:
            return r
    dev = _same_device(h=h, w=w, scales=scales, biases=biases, ids=ids)
    M, V, K, k, ptrs = _score_operands(h, w, scales, biases, ids, group_size, bits)
    top = min(max(int(top), -1), 2**31 - 1)  # outside 0 .. 64 the library refuses
    lib = load()
    with torch.cuda.device(dev):
        ws, n, keep = _workspace(lib.fmxq_head_logprobs_workspace, dev, M, V, K, k, top)
        logp = torch.empty(M, k, dtype=torch.float32, device=dev)
        entropy = torch.empty(M, dtype=torch.float32, device=dev)
        lse = torch.empty(M, dtype=torch.float32, device=dev)
        top_ids = torch.empty(M, top, dtype=torch.int32, device=dev)
        top_logp = torch.empty(M, top, dtype=torch.float32, device=dev)
        check(lib.fmxq_head_logprobs(*ptrs, logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
                                     top_ids.data_ptr(), top_logp.data_ptr(), M, V, K, k, top,
                                     temperature, group_size, bits, ws, n, _stream(h)))
    return (logp, entropy, lse, top_ids, top_logp) if top else (logp, entropy, lse)


def head_logprobs_grad(h, w, scales, biases, ids, logp, entropy, lse, grad_logp, grad_entropy=None,
                       temperature: float = 1.0, group_size: int = 64, bits: int = 4):
    """Gradient of h in head_logprobs: from those of logp [M, k] (k >= 1) and entropy [M] (None: no
    gradient), float32, and the logp, entropy and lse that head_logprobs returned for the same
    operands.  Returns dh [M, K] bf16; absent entries pass nothing back."""
    if _fast is not None:
        r = _fast.head_logprobs_grad(h, w, scales, biases, ids, logp, entropy, lse, grad_logp,
                                     grad_entropy, float(temperature), group_size, bits)
        if r is not None:
            return r
    more = {} if grad_entropy is None else {"grad_entropy": grad_entropy}
    dev = _same_device(h=h, w=w, scales=scales, biases=biases, ids=ids, logp=logp, entropy=entropy,
                       lse=lse, grad_logp=grad_logp, **more)
    M, V, K, k, ptrs = _score_operands(h, w, scales, biases, ids, group_size, bits)
    f32 = (torch.float32,)
    _shape("logp", logp, M, k)
    _shape("grad_logp", grad_logp, M, k)
    _shape("entropy", entropy, M)
    _shape("lse", lse, M)
    if grad_entropy is not None:
        _shape("grad_entropy", grad_entropy, M)
        _dev(grad_entropy, "grad_entropy", f32)
    ptrs += (_dev(logp, "logp", f32), _dev(entropy, "entropy", f32), _dev(lse, "lse", f32),
             _dev(grad_logp, "grad_logp", f32), _ptr(grad_entropy))
    lib = load()
    with torch.cuda.device(dev):
        ws, n, keep = _workspace(lib.fmxq_head_logprobs_grad_workspace, dev, M, V, K, k)
        dh = torch.empty(M, K, dtype=torch.bfloat16, device=dev)
        check(lib.fmxq_head_logprobs_grad(*ptrs, dh.data_ptr(), M, V, K, k, temperature, group_size,
                                          bits, ws, n, _stream(h)))
    return dh


def quantized_matmul_grad(dy, w, scales, biases, group_size: int = 64, bits: int = 4):
    """Gradient of x in quantized_matmul: dx = dy @ deq(W), dy [..., N] bf16, w [N, K*bits/32];
    dx [..., K] bf16."""
    if _fast is not None:
        r = _fast.qmm_grad(dy, w, scales, biases, None, group_size, bits)
        if r is not None:
            return r
    dev = _same_device(dy=dy, w=w, scales=scales, biases=biases)
    if w.dim() != 2 or dy.dim() < 1:
        raise ValueError("dy must be [..., N] and w [N, K*bits/32]")
    N, K = w.shape[0], w.shape[1] * 32 // bits if bits in (4, 8) else 0
    if dy.shape[-1] != N:
        raise ValueError(f"dy has {dy.shape[-1]} columns but w {N} rows")
    _quant_shapes(w, scales, biases, (N,), K, group_size, bits)
    M = 1
    for d in dy.shape[:-1]:
        M *= d
    args = (_dev(dy, "dy", _BF16_LIKE), _dev(w, "w", _U32_LIKE),
            _dev(scales, "scales", _BF16_LIKE), _dev(biases, "biases", _BF16_LIKE))
    lib = load()
    with torch.cuda.device(dev):
        dx = torch.empty(*dy.shape[:-1], K, dtype=torch.bfloat16, device=dev)
        ws, n, keep = _workspace(lib.fmxq_quantized_matmul_grad_workspace, dev, M, N, K,
                                 more=_moved(dy))
        check(lib.fmxq_quantized_matmul_grad(*args, dx.data_ptr(), M, N, K, group_size, bits, ws,
                                             n, _stream(dy)))
    return dx


def gather_qmm_grad(dy, w, scales, biases, offsets, group_size: int = 64, bits: int = 4):
    """Gradient of x in gather_qmm over rows sorted by expert (moe_sort): rows offsets[e] ..
    offsets[e + 1] of dx are dy @ deq(W[e]).  dy [S, N] bf16; w [E, N, K*bits/32]; offsets
    [E + 1] int32; dx [S, K] bf16, zero in rows of no expert."""
    if _fast is not None and offsets is not None:
        r = _fast.qmm_grad(dy, w, scales, biases, offsets, group_size, bits)
        if r is not None:
            return r
    dev = _same_device(dy=dy, w=w, scales=scales, biases=biases, offsets=offsets)
    if w.dim() != 3 or dy.dim() != 2:
        raise ValueError("dy must be [S, N] and w [E, N, K*bits/32]")
    E, N = w.shape[:2]
    K = w.shape[2] * 32 // bits if bits in (4, 8) else 0
    S = dy.shape[0]
    _shape("dy", dy, S, N)
    _shape("offsets", offsets, E + 1)
    _quant_shapes(w, scales, biases, (E, N), K, group_size, bits)
    args = (_dev(dy, "dy", _BF16_LIKE), _dev(w, "w", _U32_LIKE),
            _dev(scales, "scales", _BF16_LIKE), _dev(biases, "biases", _BF16_LIKE),
            _dev(offsets, "offsets", (torch.int32,)))
    lib = load()
    with torch.cuda.device(dev):
        dx = torch.empty(S, K, dtype=torch.bfloat16, device=dev)
        ws, n, keep = _workspace(lib.fmxq_gather_qmm_grad_workspace, dev, S, E, N, K,
                                 more=_moved(dy))
        check(lib.fmxq_gather_qmm_grad(*args, dx.data_ptr(), S, E, N, K, group_size, bits, ws, n,
                                       _stream(dy)))
    return dx


def moe_sort(x, inds, n_experts: int):
    """Token rows sorted by expert: x [T, D] bf16, inds [T, k] int32/uint32 ->
    (xs [T k, D], order [T k], pos [T, k], offsets [n_experts + 1]), the last three int32.

    Slot t k + j goes to row pos[t, j]; order is the stable argsort of the ids; expert e has
    rows offsets[e] .. offsets[e + 1].  Ids out of range sort last with zero rows, and
    device_error reports them."""
    if _fast is not None:
        r = _fast.moe_sort(x, inds, n_experts)
        if r is not None:
            return r
    dev = _same_device(x=x, inds=inds)
    if x.dim() != 2 or inds.dim() != 2:
        raise ValueError("x must be [T, D] and inds [T, k]")
    T, D = x.shape
    k = inds.shape[1]
    _shape("inds", inds, T, k)
    xp, ip = _dev(x, "x", _BF16_LIKE), _dev(inds, "inds", _U32_LIKE)
    lib = load()
    with torch.cuda.device(dev):
        ws, n, keep = _workspace(lib.fmxq_moe_sort_workspace, dev, T, k, n_experts)
        xs = torch.empty(T * k, D, dtype=torch.bfloat16, device=dev)
        order = torch.empty(T * k, dtype=torch.int32, device=dev)
        pos = torch.empty(T, k, dtype=torch.int32, device=dev)
        offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
        check(lib.fmxq_moe_sort(xp, ip, xs.data_ptr(), order.data_ptr(), pos.data_ptr(),
                                offsets.data_ptr(), T, k, n_experts, D, ws, n, _stream(x)))
    return xs, order, pos, offsets


def _sorted_rows(name, y, pos):
    if y.dim() != 2 or pos.dim() != 2:
        raise ValueError(f"{name} must be [T k, D] and pos [T, k]")
    T, k = pos.shape
    _shape(name, y, T * k, y.shape[1])
    return T, k, y.shape[1], _dev(y, name, _BF16_LIKE), _dev(pos, "pos", _U32_LIKE)


def _row_weights(weights, T, k):
    _shape("weights", weights, T, k)
    return (_dev(weights, "weights", (torch.bfloat16, torch.float32)),
            int(weights.dtype == torch.bfloat16))


def moe_sort_grad(dxs, pos):
    """Gradient of moe_sort's x: dxs [T k, D] bf16 -> dx [T, D] bf16, each token's slots summed
    in float32."""
    if _fast is not None:
        r = _fast.moe_unsort(dxs, pos, None)
        if r is not None:
            return r
    dev = _same_device(dxs=dxs, pos=pos)
    T, k, D, yp, pp = _sorted_rows("dxs", dxs, pos)
    with torch.cuda.device(dev):
        dx = torch.empty(T, D, dtype=torch.bfloat16, device=dev)
        check(load().fmxq_moe_sort_grad(yp, pp, dx.data_ptr(), T, k, D, _stream(dxs)))
    return dx


def moe_unsort(y, pos, weights):
    """Sorted rows back to tokens: out[t] = sum_j weights[t, j] y[pos[t, j]] in float32, rounded
    once.  y [T k, D] bf16; weights [T, k] bfloat16 or float32; out [T, D] bf16."""
    if _fast is not None and weights is not None:
        r = _fast.moe_unsort(y, pos, weights)
        if r is not None:
            return r
    dev = _same_device(y=y, pos=pos, weights=weights)
    T, k, D, yp, pp = _sorted_rows("y", y, pos)
    wp, wb = _row_weights(weights, T, k)
    with torch.cuda.device(dev):
        out = torch.empty(T, D, dtype=torch.bfloat16, device=dev)
        check(load().fmxq_moe_unsort(yp, pp, wp, wb, out.data_ptr(), T, k, D, _stream(y)))
    return out


def moe_unsort_grad(dout, y, pos, weights):
    """Gradients of moe_unsort: dout [T, D] bf16 -> (dy [T k, D] bf16, dweights [T, k] in the
    weights' type).  The positions are those of moe_sort, all different: rows of dy that none names
    (where one is out of range, which device_error reports) are not written."""
    if _fast is not None:
        r = _fast.moe_unsort_grad(dout, y, pos, weights)
        if r is not None:
            return r
    dev = _same_device(dout=dout, y=y, pos=pos, weights=weights)
    T, k, D, yp, pp = _sorted_rows("y", y, pos)
    _shape("dout", dout, T, D)
    dp = _dev(dout, "dout", _BF16_LIKE)
    wp, wb = _row_weights(weights, T, k)
    with torch.cuda.device(dev):
        dy = torch.empty(T * k, D, dtype=torch.bfloat16, device=dev)
        dw = torch.empty(T, k, dtype=weights.dtype, device=dev)
        check(load().fmxq_moe_unsort_grad(dp, yp, pp, wp, wb, dy.data_ptr(), dw.data_ptr(), T, k, D,
                                          _stream(dout)))
    return dy, dw


# ---- adapters beside quantized weights, and clipped gradients ---------------------


def _lora_operands(x, N, w, scales, biases, a, b, adapters, lora_scales, group_size, bits):
    if w.dim() != 2 or a.dim() != 3 or b.dim() != 3 or x.dim() < 1:
        raise ValueError("x must be [..., K], w [N, K*bits/32], a [E, r, K] and b [E, N, r]")
    K = x.shape[-1]
    E, r = a.shape[0], min(a.shape[1], 2**31 - 1)  # more than 128 are refused by the library
    _quant_shapes(w, scales, biases, (N,), K, group_size, bits)
    _shape("a", a, E, r, K)
    _shape("b", b, E, N, r)
    _shape("adapters", adapters, *x.shape[:-1])
    _shape("lora_scales", lora_scales, E)
    M = adapters.numel()
    ptrs = (_dev(x, "x", _BF16_LIKE), _dev(w, "w", _U32_LIKE), _dev(scales, "scales", _BF16_LIKE),
            _dev(biases, "biases", _BF16_LIKE), _dev(a, "a", _BF16_LIKE), _dev(b, "b", _BF16_LIKE),
            _dev(adapters, "adapters", (torch.int32,)),
            _dev(lora_scales, "lora_scales", (torch.float32,)))
    return M, K, E, r, ptrs


def quantized_matmul_lora(x, w, scales, biases, a, b, adapters, lora_scales, group_size: int = 64,
                          bits: int = 4):
    """quantized_matmul with a low-rank adapter for each row:
    y[m] = x[m] @ deq(W)^T + lora_scales[e] (x[m] @ A[e]^T) @ B[e]^T with e = adapters[m].

    x [..., K] bf16; w [N, K*bits/32]; a [E, r, K] and b [E, N, r] bf16, r a multiple of 8 up to
    128 (zeros fill smaller ranks); adapters [...] int32, below zero for a row without one;
    lora_scales [E] float32.  Returns y [..., N] bf16, summed in float32 and rounded once.  An adapter
    past the last counts as none, and device_error reports it.  y is not finite exactly where the
    formula is not, but an infinite operand may give NaN in place of an infinity."""
    if _fast is not None:
        r = _fast.qmm_lora(x, w, scales, biases, a, b, adapters, lora_scales, group_size, bits)
        if r is not None:
            return r
    dev = _same_device(x=x, w=w, scales=scales, biases=biases, a=a, b=b, adapters=adapters,
                       lora_scales=lora_scales)
    N = w.shape[0] if w.dim() else 0
    M, K, E, r, ptrs = _lora_operands(x, N, w, scales, biases, a, b, adapters, lora_scales,
                                      group_size, bits)
    lib = load()
    with torch.cuda.device(dev):
        y = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=dev)
        ws, n, keep = _workspace(lib.fmxq_quantized_matmul_lora_workspace, dev, M, N, K, E, r)
        check(lib.fmxq_quantized_matmul_lora(*ptrs, y.data_ptr(), M, N, K, E, r, group_size, bits, ws,
                                             n, _stream(x)))
    return y


def quantized_matmul_lora_grad(dy, x, w, scales, biases, a, b, adapters, lora_scales,
                               group_size: int = 64, bits: int = 4):
    """Gradients of quantized_matmul_lora, W frozen: dy [..., N] bf16 and its operands ->
    (dx [..., K] bf16, da [E, r, K] float32, db [E, N, r] float32), the adapters' sums over their
    rows and zeros for one without."""
    if _fast is not None:
        r = _fast.qmm_lora_grad(dy, x, w, scales, biases, a, b, adapters, lora_scales, group_size,
                                bits)
        if r is not None:
            return r
    dev = _same_device(dy=dy, x=x, w=w, scales=scales, biases=biases, a=a, b=b, adapters=adapters,
                       lora_scales=lora_scales)
    N = w.shape[0] if w.dim() else 0
    M, K, E, r, ptrs = _lora_operands(x, N, w, scales, biases, a, b, adapters, lora_scales,
                                      group_size, bits)
    _shape("dy", dy, *x.shape[:-1], N)
    dyp = _dev(dy, "dy", _BF16_LIKE)
    lib = load()
    with torch.cuda.device(dev):
        dx = torch.empty(*x.shape, dtype=torch.bfloat16, device=dev)
        da = torch.empty(E, r, K, dtype=torch.float32, device=dev)
        db = torch.empty(E, N, r, dtype=torch.float32, device=dev)
        ws, n, keep = _workspace(lib.fmxq_quantized_matmul_lora_grad_workspace, dev, M, N, K, E, r,
                                 more=_moved(dy) if N else 0)
        check(lib.fmxq_quantized_matmul_lora_grad(dyp, *ptrs, dx.data_ptr(), da.data_ptr(),
                                                  db.data_ptr(), M, N, K, E, r, group_size, bits, ws,
                                                  n, _stream(dy)))
    return dx, da, db


def _clip_call(grads, outs, max_norm):
    """grad_norm (outs None) or clip_grad_norm of lists of tensors."""
    import ctypes

    types = (torch.float32, torch.bfloat16)
    if not grads:
        raise ValueError("no gradients")
    dev = _same_device(**{f"grads[{i}]": g for i, g in enumerate(grads)})
    ptrs = [_dev(g, f"grads[{i}]", types) for i, g in enumerate(grads)]
    n = len(grads)
    if outs is not None:
        if len(outs) != n:
            raise ValueError(f"{len(outs)} results for {n} gradients")
        _same_device(**{"grads[0]": grads[0]}, **{f"outs[{i}]": o for i, o in enumerate(outs)})
        for i, (g, o) in enumerate(zip(grads, outs)):
            _shape(f"outs[{i}]", o, *g.shape)
            _dev(o, f"outs[{i}]", (g.dtype,))
    P = ctypes.c_void_p * n
    counts = (ctypes.c_int64 * n)(*[g.numel() for g in grads])
    bf16 = (ctypes.c_int * n)(*[int(g.dtype is torch.bfloat16) for g in grads])
    lib = load()
    with torch.cuda.device(dev):
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ws, size, keep = _workspace(lib.fmxq_grad_norm_workspace, dev)
        if outs is None:
            check(lib.fmxq_grad_norm(P(*ptrs), counts, bf16, n, norm.data_ptr(), ws, size,
                                     _stream(grads[0])))
        else:
            check(lib.fmxq_clip_grad_norm(P(*ptrs), P(*[o.data_ptr() for o in outs]), counts, bf16, n,
                                          max_norm, norm.data_ptr(), ws, size, _stream(grads[0])))
    return norm


def grad_norm(grads):
    """The norm over many gradients: the root of the sum of all their squares, summed in 64 bits.
    grads: float32 or bfloat16 tensors of one device.  Returns a float32 scalar tensor, without
    waiting for it."""
    if _fast is not None:
        r = _fast.clip(grads, None, 0.0)
        if r is not None:
            return r
    return _clip_call(list(grads), None, 0.0)


def clip_grad_norm(grads, max_norm: float, outs=None):
    """Gradients scaled by min(1, max_norm / norm), norm as grad_norm has it -> (outs, norm).

    outs: the results' tensors, of the gradients' shapes and types (new ones without); they may
    be the gradients themselves.  Values stay as they are where the norm is zero, or where an infinity
    or NaN among them makes it one, so a step can be skipped by the norm alone.  (Finite gradients whose
    norm is past float32's range are scaled by its 64-bit value; the norm returned is infinite.)"""
    many = (list, tuple)  # others (a generator, for one) are walked once
    if not isinstance(grads, many):
        grads = list(grads)
    if outs is None:
        outs = [torch.empty_like(g) for g in grads]
    elif not isinstance(outs, many):
        outs = list(outs)
    if _fast is not None:
        r = _fast.clip(grads, outs, float(max_norm))
        if r is not None:
            return outs, r
    return outs, _clip_call(list(grads), list(outs), float(max_norm))


def device_error(device=None) -> None:
    """Raise FmxqError(FMXQ_ERR_INDEX) if a gather met an out-of-range index."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    check(load().fmxq_device_error(torch.cuda.current_stream(dev).cuda_stream))
