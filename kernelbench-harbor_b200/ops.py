"""torch custom ops over the C ABI (include/b200q.h).

Each op validates its tensors the way the reference operator would see them
(shapes of QUANT_REF.forward, generate_tasks.py:54-61), makes them contiguous
(as the reference Triton oracle does, common/oracles/quant_w4a16_pa.py:74-77),
allocates the output (callee-allocated, like the oracle's torch.empty at :79)
and calls the library on the current CUDA stream.  No CPU path exists: a CPU
tensor is an error."""
from __future__ import annotations

import functools
import threading
from typing import Optional, Union

import torch
from torch.autograd import forward_ad

from . import _lib

_ws_lock = threading.Lock()
_ws: dict = {}
_ws_captured: dict = {}  # workspaces made inside a graph capture: the capture that zeroed them last
_ws_outgrown: list = []  # captured graphs may use them still


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Zero-initialised scratch owned by this process, one per (device, stream).
    Kernels return it to the zero state, so it is allocated (and zeroed) once
    and reused; it is never shared by two streams, whose launches could overlap.

    Inside a graph capture the zeroing becomes a node of that graph: a workspace
    made there is zeroed in every graph that is captured with it (they may be
    replayed in any order), and calls outside a capture take another."""
    key = (_index(device), _stream_ptr(device))
    with _ws_lock:
        buf = _ws.get(key)
        if buf is not None and buf.numel() >= nbytes and key not in _ws_captured:
            return buf
        capture = _lib.lib().b200q_capture_id(key[1])
        if buf is None or buf.numel() < nbytes or not capture:
            if buf is not None:
                _ws_outgrown.append(buf)
            buf = torch.zeros(max(nbytes, 4096), dtype=torch.uint8, device=device)
            _ws[key] = buf
        elif _ws_captured[key] != capture:
            buf.zero_()
        if capture:
            _ws_captured[key] = capture
        else:
            _ws_captured.pop(key, None)
        return buf


def reset_workspaces() -> None:
    """Drops all workspaces; graphs captured before must not be replayed again."""
    with _ws_lock:
        _ws.clear()
        _ws_captured.clear()
        _ws_outgrown.clear()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _dtype_code(dt: torch.dtype) -> int:
    if dt == torch.float16:
        return _lib.DTYPE_FP16
    if dt == torch.bfloat16:
        return _lib.DTYPE_BF16
    raise TypeError(f"activations must be float16 or bfloat16, got {dt}")


def _index(device: torch.device) -> int:
    return torch.cuda.current_device() if device.index is None else device.index


def _stream_ptr(device: torch.device) -> int:
    # torch.cuda.current_stream(device).cuda_stream without the Stream object (0.1 us instead of 2.2)
    return torch._C._cuda_getCurrentRawStream(_index(device))


class _NoSwitch:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_no_switch = _NoSwitch()


def _device(device: torch.device):
    """Context in which ``device`` is the current one (kernels launch on the current device)."""
    # a CUDA tensor exists, so what torch.cuda.current_device() first looks up is there
    return _no_switch if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _no_tangent(op: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses dual tensors (forward-mode differentiation, _current_level >= 0), whose tangents the kernels do not see."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{op} has no forward-mode derivative")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    pa, pb = a.data_ptr(), b.data_ptr()
    return pa < pb + b.numel() * b.element_size() and pb < pa + a.numel() * a.element_size()


def _same_device(op: str, first: torch.Tensor, *rest: Optional[torch.Tensor]) -> None:
    d = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != d:
            raise ValueError(f"{op}: tensors on {first.device} and {t.device}")


@torch.library.custom_op("b200q::w4a16_gemm", mutates_args=())
def w4a16_gemm(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor,
               group: int) -> torch.Tensor:
    """y[M, N] = x[M, K] . ((unpack(qweight) - zeros) * scales), y in x.dtype."""
    if forward_ad._current_level >= 0:
        _no_tangent("w4a16_gemm", x)
    if not x.is_cuda:
        raise RuntimeError("b200q::w4a16_gemm runs on CUDA tensors only (no CPU implementation)")
    if x.dim() != 2 or qweight.dim() != 2:
        raise ValueError("x must be [M, K] and qweight [K, N/8]")
    if qweight.dtype != torch.int32:
        raise TypeError("qweight must be int32")
    M, K = x.shape
    if qweight.shape[0] != K:
        raise ValueError(f"qweight has {qweight.shape[0]} rows, x has K={K}")
    N = qweight.shape[1] * 8
    if group <= 0 or K % group:
        raise ValueError(f"K={K} is not a multiple of group={group}")
    for name, t in (("scales", scales), ("zeros", zeros)):
        if tuple(t.shape) != (K // group, N):
            raise ValueError(f"{name} must be [{K // group}, {N}], got {tuple(t.shape)}")
    dt = _dtype_code(x.dtype)
    scales = scales.to(x.dtype)
    zeros = zeros.to(x.dtype)
    x, qweight, scales, zeros = (_aligned(t) for t in (x, qweight, scales, zeros))
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    if M == 0:
        return y
    L = _lib.lib()
    nbytes = L.b200q_w4a16_workspace_bytes(M, N, K, group, x.device.index)
    with _device(x.device):
        ws = workspace(x.device, nbytes)
        _lib.check(L.b200q_w4a16_gemm(x.data_ptr(), qweight.data_ptr(), scales.data_ptr(), zeros.data_ptr(),
                                      y.data_ptr(), M, N, K, group, dt, ws.data_ptr(), ws.numel(),
                                      _stream_ptr(x.device)))
    return y


@w4a16_gemm.register_fake
def _(x, qweight, scales, zeros, group):
    return x.new_empty((x.shape[0], qweight.shape[1] * 8))


_is_compiling, _dispatch_modes = torch.compiler.is_compiling, torch._C._len_torch_dispatch_stack
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _dispatched(t: torch.Tensor) -> bool:
    """Whether a call on t has to go through PyTorch's dispatcher as a registered
    operator: while a program is traced (torch.compile, export, fake tensors),
    under a dispatch mode, or for a tensor subclass.  Other calls take the
    library directly (a registered operator costs 10 us more on the host)."""
    return _is_compiling() or type(t) not in _PLAIN or _dispatch_modes() > 0


def w4a16_dgrad(dy: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor,
                group: int) -> torch.Tensor:
    """dx[M, K] = dy[M, N] . ((unpack(qweight) - zeros) * scales)^T, dx in dy.dtype:
    the input gradient of w4a16_gemm (the weights are frozen).  Differentiable
    in dy, w4a16_gemm being its gradient in turn."""
    if forward_ad._current_level >= 0:
        _no_tangent("w4a16_dgrad", dy)
    if (torch.is_grad_enabled() and (dy.requires_grad or scales.requires_grad or zeros.requires_grad)) or _dispatched(dy):
        return w4a16_dgrad_op(dy, qweight, scales, zeros, group)
    return _w4a16_dgrad(dy, qweight, scales, zeros, group)


def _w4a16_dgrad(dy, qweight, scales, zeros, group):
    if not dy.is_cuda:
        raise RuntimeError("b200q w4a16_dgrad runs on CUDA tensors only (no CPU implementation)")
    if dy.dim() != 2 or qweight.dim() != 2:
        raise ValueError("dy must be [M, N] and qweight [K, N/8]")
    if qweight.dtype != torch.int32:
        raise TypeError("qweight must be int32")
    M, N = dy.shape
    K = qweight.shape[0]
    if qweight.shape[1] * 8 != N:
        raise ValueError(f"qweight has {qweight.shape[1] * 8} columns, dy has N={N}")
    if group <= 0 or K % group:
        raise ValueError(f"K={K} is not a multiple of group={group}")
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t.shape != (K // group, N):
            raise ValueError(f"{name} must be [{K // group}, {N}], got {tuple(t.shape)}")
    dt = _dtype_code(dy.dtype)
    _same_device("w4a16_dgrad", dy, qweight, scales, zeros)
    if scales.dtype != dy.dtype:
        scales = scales.to(dy.dtype)
    if zeros.dtype != dy.dtype:
        zeros = zeros.to(dy.dtype)
    dy, qweight, scales, zeros = _aligned(dy), _aligned(qweight), _aligned(scales), _aligned(zeros)
    dx = dy.new_empty((M, K))
    if M == 0:
        return dx
    with _device(dy.device):
        ws = workspace(dy.device, 256)
        _lib.check(_lib.lib().b200q_w4a16_dgrad(dy.data_ptr(), qweight.data_ptr(), scales.data_ptr(),
                                                zeros.data_ptr(), dx.data_ptr(), M, N, K, group, dt, ws.data_ptr(),
                                                ws.numel(), _stream_ptr(dy.device)))
    return dx


@torch.library.custom_op("b200q::w4a16_dgrad", mutates_args=())
def w4a16_dgrad_op(dy: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor,
                   group: int) -> torch.Tensor:
    """w4a16_dgrad as a registered operator."""
    return _w4a16_dgrad(dy, qweight, scales, zeros, group)


@w4a16_dgrad_op.register_fake
def _(dy, qweight, scales, zeros, group):
    return dy.new_empty((dy.shape[0], qweight.shape[0]))


def _w4a16_setup(ctx, inputs, output):
    _, qweight, scales, zeros, group = inputs
    ctx.save_for_backward(qweight, scales, zeros)
    ctx.group = group


def _frozen(ctx, op):
    if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
        raise RuntimeError(f"{op}: the quantised weight is frozen, scales and zeros have no gradient")


# The two are linear, and each other's gradient: gradients of any order.
def _w4a16_backward(ctx, dy):
    _frozen(ctx, "w4a16_gemm")
    qweight, scales, zeros = ctx.saved_tensors
    dx = w4a16_dgrad(dy, qweight, scales, zeros, ctx.group) if ctx.needs_input_grad[0] else None
    return dx, None, None, None, None


def _w4a16_dgrad_backward(ctx, ddx):
    _frozen(ctx, "w4a16_dgrad")
    qweight, scales, zeros = ctx.saved_tensors
    ddy = w4a16_gemm(ddx, qweight, scales, zeros, ctx.group) if ctx.needs_input_grad[0] else None
    return ddy, None, None, None, None


w4a16_dgrad_op.register_autograd(_w4a16_dgrad_backward, setup_context=_w4a16_setup)
w4a16_gemm.register_autograd(_w4a16_backward, setup_context=_w4a16_setup)


def _ptr_array(ptrs) -> "ctypes.Array":
    import ctypes
    return (ctypes.c_void_p * len(ptrs))(*[int(p) for p in ptrs])


def w4a16_gemm_peers(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor,
                     group: int, y_ptrs, ldy: int, col0: int, pad_ptrs=None, rank: int = 0) -> None:
    """Columns [col0, col0 + N) of y = x . W from this rank's shard, stored
    into every buffer of ``y_ptrs`` (device addresses of [M, ldy] arrays in
    x.dtype, peers' included).  With ``pad_ptrs`` (every rank's signal pad)
    the kernel orders itself against the peers; without, the caller does
    (``peer_barrier`` before and after)."""
    if not x.is_cuda:
        raise RuntimeError("w4a16_gemm_peers runs on CUDA tensors only (no CPU implementation)")
    M, K = x.shape
    N = qweight.shape[1] * 8
    if qweight.dtype != torch.int32 or qweight.shape[0] != K:
        raise ValueError("qweight must be int32 [K, N/8]")
    dt = _dtype_code(x.dtype)
    scales = scales.to(x.dtype)
    zeros = zeros.to(x.dtype)
    x, qweight, scales, zeros = (_aligned(t) for t in (x, qweight, scales, zeros))
    if M == 0:
        return
    L = _lib.lib()
    ws = workspace(x.device, L.b200q_w4a16_workspace_bytes(M, N, K, group, x.device.index))
    arr = _ptr_array(y_ptrs)
    pads = _ptr_array(pad_ptrs) if pad_ptrs is not None else None
    _lib.check(L.b200q_w4a16_gemm_peers(x.data_ptr(), qweight.data_ptr(), scales.data_ptr(), zeros.data_ptr(),
                                        arr, len(y_ptrs), ldy, col0, pads, rank, M, N, K, group, dt,
                                        ws.data_ptr(), ws.numel(), _stream_ptr(x.device)))


def peer_barrier(pad_ptrs, rank: int, device: torch.device) -> None:
    """Barrier of the len(pad_ptrs) ranks on the current stream (signal pads
    of 64 zeroed uint32 words, every rank's mapped into this process)."""
    L = _lib.lib()
    ws = workspace(device, 256)
    _lib.check(L.b200q_peer_barrier(_ptr_array(pad_ptrs), len(pad_ptrs), rank, ws.data_ptr(),
                                    _stream_ptr(device)))


@torch.library.custom_op("b200q::w8a8_gemm", mutates_args=())
def w8a8_gemm(x_int8: torch.Tensor, w_int8: torch.Tensor, x_scale: torch.Tensor,
              w_scale: torch.Tensor) -> torch.Tensor:
    """y[M, N] = fp16((x_int8 . w_int8) * x_scale * w_scale) (W8A8_REF.forward,
    generate_tasks.py:204-206); x_scale [M, 1] or [M], w_scale [1, N] or [N]."""
    if not x_int8.is_cuda:
        raise RuntimeError("b200q::w8a8_gemm runs on CUDA tensors only (no CPU implementation)")
    if x_int8.dtype != torch.int8 or w_int8.dtype != torch.int8:
        raise TypeError("x_int8 and w_int8 must be int8")
    M, K = x_int8.shape
    if w_int8.shape[0] != K:
        raise ValueError(f"w_int8 has {w_int8.shape[0]} rows, x has K={K}")
    N = w_int8.shape[1]
    xs = x_scale.reshape(-1).to(torch.float16)
    wsc = w_scale.reshape(-1).to(torch.float16)
    if xs.numel() != M or wsc.numel() != N:
        raise ValueError("x_scale must have M entries and w_scale N entries")
    x_int8, w_int8, xs, wsc = (_aligned(t) for t in (x_int8, w_int8, xs, wsc))
    y = torch.empty((M, N), dtype=torch.float16, device=x_int8.device)
    if M == 0:
        return y
    L = _lib.lib()
    ws = workspace(x_int8.device, L.b200q_w8a8_workspace_bytes(M, N, K, x_int8.device.index))
    _lib.check(L.b200q_w8a8_gemm(x_int8.data_ptr(), w_int8.data_ptr(), xs.data_ptr(), wsc.data_ptr(),
                                 y.data_ptr(), M, N, K, ws.data_ptr(), ws.numel(), _stream_ptr(x_int8.device)))
    return y


@w8a8_gemm.register_fake
def _(x_int8, w_int8, x_scale, w_scale):
    return x_int8.new_empty((x_int8.shape[0], w_int8.shape[1]), dtype=torch.float16)


@torch.library.custom_op("b200q::mxfp8_gemm", mutates_args=())
def mxfp8_gemm(a: torch.Tensor, scales_a: torch.Tensor, b: torch.Tensor, scales_b: torch.Tensor) -> torch.Tensor:
    """y[M, N] = fp16(A_deq . B_deq^T) for OCP-MX e4m3 operands (codes as uint8 or
    float8_e4m3fn [M, K] / [N, K], E8M0 scales uint8 [M, K/32] / [N, K/32])."""
    if not a.is_cuda:
        raise RuntimeError("b200q mxfp8_gemm runs on CUDA tensors only")
    a, b = (t.view(torch.uint8) if t.dtype != torch.uint8 else t for t in (a, b))
    M, K = a.shape
    N = b.shape[0]
    if b.shape[1] != K or scales_a.shape != (M, K // 32) or scales_b.shape != (N, K // 32):
        raise ValueError("mxfp8_gemm: shapes must be A [M,K], B [N,K], scales [*, K/32]")
    a, b, scales_a, scales_b = (_aligned(t) for t in (a, b, scales_a, scales_b))
    y = torch.empty((M, N), dtype=torch.float16, device=a.device)
    if M == 0:
        return y
    L = _lib.lib()
    ws = workspace(a.device, L.b200q_mxfp8_workspace_bytes(M, N, K, a.device.index))
    _lib.check(L.b200q_mxfp8_gemm(a.data_ptr(), scales_a.data_ptr(), b.data_ptr(), scales_b.data_ptr(),
                                  y.data_ptr(), M, N, K, ws.data_ptr(), ws.numel(), _stream_ptr(a.device)))
    return y


@mxfp8_gemm.register_fake
def _(a, scales_a, b, scales_b):
    return a.new_empty((a.shape[0], b.shape[0]), dtype=torch.float16)


def mxfp8_gemm_peers(a: torch.Tensor, scales_a: torch.Tensor, b: torch.Tensor, scales_b: torch.Tensor,
                     y_ptrs, ldy: int, col0: int, pad_ptrs=None, rank: int = 0) -> None:
    """Columns [col0, col0 + N) of y = A . B^T from this rank's B shard [N, K],
    stored into every buffer of ``y_ptrs`` ([M, ldy] fp16, peers' included),
    ordered against the peers through ``pad_ptrs`` as in w4a16_gemm_peers."""
    if not a.is_cuda:
        raise RuntimeError("mxfp8_gemm_peers runs on CUDA tensors only (no CPU implementation)")
    a, b = (t.view(torch.uint8) if t.dtype != torch.uint8 else t for t in (a, b))
    M, K = a.shape
    N = b.shape[0]
    if b.shape[1] != K or scales_a.shape != (M, K // 32) or scales_b.shape != (N, K // 32):
        raise ValueError("mxfp8_gemm_peers: shapes must be A [M,K], B [N,K], scales [*, K/32]")
    a, b, scales_a, scales_b = (_aligned(t) for t in (a, b, scales_a, scales_b))
    if M == 0:
        return
    L = _lib.lib()
    ws = workspace(a.device, L.b200q_mxfp8_workspace_bytes(M, N, K, a.device.index))
    pads = _ptr_array(pad_ptrs) if pad_ptrs is not None else None
    _lib.check(L.b200q_mxfp8_gemm_peers(a.data_ptr(), scales_a.data_ptr(), b.data_ptr(), scales_b.data_ptr(),
                                        _ptr_array(y_ptrs), len(y_ptrs), ldy, col0, pads, rank, M, N, K,
                                        ws.data_ptr(), ws.numel(), _stream_ptr(a.device)))


@torch.library.custom_op("b200q::moe_route", mutates_args=())
def moe_route(router_logits: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                                     torch.Tensor]:
    """Top-2 routing + expert-grouped permutation (see include/b200q.h).
    Returns topi [T,2] int32, gates [T,2] (logits dtype), offsets [E+1] int32,
    slot_token [2T] int32, token_slot [T,2] int32."""
    if not router_logits.is_cuda:
        raise RuntimeError("b200q moe_route runs on CUDA tensors only")
    lg = _aligned(router_logits)
    T, E = lg.shape
    dev = lg.device
    topi = torch.empty((T, 2), dtype=torch.int32, device=dev)
    gates = torch.empty((T, 2), dtype=lg.dtype, device=dev)
    offsets = torch.empty((E + 1,), dtype=torch.int32, device=dev)
    slot_token = torch.empty((2 * T,), dtype=torch.int32, device=dev)
    token_slot = torch.empty((T, 2), dtype=torch.int32, device=dev)
    _lib.check(_lib.lib().b200q_moe_route(lg.data_ptr(), T, E, _dtype_code(lg.dtype), topi.data_ptr(),
                                          gates.data_ptr(), offsets.data_ptr(), slot_token.data_ptr(),
                                          token_slot.data_ptr(), _stream_ptr(dev)))
    return topi, gates, offsets, slot_token, token_slot


@moe_route.register_fake
def _(router_logits):
    T, E = router_logits.shape
    i32 = dict(dtype=torch.int32)
    return (router_logits.new_empty((T, 2), **i32), router_logits.new_empty((T, 2)),
            router_logits.new_empty((E + 1,), **i32), router_logits.new_empty((2 * T,), **i32),
            router_logits.new_empty((T, 2), **i32))


_LOGITS_CODES = {torch.float16: _lib.DTYPE_FP16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_FP32}


@functools.lru_cache(maxsize=256)
def _balance_scratch(T: int, E: int) -> int:
    return _lib.lib().b200q_moe_balance_scratch_bytes(T, E)


def _balance_forward(logits, topi, mask):
    T, E = logits.shape
    dev = logits.device
    L = _lib.lib()
    nbytes = _balance_scratch(T, E)
    loss = logits.new_empty((), dtype=torch.float32)
    # 32-bit words like topi's, so that there is no type to look up; the kernel's scratch behind coef
    coef, counts = topi.new_empty(E + nbytes // 4), topi.new_empty(E)
    with _device(dev):
        ws = workspace(dev, 256)
        p = coef.data_ptr()
        _lib.check(L.b200q_moe_balance(logits.data_ptr(), topi.data_ptr(), _ptr(mask), T, E, topi.shape[1],
                                       _LOGITS_CODES[logits.dtype], loss.data_ptr(), counts.data_ptr(), p, p + 4 * E,
                                       nbytes, ws.data_ptr(), _stream_ptr(dev)))
    return loss, counts, coef


def _balance_grad(lg, mask, coef, dloss):
    T, E = lg.shape
    d = torch.empty_like(lg)
    with _device(lg.device):
        _lib.check(_lib.lib().b200q_moe_balance_grad(lg.data_ptr(), _ptr(mask), coef.data_ptr(), dloss.data_ptr(), T, E,
                                                     _LOGITS_CODES[lg.dtype], d.data_ptr(), _stream_ptr(lg.device)))
    return d


@torch.library.custom_op("b200q::moe_balance_grad", mutates_args=())
def moe_balance_grad_op(logits: torch.Tensor, mask: Optional[torch.Tensor], coef: torch.Tensor,
                        dloss: torch.Tensor) -> torch.Tensor:
    """moe_balance_loss's gradient of contiguous logits; coef (32-bit words, the
    first E used) from its forward pass, dloss fp32 [].  It has no derivative
    of its own: differentiating its output raises."""
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in _LOGITS_CODES:
        raise TypeError("moe_balance_grad: router_logits must be [T, E] float16, bfloat16 or float32 on a GPU")
    if coef.dtype not in (torch.int32, torch.float32) or coef.numel() < logits.shape[1] or not coef.is_contiguous():
        raise ValueError("moe_balance_grad: coef must hold E contiguous 32-bit words")
    if dloss.dtype != torch.float32 or dloss.numel() != 1:
        raise ValueError("moe_balance_grad: dloss must be one float32")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != logits.shape[:1] or not mask.is_contiguous()):
        raise ValueError("moe_balance_grad: mask must be contiguous bool [T]")
    _same_device("moe_balance_grad", logits, mask, coef, dloss)
    return _balance_grad(logits.contiguous(), mask, coef, dloss)


@moe_balance_grad_op.register_fake
def _(logits, mask, coef, dloss):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topi, mask):
        loss, counts, coef = _balance_forward(logits, topi, mask)
        ctx.save_for_backward(logits, mask, coef)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)  # no zeros for counts
        return loss, counts

    @staticmethod
    def backward(ctx, dloss, _):
        if dloss is None:
            return None, None, None
        # under create_graph as an operator that refuses to be differentiated again
        grad = moe_balance_grad_op if torch.is_grad_enabled() else _balance_grad
        return grad(*ctx.saved_tensors, dloss), None, None


@torch.library.custom_op("b200q::moe_balance", mutates_args=())
def moe_balance_op(logits: torch.Tensor, topi: torch.Tensor,
                   mask: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """moe_balance_loss as a registered operator: topi int32; (loss, counts, coef [E], which the gradient takes)."""
    if not logits.is_cuda or logits.dim() != 2 or topi.dim() != 2 or topi.shape[0] != logits.shape[0]:
        raise ValueError("moe_balance: router_logits [T, E] and topi [T, k] on a GPU expected")
    if logits.dtype not in _LOGITS_CODES or topi.dtype != torch.int32:
        raise TypeError("moe_balance: router_logits must be float16, bfloat16 or float32, topi int32")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != logits.shape[:1]):
        raise ValueError("moe_balance: mask must be bool [T]")
    _same_device("moe_balance", logits, topi, mask)
    loss, counts, coef = _balance_forward(logits.contiguous(), topi.contiguous(), None if mask is None else mask.contiguous())
    return loss, counts, coef[:logits.shape[1]].clone()  # without the kernel's scratch


@moe_balance_op.register_fake
def _(logits, topi, mask):
    E = logits.shape[1]
    return logits.new_empty((), dtype=torch.float32), topi.new_empty(E), topi.new_empty(E)


def _balance_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[0], inputs[2], output[2])


def _balance_op_backward(ctx, dloss, *_):
    lg, mask, coef = ctx.saved_tensors
    return moe_balance_grad_op(lg, mask, coef, dloss), None, None


moe_balance_op.register_autograd(_balance_op_backward, setup_context=_balance_setup)


def moe_balance_loss(router_logits: torch.Tensor, topi: torch.Tensor,
                     token_mask: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Load-balance loss of a top-k router and the per-expert token counts.

    router_logits [T, E] fp16 / bf16 / fp32, topi [T, k] integer (moe_route's
    first output for k = 2; -1 is a dropped choice), token_mask [T] bool (False:
    padding, counts nowhere).  loss = E sum_e f_e P_e, fp32 scalar, with f_e the
    share of the live choices that went to expert e and P_e the mean softmax
    probability of e; counts [E] int32.  The loss is differentiable in
    router_logits (f is a count and carries no gradient); see include/b200q.h
    for rows that are all -inf and for indices out of range."""
    if forward_ad._current_level >= 0:
        _no_tangent("moe_balance_loss", router_logits)
    if not router_logits.is_cuda:
        raise RuntimeError("b200q moe_balance_loss runs on CUDA tensors only")
    if router_logits.dim() != 2 or topi.dim() != 2 or topi.shape[0] != router_logits.shape[0]:
        raise ValueError("router_logits must be [T, E] and topi [T, k]")
    if router_logits.dtype not in _LOGITS_CODES:
        raise TypeError(f"router_logits must be float16, bfloat16 or float32, got {router_logits.dtype}")
    if topi.dtype not in (torch.int32, torch.int64):
        raise TypeError("topi must be int32 or int64")
    _same_device("moe_balance_loss", router_logits, topi, token_mask)
    if token_mask is not None:
        if token_mask.dtype != torch.bool or tuple(token_mask.shape) != (router_logits.shape[0],):
            raise ValueError("token_mask must be bool [T]")
        token_mask = token_mask.contiguous()
    if topi.dtype == torch.int64:  # what 32 bits do not hold stays out of range
        topi = topi.clamp(-2, router_logits.shape[1]).to(torch.int32)
    topi = topi.contiguous()
    logits = router_logits.contiguous()
    if _dispatched(logits):
        return moe_balance_op(logits, topi, token_mask)[:2]
    if torch.is_grad_enabled() and logits.requires_grad:
        return _BalanceLoss.apply(logits, topi, token_mask)
    return _balance_forward(logits, topi, token_mask)[:2]


def moe_grouped_gemm(x: torch.Tensor, offsets: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,
                     zeros: torch.Tensor, group: int, up=None) -> torch.Tensor:
    """See moe_grouped_gemm_op; ``up`` = (qweight_up, scales_up, zeros_up) or None."""
    u = up if up is not None else (None, None, None)
    return moe_grouped_gemm_op(x, offsets, qweight, scales, zeros, group, u[0], u[1], u[2])


@torch.library.custom_op("b200q::moe_grouped_gemm", mutates_args=())
def moe_grouped_gemm_op(x: torch.Tensor, offsets: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,
                        zeros: torch.Tensor, group: int, qweight_up: Optional[torch.Tensor] = None,
                        scales_up: Optional[torch.Tensor] = None,
                        zeros_up: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One launch over all experts.  x [rows, K] grouped by expert (rows of
    expert e at [offsets[e], offsets[e+1]), offsets on the device); qweight
    [E, K, N/8], scales / zeros [E, K/group, N].  Returns y [rows, N] =
    x . W_e, or with ``up = (qweight_up, scales_up, zeros_up)`` the fused
    SiLU(x . Wg_e) * (x . Wu_e)."""
    up = None if qweight_up is None else (qweight_up, scales_up, zeros_up)
    if not x.is_cuda:
        raise RuntimeError("b200q moe_grouped_gemm runs on CUDA tensors only")
    rows, K = x.shape
    E = qweight.shape[0]
    if qweight.dim() != 3 or qweight.shape[1] != K or qweight.dtype != torch.int32:
        raise ValueError("qweight must be int32 [E, K, N/8]")
    N = qweight.shape[2] * 8
    if offsets.dtype != torch.int32 or offsets.numel() != E + 1:
        raise ValueError("offsets must be int32 [E + 1]")
    dt = _dtype_code(x.dtype)
    ts = [_aligned(t) for t in (x, qweight, scales.to(x.dtype), zeros.to(x.dtype), offsets)]
    if up is not None:
        ts += [_aligned(up[0]), _aligned(up[1].to(x.dtype)), _aligned(up[2].to(x.dtype))]
        if tuple(ts[5].shape) != tuple(qweight.shape):
            raise ValueError("up-projection qweight must match the gate's shape")
    y = torch.empty((rows, N), dtype=x.dtype, device=x.device)
    if rows == 0:
        return y
    ws = workspace(x.device, 256)
    ptr = lambda i: ts[i].data_ptr() if i < len(ts) else None  # noqa: E731
    _lib.check(_lib.lib().b200q_moe_grouped_gemm(ptr(0), ptr(1), ptr(2), ptr(3), ptr(5), ptr(6), ptr(7), ptr(4), E,
                                                 y.data_ptr(), rows, N, K, group, dt, ws.data_ptr(), ws.numel(),
                                                 _stream_ptr(x.device)))
    return y


@moe_grouped_gemm_op.register_fake
def _(x, offsets, qweight, scales, zeros, group, qweight_up=None, scales_up=None, zeros_up=None):
    return x.new_empty((x.shape[0], qweight.shape[2] * 8))


def ep_pack(x: torch.Tensor, offsets: torch.Tensor, slot_token: torch.Tensor, token_slot: torch.Tensor,
            n_experts: int, world: int, capacity: int):
    """Send buffer [world * capacity, D + 8] of an expert-parallel exchange
    (see include/b200q.h) and pair_slot [T, 2] int32."""
    T, D = x.shape
    x = _aligned(x)
    send = torch.empty((world * capacity, D + 8), dtype=x.dtype, device=x.device)
    pair_slot = torch.empty((T, 2), dtype=torch.int32, device=x.device)
    _lib.check(_lib.lib().b200q_ep_pack(x.data_ptr(), T, D, _dtype_code(x.dtype), offsets.data_ptr(),
                                        slot_token.data_ptr(), token_slot.data_ptr(), n_experts, world, capacity,
                                        send.data_ptr(), pair_slot.data_ptr(), _stream_ptr(x.device)))
    return send, pair_slot


def ep_regroup(recv: torch.Tensor, n_local: int):
    """(loc_offsets [n_local + 1], src [R], row_pos [R]) int32 for received rows [R, D + 8]."""
    R, D8 = recv.shape
    dev = recv.device
    loc = torch.empty(n_local + 1, dtype=torch.int32, device=dev)
    src = torch.empty(R, dtype=torch.int32, device=dev)
    pos = torch.empty(R, dtype=torch.int32, device=dev)
    _lib.check(_lib.lib().b200q_ep_regroup(recv.data_ptr(), R, D8 - 8, _dtype_code(recv.dtype), n_local,
                                           loc.data_ptr(), src.data_ptr(), pos.data_ptr(), _stream_ptr(dev)))
    return loc, src, pos


def ep_gather(src: torch.Tensor, idx: torch.Tensor, D: int, out: torch.Tensor) -> torch.Tensor:
    """out[j, :D] = src[idx[j], :D] where idx[j] >= 0 (2-D row-pitched tensors)."""
    _lib.check(_lib.lib().b200q_ep_gather(src.data_ptr(), src.stride(0), idx.data_ptr(), idx.numel(), D,
                                          out.data_ptr(), out.stride(0), _stream_ptr(src.device)))
    return out


def pack_int4(codes: torch.Tensor, offset: int = 0) -> torch.Tensor:
    """4-bit codes [..., N] (int8 / uint8, one per byte) -> int32 [..., N/8]
    packed along N (nibble i of word j = column 8j + i).  offset 0: unsigned
    codes in [0, 15]; offset 8: signed int4 in [-8, 7] stored as q + 8 (use
    zero point 8).  Codes out of range set the device status bit."""
    if not codes.is_cuda:
        raise RuntimeError("b200q pack_int4 runs on CUDA tensors only")
    if codes.dtype not in (torch.int8, torch.uint8):
        raise TypeError("codes must be int8 or uint8")
    N = codes.shape[-1]
    c = _aligned(codes).reshape(-1, N)
    out = torch.empty(codes.shape[:-1] + (N // 8,), dtype=torch.int32, device=codes.device)
    ws = workspace(codes.device, 256)
    _lib.check(_lib.lib().b200q_pack_int4(c.data_ptr(), c.shape[0], N, offset, out.data_ptr(), ws.data_ptr(),
                                          _stream_ptr(codes.device)))
    return out


def silu_mul_fp8(y: torch.Tensor, codes: bool = False):
    """FUSED_SILU_REF: y [T, 2H] -> SiLU(gate) * up quantised per 128 columns
    to e4m3 and dequantised, fp32 [T, H].  With ``codes`` also returns the
    e4m3 codes (torch.float8_e4m3fn [T, H]) and scales (fp32 [T, H/128])."""
    if not y.is_cuda:
        raise RuntimeError("b200q silu_mul_fp8 runs on CUDA tensors only")
    T, H2 = y.shape
    H = H2 // 2
    y = _aligned(y)
    out = torch.empty((T, H), dtype=torch.float32, device=y.device)
    q = torch.empty((T, H), dtype=torch.uint8, device=y.device) if codes else None
    sc = torch.empty((T, H // 128), dtype=torch.float32, device=y.device) if codes else None
    _lib.check(_lib.lib().b200q_silu_mul_fp8(y.data_ptr(), T, H, _dtype_code(y.dtype), out.data_ptr(),
                                             q.data_ptr() if codes else None, sc.data_ptr() if codes else None,
                                             _stream_ptr(y.device)))
    if codes:
        return out, q.view(torch.float8_e4m3fn), sc
    return out


def lora_shrink(x: torch.Tensor, A: torch.Tensor, lora_ids: torch.Tensor) -> torch.Tensor:
    """lo [T, r] = x[t] . A[lora_ids[t]] per token (A [L, D, r]), x's dtype."""
    T, D = x.shape
    L, _, r = A.shape
    ids = lora_ids.to(torch.int64).contiguous()
    x, A = _aligned(x), _aligned(A.to(x.dtype))
    lo = torch.empty((T, r), dtype=x.dtype, device=x.device)
    ws = workspace(x.device, 256)
    _lib.check(_lib.lib().b200q_lora_shrink(x.data_ptr(), A.data_ptr(), ids.data_ptr(), T, D, r, L,
                                            _dtype_code(x.dtype), lo.data_ptr(), ws.data_ptr(),
                                            _stream_ptr(x.device)))
    return lo


def _written(out: torch.Tensor) -> None:
    """Tells autograd that a kernel has written over out: what saved it refuses its new contents."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


class _Overwritten(torch.autograd.Function):
    """A tensor with a gradient history that an operator without a gradient has written over."""

    @staticmethod
    def forward(ctx, op, t):
        ctx.op = op
        ctx.mark_dirty(t)
        return t

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.op} has no gradient (lora_apply and lora_w4a16 have)")


def lora_expand_add(base: torch.Tensor, lo: torch.Tensor, B: torch.Tensor, lora_ids: torch.Tensor,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, N] = base + round(lo[t] . B[lora_ids[t]]) (B [L, r, N])."""
    T, N = base.shape
    L, r, _ = B.shape
    ids = lora_ids.to(torch.int64).contiguous()
    base, lo, B = _aligned(base), _aligned(lo), _aligned(B.to(base.dtype))
    y = out if out is not None else torch.empty_like(base)
    _lib.check(_lib.lib().b200q_lora_expand_add(base.data_ptr(), lo.data_ptr(), B.data_ptr(), ids.data_ptr(), T, r,
                                                N, L, _dtype_code(base.dtype), y.data_ptr(),
                                                _stream_ptr(base.device)))
    if out is not None:
        if out.requires_grad and torch.is_grad_enabled():  # its history ends here
            return _Overwritten.apply("lora_expand_add", out)
        _written(out)
    return y


def _one_launch(T: int, r: int) -> bool:
    """Whether b200q_lora_apply runs as one launch: it needs no room for the row between, and has no wait that could run out."""
    return T <= (256 if r <= 32 else 128)


class LoraPlan:
    """A batch's tokens grouped by adapter: made once by lora_plan, used by
    every projection that the batch passes through."""

    __slots__ = ("data", "tokens", "adapters", "device")

    def __init__(self, data: torch.Tensor, tokens: int, adapters: int):
        self.data, self.tokens, self.adapters, self.device = data, tokens, adapters, data.device


def lora_plan(lora_ids: torch.Tensor, n_adapters: int) -> LoraPlan:
    """Groups the tokens of lora_ids [T] (integer; -1 = no adapter) for
    lora_apply over ``n_adapters`` adapters.  Any other id outside
    [0, n_adapters) counts as none and sets the device status bit.  The ids
    are read on the device: no host synchronisation."""
    if not lora_ids.is_cuda:
        raise RuntimeError("b200q lora_plan runs on CUDA tensors only")
    if lora_ids.dim() != 1 or lora_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("lora_ids must be int32 or int64 [T]")
    ids = lora_ids.to(torch.int64).contiguous()
    data = (lora_plan_op if _dispatched(ids) else _lora_plan)(ids, n_adapters)
    return LoraPlan(data, ids.shape[0], n_adapters)


def _lora_plan(ids, n_adapters):
    T, dev = ids.numel(), ids.device
    L = _lib.lib()
    nbytes = L.b200q_lora_plan_bytes(T, n_adapters)
    data = torch.empty((max(nbytes, 4) // 4,), dtype=torch.int32, device=dev)
    with _device(dev):
        ws = workspace(dev, 256)
        _lib.check(L.b200q_lora_plan(ids.data_ptr(), T, n_adapters, data.data_ptr(), nbytes, ws.data_ptr(),
                                     _stream_ptr(dev)))
    return data


@torch.library.custom_op("b200q::lora_plan", mutates_args=())
def lora_plan_op(lora_ids: torch.Tensor, n_adapters: int) -> torch.Tensor:
    """lora_plan's words as a registered operator: lora_ids int64 [T]."""
    if not lora_ids.is_cuda or lora_ids.dim() != 1 or lora_ids.dtype != torch.int64:
        raise ValueError("lora_plan: lora_ids int64 [T] on a GPU expected")
    return _lora_plan(lora_ids.contiguous(), n_adapters)


def _plan_words(T, n_adapters):
    """b200q_lora_plan_bytes / 4 (the layout is in lora_seg.cuh); T may be symbolic."""
    up4 = lambda v: (v + 3) // 4 * 4  # noqa: E731
    tiles = lambda rows: torch.sym_min(T // rows + n_adapters + 1, T)  # noqa: E731
    return up4(up4(8 + n_adapters + 2) + T) + 4 * (tiles(16) + tiles(128))


@lora_plan_op.register_fake
def _(lora_ids, n_adapters):
    return lora_ids.new_empty(_plan_words(lora_ids.shape[0], n_adapters), dtype=torch.int32)


def _lora_run(x, base, A, B, scaling, plan, out, lo):
    """One b200q_lora_apply call on contiguous, aligned tensors; returns the
    sizes as the library takes them."""
    n_adapters, D, r = A.shape
    T = x.shape[0]
    dev = x.device
    sizes = (T, D, B.shape[2], r, n_adapters, _dtype_code(x.dtype))
    with _device(dev):
        status = None if _one_launch(T, r) else workspace(dev, 256).data_ptr()
        _lib.check(_lib.lib().b200q_lora_apply(x.data_ptr(), base.data_ptr(), A.data_ptr(), B.data_ptr(), _ptr(scaling),
                                               plan.data_ptr(), *sizes, out.data_ptr(), _ptr(lo), status,
                                               _stream_ptr(dev)))
    return sizes


@functools.lru_cache(maxsize=256)
def _lora_mid_values(T: int, r: int) -> int:
    return _lib.lib().b200q_lora_mid_bytes(T, r) // 4


def _lora_mid(plan: LoraPlan, r: int) -> torch.Tensor:
    # 32-bit words beside the plan's: new_empty without a type or device to look up takes 1.5 us less than torch.empty
    return plan.data.new_empty(_lora_mid_values(plan.tokens, r))


@functools.lru_cache(maxsize=256)
def _lora_scratch(T: int, D: int, N: int, r: int, n_adapters: int, dtype: int, device: int) -> int:
    # the split of the token sums depends on the device (the current one)
    return _lib.lib().b200q_lora_backward_scratch_bytes(T, D, N, r, n_adapters, dtype)


def _lora_grads(sizes, x, d, base, A, B, scaling, plan, lo, dx, want_A, want_B):
    """dA and dB; and dx (if given) = base (None: 0) + the adapters' part."""
    dA = torch.empty_like(A) if want_A else None
    dB = torch.empty_like(B) if want_B else None
    dev = x.device
    with _device(dev):
        nbytes = _lora_scratch(*sizes, dev.index)
        scratch = plan.new_empty(nbytes // 4)  # fp32 sums
        status = None if _one_launch(sizes[0], sizes[3]) else workspace(dev, 256).data_ptr()
        _lib.check(_lib.lib().b200q_lora_backward(
            x.data_ptr(), d.data_ptr(), _ptr(base), A.data_ptr(), B.data_ptr(), _ptr(scaling), plan.data_ptr(),
            lo.data_ptr(), *sizes, scratch.data_ptr(), nbytes, _ptr(dx), _ptr(dA), _ptr(dB), status, _stream_ptr(dev)))
    return dA, dB


@torch.library.custom_op("b200q::lora_backward", mutates_args=())
def lora_backward_op(x: torch.Tensor, dy: torch.Tensor, base: Optional[torch.Tensor], A: torch.Tensor, B: torch.Tensor,
                     scaling: Optional[torch.Tensor], plan: torch.Tensor, lo: torch.Tensor, want_x: bool, want_A: bool,
                     want_B: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """lora_apply's gradients (dx = base + its part, dA, dB), empty where one is not
    wanted; plan and lo from the forward pass.  They have no derivative of
    their own: differentiating them raises."""
    sizes = _lora_operands("lora_backward", x, A, B, scaling, plan, dy=dy, base=base, lo=lo)
    x, dy, A, B = _aligned(x), _aligned(dy), _aligned(A), _aligned(B)
    dx = torch.empty_like(x) if want_x else x.new_empty(0)
    dA, dB = _lora_grads(sizes, x, dy, None if base is None else _aligned(base), A, B, scaling, plan, lo,
                         dx if want_x else None, want_A, want_B)
    return dx, dA if want_A else A.new_empty(0), dB if want_B else B.new_empty(0)


@lora_backward_op.register_fake
def _(x, dy, base, A, B, scaling, plan, lo, want_x, want_A, want_B):
    return tuple(t.new_empty(t.shape) if want else t.new_empty(0) for t, want in ((x, want_x), (A, want_A), (B, want_B)))


def _lora_operands(op, x, A, B, scaling, plan, *, dy=None, base=None, lo=None):
    """Checks what a registered operator is given; returns the sizes as the library takes them."""
    if not x.is_cuda or x.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise ValueError(f"{op}: x [T, D], A [L, D, r] and B [L, r, N] on a GPU expected")
    (T, D), (n_adapters, _, r), N = x.shape, A.shape, B.shape[2]
    code = _dtype_code(x.dtype)
    for t, shape in ((A, (n_adapters, D, r)), (B, (n_adapters, r, N)), (dy, (T, N)), (base, (T, D) if dy is not None else (T, N))):
        if t is not None and (tuple(t.shape) != shape or t.dtype != x.dtype):
            raise ValueError(f"{op}: {list(shape)} of {x.dtype} expected, got {tuple(t.shape)} of {t.dtype}")
    if plan.dtype != torch.int32 or not plan.is_contiguous() or plan.data_ptr() % 16 or \
            4 * plan.numel() < max(1, _lib.lib().b200q_lora_plan_bytes(T, n_adapters)):
        raise ValueError(f"{op}: not a plan of {T} tokens and {n_adapters} adapters")
    if lo is not None and (lo.dtype not in (torch.int32, torch.float32) or not lo.is_contiguous() or
                           4 * lo.numel() < _lib.lib().b200q_lora_mid_bytes(T, r)):
        raise ValueError(f"{op}: lo is not the forward pass's")
    if scaling is not None and (scaling.dtype != torch.float32 or tuple(scaling.shape) != (n_adapters,) or
                                not scaling.is_contiguous()):
        raise ValueError(f"{op}: scaling must be contiguous float32 [{n_adapters}]")
    _same_device(op, x, A, B, scaling, plan, dy, base, lo)
    return T, D, N, r, n_adapters, code


def _lora_backward(sizes, x, d, base, A, B, scaling, plan, lo, dx, want_x, want_A, want_B):
    """(dx, dA, dB) for a backward pass; dx: where to put it (base itself), or None.
    sizes: None in a registered operator's formula."""
    if torch.is_grad_enabled():
        # create_graph: operators that refuse to be differentiated again, one for each
        # gradient, so that each refuses exactly where it depends on something that
        # asks for a gradient of its own
        rest = (scaling, plan, lo)
        return (lora_backward_op(x.detach(), d, base, A, B, *rest, True, False, False)[0] if want_x else None,
                lora_backward_op(x, d, None, A.detach(), B, *rest, False, True, False)[1] if want_A else None,
                lora_backward_op(x, d, None, A, B.detach(), *rest, False, False, True)[2] if want_B else None)
    if sizes is None:
        out = lora_backward_op(x, d, base, A, B, scaling, plan, lo, want_x, want_A, want_B)
        return tuple(g if want else None for g, want in zip(out, (want_x, want_A, want_B)))
    if dx is None and want_x:
        dx = torch.empty_like(x)
    if not (want_x or want_A or want_B):
        return None, None, None
    return (dx, *_lora_grads(sizes, x, d, base, A, B, scaling, plan, lo, dx, want_A, want_B))


def _saveable(plan: LoraPlan) -> LoraPlan:
    """The plan, copied where autograd could not save it (made in inference mode)."""
    return LoraPlan(plan.data.clone(), plan.tokens, plan.adapters) if plan.data.is_inference() else plan


class _LoraApply(torch.autograd.Function):
    @staticmethod
    def forward(ctx, base, x, A, B, scaling, plan):
        y, lo = torch.empty_like(base), _lora_mid(plan, A.shape[2])
        ctx.sizes = _lora_run(x, base, A, B, scaling, plan.data, y, lo)
        ctx.save_for_backward(x, A, B, scaling, plan.data, lo)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, A, B, scaling, plan, lo = ctx.saved_tensors
        want_base, *want = ctx.needs_input_grad[:4]
        grads = _lora_backward(ctx.sizes, x, _aligned(dy), None, A, B, scaling, plan, lo, None, *want)
        return (dy if want_base else None, *grads, None, None)


class _LoRAW4A16(torch.autograd.Function):
    """w4a16_gemm with lora_apply in place on its output; one gradient of x for both."""

    @staticmethod
    def forward(ctx, x, A, B, qweight, scales, zeros, group, scaling, plan):
        y, lo = w4a16_gemm(x, qweight, scales, zeros, group), _lora_mid(plan, A.shape[2])
        ctx.sizes = _lora_run(x, y, A, B, scaling, plan.data, y, lo)
        ctx.save_for_backward(x, A, B, scaling, qweight, scales, zeros, plan.data, lo)
        ctx.group = group
        return y

    @staticmethod
    def backward(ctx, dy):
        x, A, B, scaling, qweight, scales, zeros, plan, lo = ctx.saved_tensors
        *want, _, need_scales, need_zeros = ctx.needs_input_grad[:6]
        if need_scales or need_zeros:
            raise RuntimeError("lora_w4a16: the quantised weight is frozen, scales and zeros have no gradient")
        d = _aligned(dy)
        dx = w4a16_dgrad(d, qweight, scales, zeros, ctx.group) if want[0] else None
        grads = _lora_backward(ctx.sizes, x, d, dx, A, B, scaling, plan, lo, dx, *want)
        return (*grads, None, None, None, None, None, None)


@torch.library.custom_op("b200q::lora_apply", mutates_args=())
def lora_apply_op(base: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, scaling: Optional[torch.Tensor],
                  plan: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """lora_apply as a registered operator, on a plan's words: (y, lo), lo as b200q_lora_apply leaves it."""
    sizes = _lora_operands("lora_apply", x, A, B, scaling, plan, base=base)
    base, x, A, B = _aligned(base), _aligned(x), _aligned(A), _aligned(B)
    y, lo = torch.empty_like(base), plan.new_empty(_lora_mid_values(sizes[0], sizes[3]))
    _lora_run(x, base, A, B, scaling, plan, y, lo)
    return y, lo


@torch.library.custom_op("b200q::lora_w4a16", mutates_args=())
def lora_w4a16_op(x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,
                  zeros: torch.Tensor, group: int, scaling: Optional[torch.Tensor],
                  plan: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """lora_w4a16 as a registered operator, on a plan's words: (y, lo)."""
    sizes = _lora_operands("lora_w4a16", x, A, B, scaling, plan)
    if qweight.dim() != 2 or qweight.shape[1] * 8 != B.shape[2]:
        raise ValueError(f"lora_w4a16: qweight {tuple(qweight.shape)} does not fit B {tuple(B.shape)}")
    x, A, B = _aligned(x), _aligned(A), _aligned(B)
    y, lo = w4a16_gemm(x, qweight, scales, zeros, group), plan.new_empty(_lora_mid_values(sizes[0], sizes[3]))
    _lora_run(x, y, A, B, scaling, plan, y, lo)
    return y, lo


def _lo_words(x, A, plan):
    r = A.shape[2]
    return plan.new_empty(x.shape[0] * (16 if r <= 16 else 32 if r <= 32 else 64))  # b200q_lora_mid_bytes / 4


@lora_apply_op.register_fake
def _(base, x, A, B, scaling, plan):
    return base.new_empty(base.shape), _lo_words(x, A, plan)


@lora_w4a16_op.register_fake
def _(x, A, B, qweight, scales, zeros, group, scaling, plan):
    return x.new_empty((x.shape[0], B.shape[2])), _lo_words(x, A, plan)


def _lora_apply_setup(ctx, inputs, output):
    _, x, A, B, scaling, plan = inputs
    ctx.save_for_backward(x, A, B, scaling, plan, output[1])


def _lora_apply_backward(ctx, dy, _):
    x, A, B, scaling, plan, lo = ctx.saved_tensors
    want_base, *want = ctx.needs_input_grad[:4]
    grads = _lora_backward(None, x, dy, None, A, B, scaling, plan, lo, None, *want)
    return (dy if want_base else None, *grads, None, None)


def _lora_w4a16_setup(ctx, inputs, output):
    x, A, B, qweight, scales, zeros, ctx.group, scaling, plan = inputs
    ctx.save_for_backward(x, A, B, qweight, scales, zeros, scaling, plan, output[1])


def _lora_w4a16_backward(ctx, dy, _):
    x, A, B, qweight, scales, zeros, scaling, plan, lo = ctx.saved_tensors
    *want, _, need_scales, need_zeros = ctx.needs_input_grad[:6]
    if need_scales or need_zeros:
        raise RuntimeError("lora_w4a16: the quantised weight is frozen, scales and zeros have no gradient")
    dx = w4a16_dgrad(dy, qweight, scales, zeros, ctx.group) if want[0] else None
    grads = _lora_backward(None, x, dy, dx, A, B, scaling, plan, lo, dx, *want)
    return (*grads, None, None, None, None, None, None)


lora_apply_op.register_autograd(_lora_apply_backward, setup_context=_lora_apply_setup)
lora_w4a16_op.register_autograd(_lora_w4a16_backward, setup_context=_lora_w4a16_setup)


def _lora_check(op, x, A, B, plan, scaling):
    """Checks the adapter operands that lora_apply and lora_w4a16 share; returns
    A and B in x's dtype, the plan and scaling as fp32."""
    if forward_ad._current_level >= 0:
        _no_tangent(op, x, A, B)
    if not x.is_cuda:
        raise RuntimeError(f"b200q {op} runs on CUDA tensors only")
    if x.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise ValueError(f"{op}: x [T, D], A [L, D, r] and B [L, r, N] expected")
    T, D = x.shape
    n_adapters, Da, r = A.shape
    Lb, rb, _ = B.shape
    if Da != D or Lb != n_adapters or rb != r:
        raise ValueError(f"{op}: shapes do not fit: x {tuple(x.shape)}, A {tuple(A.shape)}, B {tuple(B.shape)}")
    dt = x.dtype
    _dtype_code(dt)
    if isinstance(plan, torch.Tensor):
        plan = lora_plan(plan, n_adapters)
    if plan.tokens != T or plan.adapters != n_adapters:
        raise ValueError(f"{op}: the plan is for {plan.tokens} tokens and {plan.adapters} adapters, "
                         f"not {T} and {n_adapters}")
    _same_device(op, x, A, B, plan.data, scaling)
    if scaling is not None:
        if scaling.shape != (n_adapters,):
            raise ValueError(f"{op}: scaling must be [{n_adapters}]")
        if scaling.requires_grad:
            raise ValueError(f"{op}: scaling is a constant and has no gradient")
        if scaling.dtype != torch.float32 or not scaling.is_contiguous():
            scaling = scaling.to(torch.float32).contiguous()
    if A.dtype != dt:
        A = A.to(dt)
    if B.dtype != dt:
        B = B.to(dt)
    return A, B, plan, scaling


def lora_apply(base: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
               plan: Union[LoraPlan, torch.Tensor], scaling: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = base[t] + scaling[id_t] * (x[t] . A[id_t]) . B[id_t]: the adapters
    of many requests beside one shared projection's output ``base``.

    base [T, N] and x [T, D] fp16 / bf16, A [L, D, r], B [L, r, N] (r <= 64),
    plan: lora_plan's result, or the ids [T] themselves (-1 = no adapter: y =
    base), scaling [L] or None (1).  The row between the two products stays in
    fp32; y is rounded once.  Differentiable in base, x, A and B (scaling is a
    constant).  ``out`` (which may be ``base``: in place) takes the result
    where no gradient is wanted."""
    if forward_ad._current_level >= 0:
        _no_tangent("lora_apply", base)
    A, B, plan, scaling = _lora_check("lora_apply", x, A, B, plan, scaling)
    T, dt = x.shape[0], x.dtype
    if base.shape != (T, B.shape[2]):
        raise ValueError(f"lora_apply: base must be [{T}, {B.shape[2]}], got {tuple(base.shape)}")
    if base.dtype != dt:
        raise TypeError(f"lora_apply: base is {base.dtype}, x is {dt}")
    _same_device("lora_apply", x, base, out)
    wanted = torch.is_grad_enabled() and (x.requires_grad or A.requires_grad or B.requires_grad or base.requires_grad or
                                          (out is not None and out.requires_grad))
    if wanted and out is not None:
        raise ValueError("lora_apply: out cannot be given where a gradient is wanted")
    if _dispatched(x):
        y = lora_apply_op(base, x, A, B, scaling, plan.data)[0]
        if out is None:
            return y
        if out.shape != base.shape or out.dtype != dt:
            raise ValueError("lora_apply: out must be a [T, N] tensor of x's dtype")
        return out.copy_(y)
    if wanted:
        return _LoraApply.apply(_aligned(base), _aligned(x), _aligned(A), _aligned(B), scaling, _saveable(plan))
    out_given = out is not None
    if not out_given:
        base = _aligned(base)
        out = torch.empty_like(base)
    else:
        if out.shape != base.shape or out.dtype != dt or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("lora_apply: out must be a contiguous, 16-byte aligned [T, N] tensor of x's dtype")
        if out is not base:
            base = _aligned(base)
    x, A, B = _aligned(x), _aligned(A), _aligned(B)
    if out_given and (any(t is not None and _overlap(out, t) for t in (x, A, B, scaling, plan.data)) or
                      (out.data_ptr() != base.data_ptr() and _overlap(out, base))):
        raise ValueError("lora_apply: out shares memory with an input (it may be base itself)")
    r = A.shape[2]
    lo = None if _one_launch(T, r) else _lora_mid(plan, r)
    _lora_run(x, base, A, B, scaling, plan.data, out, lo)
    if out_given:
        _written(out)
    return out


def lora_w4a16(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor, group: int,
               A: torch.Tensor, B: torch.Tensor, plan: Union[LoraPlan, torch.Tensor],
               scaling: Optional[torch.Tensor] = None) -> torch.Tensor:
    """w4a16_gemm(x, qweight, scales, zeros, group) with lora_apply's adapters
    beside it, in place on the projection's output.  Differentiable in x, A and
    B: x's gradient is w4a16_dgrad's with the adapters' part added to it in
    place.  Both results are rounded twice: as the projection's (the input
    gradient's) output, and with the adapters' part."""
    A, B, plan, scaling = _lora_check("lora_w4a16", x, A, B, plan, scaling)
    if qweight.dim() != 2 or qweight.shape[1] * 8 != B.shape[2]:
        raise ValueError(f"lora_w4a16: qweight {tuple(qweight.shape)} does not fit B {tuple(B.shape)}")
    _same_device("lora_w4a16", x, qweight, scales, zeros)
    if _dispatched(x):
        return lora_w4a16_op(x, A, B, qweight, scales, zeros, group, scaling, plan.data)[0]
    if torch.is_grad_enabled() and (x.requires_grad or A.requires_grad or B.requires_grad):
        return _LoRAW4A16.apply(_aligned(x), _aligned(A), _aligned(B), qweight, scales, zeros, group, scaling,
                                _saveable(plan))
    y = w4a16_gemm(x, qweight, scales, zeros, group)
    x = _aligned(x)
    r = A.shape[2]
    lo = None if _one_launch(x.shape[0], r) else _lora_mid(plan, r)
    with torch.no_grad():
        _lora_run(x, y, _aligned(A), _aligned(B), scaling, plan.data, y, lo)
    return y


def moe_gather(x: torch.Tensor, slot_token: torch.Tensor) -> torch.Tensor:
    x = _aligned(x)
    xg = torch.empty((slot_token.numel(), x.shape[1]), dtype=x.dtype, device=x.device)
    _lib.check(_lib.lib().b200q_moe_gather(x.data_ptr(), slot_token.data_ptr(), slot_token.numel(), x.shape[1],
                                           xg.data_ptr(), _stream_ptr(x.device)))
    return xg


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    gate, up = gate.contiguous(), up.contiguous()
    h = torch.empty_like(gate)
    _lib.check(_lib.lib().b200q_silu_mul(gate.data_ptr(), up.data_ptr(), h.data_ptr(), gate.numel(),
                                         _dtype_code(gate.dtype), _stream_ptr(gate.device)))
    return h


def moe_combine(ye: torch.Tensor, token_slot: torch.Tensor, gates: torch.Tensor) -> torch.Tensor:
    ye = ye.contiguous()
    T = token_slot.shape[0]
    y = torch.empty((T, ye.shape[1]), dtype=ye.dtype, device=ye.device)
    _lib.check(_lib.lib().b200q_moe_combine(ye.data_ptr(), token_slot.data_ptr(), gates.contiguous().data_ptr(),
                                            y.data_ptr(), T, ye.shape[1], _dtype_code(ye.dtype),
                                            _stream_ptr(ye.device)))
    return y


def set_weight_prefetch(enable: bool) -> bool:
    """Lets small-M W4A16 calls stream their weights while the previous kernel
    in the stream is still running (programmatic dependent launch).  Only valid
    when the kernel just before each call does not write that call's weights,
    scales or zeros.  Process-wide; returns the previous setting."""
    return bool(_lib.lib().b200q_set_weight_prefetch(1 if enable else 0))


def device_status(device: torch.device | None = None) -> int:
    """Reads and clears the device error word of this stream's workspace
    (synchronises the stream).  0 means no kernel reported an error."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    ws = workspace(device, 4096)
    r = _lib.lib().b200q_workspace_status(ws.data_ptr(), _stream_ptr(device))
    if r < 0:
        _lib.check(r)
    if r > 0:
        ws.zero_()  # a kernel that gave up may have left split-K counters behind
    return r
