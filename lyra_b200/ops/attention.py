"""Python face of the sm_100a attention kernels (``csrc/attn``). Tensors are token-major ``[B, T, N, D]``;
heads-first views (``x.transpose(1, 2)``) of such tensors are accepted without a copy."""

from __future__ import annotations

import functools

import torch

from lyra_b200.nn.quant import QArray
from lyra_b200.ops import native
from lyra_b200.ops.native import c_float, c_int, c_ll, ptr


def _btnd(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """``x`` is heads-first ``[B, N, T, D]`` (any strides with unit inner stride). Returns (tensor, (sb, st, sn))."""
    if x.stride(-1) != 1 or x.data_ptr() % 16 or any(s % 8 for s in x.stride()[:-1]):
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    return x, (x.stride(0), x.stride(2), x.stride(1))


def flash_fwd(q, k, v, sinks, scale: float, window: int, q_start: int = 0):
    """``q [B, Nq, T, D]``, ``k, v [B, Nkv, S, D]`` bf16 -> ``(out [B, Nq, T, D] (token-major storage), lse [B, Nq, T] fp32)``."""
    B, Nq, T, D = q.shape
    Nkv, S = k.shape[1], k.shape[2]
    q, qs = _btnd(q)
    k, ks = _btnd(k)
    v, vs = _btnd(v)
    out = torch.empty(B, T, Nq, D, dtype=torch.bfloat16, device=q.device)
    lse = torch.empty(B, Nq, T, dtype=torch.float32, device=q.device)
    fn = native.kernels().lyra_flash_fwd
    fn.restype = c_int
    rc = fn(ptr(q), c_ll(qs[0]), c_ll(qs[1]), c_ll(qs[2]), ptr(k), c_ll(ks[0]), c_ll(ks[1]), c_ll(ks[2]),
            ptr(v), c_ll(vs[0]), c_ll(vs[1]), c_ll(vs[2]), ptr(sinks.float().contiguous()), ptr(out), ptr(lse),
            c_int(B), c_int(T), c_int(S), c_int(Nq), c_int(Nkv), c_int(D), c_float(scale), c_int(window), c_int(int(q_start)),
            ptr(native.status_word()), native.stream_ptr())
    native.check(rc, "lyra_flash_fwd")
    native.count_launch()
    return out.transpose(1, 2), lse


def _strides3(x: torch.Tensor):
    import ctypes

    return (ctypes.c_longlong * 3)(x.stride(0), x.stride(2), x.stride(1))


def flash_bwd(q, k, v, out, d_out, lse, sinks, scale: float, window: int, q_start: int = 0):
    """Gradients of :func:`flash_fwd`. All tensors heads-first views; ``out`` must be the forward's output.
    Returns ``(dq, dk, dv, dsinks)`` (heads-first views of token-major storage, dsinks fp32 ``[Nq]``)."""
    B, Nq, T, D = q.shape
    Nkv, S = k.shape[1], k.shape[2]
    q, _ = _btnd(q)
    k, _ = _btnd(k)
    v, _ = _btnd(v)
    d_out, _ = _btnd(d_out)
    out_t = out.transpose(1, 2)
    if not out_t.is_contiguous():
        out_t = out_t.contiguous()
    dq = torch.empty(B, T, Nq, D, dtype=torch.bfloat16, device=q.device)
    dk = torch.empty(B, S, Nkv, D, dtype=torch.bfloat16, device=q.device)
    dv = torch.empty(B, S, Nkv, D, dtype=torch.bfloat16, device=q.device)
    delta = torch.empty(B, Nq, T, dtype=torch.float32, device=q.device)
    fn = native.kernels().lyra_flash_bwd
    fn.restype = c_int
    rc = fn(ptr(q), _strides3(q), ptr(k), _strides3(k), ptr(v), _strides3(v), ptr(out_t), ptr(d_out), _strides3(d_out),
            ptr(lse), ptr(delta), ptr(dq), ptr(dk), ptr(dv),
            c_int(B), c_int(T), c_int(S), c_int(Nq), c_int(Nkv), c_int(D), c_float(scale), c_int(window), c_int(int(q_start)),
            ptr(native.status_word()), native.stream_ptr())
    native.check(rc, "lyra_flash_bwd")
    native.count_launch(3)
    # dsink_h = -sum_{b,t} exp(sink_h - lse) * delta  (lyra/kernels/flash_attention.py:653-659)
    dsinks = -(torch.exp(sinks.float()[None, :, None] - lse) * delta).sum(dim=(0, 2))
    return dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2), dsinks


class FlashAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sinks, scale, window, q_start):
        out, lse = flash_fwd(q, k, v, sinks, scale, window, q_start)
        ctx.save_for_backward(q, k, v, out, lse, sinks)
        ctx.args = (scale, window, q_start)
        return out

    @staticmethod
    def backward(ctx, d_out):
        q, k, v, out, lse, sinks = ctx.saved_tensors
        scale, window, q_start = ctx.args
        dq, dk, dv, dsinks = flash_bwd(q, k, v, out, d_out, lse, sinks, scale, window, q_start)
        return dq, dk, dv, dsinks.to(sinks.dtype), None, None, None


def flash_attention(q, k, v, sinks, scale: float, window: int, q_start: int = 0):
    return FlashAttention.apply(q, k, v, sinks, scale, window, q_start)


# --------------------------------------------------------------------------- shared prefix (csrc/attn/prefix_attn.cu)
def check_prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, sinks, scale: float, window: int, pos) -> None:
    """Refuses arguments that do not describe a batch with a shared prefix."""
    if q.ndim != 4 or not q.is_floating_point():
        raise ValueError(f"q must be a floating-point [B, Nq, T, D], got {tuple(q.shape)} {q.dtype}")
    B, Nq, T, D = q.shape
    device, tensors = q.device, [q]
    for name, keys, values, axes in (("prefix", prefix_k, prefix_v, 3), ("own cache", k_cache, v_cache, 4)):
        quantised = isinstance(keys, QArray)
        if quantised != isinstance(values, QArray):
            raise ValueError(f"{name}: keys and values must both be quantised or both not")
        shape = keys.shape
        if len(shape) != axes or values.shape != shape or shape[-1] != D or shape[-3] < 1 or Nq % shape[-3] or (axes == 4 and shape[0] != B):
            raise ValueError(f"{name}: keys {tuple(shape)} and values {tuple(values.shape)} must be {['B', 'Nkv', 'positions', D][4 - axes:]} with B {B} and "
                             f"Nkv a divisor of {Nq}")
        if quantised:
            for t in (keys, values):
                if tuple(t.block) != (1, D) or tuple(t.scale.shape) != (*shape[:-1], 1):
                    raise ValueError(f"{name}: a quantised cache has blocks (1, {D}), got {t.block} with scales {tuple(t.scale.shape)}")
                tensors += (t.qval, t.scale)
        else:
            tensors += (keys, values)
    if prefix_k.shape[0] != k_cache.shape[1]:
        raise ValueError(f"{prefix_k.shape[0]} kv heads in the prefix, {k_cache.shape[1]} in the caches")
    if sinks is not None:
        if sinks.shape != (Nq,):
            raise ValueError(f"sinks {tuple(sinks.shape)} must be [{Nq}]")
        tensors.append(sinks)
    if not scale > 0 or window < 0 or window != int(window):
        raise ValueError(f"scale {scale} must be positive and window {window} a number of positions (0: none)")
    if isinstance(pos, torch.Tensor):
        if pos.dtype not in (torch.int32, torch.int64) or pos.numel() not in (1, B):
            raise ValueError(f"pos must hold 1 or {B} integers, got {tuple(pos.shape)} {pos.dtype}")
        tensors.append(pos)
    elif not hasattr(pos, "__index__"):
        raise ValueError(f"pos must be an int or a tensor of integers, got {type(pos).__name__}")
    elif pos + T > k_cache.shape[2]:
        raise ValueError(f"{T} tokens from position {pos} on do not fit a cache of {k_cache.shape[2]}")
    for t in tensors:
        if t.device != device:
            raise ValueError(f"all arguments must be on {device}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("prefix_attention has no backward pass: call it under torch.no_grad()")


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit inner stride and 16-byte steps on every other axis (copied if it is not so already)."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous() and t.shape[-1] * t.element_size() % 16 == 0:
            return t
        unit, strides = 16 // t.element_size(), t.stride()
        if strides[-1] == 1 and all(s > 0 and s % unit == 0 for s, n in zip(strides[:-1], t.shape) if n > 1):
            return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _scales(t: QArray, contiguous: bool) -> torch.Tensor:
    """fp32 ``[..., positions, 1]`` of a cache's scales, neighbouring positions side by side."""
    s = t.scale if t.scale.dtype == torch.float32 else t.scale.float()
    ready = s.is_contiguous() or (not contiguous and (s.stride(-2) == 1 or s.shape[-2] <= 1))
    return s if ready else s.contiguous()


@functools.lru_cache(maxsize=256)
def _prefix_workspace(*shape: int) -> int:
    return native.function("lyra_prefix_attention_workspace", "iiiiiii", c_ll)(*shape)


def prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, sinks, scale: float, window: int, pos):
    """CUDA path; the arguments have passed :func:`check_prefix_attention`. The workspace is allocated per call."""
    B, Nq, T, D = q.shape
    quant, own_quant = isinstance(prefix_k, QArray), isinstance(k_cache, QArray)
    pk, pv = (prefix_k.qval, prefix_v.qval) if quant else (prefix_k, prefix_v)
    kc, vc = (k_cache.qval, v_cache.qval) if own_quant else (k_cache, v_cache)
    if D not in (64, 128):
        raise ValueError(f"prefix_attention takes head dim 64 or 128 on a GPU, got {D}")
    for t, q8 in ((pk, quant), (pv, quant), (kc, own_quant), (vc, own_quant)):
        if t.dtype != (torch.float8_e4m3fn if q8 else torch.bfloat16):
            raise ValueError(f"prefix and caches must be bf16, or e4m3 with scales, on a GPU; got {t.dtype}")
    Nkv, P = pk.shape[0], pk.shape[1]
    S = kc.shape[2]
    dev = q.device
    window = 0 if window >= P + S else int(window)            # a window of everything is none
    out = torch.empty((B, T, Nq, D), dtype=torch.bfloat16, device=dev)
    if out.numel() == 0:
        return out.transpose(1, 2).to(q.dtype)
    with native.on_device(q):
        need = _prefix_workspace(B, T, P, Nq, Nkv, D, window)
        if need < 0:
            raise ValueError(f"prefix_attention does not take B {B}, T {T}, {Nq} / {Nkv} heads on a GPU")
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        qb, pk, pv = _rows16(q if q.dtype == torch.bfloat16 else q.to(torch.bfloat16)), _rows16(pk), _rows16(pv)
        kc, vc = _rows16(kc.contiguous()), _rows16(vc.contiguous())
        pks = pvs = ks = vs = sk = at = None
        pks_step = pvs_step = 0
        if quant and P:
            pks, pvs = _scales(prefix_k, False), _scales(prefix_v, False)
            pks_step, pvs_step = pks.stride(0), pvs.stride(0)
        if own_quant:
            ks, vs = _scales(k_cache, True), _scales(v_cache, True)
        if sinks is not None:
            sk = sinks if sinks.dtype == torch.float32 and sinks.is_contiguous() else sinks.float().contiguous()
        if isinstance(pos, torch.Tensor):
            at = pos if pos.dtype == torch.int32 and pos.is_contiguous() else pos.to(torch.int32).contiguous()
        address = lambda t: t.data_ptr() if t is not None else None
        fn = native.function("lyra_prefix_attention", _PREFIX_ARGS)
        qs, ps, vs_ = qb.stride(), _steps(pk), _steps(pv)
        rc = fn(qb.data_ptr(), qs[0], qs[1], qs[2], pk.data_ptr(), ps[0], ps[1], pv.data_ptr(), vs_[0], vs_[1], address(pks), pks_step, address(pvs), pvs_step,
                quant, kc.data_ptr(), vc.data_ptr(), address(ks), address(vs), own_quant, address(sk), address(at), at.numel() if at is not None else 0,
                max(int(pos), -1) if at is None else 0, out.data_ptr(), ws.data_ptr(), need, B, T, P, S, Nq, Nkv, D, scale, window, native.status_word().data_ptr(),
                native.stream_address())
    native.check(rc, "lyra_prefix_attention")
    native.count_launch(2 if P else 1)
    out = out.transpose(1, 2)
    return out if q.dtype == torch.bfloat16 else out.to(q.dtype)


_PREFIX_ARGS = "plllpllpllplpl" + "ippppippii" + "ppliiiiiiifipp"


def _steps(t: torch.Tensor) -> tuple[int, int]:
    """(head, position) strides of a prefix; an axis of length one has none that matters, but a TMA map wants one it can use."""
    row = t.shape[2] if t.shape[1] <= 1 else t.stride(1)
    return (row * max(t.shape[1], 1) if t.shape[0] <= 1 else t.stride(0)), row
