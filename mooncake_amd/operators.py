"""The router in front of dispatch and the experts between dispatch and combine, on torch tensors.

    topk_idx, topk_weights = route(logits, num_topk)
    recv_x, recv_count, handle, event, hook = buffer.dispatch(x, topk_idx, ...)
    expert_out = expert_mlp(recv_x, recv_count, w_gate_up, w_down)
    combined, event, hook = buffer.combine(expert_out, topk_idx, topk_weights, ..., handle)

Everything is enqueued on the current stream and nothing waits for it; outputs that are not handed in are allocated for
that stream by torch.  All of it runs on libmooncake_ep_hip.so (mc_ep_route, mc_ep_expert_gate_up, mc_ep_expert_down).
Arguments of a wrong shape, type, stride or device raise AssertionError, as `Buffer`'s do; sizes beyond what the library
takes raise RuntimeError.

These are operators of serving: no gradients, as dispatch and combine have none.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib, ep

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)
_native = ep._native if _raw_stream is not None and _raw_device is not None else None

_BF16, _F32, _FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn

# packed rows, activations or weights: bf16, or fp8 e4m3 values and their f32 scales
Scaled = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _here() -> Tuple[int, int]:
    """The current device and its current stream."""
    if _native is not None:
        device = _raw_device()
        return device, _raw_stream(device)
    return torch.cuda.current_device(), int(torch.cuda.current_stream().cuda_stream)


def _parts(v: Scaled) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    if isinstance(v, (tuple, list)):
        values, scales = v
        assert scales is not None
        return values, scales
    return v, None


def route(logits: torch.Tensor, num_topk: int, score: str = "softmax", bias: Optional[torch.Tensor] = None,
          num_groups: int = 1, topk_groups: int = 1, renormalize: bool = True, scale: float = 1.0,
          token_mask: Optional[torch.Tensor] = None, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Router logits [T, E] (f32 or bf16, rows any E or more elements apart) -> (topk_idx int64, topk_weights f32), both [T, num_topk]:
    what `Buffer.dispatch` and `Buffer.combine` take.

    The scores are softmax (over the experts) or sigmoid of the logits, in 32 bits (a sigmoid is zero for logits below
    -88.72).  Experts are chosen by score + bias (bias f32 [E]) or, without one, by their logits - the same order -, in
    falling order, the lowest index first among equals.  With num_groups > 1 the experts are that many equal groups of
    consecutive ones and only those of the best topk_groups groups can be chosen; a group counts as its best expert, with
    a bias as its best two together.  The weights are the chosen experts' scores without the bias, divided by their sum if
    `renormalize`, times `scale`.

    token_mask (bool [T]): False leaves a token out.  Logits of -inf or NaN, and choices of -inf or NaN (a bias of -inf
    takes an expert out of service), are never chosen; +inf counts as the largest finite number.  Places that stay empty
    hold index -1, which dispatch and combine skip, and weight 0.  `out`: (topk_idx, topk_weights) to write to."""
    assert score in ("softmax", "sigmoid")
    idx, weights = (None, None) if out is None else out
    device, stream = _here()
    if _native is not None:
        return _native.route_tensors(logits, num_topk, score == "sigmoid", bias, num_groups, topk_groups, renormalize, scale,
                                     token_mask, idx, weights, device, stream)
    # the compiled module's checks
    assert logits.dim() == 2 and logits.dtype in (_F32, _BF16)
    assert logits.is_cuda and logits.get_device() == device
    T, E = logits.shape
    assert E <= 1 or logits.stride(1) == 1
    assert 0 < num_topk <= E
    assert num_groups > 0 and E % num_groups == 0
    assert 0 < topk_groups <= num_groups
    if bias is not None:
        _need(bias, (E,), _F32, device)
    if token_mask is not None:
        _need(token_mask, (T,), torch.bool, device)
    if idx is None:
        idx = torch.empty((T, num_topk), dtype=torch.int64, device=logits.device)
    if weights is None:
        weights = torch.empty((T, num_topk), dtype=_F32, device=logits.device)
    _need(idx, (T, num_topk), torch.int64, device)
    _need(weights, (T, num_topk), _F32, device)
    _lib.check(_lib.lib().mc_ep_route(
        logits.data_ptr(), int(logits.dtype == _BF16), logits.stride(0) if T > 1 else E, _address(bias),
        _address(token_mask), T, E, num_topk, int(score == "sigmoid"), num_groups, topk_groups, int(bool(renormalize)),
        scale, idx.data_ptr(), weights.data_ptr(), stream))
    return idx, weights


def expert_gate_up(packed_recv_x: Scaled, packed_recv_count: torch.Tensor, w_gate_up: Scaled,
                   act: Optional[Scaled] = None) -> Scaled:
    """act[e] = silu(x[e] Wg[e]^T) * (x[e] Wu[e]^T) for the first packed_recv_count[e] rows of every local expert; other
    rows are neither read nor written.

    packed_recv_x: dispatch's first output, bf16 [L, R*max, H] or (fp8 values, f32 scales [L, R*max, H/128] stored
    column-major per expert).  w_gate_up: [L, 2I, H], Wg's rows first - bf16, or (fp8 values, f32 scales of their 128 x 128
    blocks [L, 2I/128, H/128]) for an fp8 payload.  Returns (or writes to `act`) bf16 [L, R*max, I], or (fp8 values, f32
    scales [L, R*max, I/128]) laid out like the payload, a scale being amax / 448 with amax at least 1e-4.  I is a multiple
    of 128 in fp8, of 8 in bf16.  `act` may not lie on the payload.

    bf16 products are summed in 32 bits.  In fp8 the matrix instruction cuts each of eight consecutive products off 2^-13
    below the largest of the eight (an error of at most 7 * 2^-13 of that one per eight); all other sums have 32 bits."""
    x, scales = _parts(packed_recv_x)
    w, w_scales = _parts(w_gate_up)
    a, a_scales = (None, None) if act is None else _parts(act)
    device, stream = _here()
    if _native is not None:
        a, a_scales = _native.expert_gate_up_tensors(x, scales, packed_recv_count, w, w_scales, a, a_scales, device, stream)
        return a if a_scales is None else (a, a_scales)
    L, rows, H, I, fp8 = _gate_up_shape(x, scales, packed_recv_count, w, w_scales, device)
    if a is None:
        a = torch.empty((L, rows, I), dtype=x.dtype, device=x.device)
        if fp8:
            a_scales = torch.empty((L, I // 128, rows), dtype=_F32, device=x.device).transpose(1, 2)
    _need(a, (L, rows, I), x.dtype, device)
    assert fp8 == (a_scales is not None)
    if fp8:
        _need_scales(a_scales, (L, rows, I // 128), device)
    _lib.check(_lib.lib().mc_ep_expert_gate_up(
        x.data_ptr(), _address(scales), packed_recv_count.data_ptr(), w.data_ptr(), _address(w_scales), a.data_ptr(),
        _address(a_scales), L, rows, H, I, int(fp8), stream))
    return (a, a_scales) if fp8 else a


def expert_down(act: Scaled, packed_recv_count: torch.Tensor, w_down: Scaled,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[e] = act[e] Wd[e]^T, bf16 [L, R*max, H], for the first packed_recv_count[e] rows of every local expert: what
    combine reads.  act as `expert_gate_up` returns it; w_down [L, H, I], bf16 or (fp8 values, f32 scales of their
    128 x 128 blocks [L, H/128, I/128]).  `out` may not lie on the activations."""
    a, a_scales = _parts(act)
    w, w_scales = _parts(w_down)
    device, stream = _here()
    if _native is not None:
        return _native.expert_down_tensors(a, a_scales, packed_recv_count, w, w_scales, out, device, stream)
    assert a.dim() == 3 and w.dim() == 3
    L, rows, I = a.shape
    H, fp8 = w.shape[1], a_scales is not None
    _need(a, (L, rows, I), _FP8 if fp8 else _BF16, device)
    assert H % 128 == 0 and I % (128 if fp8 else 8) == 0
    _need_weights(w, w_scales, L, H, I, fp8, device)
    _need(packed_recv_count, (L,), torch.int32, device)
    if fp8:
        _need_scales(a_scales, (L, rows, I // 128), device)
    if out is None:
        out = torch.empty((L, rows, H), dtype=_BF16, device=a.device)
    _need(out, (L, rows, H), _BF16, device)
    _lib.check(_lib.lib().mc_ep_expert_down(
        a.data_ptr(), _address(a_scales), packed_recv_count.data_ptr(), w.data_ptr(), _address(w_scales), out.data_ptr(),
        L, rows, H, I, int(fp8), stream))
    return out


def expert_mlp(packed_recv_x: Scaled, packed_recv_count: torch.Tensor, w_gate_up: Scaled, w_down: Scaled,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`expert_down` of `expert_gate_up`: dispatch's packed rows -> the rows combine reads.  The activations between the
    two live in memory that torch lends for the call, rounded to the payload's type.  A bf16 `out` may be the payload itself."""
    return expert_down(expert_gate_up(packed_recv_x, packed_recv_count, w_gate_up), packed_recv_count, w_down, out)


# --- the compiled module's checks, for the ctypes binding ---------------------------------------------------------


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _need(t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: int) -> None:
    assert tuple(t.shape) == shape
    assert t.dtype == dtype
    assert t.is_cuda and t.get_device() == device
    assert t.is_contiguous()


def _need_scales(t: torch.Tensor, shape: tuple, device: int) -> None:
    assert tuple(t.shape) == shape
    _need(t.transpose(1, 2), (shape[0], shape[2], shape[1]), _F32, device)


def _need_weights(w: torch.Tensor, scales: Optional[torch.Tensor], L: int, rows: int, columns: int, fp8: bool,
                  device: int) -> None:
    _need(w, (L, rows, columns), _FP8 if fp8 else _BF16, device)
    assert fp8 == (scales is not None)
    if fp8:
        assert rows % 128 == 0 and columns % 128 == 0
        _need(scales, (L, rows // 128, columns // 128), _F32, device)


def _gate_up_shape(x, scales, count, w, w_scales, device) -> tuple:
    assert x.dim() == 3 and w.dim() == 3
    L, rows, H = x.shape
    fp8 = scales is not None
    _need(x, (L, rows, H), _FP8 if fp8 else _BF16, device)
    assert H % 128 == 0 and w.shape[1] % 2 == 0
    I = w.shape[1] // 2
    _need_weights(w, w_scales, L, 2 * I, H, fp8, device)
    assert I % (128 if fp8 else 8) == 0
    _need(count, (L,), torch.int32, device)
    if fp8:
        _need_scales(scales, (L, rows, H // 128), device)
    return L, rows, H, I, fp8
