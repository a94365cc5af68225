"""Attention of query tokens to a context of another length: an encoder's states (`cross_attention`) or a cached clip that
the whole batch shares followed by each sample's own tokens (`prefix_attention`).

Beyond `functional.attention` these take what conditioning brings along: samples of different lengths (padded, packed one
after the other, or masked), grouped heads without repeating K / V, and one copy of a shared prefix. Layout BSHD as there.
CUDA bf16 / fp16 tensors with a head dim that is a multiple of 8 up to 128 run on the kernels of `csrc/context_attn_*.cu`;
everything else (CPU, fp32, other head dims) takes the fp32 evaluation of `context_attention_reference`, in query blocks.

A query that sees no key gives a zero row, and -inf as its log-sum-exp. What lies in padded or masked places does not
matter, infinities and NaN included; what lies in visible ones reaches the results as in a plain evaluation. Inference only: the kernels
record no gradient. On the kernels neither call synchronises with the host when lengths are given as device tensors, so both
can be captured in a CUDA graph (the fp32 evaluation reads `cu_kv` on the host).

Role parity: telefuser/ops/attention/attention_impl.py:112-315 (variable-length forms of the attention back ends).
"""

from __future__ import annotations

import functools
import math
import struct

import torch

from . import native
from .functional import _native

# tfb_context_attn_args of csrc/tfb_api.h: 11 pointers, 14 strides, 8 sizes, the scale, one reserved word. Packed in one
# step: a ctypes structure filled field by field costs a short call several microseconds.
_ARGS = struct.Struct("@11P14l8ifi")


def context_attention_reference(q, k, v, visible=None, scale=None, return_lse=False, q_block: int | None = None):
    """fp32 evaluation: q [B, Sq, H, D], k / v [B, Skv, Hkv, D] (H a multiple of Hkv), visible bool [B, Skv] or None."""
    B, Sq, H, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    if 0 in (B, Sq, H):
        out, lse = torch.empty_like(q), q.new_empty(B, H, Sq, dtype=torch.float32)
        return (out, lse) if return_lse else out
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    kf, vf = k.float().permute(0, 2, 3, 1), v.float().transpose(1, 2)  # [B, Hkv, D, Skv], [B, Hkv, Skv, D]
    if visible is not None:  # hidden rows may hold anything
        kf = kf.masked_fill(~visible[:, None, None, :], 0.0)
        vf = vf.masked_fill(~visible[:, None, :, None], 0.0)
    out = torch.empty(B, Sq, H, D, device=q.device, dtype=q.dtype)
    lse = torch.empty(B, H, Sq, device=q.device, dtype=torch.float32)
    step = q_block or max(Sq, 1)
    for s0 in range(0, Sq, step):
        qf = q[:, s0 : s0 + step].float()
        n = qf.shape[1]
        qf = qf.reshape(B, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
        s = (qf @ kf) * scale
        if visible is not None:
            s = s.masked_fill(~visible[:, None, None, :], float("-inf"))
        ls = torch.logsumexp(s, dim=-1) if Skv else s.new_full(s.shape[:-1], float("-inf"))
        p = torch.exp(s - ls.masked_fill(ls == float("-inf"), 0.0)[..., None])
        out[:, s0 : s0 + n] = (p @ vf).reshape(B, H, n, D).transpose(1, 2).to(q.dtype)
        lse[:, :, s0 : s0 + n] = ls.reshape(B, H, n)
    return (out, lse) if return_lse else out


def _q_block(q, keys: int) -> int | None:
    return max(128, (1 << 24) // max(keys, 1)) if q.is_cuda and q.shape[1] * keys > (1 << 24) else None


def _check(q, k, v, what: str) -> None:
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape:
        raise ValueError(f"{what}: q [B, Sq, H, D] and k / v of one shape [B, Skv, Hkv, D], got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    _, _, H, D = qs
    _, _, Hkv, Dk = ks
    if Dk != D or Hkv < 1 or H % Hkv:
        raise ValueError(f"{what}: heads {H} x {D} do not fit key heads {Hkv} x {Dk}")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"{what}: q, k and v have one type, got {dtype}, {k.dtype}, {v.dtype}")
    native.same_device(q, k, v)


def _scale(scale, D: int) -> float:
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 2.0**-126 <= scale <= 2.0**127:  # the kernels hold it, times log2(e), in fp32
        raise ValueError(f"the score scale must be positive, finite and a normal number in fp32, got {scale}")
    return scale


def _lengths(lens, n: int, most: int, device, what: str):
    """-> int32 [n] on `device`. Values that the host holds are checked; values on the device are clamped by the kernels."""
    if not torch.is_tensor(lens) or lens.device.type == "cpu":
        values = lens.tolist() if torch.is_tensor(lens) else list(lens)
        if len(values) != n or any(isinstance(x, list) or x != int(x) or not 0 <= x <= most for x in values):
            raise ValueError(f"{what}: {n} whole numbers in [0, {most}] expected, got {values}")
        return torch.tensor([int(x) for x in values], dtype=torch.int32, device=device)
    if lens.shape != (n,) or lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: an integer tensor of shape ({n},) expected, got {lens.dtype} {tuple(lens.shape)}")
    if lens.device != device:
        raise ValueError(f"{what} is on {lens.device}, the queries are on {device}")
    return lens.contiguous() if lens.dtype == torch.int32 else lens.clamp(-1, 2**31 - 1).to(torch.int32)


def _operand(t, rows: int, heads: int, D: int):
    """t [n, rows, heads, D] -> (tensor, address, batch, token and head strides), with unit channel stride, 16-byte rows and no
    broadcast dimension: copied only if it is not so already. A dimension of one entry may get any stride."""
    at = t.data_ptr()
    if t.is_contiguous() and not at & 15:  # D is a multiple of 8
        return t, at, rows * heads * D, heads * D, D
    strides = [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]
    if at & 15 or strides[3] != 1 or any(n > 1 and (s <= 0 or s % 8) for n, s in zip(t.shape[:3], strides)):
        return _operand(t.clone(memory_format=torch.contiguous_format), rows, heads, D)
    return t, at, strides[0], strides[1], strides[2]


def _runs_native(q) -> bool:
    return _native(q) and q.dtype in (torch.bfloat16, torch.float16) and q.shape[3] % 8 == 0 and 8 <= q.shape[3] <= 128


@functools.lru_cache(maxsize=4096)
def _work_bytes(device: int, packed: bool, masked: bool, sizes: tuple) -> int:
    """Scratch of a call of these sizes (the key splits depend on nothing else)."""
    some = 16  # an address that is not looked at
    args = _ARGS.pack(some, some, some, some, some, some, 0, 0, some if packed else 0, some if masked else 0, 0, *(0,) * 14,
                      *sizes, 1.0, 0)  # fmt: skip
    need = native.load().tfb_context_attn_work(args)
    if need < 0:
        native.check(-need, "tfb_context_attn_work")
    return need


def _launch(q, k, v, kp, vp, kv_lens, cu_kv, key_mask, scale, return_lse):
    dev = q.device.index
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _launch(q, k, v, kp, vp, kv_lens, cu_kv, key_mask, scale, return_lse)
    B, Sq, H, D = q.shape
    _, Skv, Hkv, _ = k.shape
    P = 0 if kp is None else kp.shape[1]
    if P and B > 1 and Sq > 1 and q.stride(0) != Sq * q.stride(1):
        q = q.contiguous()  # the shared prefix sees the tokens of all samples as one row after the other
    out = torch.empty_like(q) if q.is_contiguous() else torch.empty((B, Sq, H, D), device=q.device, dtype=q.dtype)
    lse = q.new_empty((B, H, Sq), dtype=torch.float32) if return_lse else None
    if B and Sq and H:
        q, qp, q_bs, q_ss, q_hs = _operand(q, Sq, H, D)
        k, kk, k_bs, k_ss, k_hs = _operand(k, Skv, Hkv, D)
        v, vv, v_bs, v_ss, v_hs = _operand(v, Skv, Hkv, D)
        a = b = a_ss = a_hs = b_ss = b_hs = 0
        if P:
            kp, a, _, a_ss, a_hs = _operand(kp, P, Hkv, D)
            vp, b, _, b_ss, b_hs = _operand(vp, P, Hkv, D)
        sizes = (B, Sq, H, Hkv, D, Skv, P, q.dtype == torch.float16)
        need = _work_bytes(dev, cu_kv is not None, key_mask is not None, sizes)
        work = torch.empty(need // 4, device=q.device, dtype=torch.float32) if need else None
        args = _ARGS.pack(
            qp, kk, vv, a, b, out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if kv_lens is None else kv_lens.data_ptr(),
            0 if cu_kv is None else cu_kv.data_ptr(), 0 if key_mask is None else key_mask.data_ptr(),
            0 if work is None else work.data_ptr(), q_bs, q_ss, q_hs, k_bs, k_ss, k_hs, v_bs, v_ss, v_hs, a_ss, a_hs, b_ss, b_hs,
            0 if key_mask is None else key_mask.stride(0), *sizes, scale, 0)  # fmt: skip
        native.check(native.load().tfb_context_attn(args, native.stream_ptr()), "tfb_context_attn")
    return (out, lse) if return_lse else out


def cross_attention(q, k, v, kv_lens=None, cu_kv=None, key_mask=None, scale=None, return_lse=False):
    """softmax(scale q k^T) v of q [B, Sq, H, D] over an encoder's states -> [B, Sq, H, D] (and fp32 lse [B, H, Sq]).

    k / v: [B, Skv, Hkv, D], H a multiple of Hkv (query head h reads key head h // (H / Hkv)); of these sample b sees
    the first `kv_lens[b]` (all by default), without those where `key_mask` [B, Skv] is False. Or, with `cu_kv` [B + 1],
    packed [T, Hkv, D] (or [1, T, Hkv, D]): sample b sees rows cu_kv[b] .. cu_kv[b + 1] - 1.
    `kv_lens` / `cu_kv`: lists or CPU tensors (checked, copied to the device) or int32 / int64 device tensors (used in
    place; out-of-range values are clamped to the tensors). `scale`: 1 / sqrt(D) by default, positive."""
    if cu_kv is not None:
        if kv_lens is not None or key_mask is not None:
            raise ValueError("cross_attention: packed states (cu_kv) exclude kv_lens and key_mask")
        if k.dim() == 3:
            k, v = k.unsqueeze(0), v.unsqueeze(0)
        if k.shape[0] != 1:
            raise ValueError(f"cross_attention: packed k / v are [T, Hkv, D], got {tuple(k.shape)}")
    _check(q, k, v, "cross_attention")
    B, Skv = q.shape[0], k.shape[1]
    scale = _scale(scale, q.shape[3])
    if cu_kv is not None:
        if not torch.is_tensor(cu_kv) or cu_kv.device.type == "cpu":
            values = [int(x) for x in cu_kv]
            if any(a > b for a, b in zip(values, values[1:])):
                raise ValueError(f"cross_attention: cu_kv must not decrease, got {values}")
        cu_kv = _lengths(cu_kv, B + 1, Skv, q.device, "cu_kv")
    elif k.shape[0] != B:
        raise ValueError(f"cross_attention: batch {B} of q against {k.shape[0]} of k / v")
    if kv_lens is not None:
        kv_lens = _lengths(kv_lens, B, Skv, q.device, "kv_lens")
    if key_mask is not None:
        if key_mask.shape != (B, Skv) or key_mask.dtype != torch.bool:
            raise ValueError(f"cross_attention: key_mask is bool [{B}, {Skv}], got {key_mask.dtype} {tuple(key_mask.shape)}")
        native.same_device(q, key_mask)
        key_mask = key_mask if key_mask.stride(-1) == 1 or Skv == 1 else key_mask.contiguous()
    if _runs_native(q):
        return _launch(q, k, v, None, None, kv_lens, cu_kv, key_mask, scale, return_lse)
    visible = key_mask
    if cu_kv is not None:
        cu = [min(max(x, 0), Skv) for x in cu_kv.tolist()]
        lens = [max(b - a, 0) for a, b in zip(cu, cu[1:])]
        at = torch.tensor(cu[:-1], dtype=torch.long, device=q.device)[:, None] + torch.arange(max(lens, default=0), device=q.device)
        visible = torch.arange(at.shape[1], device=q.device) < torch.tensor(lens, dtype=torch.long, device=q.device)[:, None]
        k, v = (t[0][at.clamp(max=max(Skv - 1, 0))] if Skv else t.new_zeros(B, 0, *t.shape[2:]) for t in (k, v))
    elif kv_lens is not None:
        seen = torch.arange(Skv, device=q.device) < kv_lens[:, None]
        visible = seen if visible is None else visible & seen
    return context_attention_reference(q, k, v, visible, scale, return_lse, _q_block(q, k.shape[1]))


def prefix_attention(q, k_prefix, v_prefix, k, v, kv_lens=None, scale=None, return_lse=False):
    """Attention of a batch whose samples share a prefix of keys: softmax over the P prefix keys followed by the sample's own.

    q [B, Sq, H, D]; k_prefix / v_prefix [1, P, Hkv, D] (or [P, Hkv, D]), stored once for all samples; k / v
    [B, S, Hkv, D], of which sample b sees the first `kv_lens[b]` (all by default; P or S may be 0). Equal to `cross_attention` over the
    concatenation, which is never built. Every query sees every key: causal order among the own tokens is not applied.
    With few queries per sample (single tokens) the prefix is read once for the whole batch instead of once per sample."""
    if k_prefix.dim() == 3:
        k_prefix, v_prefix = k_prefix.unsqueeze(0), v_prefix.unsqueeze(0)
    _check(q, k, v, "prefix_attention")
    _check(q, k_prefix, v_prefix, "prefix_attention (prefix)")
    if k_prefix.shape[0] != 1 or k_prefix.shape[2] != k.shape[2]:
        raise ValueError(f"prefix_attention: the shared prefix is [1, P, {k.shape[2]}, {k.shape[3]}], got {tuple(k_prefix.shape)}")
    B, S = q.shape[0], k.shape[1]
    if k.shape[0] != B:
        raise ValueError(f"prefix_attention: batch {B} of q against {k.shape[0]} of k / v")
    scale = _scale(scale, q.shape[3])
    if kv_lens is not None:
        kv_lens = _lengths(kv_lens, B, S, q.device, "kv_lens")
    if _runs_native(q):
        return _launch(q, k, v, k_prefix, v_prefix, kv_lens, None, None, scale, return_lse)
    visible = None
    if kv_lens is not None:
        P = k_prefix.shape[1]
        visible = torch.arange(P + S, device=q.device) < P + kv_lens.clamp(0, S)[:, None]
    k, v = (torch.cat([a.expand(B, -1, -1, -1), b], dim=1) for a, b in ((k_prefix, k), (v_prefix, v)))
    return context_attention_reference(q, k, v, visible, scale, return_lse, _q_block(q, k.shape[1]))


__all__ = ["cross_attention", "prefix_attention", "context_attention_reference"]
