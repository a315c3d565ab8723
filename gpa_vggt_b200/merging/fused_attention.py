"""Flash attention with a per-key additive bias (drop-in for
merging/fused_attention.py).

``attention_keybias(q, k, v, bias, sm_scale, return_lse)`` follows the
reference's merging/fused_attention.py:130-180: SDPA(q, k, v, attn_mask=bias)
for a per-key bias [B, H, 1, N] (or None), fp32 q/k/v/bias first cast to the
autocast dtype (bf16 by default), optional log2 softmax denominators
[B, H, M] fp32.  The kernel is ``gpa_attention_keybias`` (tcgen05, head_dim 64).

``attention_shared_prefix`` is the same attention for a batch of requests whose
keys are a shared set, merged once, and a cache of their own.
"""
import torch

from .. import kernels

LOG2E = 1.4426950408889634


def attention_keybias(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      bias, sm_scale: float, return_lse: bool = False):
    """SDPA(q, k, v, attn_mask=bias) where bias is per-key: [B, H, 1, N].

    q [B, H, M, D], k/v [B, H, N, D] (CUDA, bf16; fp32 is cast first as in the
    reference).  Returns [B, H, M, D] bf16, and with return_lse also
    [B, H, M] fp32 log2 softmax denominators.  `bias` may be None.
    """
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("attention_keybias: CUDA tensors required (no CPU fallback)")
    if q.dtype == torch.float32:
        dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else torch.bfloat16
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
        bias = None if bias is None else bias.to(dt)
    if q.dtype == torch.float16:
        raise NotImplementedError("attention_keybias: fp16 inputs are not supported (bf16 only)")
    v = v.to(q.dtype)
    return kernels.attention(q, k, v, bias, sm_scale, return_lse=return_lse)


def attention_shared_prefix(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                            k_own: torch.Tensor, v_own: torch.Tensor, bias, sm_scale: float,
                            own_len=None, q_len=None, causal: bool = False, return_lse: bool = False):
    """attention_keybias for a batch of requests that share most of their keys:
    one softmax over k_prefix [Hk, P, D] with a per-key bias ([P], [1, P] or
    [Hk, P], or None: the log counts of merged keys) and over each request's own
    k_own [R, Hk, N, D].  q [R, H, M, D] -> [R, H, M, D] bf16, with return_lse
    also [R, H, M] fp32 log2 softmax denominators.  The prefix, merged once, is
    read once for all requests.  Lengths, order and masks as in
    ``kernels.attention_shared_prefix``; fp32 q/k/v/bias are cast first, as in
    attention_keybias.
    """
    if not all(t.is_cuda for t in (q, k_prefix, v_prefix, k_own, v_own)):
        raise ValueError("attention_shared_prefix: CUDA tensors required (no CPU fallback)")
    if q.dtype == torch.float32:
        dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else torch.bfloat16
        q, k_prefix, v_prefix, k_own, v_own = (t.to(dt) for t in (q, k_prefix, v_prefix, k_own, v_own))
        if bias is not None:   # fp32's lowest value would round to -inf, which takes a key out
            most = torch.finfo(dt).max
            bias = torch.where(bias > -float("inf"), bias.clamp(-most, most), bias).to(dt)
    if q.dtype == torch.float16:
        raise NotImplementedError("attention_shared_prefix: fp16 inputs are not supported (bf16 only)")
    return kernels.attention_shared_prefix(q, k_prefix, v_prefix, k_own, v_own, sm_scale, own_len=own_len,
                                           q_len=q_len, bias=bias, causal=causal, return_lse=return_lse)
