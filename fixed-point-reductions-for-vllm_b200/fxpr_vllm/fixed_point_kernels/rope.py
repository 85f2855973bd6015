"""Rotary position launchers: with the per-head fixed-point RMSNorm of queries
and keys in the same pass, and with the paged-cache append. The reference has
neither (vLLM's own rotary and cache kernels run there).

Both round once: norm and rotation are computed in fp32 from the inputs and
the result is rounded to the output (or cache) type, with every product and
sum rounded by itself, so the bits do not depend on a compiler's contraction
or on the batch."""

from __future__ import annotations

import ctypes

import torch

from .. import _native as N
from .fixed_point import int_bits_of

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _check(what: str, ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(f"{what}: {text}")


def _params(what: str, q, k, positions, cos_sin_cache, is_neox, q_weight, k_weight, eps, frac_bits,
            fxp_int_bits) -> tuple[N.RopeParams, list]:
    """Checked parameters of both forms, and the tensors that must outlive the launch."""
    _check(what, q.dim() == 3 and k.dim() == 3 and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2],
           f"q and k must be [tokens, heads, head_dim]; got {tuple(q.shape)} and {tuple(k.shape)}")
    _check(what, q.dtype == k.dtype and q.dtype in _FLOATS,
           f"q and k must share a type of float16/bfloat16/float32; got {q.dtype} and {k.dtype}")
    tokens, heads, dim = q.shape
    _check(what, tuple(positions.shape) == (tokens,) and positions.dtype in (torch.int32, torch.int64),
           f"positions must be int32/int64 [{tokens}]; got {positions.dtype} {tuple(positions.shape)}")
    _check(what, cos_sin_cache.dim() == 2 and cos_sin_cache.dtype in _FLOATS,
           f"cos_sin_cache must be a float [positions, rot_dim]; got {tuple(cos_sin_cache.shape)}")
    rot = cos_sin_cache.shape[1]
    _check(what, rot % 2 == 0 and rot <= dim, f"rot_dim must be even and at most head_dim {dim}; got {rot}")
    _check(what, (q_weight is None) == (k_weight is None), "give both norm weights or neither")
    p = N.RopeParams()
    q, k, table, pos = _rows(q), _rows(k), _rows(cos_sin_cache), positions.contiguous()
    keep = [q, k, table, pos]
    if q_weight is not None:
        _check(what, q_weight.shape == k_weight.shape == (dim,) and q_weight.dtype == k_weight.dtype
               and q_weight.dtype in _FLOATS,
               f"norm weights must share a float type and be [{dim}]; got {q_weight.dtype} "
               f"{tuple(q_weight.shape)} and {k_weight.dtype} {tuple(k_weight.shape)}")
        qw, kw = q_weight.contiguous(), k_weight.contiguous()
        keep += [qw, kw]
        p.q_weight, p.k_weight, p.weight_dtype = qw.data_ptr(), kw.data_ptr(), N.dcode(qw)
        p.frac_bits, p.int_bits = int(frac_bits), int_bits_of(fxp_int_bits)
    p.q, p.k, p.dtype = q.data_ptr(), k.data_ptr(), N.dcode(q)
    p.q_stride_tok, p.q_stride_head = q.stride(0), q.stride(1)
    p.k_stride_tok, p.k_stride_head = k.stride(0), k.stride(1)
    p.positions, p.positions_64 = pos.data_ptr(), 1 if pos.dtype == torch.int64 else 0
    p.table, p.table_dtype = table.data_ptr(), N.dcode(table)
    p.table_rows, p.table_stride = table.shape[0], table.stride(0)
    p.rot_dim, p.is_neox = rot, 1 if is_neox else 0
    p.tokens, p.num_heads, p.num_kv_heads, p.head_dim = tokens, heads, k.shape[1], dim
    p.eps = float(eps)
    return p, keep


def _out(what: str, name: str, out: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _check(what, out.shape == like.shape and out.dtype == like.dtype and (out.stride(-1) == 1 or out.shape[-1] == 1),
           f"{name} must have the input's shape and type, with head_dim contiguous")
    return out


def qk_norm_rope_fxp(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                     positions: torch.Tensor, cos_sin_cache: torch.Tensor, is_neox: bool = True,
                     eps: float = 1e-6, frac_bits: int = 16, fxp_int_bits: int = 32,
                     q_out: torch.Tensor | None = None,
                     k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Each head of q ``[tokens, heads, head_dim]`` and k normed by the
    fixed-point RMSNorm over head_dim (the arithmetic of ``rms_norm_fxp``) and
    its first rot_dim dims turned by the row ``[cos | sin]`` of
    ``cos_sin_cache`` at the token's position: pairs ``(i, i + rot_dim/2)``, or
    ``(2i, 2i + 1)`` when ``is_neox`` is false. Returns new tensors unless
    ``q_out`` / ``k_out`` are given (they may be q and k themselves). A
    position outside the table makes the rotated dims of its row NaN."""
    what = "qk_norm_rope_fxp"
    _check(what, q_weight is not None and k_weight is not None, "q_weight and k_weight are needed")
    p, keep = _params(what, q, k, positions, cos_sin_cache, is_neox, q_weight, k_weight, eps, frac_bits,
                      fxp_int_bits)
    yq, yk = _out(what, "q_out", q_out, q), _out(what, "k_out", k_out, k)
    p.q_out, p.qo_stride_tok, p.qo_stride_head = yq.data_ptr(), yq.stride(0), yq.stride(1)
    p.k_out, p.ko_stride_tok, p.ko_stride_head = yk.data_ptr(), yk.stride(0), yk.stride(1)
    dev = N.same_device(q, k, q_weight, k_weight, positions, cos_sin_cache, yq, yk)
    with N.on_device(dev):
        rc = N.load().fxpr_qk_norm_rope_fxp(ctypes.byref(p), N.stream_ptr(dev))
    N.check(rc, what)
    return yq, yk


def rope_append_kv_fxp(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_cache: torch.Tensor,
                       slot_mapping: torch.Tensor, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                       is_neox: bool = True, q_weight: torch.Tensor | None = None,
                       k_weight: torch.Tensor | None = None, eps: float = 1e-6, frac_bits: int = 16,
                       fxp_int_bits: int = 32, q_out: torch.Tensor | None = None,
                       k_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary position of q and k (normed first as in :func:`qk_norm_rope_fxp`
    when the weights are given), each token's rotated k and its v written to
    the paged cache ``[blocks, 2, page, kv_heads, head_dim]`` in the cache's
    type. Returns the rotated q (a new tensor unless ``q_out`` is given);
    ``k_out`` also receives the rotated k.

    ``slot_mapping[t] = block * page + offset``; a negative slot is padding and
    one beyond the cache writes nothing either, and tokens behind the mapping's
    end are rotated but not cached. Slots must be distinct: of two tokens with
    the same slot, each value comes from either of them."""
    what = "rope_append_kv_fxp"
    p, keep = _params(what, q, k, positions, cos_sin_cache, is_neox, q_weight, k_weight, eps, frac_bits,
                      fxp_int_bits)
    _check(what, v.shape == k.shape and v.dtype == k.dtype,
           f"v must have k's shape and type; got {v.dtype} {tuple(v.shape)}")
    _check(what, kv_cache.dim() == 5 and kv_cache.shape[1] == 2 and tuple(kv_cache.shape[3:]) == tuple(k.shape[1:])
           and kv_cache.shape[2] > 0 and kv_cache.dtype in _FLOATS,
           f"kv_cache must be a float [blocks, 2, page, {k.shape[1]}, {k.shape[2]}]; got {kv_cache.dtype} "
           f"{tuple(kv_cache.shape)}")
    _check(what, kv_cache.stride(-1) == 1 or kv_cache.shape[-1] == 1, "head_dim of kv_cache must be contiguous")
    _check(what, slot_mapping.dim() == 1 and slot_mapping.shape[0] <= q.shape[0]
           and slot_mapping.dtype in (torch.int32, torch.int64),
           f"slot_mapping must be int32/int64 of at most {q.shape[0]} entries; got {slot_mapping.dtype} "
           f"{tuple(slot_mapping.shape)}")
    v, slots = _rows(v), slot_mapping.to(torch.int64).contiguous()
    yq = _out(what, "q_out", q_out, q)
    p.v, p.v_stride_tok, p.v_stride_head = v.data_ptr(), v.stride(0), v.stride(1)
    p.q_out, p.qo_stride_tok, p.qo_stride_head = yq.data_ptr(), yq.stride(0), yq.stride(1)
    if k_out is not None:
        yk = _out(what, "k_out", k_out, k)
        p.k_out, p.ko_stride_tok, p.ko_stride_head = yk.data_ptr(), yk.stride(0), yk.stride(1)
    es, (sb, s2, ss, sh, _) = kv_cache.element_size(), kv_cache.stride()
    p.k_cache, p.v_cache, p.cache_dtype = kv_cache.data_ptr(), kv_cache.data_ptr() + s2 * es, N.dcode(kv_cache)
    p.kc_stride_blk, p.kc_stride_slot, p.kc_stride_head = sb, ss, sh
    p.vc_stride_blk, p.vc_stride_slot, p.vc_stride_head = sb, ss, sh
    p.num_blocks, p.page_size = kv_cache.shape[0], kv_cache.shape[2]
    p.slot_mapping, p.num_slots = slots.data_ptr(), slots.shape[0]
    dev = N.same_device(q, k, v, kv_cache, slot_mapping, positions, cos_sin_cache, q_weight, k_weight, yq, k_out)
    with N.on_device(dev):
        rc = N.load().fxpr_rope_append_kv_fxp(ctypes.byref(p), N.stream_ptr(dev))
    N.check(rc, what)
    return yq
