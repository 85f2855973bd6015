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
_INTS = (torch.int32, torch.int64)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _seen(x: torch.Tensor | None) -> str:
    return "None" if x is None else f"{x.dtype} {tuple(x.shape)}"


def _params(what: str, q, k, positions, cos_sin_cache, is_neox, q_weight, k_weight, eps, frac_bits,
            fxp_int_bits) -> tuple[N.RopeParams, list]:
    """Checked parameters of both forms, and the tensors that must outlive the launch."""
    qs, ks, dt = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2]:
        raise ValueError(f"{what}: q and k must be [tokens, heads, head_dim]; got {_seen(q)} and {_seen(k)}")
    if k.dtype != dt or dt not in _FLOATS:
        raise ValueError(f"{what}: q and k must share a type of float16/bfloat16/float32; got {_seen(q)} and {_seen(k)}")
    tokens, heads, dim = qs
    if positions.dim() != 1 or positions.shape[0] != tokens or positions.dtype not in _INTS:
        raise ValueError(f"{what}: positions must be int32/int64 [{tokens}]; got {_seen(positions)}")
    if cos_sin_cache.dim() != 2 or cos_sin_cache.dtype not in _FLOATS:
        raise ValueError(f"{what}: cos_sin_cache must be a float [positions, rot_dim]; got {_seen(cos_sin_cache)}")
    rows, rot = cos_sin_cache.shape
    if rot % 2 != 0 or rot > dim:
        raise ValueError(f"{what}: rot_dim must be even and at most head_dim {dim}; got {rot}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError(f"{what}: give both norm weights or neither")
    p = N.RopeParams()
    q, k, table, pos = _rows(q), _rows(k), _rows(cos_sin_cache), positions.contiguous()
    keep = [q, k, table, pos]
    if q_weight is not None:
        if (q_weight.dim() != 1 or q_weight.shape != k_weight.shape or q_weight.shape[0] != dim
                or q_weight.dtype != k_weight.dtype or q_weight.dtype not in _FLOATS):
            raise ValueError(f"{what}: norm weights must share a float type and be [{dim}]; got {_seen(q_weight)} "
                             f"and {_seen(k_weight)}")
        qw, kw = q_weight.contiguous(), k_weight.contiguous()
        keep += [qw, kw]
        p.q_weight, p.k_weight, p.weight_dtype = qw.data_ptr(), kw.data_ptr(), N.DTYPE_CODE[qw.dtype]
        p.frac_bits, p.int_bits, p.eps = frac_bits, int_bits_of(fxp_int_bits), eps
    p.q, p.k, p.dtype = q.data_ptr(), k.data_ptr(), N.DTYPE_CODE[dt]
    p.q_stride_tok, p.q_stride_head, _ = q.stride()
    p.k_stride_tok, p.k_stride_head, _ = k.stride()
    p.positions, p.positions_64 = pos.data_ptr(), 1 if pos.dtype == torch.int64 else 0
    p.table, p.table_dtype = table.data_ptr(), N.DTYPE_CODE[table.dtype]
    p.table_rows, p.table_stride = rows, table.stride(0)
    p.rot_dim, p.is_neox = rot, 1 if is_neox else 0
    p.tokens, p.num_heads, p.num_kv_heads, p.head_dim = tokens, heads, ks[1], dim
    return p, keep


def _out(what: str, name: str, out: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if out.shape != like.shape or out.dtype != like.dtype or (out.stride(-1) != 1 and out.shape[-1] != 1):
        raise ValueError(f"{what}: {name} must have the input's shape and type, with head_dim contiguous")
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
    if q_weight is None or k_weight is None:
        raise ValueError(f"{what}: q_weight and k_weight are needed")
    p, keep = _params(what, q, k, positions, cos_sin_cache, is_neox, q_weight, k_weight, eps, frac_bits,
                      fxp_int_bits)
    yq, yk = _out(what, "q_out", q_out, q), _out(what, "k_out", k_out, k)
    p.q_out, p.k_out = yq.data_ptr(), yk.data_ptr()
    p.qo_stride_tok, p.qo_stride_head, _ = yq.stride()
    p.ko_stride_tok, p.ko_stride_head, _ = yk.stride()
    dev = N.same_device(q, k, q_weight, k_weight, positions, cos_sin_cache, yq, yk)
    rc = N.launch(N.load().fxpr_qk_norm_rope_fxp, dev, ctypes.byref(p))
    if rc:
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
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must have k's shape and type; got {_seen(v)}")
    cs, (_, kv_heads, dim) = kv_cache.shape, k.shape
    if len(cs) != 5 or cs[1] != 2 or cs[2] == 0 or cs[3] != kv_heads or cs[4] != dim or kv_cache.dtype not in _FLOATS:
        raise ValueError(f"{what}: kv_cache must be a float [blocks, 2, page, {kv_heads}, {dim}]; got {_seen(kv_cache)}")
    sb, s2, ss, sh, s1 = kv_cache.stride()
    if s1 != 1 and dim != 1:
        raise ValueError(f"{what}: head_dim of kv_cache must be contiguous")
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] > q.shape[0] or slot_mapping.dtype not in _INTS:
        raise ValueError(f"{what}: slot_mapping must be int32/int64 of at most {q.shape[0]} entries; got {_seen(slot_mapping)}")
    v, slots = _rows(v), slot_mapping.to(torch.int64).contiguous()
    yq = _out(what, "q_out", q_out, q)
    p.v, p.q_out = v.data_ptr(), yq.data_ptr()
    p.v_stride_tok, p.v_stride_head, _ = v.stride()
    p.qo_stride_tok, p.qo_stride_head, _ = yq.stride()
    if k_out is not None:
        yk = _out(what, "k_out", k_out, k)
        p.k_out = yk.data_ptr()
        p.ko_stride_tok, p.ko_stride_head, _ = yk.stride()
    base = kv_cache.data_ptr()
    p.k_cache, p.v_cache, p.cache_dtype = base, base + s2 * kv_cache.element_size(), N.DTYPE_CODE[kv_cache.dtype]
    p.kc_stride_blk = p.vc_stride_blk = sb
    p.kc_stride_slot = p.vc_stride_slot = ss
    p.kc_stride_head = p.vc_stride_head = sh
    p.num_blocks, p.page_size = cs[0], cs[2]
    p.slot_mapping, p.num_slots = slots.data_ptr(), slots.shape[0]
    dev = N.same_device(q, k, v, kv_cache, slot_mapping, positions, cos_sin_cache, q_weight, k_weight, yq, k_out)
    rc = N.launch(N.load().fxpr_rope_append_kv_fxp, dev, ctypes.byref(p))
    if rc:
        N.check(rc, what)
    return yq
