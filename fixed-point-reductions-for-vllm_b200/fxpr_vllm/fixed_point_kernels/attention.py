"""Paged unified attention launcher (reference: fixed_point_kernels/attention.py:13-15,
398-489). Same signature as the reference's ``unified_attention_fxp`` plus two
optional performance hints (``num_kv_splits``, ``max_seq_len``); results do not
depend on either.
"""

from __future__ import annotations

import ctypes
import os

import torch

from .. import _native as N
from .fixed_point import RCP_LN2, int_bits_of


def _validate_hints() -> bool:
    return os.environ.get("FXPR_VALIDATE_HINTS", "0") not in ("", "0")


def check_max_seq_len_hint(seq_lens: torch.Tensor, max_seq_len: int) -> None:
    """Raise ``ValueError`` if ``max_seq_len`` is below any entry of ``seq_lens``."""
    longest = int(seq_lens.max()) if seq_lens.numel() else 0
    if longest > int(max_seq_len):
        raise ValueError(f"unified_attention_fxp: max_seq_len={int(max_seq_len)} is below the "
                         f"longest context in seq_lens ({longest})")


def prepare_log2_softmax_scale(head_dim, softmax_scale=None):
    """attention.py:13-15."""
    scale = 1.0 / (head_dim**0.5) if softmax_scale is None else softmax_scale
    return scale * RCP_LN2


def unified_attention_fxp(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    o: torch.Tensor,
    query_start_loc: torch.Tensor,
    seq_lens: torch.Tensor,
    block_table: torch.Tensor,
    max_query_len: int,
    *,
    alibi_slopes: torch.Tensor | None = None,
    fxp_dtype=torch.int32,
    is_causal: bool = True,
    softmax_scale: float | None = None,
    frac_bits: int = 14,
    block_n: int = 64,
    d_chunk: int = 64,
    logits_soft_cap: float = 0.0,
    window_size: int = 0,
    num_kv_splits: int | None = None,
    max_seq_len: int | None = None,
    use_workspace: bool = True,
):
    """Run unified prefill + decode attention on a vLLM-layout paged KV cache,
    writing into ``o``. ``block_n``/``d_chunk`` are accepted for signature
    compatibility (the reference's tile sizes; they do not change results).
    ``max_seq_len`` must bound every ``seq_lens`` entry when given: keys
    beyond it are not read (the kernels cut each context at the workspace
    sized from the hint rather than overrun it). With ``FXPR_VALIDATE_HINTS=1``
    in the environment the hint is checked against ``seq_lens`` before the
    launch (a device-to-host read, so not during stream capture) and a
    violation raises ``ValueError``.
    ``use_workspace=False`` selects the scratch-free cluster path (same
    results; the chunked path is faster for decode)."""
    assert q.is_cuda and kv_cache.is_cuda, "unified_attention_fxp requires CUDA tensors"
    assert kv_cache.ndim == 5 and kv_cache.shape[1] == 2, (
        "kv_cache must be (num_blocks, 2, block_size, num_kv_heads, head_dim); "
        f"got {tuple(kv_cache.shape)}"
    )
    key_cache, value_cache = kv_cache.unbind(1)
    head_dim_query, head_dim = q.shape[-1], key_cache.shape[-1]
    assert head_dim_query == head_dim, "head_dim mismatch between q and key_cache"
    bits = int_bits_of(fxp_dtype)
    if alibi_slopes is not None:
        assert alibi_slopes.is_cuda and alibi_slopes.dtype == torch.float32, (
            "alibi_slopes must be a float32 CUDA tensor (pre-scaled by RCP_LN2)"
        )
        alibi_slopes = alibi_slopes.contiguous()
    num_requests = seq_lens.shape[0]
    if num_requests == 0 or max_query_len <= 0:
        return
    if max_seq_len and _validate_hints() and not torch.cuda.is_current_stream_capturing():
        check_max_seq_len_hint(seq_lens, max_seq_len)
    assert key_cache.stride(-1) == 1 and value_cache.stride(-1) == 1 and q.stride(-1) == 1 \
        and o.stride(-1) == 1, "head_dim must be the innermost (contiguous) dimension"
    if num_kv_splits is None:
        from ..vllm_modules.config import get_runtime_config

        num_kv_splits = get_runtime_config().num_kv_splits
    qsl = query_start_loc if query_start_loc.dtype == torch.int32 else query_start_loc.to(torch.int32)
    sl = seq_lens if seq_lens.dtype == torch.int32 else seq_lens.to(torch.int32)
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    qsl, sl = qsl.contiguous(), sl.contiguous()
    if bt.stride(-1) != 1:
        bt = bt.contiguous()
    p = N.AttentionParams()
    p.q, p.q_dtype, p.q_stride_tok, p.q_stride_head = q.data_ptr(), N.dcode(q), q.stride(0), q.stride(1)
    p.k_cache, p.v_cache, p.kv_dtype = key_cache.data_ptr(), value_cache.data_ptr(), N.dcode(key_cache)
    p.k_stride_blk, p.k_stride_slot, p.k_stride_head = key_cache.stride()[:3]
    p.v_stride_blk, p.v_stride_slot, p.v_stride_head = value_cache.stride()[:3]
    p.o, p.o_dtype, p.o_stride_tok, p.o_stride_head = o.data_ptr(), N.dcode(o), o.stride(0), o.stride(1)
    p.query_start_loc, p.seq_lens, p.block_table = qsl.data_ptr(), sl.data_ptr(), bt.data_ptr()
    p.bt_stride = bt.stride(0)
    p.block_table_cols = bt.shape[1]
    p.max_seq_len = int(max_seq_len) if max_seq_len else 0
    p.alibi_slopes = alibi_slopes.data_ptr() if alibi_slopes is not None else None
    p.num_requests = num_requests
    p.max_query_len = int(max_query_len)
    p.num_heads = q.shape[1]
    p.num_kv_heads = key_cache.shape[2]
    p.head_dim = head_dim
    p.page_size = key_cache.shape[1]
    p.num_blocks = key_cache.shape[0]
    p.is_causal = 1 if is_causal else 0
    p.window_size = int(window_size)
    p.scale_log2 = prepare_log2_softmax_scale(head_dim_query, softmax_scale)
    p.logits_soft_cap = logits_soft_cap * RCP_LN2 if logits_soft_cap > 0.0 else 0.0
    p.frac_bits = frac_bits
    p.int_bits = bits
    p.num_kv_splits = int(num_kv_splits)
    lib = N.load()
    if use_workspace:
        need = lib.fxpr_attention_workspace_bytes(ctypes.byref(p))
        ws = N.attention_workspace(q.device, need)
        if ws is not None:
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    rc = lib.fxpr_unified_attention_fxp(ctypes.byref(p), N.stream_ptr(q.device))
    N.check(rc, "unified_attention_fxp")


def shared_prefix_attention_fxp(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    o: torch.Tensor,
    query_start_loc: torch.Tensor,
    seq_lens: torch.Tensor,
    block_table: torch.Tensor,
    common_prefix_len: int,
    max_query_len: int,
    *,
    alibi_slopes: torch.Tensor | None = None,
    fxp_dtype=torch.int32,
    is_causal: bool = True,
    softmax_scale: float | None = None,
    frac_bits: int = 16,
    logits_soft_cap: float = 0.0,
    window_size: int = 0,
    max_seq_len: int | None = None,
) -> None:
    """:func:`unified_attention_fxp` for a batch whose requests share their
    first ``common_prefix_len`` keys, written into ``o``: the prefix's keys and
    values are read and converted once for a tile of rows of all requests.

    The first ``common_prefix_len // page`` entries of every block-table row
    are the same pages (those of row 0 are read), and the keys of a last page
    that the prefix covers in part are equal in every request's own page. With
    V finite in fp16 (to which it is cast) the result has the bits of
    ``unified_attention_fxp``; a masked key contributes nothing whatever its V
    holds, and a row which sees no key is 0, in every form that a call may run. Rows of ``o`` behind ``query_start_loc[-1]`` are
    left as they are, queries behind the rows of ``q`` are skipped, and a block
    id outside the cache reads zeros. ``max_seq_len`` bounds every ``seq_lens`` entry when
    given, as there. Scratch is a tensor of the call, so calls on several
    streams and captured graphs share nothing."""
    what = "shared_prefix_attention_fxp"

    def bad(text):
        raise ValueError(f"{what}: {text}")

    if q.dim() != 3 or o.shape != q.shape:
        bad(f"q and o must be [tokens, heads, head_dim]; got {tuple(q.shape)} and {tuple(o.shape)}")
    if kv_cache.dim() != 5 or kv_cache.shape[1] != 2 or kv_cache.shape[4] != q.shape[2]:
        bad(f"kv_cache must be [blocks, 2, page, kv_heads, {q.shape[2]}]; got {tuple(kv_cache.shape)}")
    tokens, heads, dim = q.shape
    blocks, _, page, kv_heads, _ = kv_cache.shape
    if kv_heads < 1 or heads % kv_heads != 0 or page < 1:
        bad(f"{heads} query heads do not group over {kv_heads} KV heads, or the page is empty")
    if block_table.dim() != 2 or seq_lens.dim() != 1 or query_start_loc.dim() != 1:
        bad("block_table must have two dimensions, seq_lens and query_start_loc one")
    reqs = seq_lens.shape[0]
    if query_start_loc.shape[0] != reqs + 1 or block_table.shape[0] < reqs:
        bad(f"{reqs} requests need {reqs + 1} query_start_loc entries and {reqs} block-table rows; got "
            f"{query_start_loc.shape[0]} and {block_table.shape[0]}")
    if not 0 <= common_prefix_len <= block_table.shape[1] * page:
        bad(f"common_prefix_len {common_prefix_len} outside the block table's {block_table.shape[1] * page} keys")
    if q.stride(2) != 1 or o.stride(2) != 1 or kv_cache.stride(4) != 1:
        bad("head_dim must be the innermost (contiguous) dimension")
    if alibi_slopes is not None and (alibi_slopes.dtype != torch.float32 or alibi_slopes.shape != (heads,)):
        bad(f"alibi_slopes must be float32 [{heads}] (pre-scaled by 1/ln 2)")
    dev = N.same_device(q, kv_cache, o, query_start_loc, seq_lens, block_table, alibi_slopes)
    if reqs == 0 or max_query_len <= 0 or tokens == 0:
        return
    if max_seq_len and _validate_hints() and not torch.cuda.is_current_stream_capturing():
        check_max_seq_len_hint(seq_lens, max_seq_len)
    qsl, sl, bt = (x.to(torch.int32) for x in (query_start_loc, seq_lens, block_table))
    qsl, sl = qsl.contiguous(), sl.contiguous()
    bt = bt if bt.stride(1) == 1 or bt.shape[1] == 1 else bt.contiguous()
    slopes = alibi_slopes.contiguous() if alibi_slopes is not None else None
    p = N.AttentionParams()
    es, base = kv_cache.element_size(), kv_cache.data_ptr()
    sb, s2, ss, sh, _ = kv_cache.stride()
    p.q, p.q_dtype = q.data_ptr(), N.dcode(q)
    p.q_stride_tok, p.q_stride_head, _ = q.stride()
    p.k_cache, p.v_cache, p.kv_dtype = base, base + s2 * es, N.dcode(kv_cache)
    p.k_stride_blk = p.v_stride_blk = sb
    p.k_stride_slot = p.v_stride_slot = ss
    p.k_stride_head = p.v_stride_head = sh
    p.o, p.o_dtype = o.data_ptr(), N.dcode(o)
    p.o_stride_tok, p.o_stride_head, _ = o.stride()
    p.query_start_loc, p.seq_lens, p.block_table = qsl.data_ptr(), sl.data_ptr(), bt.data_ptr()
    p.bt_stride, p.block_table_cols = bt.stride(0), bt.shape[1]
    p.max_seq_len = int(max_seq_len) if max_seq_len else 0
    p.alibi_slopes = slopes.data_ptr() if slopes is not None else None
    p.num_requests, p.max_query_len = reqs, int(max_query_len)
    p.num_heads, p.num_kv_heads, p.head_dim, p.page_size = heads, kv_heads, dim, page
    p.num_blocks = blocks
    p.is_causal, p.window_size = 1 if is_causal else 0, int(window_size)
    p.scale_log2 = prepare_log2_softmax_scale(dim, softmax_scale)
    p.logits_soft_cap = logits_soft_cap * RCP_LN2 if logits_soft_cap > 0.0 else 0.0
    p.frac_bits, p.int_bits, p.num_kv_splits = frac_bits, int_bits_of(fxp_dtype), 8
    lib = N.load()
    need = lib.fxpr_shared_prefix_attention_workspace_bytes(ctypes.byref(p), common_prefix_len, tokens)
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    if need:
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
    rc = N.launch(lib.fxpr_shared_prefix_attention_fxp, dev, ctypes.byref(p), common_prefix_len, tokens)
    if rc:
        N.check(rc, what)


def shared_prefix_takes_prefix_kernels(
    common_prefix_len: int,
    num_requests: int,
    num_tokens: int,
    max_query_len: int,
    max_seq_len: int,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    page_size: int,
    *,
    dtype: torch.dtype = torch.bfloat16,
    kv_dtype: torch.dtype | None = None,
    fxp_dtype=torch.int32,
    frac_bits: int = 16,
    logits_soft_cap: float = 0.0,
    window_size: int = 0,
    alibi: bool = False,
) -> bool:
    """Whether :func:`shared_prefix_attention_fxp` runs the prefix kernels for
    such a call (queries of ``dtype`` in rows of whole heads, a contiguous
    cache), or else the unified attention's, with the same result. The
    operator's own rule, asked on the host."""
    p = N.AttentionParams()
    p.q_dtype = p.o_dtype = N.DTYPE_CODE[dtype]
    p.kv_dtype = N.DTYPE_CODE[dtype if kv_dtype is None else kv_dtype]
    p.q_stride_tok = p.o_stride_tok = num_heads * head_dim
    p.q_stride_head = p.o_stride_head = p.k_stride_head = p.v_stride_head = head_dim
    p.k_stride_slot = p.v_stride_slot = num_kv_heads * head_dim
    p.k_stride_blk = p.v_stride_blk = 2 * page_size * num_kv_heads * head_dim
    p.num_requests, p.max_query_len, p.max_seq_len = num_requests, max_query_len, max_seq_len
    p.num_heads, p.num_kv_heads, p.head_dim, p.page_size = num_heads, num_kv_heads, head_dim, page_size
    p.block_table_cols = -(-max(max_seq_len, common_prefix_len) // page_size)
    p.num_blocks = p.block_table_cols
    p.is_causal, p.window_size, p.logits_soft_cap = 1, window_size, logits_soft_cap
    p.alibi_slopes = 16 if alibi else None  # only whether they are given
    p.frac_bits, p.int_bits = frac_bits, int_bits_of(fxp_dtype)
    return bool(N.load().fxpr_shared_prefix_attention_takes_prefix(ctypes.byref(p), common_prefix_len, num_tokens))
