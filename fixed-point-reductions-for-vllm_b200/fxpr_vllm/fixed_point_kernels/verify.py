"""Launcher of the verification of drafted tokens (speculative decoding). No
counterpart in the reference."""

from __future__ import annotations

import torch

from .. import _native as N

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_INTS = (torch.int32, torch.int64)
MAX_DRAFT_LEN = 32


def _bad(text: str):
    raise ValueError(f"verify_draft_fxp: {text}")


def _seen(x: torch.Tensor) -> str:
    return f"{x.dtype} {tuple(x.shape)}"


def verify_draft_fxp(target_probs: torch.Tensor, draft_probs: torch.Tensor | None, draft_token_ids: torch.Tensor,
                     draft_start_loc: torch.Tensor, bonus_token_ids: torch.Tensor, accept_uniform: torch.Tensor,
                     resample_uniform: torch.Tensor, max_draft_len: int,
                     frac_bits: int = 30) -> tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand, and the token after them, in integers: the
    same tokens whatever the batch, the padding or the GPU.

    ``target_probs`` and ``draft_probs`` are ``[num_drafts, vocab]``, the
    positions of all requests one after the other, request r's from
    ``draft_start_loc[r]`` to ``draft_start_loc[r + 1]`` (of which at most
    ``max_draft_len`` are looked at). Probabilities are clamped to [0, 1] and
    rounded to the ``2^-frac_bits`` grid, P and Q; random numbers, in [0, 1),
    are truncated to 24 bits. A token x is taken iff
    ``accept_uniform * Q(x) < P(x)``. At the first that is not, a token is
    drawn from ``max(P - Q, 0)`` (from P where that is zero everywhere): the
    smallest v whose running sum exceeds ``floor(resample_uniform[r] * sum)``.
    When all are taken, ``bonus_token_ids[r]`` follows. ``draft_probs=None``
    stands for a deterministic drafter (Q is 1 at the drafted token).

    Returns ``token_ids`` int32 ``[num_requests, max_draft_len + 1]`` (the
    taken tokens, the drawn or bonus token, then -1) and ``num_accepted``
    int32 ``[num_requests]``. A drafted id outside the vocabulary is never
    taken; a target row that is zero everywhere draws -1."""
    most, f = int(max_draft_len), int(frac_bits)
    if target_probs.dim() != 2 or target_probs.dtype not in _FLOATS:
        _bad(f"target_probs must be float16/bfloat16/float32 [num_drafts, vocab]; got {_seen(target_probs)}")
    n, vocab = target_probs.shape
    if draft_probs is not None and (draft_probs.shape != target_probs.shape or draft_probs.dtype != target_probs.dtype):
        _bad(f"draft_probs must have target_probs' shape and type; got {_seen(draft_probs)}")
    if draft_start_loc.dim() != 1 or draft_start_loc.dtype not in _INTS or draft_start_loc.shape[0] < 1:
        _bad(f"draft_start_loc must be int32/int64 [num_requests + 1]; got {_seen(draft_start_loc)}")
    reqs = draft_start_loc.shape[0] - 1
    for name, x, size in (("draft_token_ids", draft_token_ids, n), ("bonus_token_ids", bonus_token_ids, reqs)):
        if x.dim() != 1 or x.shape[0] != size or x.dtype not in _INTS:
            _bad(f"{name} must be int32/int64 [{size}]; got {_seen(x)}")
    for name, x, size in (("accept_uniform", accept_uniform, n), ("resample_uniform", resample_uniform, reqs)):
        if x.dim() != 1 or x.shape[0] != size or x.dtype != torch.float32:
            _bad(f"{name} must be float32 [{size}]; got {_seen(x)}")
    if not 0 <= most <= MAX_DRAFT_LEN:
        _bad(f"max_draft_len must be 0..{MAX_DRAFT_LEN}, got {most}")
    if not 1 <= f <= 30:
        _bad(f"frac_bits must be 1..30, got {f}")
    if not 1 <= vocab <= 1 << 24:
        _bad(f"the vocabulary must have 1..2^24 entries, got {vocab}")
    dev = N.same_device(target_probs, draft_probs, draft_token_ids, draft_start_loc, bonus_token_ids,
                        accept_uniform, resample_uniform)
    p = target_probs if target_probs.stride(1) == 1 or vocab == 1 else target_probs.contiguous()
    q = draft_probs
    if q is not None and q.stride(1) != 1 and vocab != 1:
        q = q.contiguous()
    ids, bonus = draft_token_ids.contiguous(), bonus_token_ids.contiguous()
    start = draft_start_loc.to(torch.int32).contiguous()
    u, r = accept_uniform.contiguous(), resample_uniform.contiguous()
    out = p.new_empty((reqs, most + 1), dtype=torch.int32)
    taken = p.new_empty((reqs,), dtype=torch.int32)
    rc = N.launch(
        N.load().fxpr_verify_draft_fxp, dev, p.data_ptr(), None if q is None else q.data_ptr(), N.DTYPE_CODE[p.dtype],
        p.stride(0), 0 if q is None else q.stride(0), n, vocab, ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0,
        start.data_ptr(), bonus.data_ptr(), 1 if bonus.dtype == torch.int64 else 0, u.data_ptr(), r.data_ptr(),
        reqs, most, f, out.data_ptr(), most + 1, taken.data_ptr())
    if rc:
        N.check(rc, "verify_draft_fxp")
    return out, taken
