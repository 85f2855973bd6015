"""Attention behind a shared prefix keeps its contract whichever kernels a call
runs: the prefix kernels, or one of the unified attention's three forms."""

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm.fixed_point_kernels import attention as A
from tests.helpers import bits_equal

BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32
PAGE = 16

# head_dim, query heads, KV heads, prefix, queries of each request, type, largest context given (0: the real one): what runs
ROUTES = {
    "prefix": (64, 8, 4, 320, [1, 3, 2, 4], BF, 0),
    "chunks, one query": (64, 8, 4, 128, [1, 1, 1, 1], BF, 0),   # a short prefix
    "chunks, several": (128, 7, 1, 128, [1, 3, 2, 4], HF, 0),
    "chunks, fp32": (64, 8, 4, 320, [1, 3, 2, 4], F4, 0),
    "clusters": (64, 8, 4, 320, [1, 3, 2, 4], BF, 1 << 21),      # a workspace beyond the limit
    "clusters, head_dim 32": (32, 16, 4, 320, [1, 3, 2, 4], HF, 1 << 21),
    "decode": (128, 8, 2, 320, [1, 1, 1, 1], BF, 0),             # few requests, groups of four
}


def _batch(route, own=(5, 40, 21, 9), seed=0):
    D, H, KVH, prefix, qlens, dtype, most = ROUTES[route]
    g = torch.Generator().manual_seed(seed)
    R, total = len(qlens), [prefix + n for n in own]
    shared, cols = prefix // PAGE, (max(total) + PAGE - 1) // PAGE
    bt = torch.empty(R, cols, dtype=torch.int32)
    bt[:, :shared] = torch.arange(shared).int()
    bt[:, shared:] = shared + torch.arange(R * (cols - shared)).int().view(R, -1)
    kv = torch.randn(shared + R * (cols - shared), 2, PAGE, KVH, D, generator=g).to(dtype)
    q = (torch.randn(sum(qlens), H, D, generator=g) * 1.5).to(dtype)
    qsl = torch.tensor([sum(qlens[:i]) for i in range(R + 1)], dtype=torch.int32)
    return [x.cuda() for x in (q, kv, qsl, torch.tensor(total, dtype=torch.int32), bt)], prefix, max(qlens), most or max(total)


def _run(batch, **kw):
    (q, kv, qsl, sl, bt), prefix, mq, ms = batch
    o = torch.full(q.shape, 7.0, device="cuda")
    A.shared_prefix_attention_fxp(q, kv, o, qsl, sl, bt, prefix, mq, max_seq_len=ms, **kw)
    return o


@pytest.mark.gpu
@pytest.mark.parametrize("route", ROUTES)
def test_block_ids_outside_the_cache_read_zeros(route):
    """In the shared pages and in a request's own: as if those pages held zeros."""
    batch = _batch(route)
    (q, kv, qsl, sl, bt), prefix, mq, ms = batch
    bad, zeroed = bt.clone(), kv.clone()
    own = prefix // PAGE
    for col, ident in ((2, kv.shape[0]), (5, -1), (6, 2**31 - 1)):
        zeroed[bt[0, col].long()] = 0
        bad[:, col] = ident
    zeroed[bt[1, own].long()] = 0
    bad[1, own] = kv.shape[0] + 7
    got = _run(((q, kv, qsl, sl, bad), prefix, mq, ms))
    assert bits_equal(got, _run(((q, zeroed, qsl, sl, bt), prefix, mq, ms)))


@pytest.mark.gpu
@pytest.mark.parametrize("route", ROUTES)
def test_queries_behind_the_rows_are_skipped(route):
    """Ranges of queries that end behind the rows of q: the missing rows are neither read nor written, the others keep their bits."""
    batch = _batch(route)
    (q, kv, qsl, sl, bt), prefix, mq, ms = batch
    want = _run(batch)
    n = q.shape[0] - (3 if mq > 1 else 2)  # within the last request's queries, or the last two requests' rows
    guard = torch.full((q.shape[0] + 8, *q.shape[1:]), 7.0, device="cuda")
    A.shared_prefix_attention_fxp(q[:n], kv, guard[:n], qsl, sl, bt, prefix, mq, max_seq_len=ms)
    assert bits_equal(guard[:n], want[:n]) and (guard[n:] == 7.0).all()
