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


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("route", ROUTES)
def test_masked_keys_contribute_nothing(route, bits):
    """V of keys that a row does not see may be infinite or NaN: a window's hidden pages, later queries' keys, places behind the end."""
    batch = _batch(route)
    (q, kv, qsl, sl, bt), prefix, mq, _ = batch
    want = _run(batch, fxp_dtype=bits)
    for r, n in enumerate(sl.tolist()):  # behind the sequence's end, on its last page
        kv[bt[r, n // PAGE].long(), 1, n % PAGE:] = float("nan")
    assert bits_equal(_run(batch, fxp_dtype=bits), want)
    if mq > 1:  # the last query's own key, hidden from the queries before it
        r = int(torch.argmax(qsl[1:] - qsl[:-1]))
        j = int(sl[r]) - 1
        kv[bt[r, j // PAGE].long(), 1, j % PAGE] = float("inf")
        got, last = _run(batch, fxp_dtype=bits), int(qsl[r + 1]) - 1
        keep = [t for t in range(q.shape[0]) if t != last]
        assert bits_equal(got[keep], want[keep])
        return
    want = _run(batch, fxp_dtype=bits, window_size=64)
    kv[bt[0, :prefix // PAGE - 5].long(), 1] = float("inf")
    kv[bt[0, 2].long(), 1] = float("nan")
    assert bits_equal(_run(batch, fxp_dtype=bits, window_size=64), want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("route", ROUTES)
def test_rows_that_see_no_key_are_zero(route, bits):
    """A request without keys, and queries in front of a sequence shorter than their number."""
    batch = _batch(route)
    (q, _, qsl, sl, _), _, mq, _ = batch
    want = _run(batch, fxp_dtype=bits)
    sl[0] = 0
    blind = [0]
    if mq > 1:
        sl[3] = 1  # four queries, one key: three rows see nothing
        blind += list(range(int(qsl[3]), int(qsl[4]) - 1))
    got = _run(batch, fxp_dtype=bits)
    assert (got[blind] == 0).all() and got.isfinite().all()
    rest = list(range(int(qsl[1]), int(qsl[3])))
    assert bits_equal(got[rest], want[rest])
    window = _run(batch, fxp_dtype=bits, window_size=64)
    assert (window[blind] == 0).all()


@pytest.mark.gpu
def test_a_request_does_not_see_its_batch():
    """Requests with infinite V behind a window, one of them without keys: the same bits by the unified kernels as by the prefix
    kernels."""
    batch = _batch("chunks, one query")
    (q, kv, qsl, sl, bt), prefix, mq, ms = batch
    kv[bt[0, :3].long(), 1] = float("inf")
    sl[2] = 0
    small = _run(batch, window_size=64)
    # the same requests behind 128 more keys that their window hides: from 256 shared keys on the prefix kernels run
    extra = torch.randn(8, *kv.shape[1:], device="cuda").to(kv.dtype)
    extra[:, 1] = float("nan")
    more = torch.cat([(kv.shape[0] + torch.arange(8, device="cuda").int()).expand(4, -1), bt], 1)
    far = torch.where(sl > 0, sl + 128, 0).int()
    large = _run(((q, torch.cat([kv, extra]), qsl, far, more), prefix + 128, mq, ms + 128), window_size=64)
    assert bits_equal(small, large)


def _time(run):
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(4):
            run()
    best = float("inf")
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


# requests, queries of each, query heads, KV heads, head_dim, shared keys, own keys
@pytest.mark.gpu
@pytest.mark.parametrize("R, ql, H, KVH, D, prefix, own", [
    (64, 1, 32, 8, 128, 1024, 3312), (64, 1, 32, 8, 128, 4096, 4096), (32, 1, 32, 8, 64, 2048, 4096), (16, 1, 32, 8, 128, 8192, 2048),
    (2, 1, 8, 8, 128, 4096, 1024), (1, 1, 16, 8, 128, 8192, 512), (2, 1, 32, 32, 64, 2048, 2048), (4, 2, 32, 8, 128, 512, 4096),
    (1, 1, 64, 8, 128, 4096, 1024), (24, 5, 32, 8, 64, 512, 2048), (64, 1, 16, 8, 128, 256, 1024),
])
def test_not_slower_than_unified_with_long_own_keys(R, ql, H, KVH, D, prefix, own):
    """Own keys run in kernels that are slower than the unified attention's decode kernels, and behind more launches: where they are
    many, the call takes the unified kernels (the rule that looked at the prefix alone took up to 2.4 times as long)."""
    shared, each = prefix // PAGE, own // PAGE
    bt = torch.empty(R, shared + each, dtype=torch.int32, device="cuda")
    bt[:, :shared] = torch.arange(shared).int()
    bt[:, shared:] = shared + torch.arange(R * each).int().view(R, each)
    kv = torch.randn(shared + R * each, 2, PAGE, KVH, D, device="cuda").to(BF)
    q = torch.randn(R * ql, H, D, device="cuda").to(BF)
    qsl = (torch.arange(R + 1, device="cuda") * ql).int()
    sl = torch.full((R,), prefix + own, dtype=torch.int32, device="cuda")
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    new = _time(lambda: A.shared_prefix_attention_fxp(q, kv, a, qsl, sl, bt, prefix, ql, max_seq_len=prefix + own))
    old = _time(lambda: A.unified_attention_fxp(q, kv, b, qsl, sl, bt, ql, frac_bits=16, max_seq_len=prefix + own))
    assert bits_equal(a, b)
    assert new < 1.2 * old, (new, old)  # calls of 30 us differ by up to that with where their scratch lies
