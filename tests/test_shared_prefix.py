"""Attention behind a shared prefix: refusals (no GPU); on the GPU the bits of
the unified attention over shapes, masks and magnitudes, and the definition in
64 bits."""

import ctypes
import math

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm import _native as N
from fxpr_vllm.fixed_point_kernels import attention as A
from tests.helpers import bits_equal

BF, HF = torch.bfloat16, torch.float16
LOG2E = 1.4426950408889634


def _batch(qlens, suffix, prefix, H, KVH, D, page=16, dtype=BF, seed=0, pad=0):
    """Requests of qlens[r] queries, the last of prefix + suffix[r] keys, on shared pages (a last, partly shared page is copied)."""
    g = torch.Generator().manual_seed(seed)
    R, total = len(qlens), [prefix + s for s in suffix]
    shared, cols = prefix // page, max(1, max((t + page - 1) // page for t in total))
    cols = max(cols, prefix // page)
    nblk = shared + R * (cols - shared) + 2
    perm = torch.randperm(nblk, generator=g).int()
    bt = torch.empty(R, cols, dtype=torch.int32)
    bt[:, :shared] = perm[:shared]
    bt[:, shared:] = perm[shared:shared + R * (cols - shared)].view(R, cols - shared)
    kv = torch.randn(nblk, 2, page, KVH, D, generator=g).to(dtype)
    if prefix % page and cols > shared:
        kv[bt[1:, shared].long(), :, :prefix % page] = kv[bt[0, shared].long(), :, :prefix % page]
    T = sum(qlens)
    q = (torch.randn(T + pad, H, D, generator=g) * 1.5).to(dtype)
    qsl = torch.tensor([sum(qlens[:i]) for i in range(R + 1)], dtype=torch.int32)
    return [x.cuda() for x in (q, kv, qsl, torch.tensor(total, dtype=torch.int32), bt)], max(qlens), max(total)


def _pair(batch, prefix, o_dtype=torch.float32, bits=32, **kw):
    (q, kv, qsl, sl, bt), mq, ms = batch
    a = torch.full(q.shape, 7.0, dtype=o_dtype, device="cuda")
    b = a.clone()
    A.shared_prefix_attention_fxp(q, kv, a, qsl, sl, bt, prefix, mq, fxp_dtype=bits, max_seq_len=ms, **kw)
    A.unified_attention_fxp(q, kv, b, qsl, sl, bt, mq, fxp_dtype=bits, max_seq_len=ms, **{"frac_bits": 16, **kw})
    return a, b


def _same(batch, prefix, **kw):
    a, b = _pair(batch, prefix, **kw)
    assert bits_equal(a, b), (a - b).abs().max()
    return a


# ------------------------------------------------------------------- refusals
@pytest.mark.parametrize("change, text", [
    (dict(q=torch.zeros(4, 256)), "tokens, heads"),
    (dict(o=torch.zeros(4, 4, 32)), "q and o"),
    (dict(kv_cache=torch.zeros(9, 2, 16, 2, 32)), "kv_cache"),
    (dict(kv_cache=torch.zeros(9, 16, 2, 64)), "kv_cache"),
    (dict(kv_cache=torch.zeros(9, 2, 16, 3, 64)), "group"),
    (dict(query_start_loc=torch.zeros(2, dtype=torch.int32)), "query_start_loc"),
    (dict(block_table=torch.zeros(1, 4, dtype=torch.int32)), "block-table"),
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), "dimensions"),
    (dict(common_prefix_len=-1), "common_prefix_len"), (dict(common_prefix_len=65), "common_prefix_len"),
    (dict(q=torch.zeros(4, 64, 4).transpose(1, 2)), "contiguous"),
    (dict(alibi_slopes=torch.zeros(3)), "alibi"),
])
def test_refuses(change, text):
    kw = dict(q=torch.zeros(4, 4, 64), kv_cache=torch.zeros(9, 2, 16, 2, 64), o=torch.zeros(4, 4, 64),
              query_start_loc=torch.zeros(3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32),
              block_table=torch.zeros(2, 4, dtype=torch.int32), common_prefix_len=32, max_query_len=2)
    with pytest.raises(ValueError, match=text):
        A.shared_prefix_attention_fxp(**{**kw, **change})
    with pytest.raises(RuntimeError, match="CUDA"):
        A.shared_prefix_attention_fxp(**kw)


def test_abi_refuses_and_sizes_its_workspace():
    lib = N.load()
    p = N.AttentionParams()
    p.num_requests, p.max_query_len, p.num_heads, p.num_kv_heads = 64, 1, 32, 8
    p.head_dim, p.page_size, p.max_seq_len, p.int_bits, p.frac_bits = 128, 16, 8192, 32, 16
    p.block_table_cols, p.num_blocks = 512, 1000
    p.q_dtype = p.kv_dtype = p.o_dtype = N.BF16
    size = lambda n=4096, t=64: lib.fxpr_shared_prefix_attention_workspace_bytes(ctypes.byref(p), n, t)  # noqa: E731
    assert size() >= 64 * 32 * 4096 * 4  # the prefix's scores
    assert size(0) == lib.fxpr_attention_workspace_bytes(ctypes.byref(p))  # no prefix: the unified attention's
    for field, value, code, text in [("frac_bits", 32, N.FXPR_ERR_INVALID, "frac_bits"), ("int_bits", 16, N.FXPR_ERR_UNSUPPORTED, "int16"),
                                     ("head_dim", 100, N.FXPR_ERR_UNSUPPORTED, "head_dim")]:
        old = getattr(p, field)
        setattr(p, field, value)
        assert lib.fxpr_shared_prefix_attention_fxp(ctypes.byref(p), 4096, 64, None) == code
        assert text in lib.fxpr_last_error().decode() and size() == 0
        setattr(p, field, old)
    for n in (-1, 512 * 16 + 1):
        assert lib.fxpr_shared_prefix_attention_fxp(ctypes.byref(p), n, 64, None) == N.FXPR_ERR_INVALID
        assert "common_prefix_len" in lib.fxpr_last_error().decode()
    p.workspace, p.workspace_bytes = 4096, 4096  # too small
    assert lib.fxpr_shared_prefix_attention_fxp(ctypes.byref(p), 4096, 64, None) == N.FXPR_ERR_INVALID
    assert "workspace" in lib.fxpr_last_error().decode()


# ------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qlens, suffix, prefix, H, KVH, page", [
    ([1] * 5, [1, 17, 200, 513, 1100], 256, 8, 4, 16),       # decode, own keys over several chunks
    ([1] * 9, [1] * 9, 256, 4, 4, 16),                       # no group, nothing but the query behind the prefix
    ([1] * 40, list(range(1, 41)), 1000, 16, 2, 16),         # ragged prefix (last page copied), several row tiles
    ([1] * 40, [3] * 40, 260, 12, 4, 16),                    # rows of a token on two tiles
    ([1] * 32, list(range(1, 33)), 4096, 16, 4, 16),         # groups of 4 with enough of a prefix
    ([1] * 6, list(range(1, 7)), 512, 8, 2, 16),             # and without: the unified decode kernels
    ([5, 1, 3, 9, 2], [5, 8, 3, 30, 2], 333, 8, 4, 8),       # verification, group of 2, small pages
    ([70, 1, 130], [70, 1, 200], 704, 7, 1, 48),             # chunked prefill, group of 7, pages across tiles
    ([1], [3], 500, 16, 2, 16),                              # one request
    ([1, 2, 1], [3, 900, 20], 397, 6, 2, 5),                 # pages of an odd number of keys
    ([2, 0, 3, 0], [2, 0, 9, 5], 290, 2, 2, 1),              # requests without queries, pages of one key
])
def test_bits_of_the_unified_attention(qlens, suffix, prefix, H, KVH, page, D, bits):
    for dtype in (BF, HF):
        b = _batch(qlens, suffix, prefix, H, KVH, D, page, dtype, seed=D + bits)
        _same(b, prefix, bits=bits)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(logits_soft_cap=20.0), dict(window_size=100), dict(window_size=3), dict(is_causal=False),
                                dict(window_size=400, logits_soft_cap=5.0), dict(softmax_scale=0.3), dict(alibi=True),
                                dict(alibi=True, window_size=300), dict(frac_bits=8), dict(frac_bits=20), dict(frac_bits=0),
                                dict(frac_bits=30)])
@pytest.mark.parametrize("qlens, suffix", [([1] * 12, [1 + 40 * (r % 3) for r in range(12)]), ([6, 1, 3], [60, 1, 3])])
def test_masks_and_scores(kw, qlens, suffix):
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = (2.0 ** -torch.arange(1.0, 9.0) * LOG2E).cuda()
    for D, bits in ((64, 32), (128, 64)):
        a = _same(_batch(qlens, suffix, 640, 8, 4, D, seed=3), 640, bits=bits, **kw)
        assert a.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
def test_values_beyond_the_fast_path(bits):
    """Tiles whose q, K or V the magic constant cannot round take the clamp-and-convert path, infinities and NaN in K too."""
    for scale_k, scale_v, scale_q in ((300.0, 1.0, 1.0), (1.0, 300.0, 1.0), (40.0, 90.0, 40.0)):
        b = _batch([1, 4, 1, 2], [9, 4, 100, 2], 320, 8, 2, 128, seed=5)
        q, kv, _, _, bt = b[0]
        q *= scale_q
        kv[bt[0, 3].long(), 0] *= scale_k
        kv[bt[0, 7].long(), 1] *= scale_v
        _same(b, 320, bits=bits)
    b = _batch([1, 4, 1, 2], [9, 4, 100, 2], 320, 8, 2, 64, dtype=HF, seed=6)
    q, kv, _, _, bt = b[0]
    kv[bt[0, 2].long(), 0, 3, 0, 5], kv[bt[0, 9].long(), 0, 1, 1, 9] = float("inf"), float("nan")
    kv[bt[0, 5].long(), 1, 3, 0, 5], kv[bt[0, 6].long(), 1, 1, 1, 9] = float("inf"), float("nan")
    a, u = _pair(b, 320, bits=bits)
    assert bits_equal(a, u)


@pytest.mark.gpu
def test_masked_places_do_not_count():
    """Infinities and NaN in V of keys that a window hides change nothing (nor in keys of a later query of the request)."""
    b = _batch([1, 2, 3], [1, 2, 70], 512, 8, 2, 128, seed=7)
    kv, bt = b[0][1], b[0][4]
    want = _same(b, 512, window_size=64)
    kv[bt[0, :25].long(), 1] = float("inf")
    kv[bt[0, 3].long(), 1] = float("nan")
    a, _ = _pair(b, 512, window_size=64)
    assert bits_equal(a, want)
    # the last query's own V, hidden from the ones before
    (q, _, qsl, sl, _) = b[0]
    j = int(sl[1]) - 1
    kv[bt[1, j // 16].long(), 1, j % 16] = float("inf")
    a, _ = _pair(b, 512, window_size=64)
    t = int(qsl[2]) - 1
    keep = [i for i in range(q.shape[0]) if i != t]
    assert bits_equal(a[keep], want[keep])


@pytest.mark.gpu
def test_short_and_padded_requests():
    """Requests shorter than the prefix, without keys or queries, and rows behind the last sequence."""
    (q, kv, qsl, sl, bt), mq, ms = _batch([1] * 20, [5] * 20, 256, 8, 4, 128, seed=8, pad=11)
    sl[3], sl[4], sl[5] = 100, 1, 64
    _same(((q, kv, qsl, sl, bt), mq, ms), 256)
    sl[6] = 0  # a request that sees nothing: 0, where the unified attention has no defined value
    a, b = _pair(((q, kv, qsl, sl, bt), mq, ms), 256)
    rows = [i for i in range(31) if i != 6]
    assert bits_equal(a[rows], b[rows]) and (a[6] == 0).all() and (a[20:] == 7.0).all()
    qsl[15:] = qsl[15].clone()  # the last five have no queries
    a, b = _pair(((q, kv, qsl, sl, bt), mq, ms), 256)
    assert bits_equal(a[:6], b[:6]) and (a[15:] == 7.0).all()


@pytest.mark.gpu
def test_definition_in_64_bits():
    """fp32 output against the formula in float64: scores differ by fp32 roundings of their 3 steps (2^-22 relative, |s| < 2^5), so p
    by less than 2^-16 relative; a rounded term p * v * 2^16 moves by |p v| at most that much more than its own rounding and
    otherwise by one grid step where it crosses a half, so |out - formula| < (2^-15 + 2^-16) * sum(p |v|) / den + 2^-16 * keys / den."""
    prefix = 448
    for D, dtype in ((64, HF), (128, BF)):
        b = _batch([3, 1, 1, 2], [30, 1, 77, 2], prefix, 8, 2, D, dtype=dtype, seed=9)
        got = _same(b, prefix).cpu().double()
        (q, kv, qsl, sl, bt), _, _ = b
        q, kv, qsl, sl, bt = (x.cpu() for x in (q, kv, qsl, sl, bt))
        for r in range(4):
            n = int(sl[r])
            k, v = (kv[bt[r].long(), i].flatten(0, 1)[:n].double() for i in (0, 1))
            for t in range(int(qsl[r]), int(qsl[r + 1])):
                vis = n - (int(qsl[r + 1]) - t - 1)
                for h in range(8):
                    kh, vh = k[:vis, h // 4], v[:vis, h // 4].half().double()
                    s = (q[t, h].double() * kh * 65536).round().sum(-1) / 65536 / math.sqrt(D) * LOG2E
                    p = torch.exp2(s - s.max())
                    den = (p * 65536).round().sum() / 65536
                    ref = (p[:, None] * vh * 65536).round().sum(0) / 65536 / den
                    lim = (2.0**-15 + 2.0**-16) * (p[:, None] * vh.abs()).sum(0) / den + 2.0**-16 * vis / den
                    assert ((got[t, h] - ref).abs() <= lim).all()


@pytest.mark.gpu
def test_strides_types_and_other_forms():
    """Query and output views, a split cache, 64-bit index tensors; head sizes and types that run the unified kernels."""
    (q, kv, qsl, sl, bt), mq, ms = _batch([1, 3, 1, 1], [4, 3, 60, 2], 384, 8, 2, 64, seed=10)
    want = _same(((q, kv, qsl, sl, bt), mq, ms), 384)
    wide = torch.zeros(6, 3, 8, 64, dtype=BF, device="cuda")
    wide[:, 1] = q
    out = torch.zeros(6, 8, 2, 64, device="cuda")
    store = kv.transpose(0, 1).contiguous().transpose(0, 1)
    tab = torch.zeros(4, 3 * bt.shape[1], dtype=torch.int64, device="cuda")
    tab[:, ::3] = bt
    A.shared_prefix_attention_fxp(wide[:, 1], store, out[:, :, 1], qsl.long(), sl.long(), tab[:, ::3], 384, mq)
    assert bits_equal(out[:, :, 1].contiguous(), want) and (out[:, :, 0] == 0).all()
    odd = torch.zeros(6, 8, 67, dtype=BF, device="cuda")
    odd[..., 1:65] = q
    _same(((odd[..., 1:65], kv, qsl, sl, bt), mq, ms), 384)
    for o_dtype in (BF, HF):
        a, b = _pair(((q, kv, qsl, sl, bt), mq, ms), 384, o_dtype=o_dtype)
        assert bits_equal(a, b)
    for D, dtype in ((32, BF), (256, BF), (64, torch.float32)):
        _same(_batch([1] * 6, [3] * 6, 256, 4, 2, D, dtype=dtype, seed=11), 256)
    mixed = _batch([1] * 6, [3] * 6, 256, 4, 2, 128, seed=12)
    mixed[0][0] = mixed[0][0].half()
    _same(mixed, 256)
    for prefix in (0, 1, 63, 300):
        _same(_batch([1] * 6, [3] * 6, prefix, 4, 2, 128, seed=13), prefix)


@pytest.mark.gpu
def test_block_ids_outside_the_cache_read_zeros():
    (q, kv, qsl, sl, bt), mq, ms = _batch([1] * 20, [5] * 20, 256, 8, 4, 128, seed=14)
    bad = bt.clone()
    bad[0, 3], bad[0, 7] = kv.shape[0], -5
    a = torch.zeros(q.shape, device="cuda")
    A.shared_prefix_attention_fxp(q, kv, a, qsl, sl, bad, 256, mq, max_seq_len=ms)
    zeroed = kv.clone()
    zeroed[bt[0, 3].long()] = 0
    zeroed[bt[0, 7].long()] = 0
    b = torch.zeros(q.shape, device="cuda")
    A.shared_prefix_attention_fxp(q, zeroed, b, qsl, sl, bt, 256, mq, max_seq_len=ms)
    assert bits_equal(a, b)


@pytest.mark.gpu
def test_batch_invariance_and_repeat():
    """A request's rows have the same bits alone, in any batch and in every repetition."""
    (q, kv, qsl, sl, bt), mq, ms = _batch([1] * 50, [7 * (r % 9) + 1 for r in range(50)], 2000, 32, 8, 128, seed=15)
    run = lambda i, n: A.shared_prefix_attention_fxp(  # noqa: E731
        q[i:i + n], kv, out[:n], qsl[:n + 1], sl[i:i + n], bt[i:i + n], 2000, 1, max_seq_len=ms)
    out = torch.zeros(50, 32, 128, device="cuda")
    run(0, 50)
    full = out.clone()
    for _ in range(3):
        run(0, 50)
        assert bits_equal(out, full)
    for i, n in ((0, 1), (17, 1), (13, 8), (30, 20)):
        out.zero_()
        run(i, n)
        assert bits_equal(out[:n], full[i:i + n])


@pytest.mark.gpu
def test_query_ranges_behind_the_queries():
    """A last request whose range ends behind the rows of q: its missing rows are skipped, the others keep their bits."""
    (q, kv, qsl, sl, bt), mq, ms = _batch([1] * 18 + [6], [5] * 18 + [9], 256, 8, 4, 128, seed=19)
    want = _same(((q, kv, qsl, sl, bt), mq, ms), 256)
    guard = torch.full((40, 8, 128), 7.0, device="cuda")
    A.shared_prefix_attention_fxp(q[:20], kv, guard[:20], qsl, sl, bt, 256, mq, max_seq_len=ms)
    assert bits_equal(guard[:20], want[:20]) and (guard[20:] == 7.0).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pages whose offsets in the cache pass 2^31 elements (a 4.7 GB cache of which a few pages are written)."""
    (q, kv, qsl, sl, bt), mq, ms = _batch([1] * 6, [9] * 6, 256, 16, 8, 128, seed=20)
    want = _same(((q, kv, qsl, sl, bt), mq, ms), 256)
    far = 2**31 // (2 * 16 * 8 * 128) + 1
    big = torch.empty(far + kv.shape[0] + 1, 2, 16, 8, 128, dtype=BF, device="cuda")
    big[far:far + kv.shape[0]] = kv
    out = torch.zeros(q.shape, device="cuda")
    A.shared_prefix_attention_fxp(q, big, out, qsl, sl, bt + far, 256, mq, max_seq_len=ms)
    assert bits_equal(out, want)


@pytest.mark.gpu
def test_many_rows_in_passes():
    """More row tiles than the scores' workspace holds (128 MB): the prefix runs in passes."""
    prefix = 2048
    b = _batch([96] * 24, [100] * 24, prefix, 8, 1, 64, seed=16)
    _same(b, prefix, o_dtype=BF)


@pytest.mark.gpu
def test_streams_and_two_captured_graphs():
    """Two captured graphs replayed at the same time on two streams, and an eager call beside them, share no scratch."""
    bs = [_batch([1] * 24, [9] * 24, 512, 8, 4, 128, seed=s) for s in (17, 18)]
    want = [_same(b, 512) for b in bs]
    outs, graphs = [torch.zeros_like(w) for w in want], []
    for b, o in zip(bs, outs):
        (q, kv, qsl, sl, bt), mq, ms = b
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            torch.ops.fxpr.shared_prefix_attention_fxp(q, kv, o, qsl, sl, bt, 512, mq, None, 32, True, None, 16, 0.0, 0, ms)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        _same(bs[0], 512)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert bits_equal(o, w)
