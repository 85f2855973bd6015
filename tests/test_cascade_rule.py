"""One rule for which shared-prefix calls run the prefix kernels: the operator
follows it, and the attention backend asks for cascade attention by it."""

import itertools

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm.fixed_point_kernels import attention as A
from tests.helpers import bits_equal

BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32


def _builder(head_dim=128, q_dtype=BF, kv_dtype=BF, page=16, cap=0.0):
    from fxpr_vllm.vllm_modules.attention_backend import DeterministicAttentionBackend

    cls = DeterministicAttentionBackend.get_builder_cls()
    b = cls.__new__(cls)
    b.headdim, b.block_size, b.q_dtype, b.kv_dtype, b.logits_soft_cap = head_dim, page, q_dtype, kv_dtype, cap
    return b


def _ask(b, prefix, lens, heads=32, kv_heads=8, alibi=False, window=False):
    return b.use_cascade_attention(prefix, lens, heads, kv_heads, alibi, window, False, 148, 1)


def test_no_cascade_where_the_operator_has_no_prefix_kernels():
    for kw in (dict(head_dim=32), dict(head_dim=256), dict(q_dtype=F4, kv_dtype=F4), dict(kv_dtype=F4), dict(q_dtype=F4)):
        assert not _ask(_builder(**kw), 4096, [5, 1, 3]) and not _ask(_builder(**kw), 8192, [1] * 64)
    assert _ask(_builder(), 4096, [5, 1, 3]) and _ask(_builder(head_dim=64, q_dtype=HF, kv_dtype=HF), 4096, [5, 1, 3])


def test_cascade_from_256_keys_where_the_decode_kernels_do_not_run():
    """Groups of four with one query a request: only a window, ALiBi, a softcap or an odd page size keeps the decode kernels out."""
    assert not _ask(_builder(), 512, [1] * 8)
    assert _ask(_builder(), 512, [1] * 8, window=True) and _ask(_builder(), 512, [1] * 8, alibi=True)
    assert _ask(_builder(cap=30.0), 512, [1] * 8) and _ask(_builder(page=24), 512, [1] * 8)
    assert not _ask(_builder(), 240, [1] * 8, window=True)


def test_backend_and_operator_agree():
    grid = itertools.product((32, 64, 128, 256), (BF, F4), ((8, 8), (32, 8), (64, 8), (7, 1)), (16, 24), (255, 256, 1000, 4096),
                             ([1, 1], [1] * 48, [5, 1, 3], [300, 2]), (False, True))
    seen = set()
    for D, dtype, (H, KVH), page, prefix, lens, window in grid:
        got = _ask(_builder(D, dtype, dtype, page), prefix, lens, H, KVH, window=window)
        want = A.shared_prefix_takes_prefix_kernels(prefix, len(lens), sum(lens), max(lens), prefix + max(lens), H, KVH, D, page,
                                                    dtype=dtype, window_size=100 if window else 0)
        assert got == want
        seen.add(got)
    assert seen == {False, True}


def test_own_keys_and_grids_in_the_rule():
    takes = lambda prefix, R, own, H=32, KVH=8, D=128, ql=1, **kw: A.shared_prefix_takes_prefix_kernels(  # noqa: E731
        prefix, R, R * ql, ql, prefix + own, H, KVH, D, 16, **kw)
    assert takes(4096, 64, 256) and not takes(4096, 64, 2048) and not takes(1024, 64, 256)
    assert takes(4096, 64, 64, frac_bits=28) and not takes(4096, 64, 64, frac_bits=30)
    assert takes(4096, 64, 64, frac_bits=38, fxp_dtype=64) and not takes(4096, 64, 64, frac_bits=40, fxp_dtype=64)
    assert takes(1024, 16, 64, H=8) and takes(1024, 64, 8192, H=8) and not takes(1024, 2, 1024, H=8)
    assert not takes(192, 64, 16, H=8) and not takes(4096, 64, 64, fxp_dtype=16)


# requests, queries of each, query heads, KV heads, head_dim, shared keys, own keys, type
SHAPES = [(40, 1, 8, 4, 64, 512, 1100, BF), (40, 1, 8, 4, 128, 1000, 1600, HF), (64, 1, 32, 8, 128, 4096, 500, BF), (12, 5, 8, 1, 128, 512, 700, BF),
          (8, 1, 32, 8, 128, 512, 64, BF), (2, 1, 8, 8, 128, 2048, 1500, BF), (6, 3, 12, 4, 64, 320, 9, HF), (5, 1, 64, 8, 64, 256, 30, BF),
          (33, 1, 40, 2, 64, 300, 520, BF), (3, 70, 6, 2, 128, 700, 100, HF)]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("R, ql, H, KVH, D, prefix, most, dtype", SHAPES)
def test_the_operator_follows_the_rule(R, ql, H, KVH, D, prefix, most, dtype, bits):
    """The kernels that a call launches, by its profile; own keys over one to several chunks, with the unified attention's bits."""
    g = torch.Generator().manual_seed(R + D)
    own = [ql + (37 * r + most) % (most - ql + 1) for r in range(R)]
    own[0] = most
    shared, cols = prefix // 16, -(-(prefix + most) // 16)
    bt = torch.empty(R, cols, dtype=torch.int32)
    bt[:, :shared] = torch.arange(shared).int()
    bt[:, shared:] = shared + torch.arange(R * (cols - shared)).int().view(R, -1)
    kv = torch.randn(shared + R * (cols - shared), 2, 16, KVH, D, generator=g).to(dtype)
    if prefix % 16:
        kv[bt[1:, shared].long(), :, :prefix % 16] = kv[bt[0, shared].long(), :, :prefix % 16]
    q = (torch.randn(R * ql, H, D, generator=g) * 1.5).to(dtype).cuda()
    kv, bt = kv.cuda(), bt.cuda()
    qsl = (torch.arange(R + 1) * ql).int().cuda()
    sl = torch.tensor([prefix + n for n in own], dtype=torch.int32).cuda()
    a, b = torch.zeros(q.shape, device="cuda"), torch.zeros(q.shape, device="cuda")
    args = dict(fxp_dtype=bits, max_seq_len=prefix + most)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        A.shared_prefix_attention_fxp(q, kv, a, qsl, sl, bt, prefix, ql, **args)
        torch.cuda.synchronize()
    names = " ".join(e.name for e in prof.events())
    takes = A.shared_prefix_takes_prefix_kernels(prefix, R, R * ql, ql, prefix + most, H, KVH, D, 16, dtype=dtype, fxp_dtype=bits)
    assert ("prefix_scores_kernel" in names) == takes, names
    A.unified_attention_fxp(q, kv, b, qsl, sl, bt, ql, frac_bits=16, **args)
    assert bits_equal(a, b)


def test_the_shapes_cover_both():
    took = [A.shared_prefix_takes_prefix_kernels(p, R, R * ql, ql, p + most, H, KVH, D, 16, dtype=t) for R, ql, H, KVH, D, p, most, t in SHAPES]
    assert took.count(True) >= 6 and took.count(False) >= 2
    assert any(t and s[6] > 1024 for t, s in zip(took, SHAPES)), "own keys over three chunks behind the prefix kernels"
