"""Attention behind a shared prefix where products leave the range of the fast
rounding: the bits of the unified attention, and no longer than it takes."""

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm.fixed_point_kernels import attention as A
from tests.helpers import bits_equal

BF, HF = torch.bfloat16, torch.float16
PAGE, PREFIX = 16, 448


def _batch(D, dtype, H=8, KVH=4, qlens=(3, 1, 6, 1, 2), prefix=PREFIX, own=9, seed=0):
    """Requests of own + queries keys each behind the prefix; groups of two, so that the prefix kernels run."""
    g = torch.Generator().manual_seed(seed)
    R, shared = len(qlens), prefix // PAGE
    cols = shared + (own + max(qlens) + PAGE - 1) // PAGE
    bt = torch.empty(R, cols, dtype=torch.int32)
    bt[:, :shared] = torch.arange(shared).int()
    bt[:, shared:] = shared + torch.arange(R * (cols - shared)).int().view(R, -1)
    kv = torch.randn(shared + R * (cols - shared), 2, PAGE, KVH, D, generator=g).to(dtype)
    q = (torch.randn(sum(qlens), H, D, generator=g) * 1.5).to(dtype)
    qsl = torch.tensor([sum(qlens[:i]) for i in range(R + 1)], dtype=torch.int32)
    sl = torch.tensor([prefix + own + n for n in qlens], dtype=torch.int32)
    return [x.cuda() for x in (q, kv, qsl, sl, bt)]


def _both(batch, bits, frac, prefix=PREFIX, **kw):
    q, kv, qsl, sl, bt = batch
    mq = int((qsl[1:] - qsl[:-1]).max())
    a, b = (torch.full(q.shape, 7.0, device="cuda") for _ in range(2))
    args = dict(fxp_dtype=bits, frac_bits=frac, max_seq_len=int(sl.max()), **kw)
    A.shared_prefix_attention_fxp(q, kv, a, qsl, sl, bt, prefix, mq, **args)
    A.unified_attention_fxp(q, kv, b, qsl, sl, bt, mq, **args)
    return a, b


CHANGES = {
    "channel of K": lambda q, kv: kv[:, 0, :, :, 5].mul_(25),
    "two channels of K, one far": lambda q, kv: (kv[:, 0, :, :, 3].mul_(25), kv[:, 0, :, :, 50].mul_(900)),
    "some keys": lambda q, kv: kv[3, 0, 2:5].mul_(400),
    "one request's queries": lambda q, kv: q[4:10].mul_(40),
    "a channel of q and of K": lambda q, kv: (q[:, :, 17].mul_(30), kv[:, 0, :, :, 17].mul_(100)),
    "channel of V": lambda q, kv: kv[:, 1, :, :, 7].mul_(80),
    "all of V": lambda q, kv: kv[:, 1].mul_(3000),
    "some of V": lambda q, kv: kv[9, 1, 3:8].mul_(6000),
    "everything": lambda q, kv: (q.mul_(60), kv.mul_(60)),
    "infinities and NaN in K": lambda q, kv: (kv[2, 0, 3, 0, 5].fill_(float("inf")), kv[5, 0, 1, 1, 9].fill_(float("nan")),
                                              kv[8, 0, 4, 2, 40].fill_(float("-inf"))),
    "infinities and NaN in q": lambda q, kv: (q[1, 0, 3].fill_(float("inf")), q[5, 3, 60].fill_(float("nan"))),
    "zeros in K beside infinities in q": lambda q, kv: (q[1, 0, 3].fill_(float("inf")), kv[:, 0, :, :, :16].zero_()),
}


@pytest.mark.gpu
@pytest.mark.parametrize("frac", [0, 16, 19, 23, 30])
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("D, dtype", [(64, BF), (64, HF), (128, BF), (128, HF)])
def test_bits(D, dtype, bits, frac):
    for name, change in CHANGES.items():
        batch = _batch(D, dtype, seed=D + frac)
        change(batch[0], batch[1])
        a, b = _both(batch, bits, frac)
        assert bits_equal(a, b), name


@pytest.mark.gpu
@pytest.mark.parametrize("frac", [32, 40, 50, 63])
def test_bits_of_fine_grids(frac):
    """64-bit accumulators with grids finer than 32 bits hold, up to the one on which 1 itself saturates."""
    for D, dtype in ((64, HF), (128, BF)):
        for name in ("channel of K", "channel of V", "everything", "some of V"):
            batch = _batch(D, dtype, seed=D + frac)
            CHANGES[name](batch[0], batch[1])
            a, b = _both(batch, 64, frac)
            assert bits_equal(a, b), name


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("D", [64, 128])
def test_bits_at_the_borders(D, bits):
    """Products whose largest lies just below, at and just above each range's end (2^22, 2^31 and 2^42 grid steps), halves between two
    grid steps of either sign among them; and queries whose scaling by 2^f leaves the fp32 range."""
    for top in (22, 31, 42):
        for eps in (-2.0**-7, 0.0, 2.0**-7):
            for dtype in (BF, HF):
                frac = 16 if top < 42 else 30
                batch = _batch(D, dtype, seed=top)
                q, kv = batch[0], batch[1]
                want = 2.0 ** (top - frac) * (1 + eps)  # max|q| * max|k|
                side = 2.0 ** ((top - frac) // 2)
                q.clamp_(-1.5, 1.5)
                kv[:, 0].clamp_(-1.5, 1.5)
                q[0, 0, 2], q[3, 5, 40] = side, -side
                kv[1, 0, 0, 0, 2] = kv[1, 0, 1, 0, 2] = kv[7, 0, 9, 2, 40] = want / side
                q[:, :, 8], kv[:, 0, :, :, 8] = 0.5, 2.0**-frac * torch.randint(-9, 10, kv[:, 0, :, :, 8].shape, device="cuda").to(dtype)
                kv[:, 1].clamp_(-1.5, 1.5)
                kv[4, 1, 2, 1, 3] = min(2.0 ** (top - frac) * (1 + eps), 60000.0)
                a, b = _both(batch, bits, frac, softmax_scale=2.0**-8)
                assert bits_equal(a, b), (top, eps, dtype)
    batch = _batch(D, BF, seed=1)
    q, kv = batch[0], batch[1]
    q[2, 1, 4], q[9, 6, 33] = 2.0**115, -2.0**120
    kv[:, 0, :, :, 4] *= 2.0**-110
    kv[:, 0, :, :, 33] = 0
    a, b = _both(batch, bits, 16)
    assert bits_equal(a, b)


def _time(run):
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
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


@pytest.mark.gpu
@pytest.mark.parametrize("frac", [16, 20, 24])
@pytest.mark.parametrize("change", ["channel of K", "one request's queries", "channel of V"])
def test_large_values_are_not_slower_than_unified(change, frac):
    """Outliers, and grids too fine for the fast rounding, where the prefix kernels run: at most the unified attention's time (the
    kernels that redid such tiles one product at a time took three to eight times as long)."""
    for H, KVH, qlens, prefix in ((64, 8, (1,) * 16, 2048), (32, 8, (1,) * 64, 4096)):
        batch = _batch(128, BF, H, KVH, qlens, prefix=prefix)
        CHANGES[change](batch[0], batch[1])
        q, kv, qsl, sl, bt = batch
        o, args = torch.zeros_like(q), dict(frac_bits=frac, max_seq_len=int(sl.max()))
        new = _time(lambda: A.shared_prefix_attention_fxp(q, kv, o, qsl, sl, bt, prefix, 1, **args))
        old = _time(lambda: A.unified_attention_fxp(q, kv, o, qsl, sl, bt, 1, **args))
        assert new < 1.2 * old, (H, new, old)
