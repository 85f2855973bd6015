"""Verification of drafted tokens: refusals (no GPU), and on the GPU the exact
tokens of the definition, restated below in Python integers."""

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm import _native as N
from fxpr_vllm.fixed_point_kernels import verify as V


def _grid(x, frac):
    x = x.double()
    x = torch.where(x.isnan(), torch.zeros_like(x), x.clamp(0, 1))
    return [int(v) for v in (x * 2.0**frac).round().long().tolist()]


def _definition(p, q, ids, start, bonus, u, r, most, frac):
    """Tokens and counts by Python integers, one request at a time (all CPU tensors)."""
    n, vocab = p.shape
    out, taken = [], []
    bits = lambda x: 0 if x != x else min(max(int(float(x) * 2**24), 0), 2**24 - 1)  # noqa: E731
    for k in range(len(start) - 1):
        a, length = int(start[k]), min(int(start[k + 1]) - int(start[k]), most)
        toks, final = [], int(bonus[k])
        for i in range(a, a + length):
            final = -1
            if not 0 <= i < n:
                break
            x = int(ids[i])
            P = _grid(p[i], frac)
            Q = _grid(q[i], frac) if q is not None else [2**frac if v == x else 0 for v in range(vocab)]
            if 0 <= x < vocab and bits(u[i]) * Q[x] < P[x] << 24:
                toks.append(x)
                final = int(bonus[k])
                continue
            left = [max(c - d, 0) for c, d in zip(P, Q)]
            if sum(left) == 0:
                left = P
            goal, run = sum(left) * bits(r[k]) >> 24, 0
            for v, c in enumerate(left):
                run += c
                if run > goal:
                    final = v
                    break
            break
        out.append((toks + [final] + [-1] * most)[:most + 1])
        taken.append(len(toks))
    return torch.tensor(out, dtype=torch.int32).view(-1, most + 1), torch.tensor(taken, dtype=torch.int32)


def _batch(lens, vocab, dtype=torch.float32, with_q=True, seed=0, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    x = torch.randn(n, vocab, generator=g) * sharp
    p = torch.softmax(x, -1).to(dtype)
    q = torch.softmax(x + torch.randn(n, vocab, generator=g), -1).to(dtype) if with_q else None
    src = q if with_q else p
    ids = torch.multinomial(src.float() + 1e-9, 1, generator=g)[:, 0].int() if n else torch.empty(0, dtype=torch.int32)
    start = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    bonus = torch.randint(0, vocab, (len(lens),), generator=g).int()
    return p, q, ids, start, bonus, torch.rand(n, generator=g), torch.rand(len(lens), generator=g)


def _both(args, most, frac=30):
    got = torch.ops.fxpr.verify_draft_fxp(*(None if a is None else a.cuda() for a in args), most, frac)
    want = _definition(*args, most, frac)
    assert got[0].dtype == got[1].dtype == torch.int32
    assert torch.equal(got[1].cpu(), want[1]), (got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0]), (got[0].cpu() != want[0]).nonzero()
    return want


# ------------------------------------------------------------------- refusals
@pytest.mark.parametrize("change, text", [
    (dict(target_probs=torch.zeros(5, 9, dtype=torch.float64)), "target_probs"),
    (dict(target_probs=torch.zeros(5)), "target_probs"),
    (dict(draft_probs=torch.zeros(5, 8)), "draft_probs"),
    (dict(draft_probs=torch.zeros(5, 9, dtype=torch.float16)), "draft_probs"),
    (dict(draft_token_ids=torch.zeros(4, dtype=torch.int32)), "draft_token_ids"),
    (dict(draft_token_ids=torch.zeros(5)), "draft_token_ids"),
    (dict(draft_start_loc=torch.zeros(0, dtype=torch.int32)), "draft_start_loc"),
    (dict(draft_start_loc=torch.zeros(3)), "draft_start_loc"),
    (dict(bonus_token_ids=torch.zeros(3, dtype=torch.int32)), "bonus_token_ids"),
    (dict(accept_uniform=torch.zeros(5, dtype=torch.float64)), "accept_uniform"),
    (dict(accept_uniform=torch.zeros(4)), "accept_uniform"),
    (dict(resample_uniform=torch.zeros(3)), "resample_uniform"),
    (dict(max_draft_len=33), "max_draft_len"), (dict(max_draft_len=-1), "max_draft_len"),
    (dict(frac_bits=31), "frac_bits"), (dict(frac_bits=0), "frac_bits"),
    (dict(target_probs=torch.zeros(5, 0), draft_probs=None), "vocabulary"),
])
def test_refuses(change, text):
    i32 = torch.int32
    kw = dict(target_probs=torch.zeros(5, 9), draft_probs=torch.zeros(5, 9), draft_token_ids=torch.zeros(5, dtype=i32),
              draft_start_loc=torch.tensor([0, 2, 5], dtype=i32), bonus_token_ids=torch.zeros(2, dtype=i32),
              accept_uniform=torch.zeros(5), resample_uniform=torch.zeros(2), max_draft_len=3, frac_bits=30)
    with pytest.raises(ValueError, match=text):
        V.verify_draft_fxp(**{**kw, **change})
    with pytest.raises(RuntimeError, match="CUDA"):
        V.verify_draft_fxp(**kw)


def test_abi_refuses_before_launch():
    lib = N.load()

    def call(dtype=N.F32, n=5, vocab=9, reqs=2, most=3, frac=30, ptr=None):
        return lib.fxpr_verify_draft_fxp(ptr, None, dtype, 9, 9, n, vocab, ptr, 0, ptr, ptr, 0, ptr, ptr, reqs, most,
                                         frac, ptr, 4, ptr, None)

    for kw, text in [(dict(dtype=N.F64), "float16"), (dict(frac=31), "frac_bits"), (dict(most=33), "max_draft_len"),
                     (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 24) + 1), "vocabulary"), (dict(), "null")]:
        assert call(**kw) == N.FXPR_ERR_INVALID
        assert text in lib.fxpr_last_error().decode()
    assert call(reqs=0) == N.FXPR_OK


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    dev = "cuda" if torch.cuda.is_available() else "cpu"
    with FakeTensorMode():
        p, i = torch.empty(5, 9, device=dev), torch.empty(5, dtype=torch.int32, device=dev)
        t, n = torch.ops.fxpr.verify_draft_fxp(p, None, i, torch.empty(3, dtype=torch.int32, device=dev), i[:2], p[:, 0],
                                               p[:2, 0], 4, 30)
        assert t.shape == (2, 5) and n.shape == (2,) and t.dtype == torch.int32


# ------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 128, 1000, 4096, 20011, 33000])
def test_definition(vocab, dtype, with_q):
    lens = [3, 0, 1, 5, 2, 4, 0, 1]
    for seed, frac in enumerate((30, 24, 12)):
        _both(_batch(lens, vocab, dtype, with_q, seed), 5, frac)


@pytest.mark.gpu
@pytest.mark.parametrize("reqs", [1, 2, 40, 700])
def test_batches(reqs):
    lens = [(7 * r + 3) % 5 for r in range(reqs)]
    out, taken = _both(_batch(lens, 517, seed=reqs), 4)
    if reqs == 700:
        assert (taken == torch.tensor(lens)).any() and (taken < torch.tensor(lens)).any()


@pytest.mark.gpu
def test_most_drafts_and_none():
    _both(_batch([32, 31, 0], 64, seed=1, sharp=0.1), 32)
    _both(_batch([0, 0], 64), 3)
    _both(_batch([0, 0], 64), 0)
    _both(_batch([4, 6], 64, seed=2, sharp=0.1), 2)  # longer than max_draft_len: only that many are looked at
    e = V.verify_draft_fxp(torch.zeros(0, 7, device="cuda"), None, *(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (0, 1, 0)),
                           torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"), 3)
    assert e[0].shape == (0, 4) and e[1].shape == (0,)


@pytest.mark.gpu
def test_edges():
    """One-hot rows (greedy), equal distributions (nothing remains), rows of zeros, NaN, inf and negative entries, draws of 0 and of
    the largest number below 1, ids outside the vocabulary."""
    p, q, ids, start, bonus, u, r = _batch([2] * 10, 300, seed=3)
    p[0] = p[1] = 0
    p[0, 7] = p[1, 299] = 1.0
    ids[0], ids[1] = 7, 5                 # greedy: taken, then replaced by 299
    q[2] = p[2]
    u[2] = 0.999                          # equal: taken
    q[4, int(ids[4])], p[4] = 1.0, 0.0    # refused, the target is empty
    p[6] = q[6] * 0.5
    u[6] = 0.9                            # refused and nothing remains: drawn from p itself
    p[8, :50], p[8, 50], q[8, 3] = float("nan"), float("inf"), float("-inf")
    p[10, 1], ids[10] = -3.0, 1
    ids[12], ids[14] = -1, 300
    u[16], r[8], u[18], r[9] = 0.0, 0.0, 1 - 2.0**-24, 1 - 2.0**-24
    out, taken = _both((p, q, ids, start, bonus, u, r), 2)
    assert out[0].tolist() == [7, 299, -1] and out[2, 0] == -1
    _both((p, None, ids, start, bonus, u, r), 2)
    u[:], r[:] = 1.5, -0.25               # outside [0, 1): clamped
    u[3] = r[3] = float("nan")
    _both((p, q, ids, start, bonus, u, r), 2)


@pytest.mark.gpu
def test_bad_start_loc_reads_nothing_outside():
    p, q, ids, start, bonus, u, r = _batch([2, 2, 2], 40, seed=4)
    for bad in ([0, 2, 9, 5], [-3, 2, 4, 6], [5, 7, 1 << 30, 0], [6, 6, 8, 8]):
        _both((p, q, ids, torch.tensor(bad, dtype=torch.int32), bonus, u, r), 2)


@pytest.mark.gpu
def test_strides_types_stream_and_graph():
    p, q, ids, start, bonus, u, r = (x.cuda() for x in _batch([4] * 9, 1001, seed=5))
    want = V.verify_draft_fxp(p, q, ids, start, bonus, u, r, 4)
    wide = torch.full((36, 2048), float("nan"), device="cuda")
    wide[:, 5:1006] = p
    two = torch.stack([q.t().contiguous()] * 2)  # vocabulary-major
    got = V.verify_draft_fxp(wide[:, 5:1006], two[1].t(), ids.long(), start.long(), bonus.long(), u, r, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = V.verify_draft_fxp(p, q, ids, start, bonus, u, r, 4)
    side.synchronize()
    assert torch.equal(got[0], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = V.verify_draft_fxp(p, q, ids, start, bonus, u, r, 4)
    u.copy_(torch.rand_like(u))
    r.copy_(torch.rand_like(r))
    graph.replay()
    want = V.verify_draft_fxp(p, q, ids, start, bonus, u, r, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_off_the_boundary(dtype):
    """Rows that start anywhere, alike in both tensors and not, next to values that must not be read as entries."""
    args = _batch([3] * 6, 1111, dtype, seed=6)
    want = _definition(*args, 3, 30)
    n = args[0].shape[0]
    for a, b, wa, wb in ((1, 1, 1117, 1117), (3, 3, 1120, 1128), (2, 5, 1117, 1117), (7, 7, 1120, 1121)):
        p, q = (torch.full((n, w), 1.0, dtype=dtype, device="cuda") for w in (wa, wb))
        pv, qv = p[:, a:a + 1111], q[:, b:b + 1111]
        pv.copy_(args[0])
        qv.copy_(args[1])
        got = V.verify_draft_fxp(pv, qv, *(x.cuda() for x in args[2:]), 3)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.gpu
def test_large_vocabulary():
    """2^18 + 3 entries and a flat distribution: the running sum passes 32 bits."""
    v = (1 << 18) + 3
    p = torch.full((2, v), 1.0)
    ids, start = torch.tensor([5, 9], dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    u, r = torch.tensor([0.5, 0.5]), torch.tensor([0.75, 1 - 2.0**-24])
    q = torch.zeros(2, v)
    p[:, 5] = p[:, 9] = 0.0
    want = _definition(p, q, ids, start, torch.zeros(2).int(), u, r, 1, 30)
    got = V.verify_draft_fxp(*(x.cuda() for x in (p, q, ids, start, torch.zeros(2).int(), u, r)), 1)
    assert torch.equal(got[0].cpu(), want[0])
