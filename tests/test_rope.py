"""Rotary position with the per-head fixed-point norm and with the paged-cache
append: refusals (no GPU), and on the GPU the kernels against the formulas in
64 bits, against the oracle's norm bit for bit, and the cache they write."""

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm import _native as N
from fxpr_vllm.fixed_point_kernels import rope as R
from oracle import fxp_oracle as O
from tests.helpers import bits_equal, device_prims

F = (torch.float16, torch.bfloat16, torch.float32)


def _inputs(T, Hq, Hk, D, rot, dtype, table=torch.float32, span=97, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, Hq + 2 * Hk, D, generator=g) * 2).to(dtype)
    w = (1 + 0.3 * torch.randn(2, D, generator=g)).to(dtype)
    ang = torch.arange(span, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))
    tab = torch.cat([ang.cos(), ang.sin()], -1).to(table)
    pos = torch.randint(0, span, (T,), generator=g)
    x, w, tab, pos = (t.to(device) for t in (x, w, tab, pos))
    return x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:], w[0], w[1], pos, tab


def _formula(x, w, pos, tab, neox, bits, eps=1e-6, frac=16):
    """Norm (w given) and rotation in float64, and a bound on the fp32 kernel's
    error before its last rounding."""
    x = x.double().cpu()
    D, rot = x.shape[-1], tab.shape[1]
    if w is not None:
        sq = (x.float() * x.float()).double()  # the squares are fp32 products in the definition
        top = {16: 32767.0, 32: 2.0**31 - 256, 64: 2.0**63 - 2.0**40}[bits]
        S = torch.minimum((sq * 2.0**frac).round(), torch.tensor(top, dtype=torch.float64)).sum(-1, keepdim=True)
        x = x * w.double().cpu() / torch.sqrt(S * 2.0**-frac / D + eps)
    cs = tab.double().cpu()[pos.cpu()][:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    ia = torch.arange(rot // 2) if neox else torch.arange(0, rot, 2)
    ib = ia + (rot // 2 if neox else 1)
    a, b = x[..., ia], x[..., ib]
    y = x.clone()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size = x.abs()
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    # three fp32 roundings (2^-24 each) in the rotation; in the norm two products, the sum's conversion, a division, a sum
    # and a square root and a division whose documented errors are at most 2 ulp (2^-22): in all below 2^-20 of |a| + |b|
    return y, size * 2.0**-20


def _assert_close(got, want, bound):
    """got is the value rounded once: half a step of its type on top of `bound`
    (fp16 also half of its smallest step, 2^-25, below its normal range)."""
    step = torch.finfo(got.dtype).eps / 2
    tiny = 2.0**-25 if got.dtype == torch.float16 else 0.0
    err = (got.double().cpu() - want).abs()
    lim = want.abs() * step + bound * (1 + step) + tiny
    assert torch.isfinite(got).all()
    assert (err <= lim).all(), (err - lim).max()


# ------------------------------------------------------------------- refusals
@pytest.mark.parametrize("change, text", [
    (dict(k=torch.zeros(4, 2, 32)), "head_dim"),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.float16)), "share a type"),
    (dict(q=torch.zeros(4, 128)), "tokens, heads, head_dim"),
    (dict(q=torch.zeros(3, 4, 64)), "tokens, heads, head_dim"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(positions=torch.zeros(4)), "positions"),
    (dict(cos_sin_cache=torch.zeros(9, 66)), "at most head_dim"),
    (dict(cos_sin_cache=torch.zeros(9, 33)), "even"),
    (dict(cos_sin_cache=torch.zeros(9, 64, dtype=torch.float64)), "cos_sin_cache"),
    (dict(q_weight=torch.ones(32)), "norm weights"),
    (dict(k_weight=None), "needed|both"),
    (dict(q_out=torch.zeros(4, 4, 32)), "q_out"),
])
def test_norm_rope_refuses(change, text):
    kw = dict(q=torch.zeros(4, 4, 64), k=torch.zeros(4, 2, 64), q_weight=torch.ones(64), k_weight=torch.ones(64),
              positions=torch.zeros(4, dtype=torch.int64), cos_sin_cache=torch.zeros(9, 64))
    with pytest.raises(ValueError, match=text):
        R.qk_norm_rope_fxp(**{**kw, **change})


@pytest.mark.parametrize("change, text", [
    (dict(v=torch.zeros(4, 4, 64)), "v must"),
    (dict(kv_cache=torch.zeros(3, 2, 16, 2, 32)), "kv_cache"),
    (dict(kv_cache=torch.zeros(3, 16, 2, 64)), "kv_cache"),
    (dict(kv_cache=torch.zeros(3, 2, 16, 2, 64, dtype=torch.int32)), "kv_cache"),
    (dict(kv_cache=torch.zeros(3, 2, 16, 64, 2).transpose(3, 4)), "contiguous"),
    (dict(slot_mapping=torch.zeros(5, dtype=torch.int64)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(4)), "slot_mapping"),
    (dict(q_weight=torch.ones(64)), "both"),
])
def test_append_refuses(change, text):
    kw = dict(q=torch.zeros(4, 4, 64), k=torch.zeros(4, 2, 64), v=torch.zeros(4, 2, 64),
              kv_cache=torch.zeros(3, 2, 16, 2, 64), slot_mapping=torch.arange(4),
              positions=torch.zeros(4, dtype=torch.int64), cos_sin_cache=torch.zeros(9, 64))
    with pytest.raises(ValueError, match=text):
        R.rope_append_kv_fxp(**{**kw, **change})


def test_cpu_tensors_refused():
    q, k, v, qw, kw, pos, tab = _inputs(4, 4, 2, 64, 64, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab)


def test_abi_refuses_before_launch():
    import ctypes

    lib = N.load()
    p = N.RopeParams()
    assert lib.fxpr_qk_norm_rope_fxp(None, None) == N.FXPR_ERR_INVALID
    p.dtype, p.table_dtype, p.weight_dtype = N.BF16, N.F32, N.BF16
    p.tokens, p.num_heads, p.num_kv_heads, p.head_dim = 1, 2, 1, 64
    for field, value, text in [("int_bits", 24, "16/32/64"), ("frac_bits", 32, "frac_bits"), ("head_dim", 1025, "head_dim"),
                               ("rot_dim", 3, "even"), ("rot_dim", 66, "even"), ("dtype", N.F64, "float16"),
                               ("q", None, "null")]:
        p.int_bits, p.frac_bits, p.rot_dim, p.head_dim, p.dtype = 32, 16, 64, 64, N.BF16
        p.q_weight = p.k_weight = p.k = p.k_out = p.q = p.q_out = p.positions = p.table = 4096
        setattr(p, field, value)
        assert lib.fxpr_qk_norm_rope_fxp(ctypes.byref(p), None) == N.FXPR_ERR_INVALID
        assert text in lib.fxpr_last_error().decode()


def test_fake_shapes():
    import fxpr_vllm.library_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    dev = "cuda" if torch.cuda.is_available() else "cpu"
    with FakeTensorMode():
        q, k, w = torch.empty(5, 4, 64, device=dev), torch.empty(5, 2, 64, device=dev), torch.empty(64, device=dev)
        pos, tab = torch.empty(5, dtype=torch.int64, device=dev), torch.empty(9, 64, device=dev)
        a, b = torch.ops.fxpr.qk_norm_rope_fxp(q, k, w, w, pos, tab, True, 1e-6, 16, 32)
        assert a.shape == q.shape and b.shape == k.shape
        kv = torch.empty(3, 2, 16, 2, 64, device=dev)
        o = torch.ops.fxpr.rope_append_kv_fxp(q, k, k, kv, pos, pos, tab, True, None, None, 1e-6, 16, 32)
        assert o.shape == q.shape


# ------------------------------------------------------------------ on the GPU
SHAPES = [  # T, Hq, Hk, D, rot: vector pieces full, ragged and partial; the general kernel from head_dim 40 on
    (1, 32, 8, 128, 128), (33, 4, 1, 64, 64), (7, 5, 5, 96, 48), (130, 8, 2, 128, 64), (3, 3, 1, 256, 256),
    (2, 2, 1, 512, 512), (5, 1, 1, 48, 16), (9, 2, 2, 40, 40), (4, 3, 1, 80, 24), (2, 1, 1, 7, 6), (3, 2, 1, 1, 0),
    (2, 1, 1, 1024, 1024), (300, 32, 8, 64, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 32, 64])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype", F)
def test_norm_rope_formula(dtype, neox, bits):
    frac = 8 if bits == 16 else 16
    for i, (T, Hq, Hk, D, rot) in enumerate(SHAPES):
        q, k, _, qw, kw, pos, tab = _inputs(T, Hq, Hk, D, rot, dtype, F[i % 3], seed=i, device="cuda")
        yq, yk = torch.ops.fxpr.qk_norm_rope_fxp(q, k, qw, kw, pos, tab, neox, 1e-6, frac, bits)
        for y, x, w in ((yq, q, qw), (yk, k, kw)):
            assert y.dtype == dtype and y.is_contiguous()
            _assert_close(y, *_formula(x, w, pos, tab, neox, bits, frac=frac))


@pytest.mark.gpu
def test_norm_is_the_rms_norm_operator():
    """With an angle of zero the norm remains: the bits of the oracle's fixed-point RMSNorm (vector and general kernel)."""
    prims = device_prims()
    for bits in (16, 32, 64):
        for D in (128, 40):
            q, k, _, qw, kw, pos, tab = _inputs(11, 4, 2, D, 8, torch.float32, seed=bits + D)
            tab[:, :4], tab[:, 4:] = 1.0, 0.0
            frac = 8 if bits == 16 else 16
            yq, yk = R.qk_norm_rope_fxp(q.cuda(), k.cuda(), qw.cuda(), kw.cuda(), pos.cuda(), tab.cuda(), True, 1e-6, frac, bits)
            for y, x, w in ((yq, q, qw), (yk, k, kw)):
                assert torch.equal(y.cpu(), O.rms_norm_fxp(x.contiguous(), w, 1e-6, frac, bits, prims=prims))


@pytest.mark.gpu
def test_norm_rope_strides_and_alignment():
    """Misaligned and transposed views give the bits of their contiguous copies; rows of a batch do not depend on it."""
    q, k, _, qw, kw, pos, tab = _inputs(40, 8, 2, 129, 64, torch.bfloat16, seed=3, device="cuda")
    q, k, qw, kw = q[..., 1:], k[..., 1:], qw[1:], kw[1:]
    want = R.qk_norm_rope_fxp(q.contiguous(), k.contiguous(), qw.contiguous(), kw.contiguous(), pos, tab)
    flip = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    inner = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    wide = torch.zeros(97, 100, device="cuda")
    wide[:, 3:67] = tab
    for f in (lambda x: x, flip, inner):
        for t in (tab, wide[:, 3:67]):
            got = R.qk_norm_rope_fxp(f(q), f(k), qw, kw, pos.int(), t)
            assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])
    one = R.qk_norm_rope_fxp(q[17:18], k[17:18], qw, kw, pos[17:18], tab)
    assert bits_equal(one[0], want[0][17:18]) and bits_equal(one[1], want[1][17:18])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 40])
def test_norm_rope_in_place_and_empty(D):
    q, k, _, qw, kw, pos, tab = _inputs(50, 8, 2, D, 32, torch.float16, seed=4, device="cuda")
    want = R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab, False)
    a, b = R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab, False, q_out=q, k_out=k)
    assert a.data_ptr() == q.data_ptr() and bits_equal(q, want[0]) and bits_equal(k, want[1])
    e = R.qk_norm_rope_fxp(q[:0], k[:0], qw, kw, pos[:0], tab)
    assert e[0].shape == (0, 8, D) and e[1].shape == (0, 2, D)
    n = R.qk_norm_rope_fxp(q[:, :0], k, qw, kw, pos, tab)
    assert n[0].numel() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 40])
def test_position_outside_the_table(D):
    q, k, _, qw, kw, pos, tab = _inputs(4, 2, 1, D, 32, torch.float32, seed=5, device="cuda")
    pos[1], pos[2] = tab.shape[0], -1
    yq, yk = R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab)
    for y in (yq, yk):
        assert y[1:3, :, :32].isnan().all() and y[1:3, :, 32:].isfinite().all() and y[[0, 3]].isfinite().all()


@pytest.mark.gpu
def test_norm_of_zeros_and_large_values():
    """A row of zeros stays zero; values beyond the accumulator's range saturate as the definition says; NaN and inf stay in their row."""
    q, k, _, qw, kw, pos, tab = _inputs(6, 2, 1, 64, 64, torch.float32, seed=6, device="cuda")
    q[0] = 0
    q[1] *= 1e4
    q[2, 0, 3], q[3, 1, 5] = float("inf"), float("nan")
    yq, _ = R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab)
    assert (yq[0] == 0).all()
    keep = torch.ones(6, dtype=torch.bool)
    keep[2:4] = False
    assert yq.cpu()[keep].isfinite().all()
    q2 = q.clone()
    q2[2:4] = 1.0
    y2, _ = R.qk_norm_rope_fxp(q2, k, qw, kw, pos, tab)
    assert bits_equal(y2.cpu()[keep], yq.cpu()[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [0, 32, 64])
@pytest.mark.parametrize("dtype, cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.bfloat16),
                                          (torch.float32, torch.float16), (torch.bfloat16, torch.float32)])
def test_append_formula(dtype, cache, norm):
    for i, (T, Hq, Hk, D, rot, page) in enumerate([(1, 4, 1, 128, 128, 16), (37, 8, 2, 64, 32, 16), (19, 3, 3, 40, 40, 5),
                                                   (200, 8, 2, 96, 96, 1), (9, 2, 2, 256, 128, 24)]):
        neox = i % 2 == 0
        q, k, v, qw, kw, pos, tab = _inputs(T, Hq, Hk, D, rot, dtype, F[i % 3], seed=i, device="cuda")
        g = torch.Generator().manual_seed(i)
        blocks = (T + page - 1) // page + 2
        kv = torch.randn(blocks, 2, page, Hk, D, generator=g).to(cache).cuda()
        before = kv.clone()
        slots = torch.randperm(blocks * page, generator=g)[:T].cuda()
        n = T - T // 5
        if T > 5:
            slots[2], slots[3], slots[4] = -1, -7, blocks * page + 5
        w = (qw, kw) if norm else (None, None)
        yq = torch.ops.fxpr.rope_append_kv_fxp(q, k, v, kv, slots[:n], pos, tab, neox, *w, 1e-6, 16, norm or 32)
        _assert_close(yq, *_formula(q, w[0], pos, tab, neox, norm))
        yk, bound = _formula(k, w[1], pos, tab, neox, norm)
        live = [t for t in range(n) if 0 <= int(slots[t]) < blocks * page]
        blk, off = slots[live] // page, slots[live] % page
        _assert_close(kv[blk, 0, off], yk[live], bound[live])
        assert torch.equal(kv[blk, 1, off], v[live].to(cache))
        kv[blk, :, off] = before[blk, :, off]
        assert torch.equal(kv, before), "a slot that no token has changed"


@pytest.mark.gpu
def test_append_is_norm_rope_in_the_cache():
    """The append form rotates with the bits of the other form; a cache seen through strides (blocks x 2 split) is written in place."""
    q, k, v, qw, kw, pos, tab = _inputs(64, 8, 2, 128, 128, torch.bfloat16, seed=7, device="cuda")
    want = R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab)
    slots = torch.randperm(160)[:64].cuda()
    store = torch.zeros(2, 10, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    kv = store.transpose(0, 1)
    ko = torch.empty_like(k)
    yq = R.rope_append_kv_fxp(q, k, v, kv, slots.int(), pos, tab, True, qw, kw, k_out=ko)
    assert bits_equal(yq, want[0]) and bits_equal(ko, want[1])
    assert bits_equal(store[0].flatten(0, 1)[slots], want[1]) and bits_equal(store[1].flatten(0, 1)[slots], v.contiguous())
    full = kv.contiguous()
    q1 = q.clone()
    R.rope_append_kv_fxp(q1, k, v, full, slots, pos, tab, True, qw, kw, q_out=q1)
    assert bits_equal(q1, want[0]) and torch.equal(full, kv)


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    q, k, v, qw, kw, pos, tab = _inputs(16, 8, 2, 64, 64, torch.bfloat16, seed=8, device="cuda")
    kv = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(16, device="cuda")
    R.rope_append_kv_fxp(q, k, v, kv, slots, pos, tab)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq = R.rope_append_kv_fxp(q, k, v, kv, slots, pos, tab)
    q.copy_(torch.randn_like(q))
    slots += 20
    graph.replay()
    torch.cuda.synchronize()
    want = torch.zeros_like(kv)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y2 = R.rope_append_kv_fxp(q, k, v, want, slots, pos, tab)
    side.synchronize()
    assert bits_equal(yq, y2) and bits_equal(kv.flatten(0, 1)[2:3], want.flatten(0, 1)[2:3])
    assert torch.equal(kv[1:], want[1:])


@pytest.mark.gpu
def test_append_offsets_beyond_32_bits():
    """Slots whose offsets in the cache pass 2^31 elements, in the vector kernel and the general one."""
    for D in (64, 40):
        q, k, v, _, _, pos, tab = _inputs(5, 2, 1, D, 8, torch.bfloat16, seed=9, device="cuda")
        blocks = 2**31 // (2 * 16 * D) + 4
        kv = torch.empty(blocks, 2, 16, 1, D, dtype=torch.bfloat16, device="cuda")
        kv[-3:] = 0
        small = torch.zeros(3, 2, 16, 1, D, dtype=torch.bfloat16, device="cuda")
        slots = torch.tensor([3, 20, 47, 0, 31], device="cuda")
        R.rope_append_kv_fxp(q, k, v, kv, slots + 16 * (blocks - 3), pos, tab)
        R.rope_append_kv_fxp(q, k, v, small, slots, pos, tab)
        assert bits_equal(kv[-3:].contiguous(), small) and (small != 0).any()


@pytest.mark.gpu
def test_the_same_call_on_two_streams_at_once():
    """Two calls in flight at the same time share nothing but their inputs."""
    q, k, v, qw, kw, pos, tab = _inputs(2000, 16, 4, 128, 128, torch.bfloat16, seed=10, device="cuda")
    want = R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab)
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, got):
            with torch.cuda.stream(s):
                g.append(R.qk_norm_rope_fxp(q, k, qw, kw, pos, tab))
    torch.cuda.synchronize()
    for a, b in got[0] + got[1]:
        assert bits_equal(a, want[0]) and bits_equal(b, want[1])
