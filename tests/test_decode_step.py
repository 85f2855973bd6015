"""The decode-step operators as they are used: the attention backend's calls,
one verification step through all four of them, and the engine with cascade
attention."""

import json
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

import fxpr_vllm.library_ops  # noqa: F401
from fxpr_vllm.fixed_point_kernels import attention as A
from fxpr_vllm.fixed_point_kernels import rope as R
from fxpr_vllm.vllm_modules.config import load_runtime_config
from tests.helpers import bits_equal

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "fixed-point-reductions-for-vllm_b200")


def test_fused_rope_is_opt_in():
    assert load_runtime_config({}).fused_rope is False
    assert load_runtime_config({"VLLM_FXP_FUSED_ROPE": "1"}).fused_rope is True
    assert load_runtime_config({"VLLM_FXP_FUSED_ROPE": "off"}).fused_rope is False


def test_backend_takes_cascade_where_the_prefix_kernels_run():
    from fxpr_vllm.vllm_modules.attention_backend import DeterministicAttentionBackend

    cls = DeterministicAttentionBackend.get_builder_cls()
    ask = lambda n, lens, heads=32, local=False, dcp=1: cls.use_cascade_attention(  # noqa: E731
        cls.__new__(cls), n, lens, heads, 8, False, False, local, 148, dcp)
    assert ask(4096, [5, 1, 1]) and ask(256, [1, 1], heads=64) and ask(4096, [1] * 16)
    assert not ask(4096, [1] * 15) and not ask(1024, [1, 1])  # decode batches with few (row, key) pairs
    assert not ask(255, [5, 1]) and not ask(4096, [5]) and not ask(4096, [5, 1], local=True)
    assert not ask(4096, [5, 1], dcp=2)


def _impl(heads, kv_heads, dim):
    from fxpr_vllm.vllm_modules.attention_backend import DeterministicAttentionImpl

    return DeterministicAttentionImpl(heads, dim, dim**-0.5, kv_heads, None, None)


@pytest.mark.gpu
def test_backend_rope_update_then_cascade_forward():
    """The backend's fused rotary and cache update, then its forward pass with and without a reported common prefix: equal bits."""
    H, KVH, D, page, prefix, R_ = 14, 2, 128, 16, 320, 6
    g = torch.Generator().manual_seed(0)
    impl = _impl(H, KVH, D)
    kv = torch.randn(60, 2, page, KVH, D, generator=g).bfloat16().cuda()
    cols = prefix // page + 1
    bt = torch.zeros(R_, cols, dtype=torch.int32)
    bt[:, :-1] = torch.randperm(20, generator=g)[:cols - 1].int() + 1
    bt[:, -1] = torch.arange(R_) + 30
    seq = torch.tensor([prefix + 1 + r for r in range(R_)], dtype=torch.int32)
    slots = (bt[:, -1].long() * page + (seq.long() - 1) % page).cuda()
    q, k, v = (torch.randn(R_, n, D, generator=g).bfloat16().cuda() for n in (H, KVH, KVH))
    pos = (seq.long() - 1).cuda()
    ang = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(D // 2) * 2 / D)
    table = torch.cat([ang.cos(), ang.sin()], -1).bfloat16().cuda()
    want_kv = kv.clone()
    want_q = R.rope_append_kv_fxp(q, k, v, want_kv, slots, pos, table)
    q2, k2 = q.clone().view(R_, H * D), k.clone().view(R_, KVH * D)
    impl.do_rope_and_kv_cache_update(None, q2, k2, v.view(R_, KVH * D), pos, table, True, kv, slots)
    assert bits_equal(q2.view(R_, H, D), want_q) and torch.equal(kv, want_kv)
    assert bits_equal(k2.view(R_, KVH, D), kv[bt[:, -1].long().cuda(), 0, ((seq.long() - 1) % page).cuda()])
    outs = []
    for cascade in (False, True):
        meta = SimpleNamespace(num_actual_tokens=R_, query_start_loc=torch.arange(R_ + 1, dtype=torch.int32, device="cuda"),
                               seq_lens=seq.cuda(), block_table=bt.cuda(), max_query_len=1, max_seq_len=int(seq.max()),
                               use_cascade=cascade, common_prefix_len=prefix if cascade else 0)
        out = torch.full((R_ + 2, H, D), 3.0, dtype=torch.bfloat16, device="cuda")
        pad = torch.cat([q2, q2[:2]])
        impl.forward(None, pad, None, None, kv, meta, output=out)
        outs.append(out)
    assert bits_equal(outs[0], outs[1]) and (outs[1][R_:] == 3.0).all()


@pytest.mark.gpu
def test_a_verification_step():
    """Norm and rotary, append, attention behind the prefix, verification: in a captured step replayed on new inputs, the same bits as
    the operators alone and as the step of every request alone."""
    H, KVH, D, page, prefix, V = 8, 2, 64, 16, 288, 515
    drafts, vocab_w = [3, 0, 2, 4], torch.randn(H * D, V, generator=torch.Generator().manual_seed(9)).cuda()
    R_, T = len(drafts), sum(drafts) + len(drafts)
    ops = torch.ops.fxpr
    g = torch.Generator().manual_seed(1)
    lens = [d + 1 for d in drafts]
    qsl = torch.tensor([sum(lens[:i]) for i in range(R_ + 1)], dtype=torch.int32)
    start = torch.tensor([sum(drafts[:i]) for i in range(R_ + 1)], dtype=torch.int32)
    own = [20, 1, 33, 5]  # keys of its own that each request has already
    seq = torch.tensor([prefix + o + n for o, n in zip(own, lens)], dtype=torch.int32)
    cols = (int(seq.max()) + page - 1) // page
    shared = prefix // page
    bt = torch.empty(R_, cols, dtype=torch.int32)
    bt[:, :shared] = torch.randperm(shared, generator=g).int()
    bt[:, shared:] = shared + torch.arange(R_ * (cols - shared)).int().view(R_, -1)
    pos = torch.tensor([int(seq[r]) - n + i for r, n in enumerate(lens) for i in range(n)])
    req = [r for r, n in enumerate(lens) for _ in range(n)]
    slots = torch.tensor([int(bt[r, p // page]) * page + int(p) % page for r, p in zip(req, pos.tolist())])
    rows = torch.tensor([int(qsl[r]) + i for r, n in enumerate(drafts) for i in range(n)])
    ang = torch.arange(400)[:, None] * 10000.0 ** (-torch.arange(D // 2) * 2 / D)
    w = (1 + 0.1 * torch.randn(2, D, generator=g)).bfloat16()
    c = {k: x.cuda() for k, x in dict(qsl=qsl, start=start, seq=seq, bt=bt, pos=pos, slots=slots, rows=rows, w=w,
                                      tab=torch.cat([ang.cos(), ang.sin()], -1), bonus=torch.arange(R_).int()).items()}

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        n = sum(drafts)
        return [x.cuda() for x in (torch.randn(T, H + 2 * KVH, D, generator=g).bfloat16(),
                                   torch.randn(int(bt.max()) + 1, 2, page, KVH, D, generator=g).bfloat16(),
                                   torch.randint(0, V, (n,), generator=g).int(), torch.rand(n, generator=g),
                                   torch.rand(R_, generator=g))]

    def step(x, kv, ids, u, r):
        q, k, v = x[:, :H], x[:, H:H + KVH], x[:, H + KVH:]
        q = ops.rope_append_kv_fxp(q, k, v, kv, c["slots"], c["pos"], c["tab"], True, c["w"][0], c["w"][1], 1e-6, 16, 32)
        o = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
        ops.shared_prefix_attention_fxp(q, kv, o, c["qsl"], c["seq"], c["bt"], prefix, max(lens), None, 32, True, None, 16, 0.0, 0,
                                        int(seq.max()))
        p = torch.softmax(o.view(T, -1)[c["rows"]].float() @ vocab_w, -1)
        return (q, o, *ops.verify_draft_fxp(p, None, ids, c["start"], c["bonus"], u, r, max(drafts), 30))

    static = inputs(2)
    step(*static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for seed in (3, 4):
        new = inputs(seed)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = step(*new)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(static[1], new[1])
        # the parts by themselves: the norm form's rotation, and the unified attention over the written cache
        q, k = ops.qk_norm_rope_fxp(new[0][:, :H], new[0][:, H:H + KVH], c["w"][0], c["w"][1], c["pos"], c["tab"], True, 1e-6, 16, 32)
        assert bits_equal(q, want[0]) and bits_equal(k, new[1].transpose(1, 2).flatten(0, 1)[c["slots"], 0])
        o = torch.zeros_like(want[1])
        A.unified_attention_fxp(q, new[1], o, c["qsl"], c["seq"], c["bt"], max(lens), frac_bits=16)
        assert bits_equal(o, want[1])


SCRIPT = r"""
import json, sys
sys.path.insert(0, {pkg!r})
import torch
from fxpr_vllm import e2e
from fxpr_vllm.vllm_modules import attention_backend as B
d = e2e.make_llama_dir({mdir!r}, "tiny", seed=0)
calls = []
orig = B.shared_prefix_attention_fxp
B.shared_prefix_attention_fxp = lambda **kw: (calls.append(kw["common_prefix_len"]), orig(**kw))[1]
from fxpr_vllm.register import register
register()
from vllm import LLM
llm = LLM(model=d, quantization="fixed_point_det", attention_backend="CUSTOM", skip_tokenizer_init=True, dtype="bfloat16",
          max_num_seqs=16, gpu_memory_utilization=0.25, enforce_eager=True, max_model_len=512, seed=0, enable_prefix_caching=True,
          disable_cascade_attn={off})
head = e2e.prompts(1, 304, 1024, seed=1)[0]
ps = [head + t for t in e2e.prompts(6, 21, 1024, seed=2)]
e2e.generate(llm, ps[:1], 2)  # the prefix is in the cache
json.dump({{"streams": e2e.generate(llm, ps, 12), "calls": calls}}, open({out!r}, "w"))
"""


@pytest.mark.gpu
def test_engine_with_cascade_attention(tmp_path):
    """Greedy streams behind a shared prompt: equal with the engine's cascade attention on (the shared-prefix operator runs) and off."""
    got = {}
    env = dict(os.environ, PYTHONPATH=PKG, VLLM_ENABLE_V1_MULTIPROCESSING="0", VLLM_HOST_IP="127.0.0.1", MASTER_ADDR="127.0.0.1",
               VLLM_USE_FLASHINFER_SAMPLER="0")
    for off in (True, False):
        out = tmp_path / f"streams_{off}.json"
        code = SCRIPT.format(pkg=PKG, mdir=str(tmp_path / "tiny"), out=str(out), off=off)
        r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-6000:]
        got[off] = json.load(open(out))
    assert got[True]["calls"] == [] and got[False]["calls"]
    assert all(n >= 256 for n in got[False]["calls"])
    assert got[True]["streams"] == got[False]["streams"]


@pytest.mark.gpu
def test_schemas_and_tracing():
    """The operators' schemas name what they change, their shapes can be traced, and a compiled function gives their bits."""
    g = torch.Generator().manual_seed(5)
    ops = torch.ops.fxpr
    x = torch.randn(6, 14, 64, generator=g).bfloat16().cuda()
    q, k, v = x[:, :10], x[:, 10:12], x[:, 12:]
    w, pos, tab = torch.ones(64, dtype=torch.bfloat16, device="cuda"), torch.arange(6, device="cuda"), torch.randn(9, 64, generator=g).cuda()
    kv = torch.randn(24, 2, 16, 2, 64, generator=g).bfloat16().cuda()
    bt = torch.cat([torch.arange(17).expand(3, -1), 17 + torch.arange(3)[:, None]], 1).int().cuda()
    qsl = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    sl = torch.full((3,), 280, dtype=torch.int32, device="cuda")
    p = torch.softmax(torch.randn(6, 33, generator=g), -1).cuda()
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    u = torch.rand(6, generator=g).cuda()
    calls = {
        ops.qk_norm_rope_fxp.default: (q, k, w, w, pos, tab, True, 1e-6, 16, 32),
        ops.rope_append_kv_fxp.default: (q, k, v, kv, pos + 275, pos, tab, False, None, None, 1e-6, 16, 32),
        ops.shared_prefix_attention_fxp.default: (q, kv, torch.zeros_like(q), qsl, sl, bt, 272, 2, None, 32, True, None, 16, 0.0, 0, 280),
        ops.verify_draft_fxp.default: (p, None, i32(1, 2, 3, 4, 5, 6), i32(0, 3, 6), i32(7, 8), u, u[:2], 3, 30),
    }
    for op, args in calls.items():
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))

    def step(q, k, v, kv, o):
        q, k = ops.qk_norm_rope_fxp(q, k, w, w, pos, tab, True, 1e-6, 16, 32)
        q = ops.rope_append_kv_fxp(q, k, v, kv, pos + 275, pos, tab, True, None, None, 1e-6, 16, 32)
        ops.shared_prefix_attention_fxp(q, kv, o, qsl, sl, bt, 272, 2, None, 32, True, None, 16, 0.0, 0, 280)
        return q, o.clone(), kv.clone()

    fresh = lambda: (q, k, v, kv.clone(), torch.zeros(q.shape, device="cuda"))  # noqa: E731
    want = step(*fresh())
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(*fresh())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
