"""Cascade attention in the engine with CUDA graphs: decode steps replay full
graphs, steps behind a shared prefix run the shared-prefix operator, and the
streams do not tell which."""

import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "fixed-point-reductions-for-vllm_b200")

SCRIPT = r"""
import json, sys
sys.path.insert(0, {pkg!r})
import torch
from fxpr_vllm import e2e
from fxpr_vllm.vllm_modules import attention_backend as B
e2e.PRESETS["model"] = dict(e2e.PRESETS["tiny"], num_key_value_heads={kv_heads})
d = e2e.make_llama_dir({mdir!r}, "model", seed=0)
calls, asked = [], []
orig = B.shared_prefix_attention_fxp
B.shared_prefix_attention_fxp = lambda **kw: (calls.append(kw["common_prefix_len"]), orig(**kw))[1]
rule = B.shared_prefix_takes_prefix_kernels
B.shared_prefix_takes_prefix_kernels = lambda *a, **kw: (asked.append([int(x) for x in a] + [str(kw["dtype"]), str(kw["kv_dtype"])]),
                                                         rule(*a, **kw))[1]
replays = [0]
replay = torch.cuda.CUDAGraph.replay
torch.cuda.CUDAGraph.replay = lambda self: (replays.__setitem__(0, replays[0] + 1), replay(self))[1]
from fxpr_vllm.register import register
register()
from vllm import LLM
llm = LLM(model=d, quantization="fixed_point_det", attention_backend="CUSTOM", skip_tokenizer_init=True, dtype="bfloat16",
          max_num_seqs=16, gpu_memory_utilization=0.25, max_model_len=512, seed=0, enable_prefix_caching=True,
          compilation_config=dict(mode=0, cudagraph_mode="FULL_DECODE_ONLY"), disable_cascade_attn={off})
head = e2e.prompts(1, 304, 1024, seed=1)[0]
ps = [head + t for t in e2e.prompts(6, 21, 1024, seed=2)]
e2e.generate(llm, ps[:1], 2)  # the prefix is in the cache
replays[0] = 0
shared = e2e.generate(llm, ps, 12)
during = replays[0]
apart = e2e.generate(llm, e2e.prompts(6, 40, 1024, seed=3), 12)
json.dump(dict(shared=shared, apart=apart, calls=calls, asked=asked, during=during, after=replays[0] - during,
               model=[llm.llm_engine.model_config.get_head_size()]), open({out!r}, "w"))
"""


@pytest.mark.parametrize("kv_heads", [2, 4])
def test_streams_with_cascade_and_cuda_graphs(tmp_path, kv_heads):
    """Groups of four heads: the prefix of six requests is too small for the decode steps, which stay in the full graphs, and only the
    step of several queries runs the shared-prefix operator. Groups of two: the decode steps run it too."""
    got = {}
    env = dict(os.environ, PYTHONPATH=PKG, VLLM_ENABLE_V1_MULTIPROCESSING="0", VLLM_HOST_IP="127.0.0.1", MASTER_ADDR="127.0.0.1",
               VLLM_USE_FLASHINFER_SAMPLER="0")
    for off in (True, False):
        out = tmp_path / f"streams_{off}.json"
        code = SCRIPT.format(pkg=PKG, mdir=str(tmp_path / "model"), out=str(out), off=off, kv_heads=kv_heads)
        r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-6000:]
        got[off] = json.load(open(out))
    on, off = got[False], got[True]
    assert off["calls"] == [] and off["asked"] == [] and off["during"] >= 10 and off["after"] >= 10
    assert on["calls"] and all(n >= 256 for n in on["calls"]) and on["after"] == off["after"]
    assert on["during"] == off["during"] if kv_heads == 2 else on["during"] < off["during"]
    assert on["asked"] and all(a[7] == on["model"][0] and a[9:] == ["torch.bfloat16"] * 2 for a in on["asked"])
    assert on["shared"] == off["shared"] and on["apart"] == off["apart"]
