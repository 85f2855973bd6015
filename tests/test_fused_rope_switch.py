"""The switch for vLLM's fused rotary and cache update says that it has no
effect, and the backend does not offer what the engine cannot use soundly."""

import dataclasses
import logging

from fxpr_vllm import register as R
from fxpr_vllm.vllm_modules.config import load_runtime_config


def test_set_switch_is_reported(caplog):
    with caplog.at_level(logging.INFO, logger="fxpr_vllm"):
        R._log_config(load_runtime_config({}))
        assert "FUSED_ROPE" not in caplog.text
        R._log_config(load_runtime_config({"VLLM_FXP_FUSED_ROPE": "1"}))
    said = [r for r in caplog.records if "VLLM_FXP_FUSED_ROPE has no effect" in r.getMessage()]
    assert len(said) == 1 and said[0].levelno == logging.WARNING


def test_backend_does_not_offer_it(monkeypatch):
    from fxpr_vllm.vllm_modules import attention_backend as B

    on = dataclasses.replace(load_runtime_config({}), fused_rope=True)
    monkeypatch.setattr(B, "get_runtime_config", lambda: on)
    impl = B.DeterministicAttentionImpl(8, 64, 0.125, 2, None, None)
    assert impl.fused_rope_kvcache_supported() is False
