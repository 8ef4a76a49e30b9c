"""Generation with device sampling where the model's numbers are broken, on the CPU."""
import pytest
import torch

from nanochat_cpp_b200.inference import GenerateParams, InferenceEngine, generate_multi

from test_serving_engine_cpu import _model


def test_logits_without_a_number_are_an_error():
    """-1 is what the operator answers for such a row; it is no token, neither to return nor to go on from."""
    cfg, m = _model()
    m.params.m("lm_head.weight").fill_(float("nan"))
    m.params.sync_compute()
    for stops in ({}, {"stop_id": 5}):
        with pytest.raises(ValueError, match="no number"):
            generate_multi(InferenceEngine(m), torch.ones(2, 3, dtype=torch.long), GenerateParams(max_tokens=4, temperature=1.0, top_p=0.9, **stops))
