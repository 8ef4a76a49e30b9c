"""The engine on the CPU: broken numbers under device sampling, steps of some of the sequences."""
import pytest
import torch

from nanochat_cpp_b200.inference import GenerateParams, InferenceEngine, generate_multi

from test_serving_engine_cpu import CUT, _model


def test_logits_without_a_number_are_an_error():
    """-1 is what the operator answers for such a row; it is no token, neither to return nor to go on from."""
    cfg, m = _model()
    m.params.m("lm_head.weight").fill_(float("nan"))
    m.params.sync_compute()
    for stops in ({}, {"stop_id": 5}):
        with pytest.raises(ValueError, match="no number"):
            generate_multi(InferenceEngine(m), torch.ones(2, 3, dtype=torch.long), GenerateParams(max_tokens=4, temperature=1.0, top_p=0.9, **stops))


@pytest.mark.parametrize("kv_dtype", ["auto", "mxfp8"])
def test_a_step_of_some_sequences(kv_dtype):
    """A step of two of three sequences through `cache.rows`, then one of all: the logits of a cache that holds the same."""
    cfg, m = _model(window=600)
    tokens = torch.randint(0, cfg.vocab_size, (3, 20), generator=torch.Generator().manual_seed(2))
    eng = InferenceEngine(m, kv_dtype=kv_dtype)
    a, b = eng.new_cache(3, 40), eng.new_cache(3, 40)
    eng.extend(a, tokens[:, :9])
    eng.extend(b, tokens[:, :10], [10, 9, 10])
    view = a.rows([0, 2])
    eng.decode(view, tokens[[0, 2], 9])
    view.commit()
    assert a.lens_host == b.lens_host == [10, 9, 10] and torch.equal(a.seq_lens, b.seq_lens)
    nxt = tokens[:, 11]
    assert (eng.decode(a, nxt) - eng.decode(b, nxt)).abs().max() < (1e-4 if kv_dtype == "auto" else CUT)
