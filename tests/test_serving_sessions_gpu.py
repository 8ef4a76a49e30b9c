"""Several conversations on one engine, and what a call holds on to."""
import pytest
import torch

from nanochat_cpp_b200 import ops
from nanochat_cpp_b200.inference import InferenceEngine

from test_serving_engine_gpu import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_dtype", ["auto", "mxfp8"])
def test_a_captured_step_outlives_a_longer_conversation(kv_dtype):
    """A captured decode step of a short conversation, replayed after a longer one has made the engine's rotary tables grow: the same
    logits as without the interruption. What the longer one freed is taken and overwritten in between."""
    cfg, m = _model()
    tokens = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(1)).cuda()

    def talk(interrupt):
        eng = InferenceEngine(m, kv_dtype=kv_dtype)
        a = eng.new_cache(2, 100)
        eng.extend(a, tokens[:, :20])
        out = [eng.decode_graphed(a, tokens[:, 20]).clone()]
        if interrupt:
            size = eng._cos.numel()
            b = eng.new_cache(1, 4 * cfg.seq_len)
            eng.extend(b, tokens[:1])
            eng.decode(b, tokens[:1, 0])
            torch.cuda.synchronize()
            junk = [torch.full((size,), float("nan"), dtype=t, device="cuda") for t in (torch.float32, torch.bfloat16) for _ in range(40)]
            torch.cuda.synchronize()
            del junk
        out += [eng.decode_graphed(a, tokens[:, t]).clone() for t in (21, 22)]
        assert eng.use_cuda_graph
        return out
    for x, y in zip(talk(True), talk(False)):
        assert torch.equal(x, y)
    ops.cuda_module().check_status()
