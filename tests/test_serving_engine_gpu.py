"""The engine's serving paths on the kernels: MXFP8 cache, ragged chunks, device sampling, graph replay."""
import pytest
import torch

from nanochat_cpp_b200 import ops
from nanochat_cpp_b200.config import Config
from nanochat_cpp_b200.inference import GenerateParams, InferenceEngine, generate_multi
from nanochat_cpp_b200.models import GPT

pytestmark = pytest.mark.gpu


def _model(head_dim=128, kv=2, window=128):
    cfg = Config(num_layers=4, num_heads=512 // head_dim, num_kv_heads=kv, hidden_dim=512, seq_len=512, vocab_size=1000,
                 padded_vocab_size=1024, window_pattern="SSSL", short_window_override=window)
    m = GPT(cfg, "cuda", torch.bfloat16, seed=2)
    g = torch.Generator().manual_seed(0)
    for s in m.params.specs:
        if s.name.endswith("c_proj.weight"):
            m.params.m(s.name).copy_((torch.randn(s.shape, generator=g) * 0.02).cuda())
    m.params.m("lm_head.weight").copy_((torch.randn(1024, 512, generator=g) * 0.05).cuda())
    m.params.sync_compute()
    return cfg, m


def _in_torch(fn):
    ops.set_mode("torch")
    try:
        return fn()
    finally:
        ops.set_mode("kernels")


@pytest.mark.parametrize("kv_dtype", ["auto", "mxfp8"])
@pytest.mark.parametrize("head_dim,kv", [(128, 2), (64, 8), (64, 4)])
def test_extend_and_decode_match_the_plain_operators(kv_dtype, head_dim, kv):
    """Ragged prompts, a further turn and single tokens: kernels against the PyTorch definitions on the same weights
    (0.15 on logits, as in the other engine tests: four layers of bf16 activations)."""
    cfg, m = _model(head_dim, kv)
    eng = InferenceEngine(m, use_cuda_graph=False, kv_dtype=kv_dtype)
    tokens = torch.randint(0, cfg.vocab_size, (4, 120), generator=torch.Generator().manual_seed(1)).cuda()

    def run():
        cache = eng.new_cache(4, 400)
        out = [eng.extend(cache, tokens, [120, 1, 64, 33]), eng.extend(cache, tokens[:, :50], [3, 50, 0, 20])]
        out.append(eng.decode(cache, tokens[:, 7]))
        out.append(eng.extend(cache, tokens[:, :5], all_logits=True))
        return out
    for a, b in zip(run(), _in_torch(run)):
        assert a.shape == b.shape and (a - b).abs().max() < 0.15
    ops.cuda_module().check_status()


def test_extend_is_prefill_on_a_bf16_cache():
    cfg, m = _model(window=256)
    eng = InferenceEngine(m, use_cuda_graph=False)
    tokens = torch.randint(0, cfg.vocab_size, (3, 200), generator=torch.Generator().manual_seed(2)).cuda()
    a, b = eng.new_cache(3, 300), eng.new_cache(3, 300)
    x, y = eng.prefill(a, tokens), eng.extend(b, tokens)
    assert (x - y).abs().max() < 0.15
    nxt = x.argmax(-1)
    assert (eng.decode(a, nxt) - eng.decode(b, nxt)).abs().max() < 0.15
    ops.cuda_module().check_status()


@pytest.mark.parametrize("head_dim", [64, 128])
def test_mxfp8_decode_graph_replay_and_generate(head_dim):
    cfg, m = _model(head_dim)
    prompts = torch.randint(0, cfg.vocab_size, (4, 70), generator=torch.Generator().manual_seed(3))
    graph, eager = (InferenceEngine(m, use_cuda_graph=g, kv_dtype="mxfp8") for g in (True, False))
    for params in (GenerateParams(max_tokens=20), GenerateParams(max_tokens=20, temperature=1.0, top_p=0.9, min_p=0.01, seed=5),
                   GenerateParams(max_tokens=20, temperature=0.8, top_k=40, seed=6, device_sampling=True)):
        a, b = (generate_multi(e, prompts, params) for e in (graph, eager))
        assert [s.tokens for s in a] == [s.tokens for s in b]
    assert graph.use_cuda_graph and graph._graph is not None
    lists = [prompts[0].tolist(), prompts[1, :5].tolist()]
    a, b = (generate_multi(e, lists, GenerateParams(max_tokens=9)) for e in (graph, eager))
    assert [s.tokens for s in a] == [s.tokens for s in b]
    ops.cuda_module().check_status()


def test_a_long_prompt_over_a_windowed_mxfp8_cache():
    """Longer than what the windowed layers hold at once: pieces, pages given back, and tokens after it."""
    cfg, m = _model(window=64)
    eng = InferenceEngine(m, use_cuda_graph=False, kv_dtype="mxfp8")
    tokens = torch.randint(0, cfg.vocab_size, (2, 1300), generator=torch.Generator().manual_seed(4)).cuda()
    cache = eng.new_cache(2, 1400)
    assert cache.chunk < 1300

    def run():
        c = eng.new_cache(2, 1400)
        x = eng.prefill(c, tokens)
        return x, eng.decode(c, tokens[:, 0])
    for a, b in zip(run(), _in_torch(run)):
        assert (a - b).abs().max() < 0.15
    ops.cuda_module().check_status()
