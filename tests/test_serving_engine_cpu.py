"""The engine over an MXFP8 cache, chunks of new tokens at any position, and sampling from given streams, on the CPU."""
import json

import pytest
import torch

from nanochat_cpp_b200.config import LOGIT_SOFTCAP, Config
from nanochat_cpp_b200.data import native
from nanochat_cpp_b200.inference import GenerateParams, InferenceEngine, generate_multi, sample
from nanochat_cpp_b200.models import GPT
from nanochat_cpp_b200.ops import ref


def _model(window=8, heads=2, hidden=128, kv=1):
    cfg = Config(num_layers=4, num_heads=heads, num_kv_heads=kv, hidden_dim=hidden, seq_len=256, vocab_size=96,
                 padded_vocab_size=128, rope_base=10000.0, window_pattern="SL", short_window_override=window)
    m = GPT(cfg, "cpu", torch.float32, seed=3)
    g = torch.Generator().manual_seed(1)
    for s in m.params.specs:
        if s.name.endswith("c_proj.weight"):
            m.params.m(s.name).copy_(torch.randn(s.shape, generator=g) * 0.05)
    m.params.m("lm_head.weight").copy_(torch.randn(128, hidden, generator=g) * 0.1)
    m.params.m("smear_lambda").fill_(0.4)
    m.params.sync_compute()
    return cfg, m


def _full(m, tokens):
    return LOGIT_SOFTCAP * torch.tanh(m.logits(tokens) / LOGIT_SOFTCAP)


@pytest.mark.parametrize("window", [5, 40])
def test_extend_at_different_positions_matches_the_full_forward(window):
    """Ragged chunks, idle sequences, single tokens and a continued prompt: every logit is the full forward's."""
    cfg, m = _model(window)
    B, total = 3, 90
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, cfg.vocab_size, (B, total), generator=g)
    full = _full(m, tokens)
    eng = InferenceEngine(m)
    cache = eng.new_cache(B, total + 2)
    at = [0] * B
    for counts in ([7, 0, 30], [1, 20, 0], [20, 1, 3], [30, 12, 40]):
        T = max(counts) + 2                                  # two columns of padding
        chunk = torch.zeros(B, T, dtype=torch.long)
        for b, n in enumerate(counts):
            chunk[b, :n] = tokens[b, at[b]:at[b] + n]
        lg = eng.extend(cache, chunk, counts, all_logits=True)
        for b, n in enumerate(counts):
            if n:
                assert (lg[b, :n] - full[b, at[b]:at[b] + n]).abs().max() < 1e-4
            assert not lg[b, n:].any()
            at[b] += n
        assert cache.lens_host == at and cache.seq_lens.tolist() == at
    nxt = torch.stack([tokens[b, at[b]] for b in range(B)])  # and single tokens go on from there
    lg = eng.decode(cache, nxt)
    assert all((lg[b] - full[b, at[b]]).abs().max() < 1e-4 for b in range(B))
    cache.reset([0])                                         # a sequence that starts anew among others
    lg = eng.extend(cache, tokens[:, :4], [4, 0, 0])
    assert (lg[0] - full[0, 3]).abs().max() < 1e-4 and not lg[1:].any()


# Two cuts of one prompt compute the same sums in another order (fp32: 1e-7 of a value). Where that moves a key or value
# across a rounding border of E4M3, one of its 64 channels changes by 2^-4 of itself: a channel of size 3 by 0.19, a score by
# 0.19 * 3 / 8 at most, and a logit, which takes it through one head's softmax weights and projections of size
# 0.05, by less than 0.05. A wrong position, page or length moves logits by whole units.
CUT = 0.05


def test_mxfp8_cache_does_not_depend_on_the_cut_into_chunks():
    cfg, m = _model(window=600)
    tokens = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(4))
    eng = InferenceEngine(m, kv_dtype="mxfp8")
    whole = eng.extend(eng.new_cache(2, 64), tokens, all_logits=True)
    cache = eng.new_cache(2, 64)
    parts = [eng.extend(cache, tokens[:, :13], all_logits=True), eng.extend(cache, tokens[:, 13:30], all_logits=True)]
    parts += [eng.decode(cache, tokens[:, t])[:, None] for t in range(30, 40)]
    assert (torch.cat(parts, 1) - whole).abs().max() < CUT
    assert (eng.prefill(eng.new_cache(2, 64), tokens) - whole[:, -1]).abs().max() < CUT
    assert cache.k[0].dtype == torch.uint8 and cache.bytes() * 3 < InferenceEngine(m).new_cache(2, 64).bytes()
    # what the cache holds are the quantised keys of the same positions
    k, v = cache.read(1, 0)
    exact = InferenceEngine(m)
    other = exact.new_cache(2, 64)
    exact.prefill(other, tokens)
    k2, v2 = other.read(1, 0)
    assert k.shape == k2.shape == (40, cfg.num_kv_heads, cfg.head_dim)
    k, k2 = cache.read(0, 0)[0], other.read(0, 0)[0]         # the first layer's keys depend on no attention
    first = ref.mx_kv_decode(*ref.mx_kv_encode(k2))
    assert ((k.float() - first).abs() <= 2.0 ** -3 * first.abs() + 2.0 ** -9).all()      # equal, or one code beside


def test_windowed_mxfp8_cache_long_prompt_and_release():
    cfg, m = _model(window=20)
    B, total = 2, 700
    tokens = torch.randint(0, cfg.vocab_size, (B, total), generator=torch.Generator().manual_seed(5))
    eng = InferenceEngine(m, kv_dtype="mxfp8")
    cache = eng.new_cache(B, total + 1)
    assert cache.chunk == 512                                # the prompt goes through in two pieces
    a = eng.prefill(cache, tokens)
    small = eng.new_cache(B, total + 1)
    for s in range(0, total, 100):
        b = eng.extend(small, tokens[:, s:s + 100])
    assert (a - b).abs().max() < CUT
    nxt = a.argmax(-1)
    assert (eng.decode(cache, nxt) - eng.decode(small, nxt)).abs().max() < CUT
    held = small.pages_in_use()["windowed"]
    assert held <= B * ((20 + 100) // 16 + 2)
    k, v = small.read(0, 1)
    assert k.shape[0] == total + 1 and not k[:400].any() and k[-10:].any()
    ragged = eng.new_cache(B, total + 1)
    lg = eng.prefill_ragged(ragged, [tokens[0, :600].tolist(), tokens[1, :7].tolist()])
    one = eng.prefill(eng.new_cache(1, total + 1), tokens[1:, :7])
    assert (lg[1] - one[0]).abs().max() < CUT and ragged.lens_host == [600, 7]


def test_uniform_streams_are_those_of_the_host_sampler():
    """Draw d of a row's stream from `sample_uniforms`, walked over the softmax, gives the host sampler's token (rows
    whose number lies within 1e-4 of a border are left out: the two sum in different precision)."""
    g = torch.Generator().manual_seed(0)
    z = torch.randn(40, 50, generator=g) * 2
    u = torch.from_numpy(native.sample_uniforms(7, range(40), 0, 3))
    assert torch.equal(u[1:], torch.from_numpy(native.sample_uniforms(7, range(40), 1, 2)))
    for step in range(3):
        host = sample(z, 0.8, 0, 7, torch.arange(40), step)
        mine = ref.sample_rows(z, u[step], 0.8)
        cum = torch.softmax(z.double() / 0.8, -1).cumsum(-1)
        clear = (cum - u[step].double()[:, None]).abs().amin(-1) > 1e-4
        assert int(clear.sum()) > 30 and torch.equal(host[clear], mine[clear])


def test_generate_with_nucleus_settings_and_mxfp8_cache():
    cfg, m = _model()
    prompts = [[1, 2, 3], [4, 5, 6, 7, 8]]
    for kv in ("auto", "mxfp8"):
        eng = InferenceEngine(m, kv_dtype=kv)
        run = lambda **k: [s.tokens for s in generate_multi(eng, prompts, GenerateParams(max_tokens=12, num_samples=2, **k))]  # noqa: E731
        greedy = run()
        assert run(temperature=1.0, top_p=1e-6) == greedy                      # the nucleus of one token
        assert run(temperature=1.0, min_p=1.0) == greedy and run(temperature=1.0, top_k=1, device_sampling=True) == greedy
        a = run(temperature=1.0, top_p=0.9, seed=3)
        assert a == run(temperature=1.0, top_p=0.9, seed=3) and a != run(temperature=1.0, top_p=0.9, seed=4)
        assert all(0 <= t < cfg.vocab_size for s in a for t in s)


def test_engine_refusals():
    cfg, m = _model()
    with pytest.raises(ValueError):
        InferenceEngine(m, kv_dtype="int8")
    eng = InferenceEngine(m)
    cache = eng.new_cache(2, 32)
    tok = torch.zeros(2, 4, dtype=torch.long)
    for bad in ((tok[:1], None), (tok[0], None), (tok, [5, 1]), (tok, [1]), (tok, [-1, 1])):
        with pytest.raises(ValueError):
            eng.extend(cache, *bad)
    with pytest.raises(ValueError):
        eng.extend(cache, torch.zeros(2, 40, dtype=torch.long))
    assert cache.lens_host == [0, 0]
    narrow = _model(heads=8, hidden=128, kv=8)[1]            # head_dim 16
    with pytest.raises(ValueError):
        InferenceEngine(narrow, kv_dtype="mxfp8").new_cache(1, 32)


def test_command_line_flags(tmp_path):
    from nanochat_cpp_b200 import cli
    from nanochat_cpp_b200.train.checkpointer import save_checkpoint
    cfg, m = _model()
    path, out = str(tmp_path / "m.ckpt"), str(tmp_path / "o.jsonl")
    save_checkpoint(path, m)
    args = ["generate", "--model", path, "--tokens", "1,2,3", "--max-tokens", "6", "--temperature", "0.9", "--top-p", "0.8",
            "--min-p", "0.01", "--kv-cache", "mxfp8", "--seed", "3", "--device", "cpu", "--out", out]
    assert cli.main(args) == 0
    rec = json.loads(open(out).readline())
    assert len(rec["tokens"]) == 9
