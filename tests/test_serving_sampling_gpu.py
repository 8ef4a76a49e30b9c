"""Sampling at the ends of its range: temperatures and logits near the largest numbers, vocabularies beyond shared memory."""
import pytest
import torch

from nanochat_cpp_b200 import ops

import serving_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("setting", [(1.0e38, 0, 0.9, 0.0), (1.0e38, 1000, 1.0, 0.0), (3.0e38, 40, 0.8, 0.0), (1.0e38, 0, 1.0, 0.2),
                                     (float("inf"), 0, 0.5, 0.0), (float("inf"), 100, 1.0, 0.0), (2.0e37, 2500, 0.95, 0.01)])
def test_sampling_at_extreme_temperatures(setting):
    """Logits all over fp32's range, and infinities, at temperatures that make them comparable."""
    V = 3000
    g = torch.Generator().manual_seed(0)
    z = (torch.rand(6, V, generator=g) * 2 - 1) * 3.4e38
    z[1, 5], z[2, 7], z[2, 9], z[3, ::2], z[4] = 3.4e38, float("inf"), float("inf"), float("-inf"), torch.randn(V, generator=g)
    z[5, 100:] = -3.4e38
    for u0 in (0.0, 0.3, 0.77, 0.99):
        u = torch.full((6,), u0)
        want = U.sample(z, u, *setting)
        if setting[0] == float("inf"):         # (inf - z) / inf is no number: the row has no definition there
            want[2] = 7 if u0 < 0.5 or setting[2] == 0.5 else 9
        assert torch.equal(ops.sample_rows(z.cuda(), u.cuda(), *setting).cpu(), want)


@pytest.mark.parametrize("bf16,V", [(False, 400001), (False, 700000), (True, 600000), (True, 900001)])
@pytest.mark.parametrize("setting", [(0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 5000, 0.99, 0.001), (1.0, 0, 1.0, 0.0)])
def test_vocabularies_that_do_not_fit_shared_memory(bf16, V, setting):
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(2, V, generator=g) * 2.5).to(torch.bfloat16)
    z = z if bf16 else z.float()
    u = torch.rand(2, generator=g)
    assert torch.equal(ops.sample_rows(z.cuda(), u.cuda(), *setting).cpu(), U.sample(z, u, *setting))
