"""Attention over the pages where scores are large, by both kernels."""
import pytest
import torch

from nanochat_cpp_b200 import ops

import serving_range_util as R
import serving_util as U

pytestmark = pytest.mark.gpu

ROWS, CHUNK = R.ROWS, R.CHUNK


@pytest.mark.parametrize("variant", [ROWS, CHUNK])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("size", [8.0, 64.0, 512.0, 8192.0, 2.0 ** 20])
def test_one_visible_key_of_any_score(variant, mx, size):
    """A row that sees one key gives that key's value, whatever the score (2^-8 for the probability's rounding against the sum of
    the unrounded ones, 2^-8 for the result's)."""
    g = torch.Generator().manual_seed(int(size) % 1000)
    B, T, H, D = 2, 150, 3, 128
    q, k = (torch.randn(B, T, H, D, generator=g) * size for _ in range(2))
    c = R.case(q, k, torch.randn(B, T, H, D, generator=g), [T, T], mx)
    out = R.run(c, variant, window=0).double()
    v = U.pool_values(c["v"], c["vs"])[c["table"].long()].flatten(1, 2)[:, :T]
    assert bool(((out - v).abs() <= 1.01 * 2.0 ** -7 * v.abs()).all())
    ops.cuda_module().check_status()


@pytest.mark.parametrize("variant", [ROWS, CHUNK])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("D,S", [(128, 700), (64, 1500)])
def test_equal_keys_of_large_scores(variant, mx, D, S):
    """Whole numbers: every score is exact, up to 5e4 after scaling. Keys come in a few kinds, so that many share the largest one and
    the result is a mean of values."""
    g = torch.Generator().manual_seed(D)
    B, T, H, KV = 2, 90, 4, 2
    q = torch.randint(-7, 8, (B, T, H, D), generator=g).float() * 8
    kinds = torch.randint(-7, 8, (B, 6, KV, D), generator=g).float() * 8       # E4M3 holds 4 significant bits
    kinds[:, 0] = q[:, 0, ::2].sign() * 56
    k = kinds[torch.arange(B)[:, None], torch.randint(0, 6, (B, S), generator=g)]
    c = R.case(q, k, torch.randn(B, S, KV, D, generator=g), [S, S - 41], mx)
    R.hold(c, variant, exact_products=True)
    R.hold(c, variant, window=300, scale=1.0, exact_products=True)
    R.hold(c, variant, scale=64.0 * D, exact_products=True)                     # up to 2^32


@pytest.mark.parametrize("variant", [ROWS, CHUNK])
@pytest.mark.parametrize("mx", [False, True])
def test_scores_where_fp32_steps_by_eight(variant, mx):
    """Whole-number scores above 2^23, scaled to above 2^26 in powers of two, where fp32 holds every eighth number: the later keys'
    scores are one step (2^8 in probability) above the first ones', so their values' mean is the result but for one part in 257."""
    D, n = 128, 16
    q = torch.full((1, 1, 1, D), 256.0)
    k = torch.full((1, 2 * n, 1, D), 256.0)
    q[..., 0] = 1
    k[..., 1:17] = 288
    k[:, :n, :, 0], k[:, n:, :, 0] = 1, 2
    scale = 8 / 1.4426950408889634
    s = (k[0, :, 0] @ q[0, 0, 0]).double()
    assert s.min() > 2 ** 23 and s[-1] - s[0] == 1
    steps = (s.float() * (torch.tensor(scale) * 1.4426950408889634)).double()
    assert steps.min() > 2 ** 26 and steps[-1] - steps[0] == 8
    v = torch.randn(1, 2 * n, 1, D, generator=torch.Generator().manual_seed(1))
    c = R.case(q, k, v, [2 * n], mx)
    out = R.run(c, variant, scale=scale).double()[0, 0, 0]
    values = U.pool_values(c["v"], c["vs"])[c["table"].long()].flatten(1, 2)[0, :2 * n, 0]
    low, high = values[:n].mean(0), values[n:].mean(0)
    assert bool(((out - (low + 256 * high) / 257).abs() <= 1.01 * 2.0 ** -7 * values.abs().mean(0) * 2).all())
    ops.cuda_module().check_status()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("S,T", [(400, 40), (3000, 40), (3000, 1)])
def test_near_scores_of_large_size(mx, S, T):
    """Whole-number scores of 7.3 million to three more in the many-rows kernel, whose differences matter: they are taken before the
    scale, inside a run of keys and where runs are joined, so that only the first tiles' reference is rounded (a score may be
    off by 2^-13)."""
    g = torch.Generator().manual_seed(S)
    q = torch.full((2, T, 2, 128), 240.0)
    k = torch.full((2, S, 2, 128), 240.0)
    q[..., 0] = 1
    k[..., 0] = torch.randint(0, 3, (2, S, 2), generator=g).float()
    k[:, S // 2:S // 2 + S // 8, :, 0] = 3          # the largest lie in one or two runs
    v = torch.randn(2, S, 2, 128, generator=g).abs()
    v[:, S // 2:S // 2 + S // 8] *= -1              # what the runs weigh shows
    c = R.case(q, k, v, [S, S - 7], mx)
    R.hold(c, CHUNK, scale=1.0, score_error=2.0 ** -13)
