"""Attention over MXFP8 pages whose blocks differ by many powers of two, and infinities and NaN, by both kernels."""
import pytest
import torch

from nanochat_cpp_b200 import ops

import serving_range_util as R

pytestmark = pytest.mark.gpu

ROWS, CHUNK = R.ROWS, R.CHUNK


def _spread(case, g, B, S, KV, D, T, H):
    """(q, k, v) with finite numbers whose blocks lie up to 80 powers of two apart."""
    q, k, v = R.unit(g, B, T, H, D), R.unit(g, B, S, KV, D), torch.randn(B, S, KV, D, generator=g)
    two = lambda e: torch.exp2(torch.tensor(e, dtype=torch.float32)).repeat_interleave(32)  # noqa: E731
    e = [30, 5, -30, 0][: D // 32]
    if case == "value blocks":                 # channels of different size
        v = v * two(e)
    elif case == "key blocks":                 # the queries' channels make up for it
        k, q = k * two(e), q * two([-x for x in e])
    elif case == "query channels":             # a channel that no key uses hides the others
        q[..., 5] = 2.0 ** 35
        k[..., 5] = 0
    elif case == "one large value":            # of a key that has no weight
        k[:, S // 2] = -60 * q[:, 0, :: H // KV]
        q[:] = q[:, :1, :: H // KV].repeat_interleave(H // KV, 2)
        v[:, S // 2] *= 2.0 ** 40
    elif case == "one large key":              # likewise
        q[:] = q[:, :1, :: H // KV].repeat_interleave(H // KV, 2)
        k[:, S // 3] = -2.0 ** 33 * q[:, 0, :: H // KV]
    elif case == "last key large":             # seen by the last row alone, where it has no weight
        q[:] = q[:, :1, :: H // KV].repeat_interleave(H // KV, 2)
        k[:, -1], v[:, -1] = -2.0 ** 35 * q[:, 0, :: H // KV], v[:, -1] * 2.0 ** 38
    elif case == "zero among small":           # an empty block stands at scale one
        k, v, q = k * 2.0 ** -25, v * 2.0 ** -30, q * 2.0 ** 25
        v[:, ::7], k[:, ::5, :, :32] = 0, 0
    elif case == "growing":                    # every page larger than the one before, seen through a window
        up = torch.exp2(torch.arange(S).float() / 8 % 80 - 40)[None, :, None, None]
        v = v * up
    elif case == "falling":
        v = v * torch.exp2(40 - torch.arange(S).float() / 8 % 80)[None, :, None, None]
    elif case == "keys of any size":
        x = torch.randint(-60, 0, (B, S, 1, 1), generator=g).float()
        k = k * torch.exp2(x)
        k[:, ::9] = R.unit(g, B, len(range(0, S, 9)), KV, D)
    return q, k, v


CASES = ["value blocks", "key blocks", "query channels", "one large value", "one large key", "last key large", "zero among small",
         "growing", "falling", "keys of any size"]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("variant", [ROWS, CHUNK])
@pytest.mark.parametrize("D,T,H,KV,S,page", [(128, 1, 4, 4, 700, 16), (128, 6, 4, 2, 300, 16), (64, 5, 8, 2, 260, 8), (64, 40, 2, 2, 1500, 32)])
def test_blocks_far_apart(case, variant, D, T, H, KV, S, page):
    if variant == CHUNK and page % 16:
        pytest.skip("pages of the other kernel")
    g = torch.Generator().manual_seed(D + T)
    c = R.case(*_spread(case, g, 2, S, KV, D, T, H), [S, S], True, page=page)
    R.hold(c, variant)
    R.hold(c, variant, window=40)


@pytest.mark.parametrize("case", ["value blocks", "one large value", "zero among small", "growing"])
def test_blocks_far_apart_decode(case):
    g = torch.Generator().manual_seed(7)
    c = R.case(*_spread(case, g, 3, 1200, 2, 128, 1, 4), [1200, 600, 33], True)
    out = ops.paged_decode_attention_mx(c["q"][:, 0], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"])
    want, bound = R.expect(c)
    assert bool(((out[:, None].double() - want).abs() <= bound).all())
    ops.cuda_module().check_status()


@pytest.mark.parametrize("variant", [ROWS, CHUNK])
def test_infinities_and_nan_that_are_seen(variant):
    """In one head's key or value: that head's rows that see it are not finite where the formula's are not; the other heads
    and the other sequence are as they were."""
    g = torch.Generator().manual_seed(3)
    B, S, H, D = 2, 200, 2, 64
    base = R.unit(g, B, 1, H, D), R.unit(g, B, S, H, D), torch.randn(B, S, H, D, generator=g)
    for mx in (False, True):
        want = R.run(R.case(*base, [S, S], mx), variant)
        for what in (float("nan"), float("inf"), float("-inf")):
            for which in ("k", "v"):
                q, k, v = (x.clone() for x in base)
                (k if which == "k" else v)[0, 100, 0, 7] = what
                out = R.run(R.case(q, k, v, [S, S], mx), variant)
                assert torch.equal(out[1], want[1]) and torch.equal(out[0, :, 1], want[0, :, 1])
                if which == "v":
                    assert not bool(out[0, 0, 0, 7].isfinite())
                elif what != what:
                    assert bool(out[0, 0, 0].isnan().all())
    ops.cuda_module().check_status()


@pytest.mark.parametrize("variant,kb,vb", [(ROWS, 0, 0), (ROWS, 0, 127)] +
                         [(v, kb, vb) for v in (ROWS, CHUNK) for kb, vb in ((127, 0), (5, 5), (100, 200), (220, 5))])
@pytest.mark.parametrize("D,page,T", [(128, 16, 1), (64, 48, 3), (64, 32, 20)])
def test_scale_bytes_at_the_ends(variant, D, page, T, kb, vb):
    """Pools that a program filled itself: any byte but 255 is a power of two. The queries bring the scores back to order one. (The
    many-rows kernel makes bf16 of a key, which holds every code from byte 3 on.)"""
    g = torch.Generator().manual_seed(kb + vb)
    B, H, KV, S = 2, 4, 2, 90
    q = R.unit(g, B, T, H, D) * 2.0 ** (127 - max(kb, 10))
    c = R.case(q, R.unit(g, B, S, KV, D), torch.randn(B, S, KV, D, generator=g), [S, 50], True, page=page)
    for n, b in (("k", kb), ("v", vb)):
        c[n + "s"] += b - 120                      # blocks of order one have a byte of 119 to 121
        if b == 0:
            c[n + "s"].zero_()
    R.hold(c, variant)


@pytest.mark.parametrize("variant", [ROWS, CHUNK])
@pytest.mark.parametrize("size,key_size", [(0.0, 1.0), (2.0 ** -125, 2.0 ** 115), (2.0 ** -132, 2.0 ** 118), (2.0 ** 110, 2.0 ** -110), (2.0 ** 60, 2.0 ** -90)])
@pytest.mark.parametrize("T", [1, 9])
def test_queries_of_any_size(variant, size, key_size, T):
    """Zeros (every key weighs the same), numbers below bf16's normal range and large ones, some channels zero."""
    g = torch.Generator().manual_seed(5)
    B, H, KV, D, S = 2, 4, 2, 128, 300
    q = R.unit(g, B, T, H, D) * size
    q[..., 3::7] = 0
    q[0, 0, 0] = 0
    R.hold(R.case(q, R.unit(g, B, S, KV, D) * key_size, torch.randn(B, S, KV, D, generator=g), [S, S - 100], True), variant)
    R.hold(R.case(q, R.unit(g, B, S, KV, D) * key_size, torch.randn(B, S, KV, D, generator=g), [S, S - 100], False), variant)
