"""The definitions of the serving operators on the CPU: against plain 64-bit forms, and what they refuse."""
import pytest
import torch

from nanochat_cpp_b200 import ops
from nanochat_cpp_b200.ops import ref
from nanochat_cpp_b200.ops.fp8 import ref_mx_dequantize, ref_mx_quantize

import serving_util as U


def test_scale_of_every_bf16_magnitude():
    """The block scale read off exponent and mantissa of the largest magnitude (as the kernels do) is the definition's,
    for every finite bf16 value."""
    bits = torch.arange(0, 0x7F80, dtype=torch.int32)
    x = bits.to(torch.int16).view(torch.bfloat16)
    e, m = bits >> 7, bits & 0x7F
    b = torch.where(m > 0x60, e - 7, e - 8).clamp(min=1)
    b = torch.where(bits == 0, torch.full_like(b, 127), b)
    rows = torch.zeros(len(x), 32, dtype=torch.bfloat16)
    rows[:, 0] = x
    _, eb = ref_mx_quantize(rows)
    assert torch.equal(eb[:, 0].int(), b)
    amax = x.double()
    holds = 448.0 * torch.exp2(b.double() - 127) >= amax
    small = (448.0 * torch.exp2(b.double() - 128) < amax) | (b == 1) | (bits == 0)
    assert bool(holds.all()) and bool(small.all())


def test_codes_spread_to_bf16():
    """E4M3 -> bf16 by moving the fields and one multiplication by 2^(b - 127 + 120), for every code and scale byte; above
    b = 134 the multiplication is in two steps, and byte 255 gives NaN."""
    code = torch.arange(256, dtype=torch.int32)
    finite = (code & 0x7F) != 0x7F
    moved = ((code & 0x80) << 8) | ((code & 0x7F) << 4)
    base = torch.where(moved >= 0x8000, moved - 0x10000, moved).to(torch.int16).view(torch.bfloat16)
    for b in list(range(1, 254)) + [255]:
        first = (b + 120 if b < 134 else 254) << 7
        second = 0x3F80 if b <= 134 else 0x7FC0 if b == 255 else (b - 134 + 127) << 7
        f1, f2 = (torch.tensor([x], dtype=torch.int32).to(torch.int16).view(torch.bfloat16) for x in (first, second))
        got = (base * f1) * f2
        want = ref_mx_dequantize(code.to(torch.uint8).view(torch.float8_e4m3fn).repeat(1, 1).view(8, 32),
                                 torch.full((8, 1), b, dtype=torch.uint8)).view(-1)
        if b == 255:
            assert bool(got.isnan().all())
            continue
        off = (got.double() - want.double()).abs()[finite]
        ok = (off == 0) | (off <= 2.0 ** -133) | (got[finite] == want[finite].to(torch.bfloat16))
        assert bool(ok.all()), b


@pytest.mark.parametrize("B,T,KV,D,page", [(2, 5, 3, 64, 16), (1, 40, 2, 128, 7)])
def test_append_and_read_back(B, T, KV, D, page):
    pages = -(-(T + 3) // page)
    k_pool = torch.full((B * pages, page, KV, D), 9, dtype=torch.uint8)
    scale = torch.full((B * pages, KV, page, D // 32), 9, dtype=torch.uint8)
    pools = [k_pool, k_pool.clone(), scale, scale.clone()]
    before = [p.clone() for p in pools]
    g = torch.Generator().manual_seed(1)
    k, v = ((torch.randn(B, T, KV, D, generator=g) * 3).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(B * pages, generator=g).to(torch.int32).view(B, pages)
    pos = torch.arange(3, T + 3, dtype=torch.int32)[None].repeat(B, 1)
    pos[:, 2] = -1
    ops.kv_append_mx(*pools, table, pos, k, v)
    for x, y in zip((k, v), ops.kv_read_mx(*pools, table, pos)):
        value = U.quantise(x)[0]
        value[:, 2] = 0
        assert torch.equal(y, value.to(torch.bfloat16))
    ops.kv_append_mx(*pools, table, torch.full_like(pos, -1), k, v)
    untouched = torch.ones(B * pages * page, dtype=torch.bool)
    slots = table.long().gather(1, pos.clamp_min(0).long() // page) * page + pos.clamp_min(0).long() % page
    untouched[slots[pos >= 0]] = False
    for a, b in zip(pools[:2], before[:2]):
        assert torch.equal(a.view(-1, KV, D)[untouched], b.view(-1, KV, D)[untouched])


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("H,KV,D,page,window", [(4, 2, 64, 16, -1), (6, 2, 128, 5, 20), (3, 3, 64, 16, 0)])
def test_chunk_attention(mx, H, KV, D, page, window):
    T = 7
    new, past = [7, 0, 1, 4], [0, 30, 90, 17]
    c = U.paged_case(3, 4, T, H, KV, D, page, [a + b for a, b in zip(new, past)], new, mx=mx)
    got = ops.paged_chunk_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["q_lens"], window, None, c["ks"], c["vs"])
    want, bound = U.attention(c["q"], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), c["table"], c["lens"],
                              c["q_lens"], window)
    assert bool(((got.double() - want).abs() <= bound).all())
    assert not got[1].any() and not got[2, 1:].any()
    if mx:
        one = ops.paged_decode_attention_mx(c["q"][:, 0], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"], window)
        want, bound = U.attention(c["q"][:, :1], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), c["table"],
                                  c["lens"], None, window)
        assert bool(((one[:, None].double() - want).abs() <= bound).all())


def test_chunk_attention_is_decode_attention_for_one_token():
    c = U.paged_case(5, 3, 1, 4, 2, 64, 16, [1, 33, 70], mx=False)
    a = ops.paged_chunk_attention(c["q"], c["k"], c["v"], c["table"], c["lens"])
    k, v = (torch.where(x.isnan(), torch.zeros_like(x), x) for x in (c["k"], c["v"]))
    b = ops.paged_decode_attention(c["q"][:, 0], k, v, c["table"], c["lens"])
    assert (a[:, 0].float() - b.float()).abs().max() <= 2.0 ** -7 * b.float().abs().max()


@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.05), (0.0, 0, 1.0, 0.0), (1.0, 3, 0.0, 1.0)])
def test_sample_rows(t, k, p, m):
    g = torch.Generator().manual_seed(0)
    z = (torch.randn(9, 700, generator=g) * 2).to(torch.bfloat16)
    z[1], z[2, 5], z[3] = float("-inf"), float("nan"), 0.0
    u = torch.rand(9, generator=g)
    assert torch.equal(ops.sample_rows(z, u, t, k, p, m), U.sample(z, u, t, k, p, m))


def test_sample_rows_follows_the_distribution():
    """20000 draws of one row against the probabilities: the counts lie within six standard deviations."""
    z = torch.tensor([[1.0, 3.0, 2.0, -1.0, 2.5]]).repeat(20000, 1)
    u = (torch.arange(20000, dtype=torch.float32) + 0.5) / 20000
    n = torch.bincount(ops.sample_rows(z, u, 0.8), minlength=5).double()
    p = torch.softmax(z[0].double() / 0.8, 0)
    assert bool(((n - 20000 * p).abs() <= 6 * (20000 * p * (1 - p)).sqrt()).all())


# ------------------------------------------------------------------------------------------------ refusals
def _cache_args(dev):
    k = torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device=dev)
    s = torch.zeros(4, 2, 16, 2, dtype=torch.uint8, device=dev)
    return dict(k_pool=k, v_pool=k.clone(), k_scale=s, v_scale=s.clone(),
                page_table=torch.zeros(2, 2, dtype=torch.int32, device=dev),
                positions=torch.zeros(2, 1, dtype=torch.int32, device=dev),
                k_new=torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device=dev),
                v_new=torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device=dev))


CACHE_FAULTS = [("k_pool", lambda x: x.float()), ("k_pool", lambda x: x[:, ::2]), ("v_pool", lambda x: x[:3]),
                ("k_scale", lambda x: x.transpose(1, 2).contiguous()), ("v_scale", lambda x: x[..., :1]),
                ("page_table", lambda x: x.long()), ("page_table", lambda x: x[:1]), ("positions", lambda x: x.long()),
                ("positions", lambda x: x[:, 0]), ("k_new", lambda x: x[:, :, :1]), ("v_new", lambda x: x[..., :32]),
                ("k_new", lambda x: x[0])]


def refusals_of_the_cache(dev):
    for name, change in CACHE_FAULTS:
        a = _cache_args(dev)
        a[name] = change(a[name])
        with pytest.raises((ValueError, RuntimeError)):
            ops.kv_append_mx(**a)
        if name not in ("k_new", "v_new"):
            with pytest.raises((ValueError, RuntimeError)):
                ops.kv_read_mx(**{n: x for n, x in a.items() if n not in ("k_new", "v_new")})
    a = _cache_args(dev)
    a["k_pool"], a["v_pool"] = a["k_pool"][..., :32].contiguous(), a["v_pool"][..., :32].contiguous()
    with pytest.raises((ValueError, RuntimeError)):
        ops.kv_append_mx(**a)


def refusals_of_attention(dev):
    def args(mx):
        c = _cache_args(dev)
        k = c["k_pool"] if mx else torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=dev)
        return dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device=dev), k_pool=k, v_pool=k.clone(),
                    page_table=c["page_table"], seq_lens=torch.ones(2, dtype=torch.int32, device=dev),
                    q_lens=torch.ones(2, dtype=torch.int32, device=dev), k_scale=c["k_scale"] if mx else None,
                    v_scale=c["v_scale"] if mx else None)
    faults = [("q", lambda x: x[:, :, :3]), ("q", lambda x: x[0]), ("q", lambda x: torch.cat([x, x], -1)),
              ("k_pool", lambda x: x.float()), ("v_pool", lambda x: x[:3]), ("k_pool", lambda x: x[..., :32]),
              ("page_table", lambda x: x.long()), ("page_table", lambda x: x[:1]), ("page_table", lambda x: x[:, :0]),
              ("seq_lens", lambda x: x.long()), ("seq_lens", lambda x: x[:1]), ("q_lens", lambda x: x[:1]),
              ("q_lens", lambda x: x.float())]
    for mx in (False, True):
        for name, change in faults:
            a = args(mx)
            a[name] = change(a[name])
            with pytest.raises((ValueError, RuntimeError)):
                ops.paged_chunk_attention(**a)
    a = args(True)
    a["v_scale"] = None
    with pytest.raises((ValueError, RuntimeError)):
        ops.paged_chunk_attention(**a)
    a = args(True)
    with pytest.raises((ValueError, RuntimeError)):       # four dimensions: one token only
        ops.paged_decode_attention_mx(a["q"], a["k_pool"], a["v_pool"], a["k_scale"], a["v_scale"], a["page_table"], a["seq_lens"])


def refusals_of_sampling(dev):
    z, u = torch.zeros(3, 10, device=dev), torch.zeros(3, device=dev)
    i3 = torch.ones(3, dtype=torch.int32, device=dev)
    for a in [(z[0], u), (z.half(), u), (z.long(), u), (z, u[:2]), (z, u.double()), (z[:, :0], u), (z.t().contiguous().t(), u),
              (z, u, i3), (z, u, 1.0, u), (z, u, 1.0, i3[:2]), (z, u, 1.0, 0, i3), (z, u, 1.0, 0, 1.0, u[:1])]:
        with pytest.raises((ValueError, RuntimeError)):
            ops.sample_rows(*a)


def test_refusals_on_the_cpu():
    refusals_of_the_cache("cpu")
    refusals_of_attention("cpu")
    refusals_of_sampling("cpu")
