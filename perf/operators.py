"""Measured cases of the serving operators: the MXFP8 key / value cache (append, read back), attention over it for single
tokens and for chunks of new tokens, and sampling with given random numbers.

`run` computes each in plain torch where `own` is false and calls the package's operators where it is true.
"""
import math

import torch

own = False

BLOCK = 32          # channels that share one power-of-two scale
PAGE = 16           # tokens a page
E4M3_MAX = 448.0


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the write of one decode step for 64 sequences of a 10-head model, and the rows read back
        dict(name="append_step_64", op="append", B=64, T=1, KV=10, D=128, span=2048),
        # prompts of up to 2048 tokens written at once
        dict(name="append_prompts_16x2048", op="append", B=16, T=2048, KV=10, D=128, span=2048),
        # one chat user, about 2000 cached tokens: latency
        dict(name="decode_1x2000", op="decode", B=1, H=10, KV=10, D=128, lo=2000, hi=2000, window=-1),
        # a batch of 64 conversations of mixed length
        dict(name="decode_64_ragged", op="decode", B=64, H=10, KV=10, D=128, lo=1, hi=2048, window=-1),
        # long documents, grouped heads: the whole cache streams through
        dict(name="decode_32_long_gqa", op="decode", B=32, H=10, KV=5, D=128, lo=8192, hi=32768, window=-1),
        # four drafted tokens a sequence are verified against a bf16 cache
        dict(name="chunk_verify_64x4", op="chunk", B=64, T=4, H=10, KV=10, D=128, tlo=1, past_lo=100, past_hi=2000,
             window=-1, mx=False),
        # ragged prompts from an empty cache on a windowed layer
        dict(name="chunk_prompts_8x2048", op="chunk", B=8, T=2048, H=10, KV=10, D=128, tlo=300, past_lo=0, past_hi=0,
             window=1024, mx=False),
        # a 2048-token piece of a long document over a quantised cache
        dict(name="chunk_long_2x2048_mx", op="chunk", B=2, T=2048, H=10, KV=5, D=128, tlo=2000, past_lo=12000,
             past_hi=16384, window=-1, mx=True),
        # small model, odd sizes, a turn of a chat continued
        dict(name="chunk_odd_3x77_mx", op="chunk", B=3, T=77, H=4, KV=2, D=64, tlo=5, past_lo=0, past_hi=700, window=300,
             mx=True),
        # one chat user: the usual settings
        dict(name="sample_1x65536", op="sample", R=1, V=65536, bf16=False, temperature=0.8, top_k=50, top_p=0.95,
             min_p=0.0, mixed=False),
        # a batch of rollouts from the nucleus
        dict(name="sample_64x65536", op="sample", R=64, V=65536, bf16=False, temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.02, mixed=False),
        # many requests, each with settings of its own, straight from bf16 logits
        dict(name="sample_512x32768_mixed", op="sample", R=512, V=32768, bf16=True, temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, mixed=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "chunk", "chunk", "chunk", "sample", "sample"])
    D = rng.choice([64, 128, 128])
    KV = rng.choice([1, 2, 4, 5, 6, 8, 10, 13])
    G = rng.choice([1, 1, 2, 3, 4, 5, 8])
    if op == "append":
        B = _log(rng, 1, 64)
        T = _log(rng, 1, max(1, 2048 * 160 // (B * KV)) if B * KV > 160 else 2048)
        return dict(op=op, B=B, T=T, KV=KV, D=D, span=T + _log(rng, 1, 2048))
    if op == "decode":
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, min(32768, 32 * 32768 * 5 // (B * KV))))
        return dict(op=op, B=B, H=KV * G, KV=KV, D=D, lo=rng.choice([0, 1, max(1, hi // 2)]), hi=hi,
                    window=rng.choice([-1, -1, rng.randint(0, 2 * hi)]))
    if op == "chunk":
        B = _log(rng, 1, 64)
        H = KV * G
        T = _log(rng, 1, max(1, min(2048, 2 * 2048 * 10 // (B * H) * 4)))
        most = 2 * 2048 * 18432 * 10 // (B * H * T)      # scores of the largest listed case
        past = _log(rng, 1, max(1, min(16384, most - T)))
        return dict(op=op, B=B, T=T, H=H, KV=KV, D=D, tlo=rng.choice([0, 1, T]), past_lo=0, past_hi=past,
                    window=rng.choice([-1, -1, rng.randint(0, T + past)]), mx=rng.random() < 0.5)
    R = _log(rng, 1, 512)
    V = _log(rng, 100, min(131072, 512 * 32768 // R))
    return dict(op=op, R=R, V=V, bf16=rng.random() < 0.5, temperature=round(rng.uniform(0.3, 1.5), 3),
                top_k=rng.choice([0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, round(rng.uniform(0.5, 1.0), 3)]),
                min_p=rng.choice([0.0, 0.05]), mixed=rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n whole numbers between lo and hi, hi first, spread by the golden ratio."""
    return [int(round(hi - (hi - lo) * ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _heads(g, *shape):
    """Rows as the query / key preparation leaves them: unit root mean square over the head, times 1.2."""
    x = torch.randn(*shape, device="cuda", generator=g)
    return (x * (1.2 / x.square().mean(-1, keepdim=True).sqrt())).to(torch.bfloat16)


def _encode(x):
    """bf16 [P, page, KV, D] -> (codes uint8 of that shape, scale bytes uint8 [P, KV, page, D / 32])."""
    P, page, KV, D = x.shape
    blocks = x.float().view(P, page, KV, D // BLOCK, BLOCK)
    amax = blocks.abs().amax(-1)
    mant, expo = torch.frexp(amax)                  # amax = mant * 2^expo, mant in [0.5, 1); 448 = 0.875 * 2^9
    b = (expo - 9 + (mant > 0.875).int() + 127).clamp(1, 253)
    b = torch.where(amax > 0, b, torch.full_like(b, 127))
    inv = torch.exp2((127 - b).float())
    codes = (blocks * inv[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).view(P, page, KV, D)
    return codes, b.to(torch.uint8).permute(0, 2, 1, 3).contiguous()


def _table(g, B, pages):
    return torch.randperm(B * pages, device="cuda", generator=g).to(torch.int32).view(B, pages)


def _cache(g, B, pages, KV, D, mx):
    k, v = _heads(g, B * pages, PAGE, KV, D), torch.randn(B * pages, PAGE, KV, D, device="cuda", generator=g).to(torch.bfloat16)
    if not mx:
        return dict(k=k, v=v, ks=None, vs=None)
    (k, ks), (v, vs) = _encode(k), _encode(v)
    return dict(k=k, v=v, ks=ks, vs=vs)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _append_starts(case):
    return _spread(case["B"], 0, case["span"] - case["T"])


def _append_counts(case):
    return _spread(case["B"], (case["T"] + 1) // 2, case["T"])


def _chunk_lens(case):
    return _spread(case["B"], case["tlo"], case["T"]), _spread(case["B"], case["past_lo"], case["past_hi"])


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "append":
        B, T, KV, D = case["B"], case["T"], case["KV"], case["D"]
        pages = -(-case["span"] // PAGE)
        s["k_new"], s["v_new"] = _heads(g, B, T, KV, D), torch.randn(B, T, KV, D, device="cuda", generator=g).to(torch.bfloat16)
        t = torch.arange(T, dtype=torch.int32, device="cuda")[None, :]
        pos = t + _ints(_append_starts(case))[:, None]
        s["pos"] = torch.where(t < _ints(_append_counts(case))[:, None], pos, torch.full_like(pos, -1)).contiguous()
        s["table"] = _table(g, B, pages)
        for n in ("k", "v"):
            s[n] = torch.zeros(B * pages, PAGE, KV, D, dtype=torch.uint8, device="cuda")
            s[n + "s"] = torch.full((B * pages, KV, PAGE, D // BLOCK), 127, dtype=torch.uint8, device="cuda")
    elif case["op"] == "decode":
        B = case["B"]
        pages = -(-max(1, case["hi"]) // PAGE)
        s.update(_cache(g, B, pages, case["KV"], case["D"], True))
        s["q"] = _heads(g, B, case["H"], case["D"])
        s["table"], s["lens"] = _table(g, B, pages), _ints(_spread(B, case["lo"], case["hi"]))
    elif case["op"] == "chunk":
        B = case["B"]
        new, past = _chunk_lens(case)
        pages = -(-max(1, case["T"] + case["past_hi"]) // PAGE)
        s.update(_cache(g, B, pages, case["KV"], case["D"], case["mx"]))
        s["q"] = _heads(g, B, case["T"], case["H"], case["D"])
        s["table"] = _table(g, B, pages)
        s["q_lens"], s["lens"] = _ints(new), _ints([a + b for a, b in zip(new, past)])
    else:
        R, V = case["R"], case["V"]
        z = torch.randn(R, V, device="cuda", generator=g) * 2.5
        likely = torch.randint(0, V, (R, 12), device="cuda", generator=g)          # what the context calls for
        z.scatter_add_(1, likely, 6 + 3 * torch.randn(R, 12, device="cuda", generator=g))
        z = z.to(torch.bfloat16)                                                   # the head's product is bf16: ties
        s["logits"] = z if case["bf16"] else 15.0 * torch.tanh(z.float() / 15.0)
        s["u"] = torch.rand(R, device="cuda", generator=g)
        if case["mixed"]:
            def pick(values, dtype):
                at = torch.randint(0, len(values), (R,), device="cuda", generator=g)
                return torch.tensor(values, dtype=dtype, device="cuda")[at]
            s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.2], torch.float32)
            s["top_k"] = pick([0, 1, 20, 50, 200], torch.int32)
            s["top_p"] = pick([0.8, 0.9, 0.95, 1.0], torch.float32)
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
    return s


# ---------------------------------------------------------------------------------------------------- the plain forms
def _values(codes, scale):
    """fp32 [P, page, KV, D] of a quantised pool."""
    P, page, KV, D = codes.shape
    f = torch.exp2(scale.float() - 127.0).permute(0, 2, 1, 3)
    return (codes.view(torch.float8_e4m3fn).float().view(P, page, KV, D // BLOCK, BLOCK) * f[..., None]).view(P, page, KV, D)


def _pages(pool, table):
    """[B, pages * page, KV, D]"""
    B, n = table.shape
    return pool[table.long()].reshape(B, n * pool.shape[1], *pool.shape[2:])


def _plain_append(s):
    pos = s["pos"].long()
    ok = pos >= 0
    at = pos.clamp_min(0)
    page, slot = torch.gather(s["table"].long(), 1, at // PAGE), at % PAGE
    back = []
    for n in ("k", "v"):
        codes, scale = _encode(s[n + "_new"])               # [B, T, KV, D], [B, KV, T, D / 32]
        s[n][page[ok], slot[ok]] = codes[ok]
        s[n + "s"][page[ok], :, slot[ok]] = scale.permute(0, 2, 1, 3)[ok]
        f = torch.exp2(s[n + "s"][page, :, slot].float() - 127.0)
        row = s[n][page, slot].view(torch.float8_e4m3fn).float().view(*f.shape, BLOCK) * f[..., None]
        row = row.view(s[n + "_new"].shape)
        back.append(torch.where(ok[..., None, None], row, torch.zeros_like(row)).to(torch.bfloat16))
    return dict(k=back[0], v=back[1])


def _plain_attention(q, k, v, qpos, window):
    """q [B, T, H, D], k / v fp32 [B, S, KV, D], qpos [B, T] (-1: an empty row)."""
    B, T, H, D = q.shape
    KV, S = k.shape[2], k.shape[1]
    qf = q.float().view(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4)             # [B, KV, G, T, D]
    s = torch.matmul(qf, k.permute(0, 2, 3, 1)[:, :, None]) * (1.0 / math.sqrt(D))
    j = torch.arange(S, device=q.device)
    seen = j <= qpos[..., None]
    if window >= 0:
        seen = seen & (qpos[..., None] - j <= window)
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    o = torch.matmul(p, v.permute(0, 2, 1, 3)[:, :, None]) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(torch.bfloat16)


def _plain_sample(s):
    V = s["logits"].shape[1]

    def column(name, dtype):
        return torch.as_tensor(s[name], dtype=dtype, device="cuda").to(torch.float64).reshape(-1, 1)
    t, k = column("temperature", torch.float32), column("top_k", torch.int32)
    top_p, min_p = column("top_p", torch.float32), column("min_p", torch.float32)
    z, order = s["logits"].double().sort(dim=1, descending=True, stable=True)
    p = torch.exp((z - z[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    rank = torch.arange(V, device="cuda")[None, :]
    p = torch.where(((rank < k) | (k <= 0)) & (p >= min_p), p, torch.zeros_like(p))
    before = p.cumsum(1) - p
    p = torch.where((before < top_p * p.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0), p, torch.zeros_like(p))
    p = torch.where((t > 0) | (rank == 0), p, torch.zeros_like(p))
    cum = torch.zeros_like(p).scatter_(1, order, p).cumsum(1)
    return (cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(1)


def _plain(s):
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "sample":
        return _plain_sample(s)
    k, v = (_pages(s[n].float() if s[n + "s"] is None else _values(s[n], s[n + "s"]), s["table"]) for n in ("k", "v"))
    if s["op"] == "decode":
        return _plain_attention(s["q"][:, None], k, v, s["lens"].long()[:, None] - 1, s["window"])[:, 0]
    t = torch.arange(s["T"], device="cuda")[None, :]
    qpos = t + (s["lens"] - s["q_lens"]).long()[:, None]
    qpos = torch.where(t < s["q_lens"][:, None], qpos, torch.full_like(qpos, -1))
    return _plain_attention(s["q"], k, v, qpos, s["window"])


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if not own:
        return _plain(state)
    from nanochat_cpp_b200 import ops
    s = state
    if s["op"] == "append":
        ops.kv_append_mx(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["pos"], s["k_new"], s["v_new"])
        k, v = ops.kv_read_mx(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["pos"])
        return dict(k=k, v=v)
    if s["op"] == "decode":
        return ops.paged_decode_attention_mx(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"], s["window"])
    if s["op"] == "chunk":
        return ops.paged_chunk_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["q_lens"], s["window"],
                                         k_scale=s["ks"], v_scale=s["vs"])
    return ops.sample_rows(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def _visible(first, n, window):
    """Key positions that queries at first .. first + n - 1 see between them, and the (query, key) pairs."""
    pairs = sum(min(p + 1, window + 1) if window >= 0 else p + 1 for p in range(first, first + n))
    lowest = max(0, first - window) if window >= 0 else 0
    return (first + n - lowest if n else 0), pairs


def work(case):
    op = case["op"]
    if op == "append":
        n = sum(_append_counts(case))
        rows = case["B"] * case["T"]
        e = case["KV"] * case["D"]
        return dict(bytes=2 * (n * e * 2 + n * (e + e // BLOCK) + rows * e * 2) + 4 * rows, flops=4 * n * e)
    if op == "sample":
        n = case["R"] * case["V"]
        return dict(bytes=n * (2 if case["bf16"] else 4) + 12 * case["R"], flops=10 * n)
    H, KV, D, window = case["H"], case["KV"], case["D"], case["window"]
    if op == "decode":
        lens, new = _spread(case["B"], case["lo"], case["hi"]), [1] * case["B"]
        rows, mx = case["B"], True
        seen = [_visible(n - 1, 1, window) if n else (0, 0) for n in lens]
    else:
        new, past = _chunk_lens(case)
        rows, mx = case["B"] * case["T"], case["mx"]
        seen = [_visible(p, n, window) for n, p in zip(new, past)]
    keys, pairs = sum(k for k, _ in seen), sum(p for _, p in seen)
    row = KV * (D + D // BLOCK if mx else 2 * D)
    return dict(bytes=2 * keys * row + sum(new) * H * D * 2 + rows * H * D * 2, flops=4 * pairs * H * D)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        out = {}
        for n in ("k", "v"):
            x = s[n + "_new"].double()
            x = x.view(*x.shape[:-1], -1, BLOCK)
            amax = x.abs().amax(-1, keepdim=True)
            scale = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(-126, 126))
            scale = torch.where(scale / 2 * E4M3_MAX >= amax, scale / 2, scale)          # the smallest that holds amax
            scale = torch.where(scale * E4M3_MAX < amax, scale * 2, scale)
            y = x / torch.where(amax > 0, scale, torch.ones_like(scale))
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # 3 bits behind the leading one
            y = torch.round(y / step) * step * scale                                      # ties to even
            out[n] = torch.where((s["pos"] >= 0)[..., None, None], y.flatten(-2), torch.zeros_like(y.flatten(-2)))
        return out
    if op == "sample":
        tokens = []
        for r in range(case["R"]):
            z = s["logits"][r].double()
            t, k, tp, mp = (float(torch.as_tensor(s[n]).to(torch.float32).reshape(-1)[r if case["mixed"] else 0])
                            for n in ("temperature", "top_k", "top_p", "min_p"))
            order = torch.argsort(z, descending=True, stable=True)
            if t <= 0:
                tokens.append(order[0])
                continue
            kept = order[: int(k)] if k > 0 else order
            p = torch.exp((z[kept] - z[order[0]]) / t)
            kept, p = kept[p >= mp], p[p >= mp]
            if tp < 1:
                n = int(torch.searchsorted(torch.cumsum(p, 0), tp * p.sum())) + 1
                kept, p = kept[:n], p[:n]
            kept, at = torch.sort(kept)
            cum = torch.cumsum(p[at], 0)
            i = torch.searchsorted(cum, s["u"][r].double() * cum[-1], right=True)
            tokens.append(kept[min(int(i), len(kept) - 1)])
        return torch.stack(tokens)
    H, KV, D, B = case["H"], case["KV"], case["D"], case["B"]
    lens = s["lens"].tolist()
    new = [1 if n else 0 for n in lens] if op == "decode" else s["q_lens"].tolist()
    q = s["q"][:, None] if op == "decode" else s["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, L = new[b], lens[b]
        if not n:
            continue
        rows = s["table"][b].long()
        kv = []
        for name in ("k", "v"):
            x = s[name][rows].double() if s[name + "s"] is None else s[name][rows].view(torch.float8_e4m3fn).double()
            if s[name + "s"] is not None:
                x = x * torch.exp2(s[name + "s"][rows].double() - 127).transpose(1, 2).repeat_interleave(BLOCK, dim=-1)
            kv.append(x.flatten(0, 1)[:L])
        at = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None, :]
        hidden = (j > at) | ((at - j > case["window"]) if case["window"] >= 0 else (j < 0))
        for h in range(H):
            c = h // (H // KV)
            w = (q[b, :n, h].double() @ kv[0][:, c].T) / math.sqrt(D)
            out[b, :n, h] = torch.softmax(w.masked_fill(hidden, float("-inf")), -1) @ kv[1][:, c]
    return out[:, 0] if op == "decode" else out
