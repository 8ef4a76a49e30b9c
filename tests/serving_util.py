"""Plain 64-bit forms of the serving operators, written from their definitions, and the error bounds of the kernels."""
import math

import torch


def quantise(x):
    """bf16 [..., D] -> (values fp64 [..., D], scale exponents). One power of two per 32 channels, the smallest with
    448 * 2^e >= the block's largest magnitude; E4M3 keeps three bits behind the leading one down to 2^-6, then steps of 2^-9."""
    y = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 448.0)) / 448.0))
    e = torch.where(torch.exp2(e - 1) * 448.0 >= amax, e - 1, e)
    e = torch.where(torch.exp2(e) * 448.0 < amax, e + 1, e)
    e = torch.where(amax > 0, e.clamp(-126, 126), torch.zeros_like(e))
    v = y * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    v = torch.round(v / step) * step * torch.exp2(e)
    return v.reshape(x.shape), e.reshape(*x.shape[:-1], -1)


def pool_values(pool, scale):
    """fp64 [P, page, KV, D] of a code pool and its scale pool."""
    if scale is None:
        return pool.double()
    f = torch.exp2(scale.double() - 127).permute(0, 2, 1, 3)
    return (pool.view(torch.float8_e4m3fn).double().reshape(*f.shape, 32) * f[..., None]).reshape(pool.shape)


def attention(q, k, v, page_table, seq_lens, q_lens, window, scale=None):
    """q [B, T, H, D], pools as fp64 values [P, page, KV, D]. Returns (out, bound): the exact result and the largest error a
    kernel may have that rounds the probabilities and the result to bf16 (u = 2^-8 each) and computes scores in fp32.

    With w_j the exact weights and A = sum_j w_j |v_j|: rounding every p_j by at most u changes sum p_j v_j by u A sum p
    and the sum of the rounded p (which divides) by u sum p, so the quotient by u (A + |o|); an error d of every score changes
    it by at most 2 d A; the result's own rounding adds u |o|. A score is a D-term fp32 sum of exact products, scaled:
    d <= (D + 2) 2^-24 |scale| sum_i |q_i k_i| + 2^-21, the last term for the exponential (rounding of its argument, up to 2^-24
    of a magnitude of 2^2, and the unit's own 2^-22). All of it to first order; 1 % is added for what is left out."""
    B, T, H, D = q.shape
    KV, page = k.shape[2], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    u = 2.0 ** -8
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n = T if q_lens is None else max(0, min(T, int(q_lens[b])))
        L = int(seq_lens[b])
        S = min(L, page_table.shape[1] * page)
        if n == 0 or S <= 0:
            continue
        j = torch.arange(S, device=q.device)
        pg = page_table[b].long()[j // page]
        usable = (pg >= 0) & (pg < k.shape[0])
        kk = k[pg.clamp(0, k.shape[0] - 1), j % page]
        vv = v[pg.clamp(0, k.shape[0] - 1), j % page]
        at = torch.arange(L - n, L, device=q.device)[:, None]
        seen = (j[None] <= at) & usable[None]
        if window >= 0:
            seen = seen & (at - j[None] <= window)
        used = seen.any(0)
        kk = torch.where(used[:, None, None], kk, torch.zeros_like(kk))
        vv = torch.where(used[:, None, None], vv, torch.zeros_like(vv))
        some = seen.any(1)
        for h in range(H):
            qh, kh, vh = q[b, :n, h].double(), kk[:, h // (H // KV)], vv[:, h // (H // KV)]
            s = (qh @ kh.T * scale).masked_fill(~seen, float("-inf"))
            w = torch.where(some[:, None], torch.softmax(s, -1), torch.zeros_like(s))
            o, A = w @ vh, w @ vh.abs()
            size = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            d = (D + 2) * 2.0 ** -24 * size + 2.0 ** -21
            out[b, :n, h] = o
            bound[b, :n, h] = 1.01 * ((u + 2 * d) * A + 2 * u * o.abs())
    return out, bound


def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row at a time, in 64 bits; settings are lists or numbers (rounded to fp32 as the operator takes them)."""
    def f32(x):
        return float(torch.tensor(x, dtype=torch.float32))
    out = []
    R, V = logits.shape
    logits, u = logits.double().cpu(), u.double().cpu()
    for r in range(R):
        t, k, tp, mp = (x[r] if isinstance(x, (list, tuple)) else x for x in (temperature, top_k, top_p, min_p))
        t, tp, mp = f32(t), f32(tp), f32(mp)
        z = torch.where(logits[r].isnan(), torch.full_like(logits[r], -math.inf), logits[r])
        order = torch.argsort(z, descending=True, stable=True)
        top = z[order[0]]
        if top == -math.inf:
            out.append(-1)
            continue
        if not t > 0:
            out.append(int(order[0]))
            continue
        kept = order[:k] if k > 0 else order
        p = torch.exp(torch.where(z[kept] == top, torch.zeros_like(z[kept]), (z[kept] - top) / t))
        p = torch.where(z[kept] == -math.inf, torch.zeros_like(p), p)
        ok = p >= mp
        ok[0] = True
        kept, p = kept[ok], p[ok]
        if tp < 1:
            before = torch.cumsum(p, 0) - p
            n = max(1, int((before < tp * p.sum()).sum()))
            kept, p = kept[:n], p[:n]
        kept, at = torch.sort(kept)
        cum = torch.cumsum(p[at], 0)
        i = int((cum <= u[r] * cum[-1]).sum())
        out.append(int(kept[min(i, int((cum < cum[-1]).sum()))]))
    return torch.tensor(out)


def paged_case(seed, B, T, H, KV, D, page, lens, q_lens=None, mx=True, device="cpu", spare=3, stride_pad=0):
    """Random pools behind a scattered page table with only as many pages mapped as each sequence has, the rest -1. The
    pool's unmapped pages and the places behind a sequence's end hold NaN."""
    from nanochat_cpp_b200.ops import ref
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1)
    P = sum(need) + spare
    perm = torch.randperm(P, generator=g)
    table = torch.full((B, width), -1, dtype=torch.int32)
    k = torch.full((P, page, KV, D), float("nan"), dtype=torch.bfloat16)
    v = k.clone()
    at = 0
    for b in range(B):
        for i in range(need[b]):
            pg = int(perm[at])
            at += 1
            table[b, i] = pg
            m = min(page, lens[b] - i * page)
            x = torch.randn(m, KV, D, generator=g)
            k[pg, :m] = (x * 1.2 / x.square().mean(-1, keepdim=True).sqrt()).to(torch.bfloat16)
            v[pg, :m] = torch.randn(m, KV, D, generator=g).to(torch.bfloat16)
    q = torch.randn(B, T, H, D + stride_pad, generator=g)
    q = (q * 1.2 / q.square().mean(-1, keepdim=True).sqrt()).to(torch.bfloat16)
    ks = vs = None
    if mx:
        k, ks = ref.mx_kv_encode(k)
        v, vs = ref.mx_kv_encode(v)
        ks, vs = ks.permute(0, 2, 1, 3).contiguous(), vs.permute(0, 2, 1, 3).contiguous()
    c = dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32),
             q_lens=None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32))
    c = {n: x.to(device) if isinstance(x, torch.Tensor) else x for n, x in c.items()}
    c["q"] = c["q"][..., :D]
    return c
