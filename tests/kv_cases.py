"""Shared helpers of the paged key-value cache's tests: caches with random pages, and the operators in 64 bits on
the CPU, from dense arrays [Hkv, tokens, D] of each sequence."""
import math

import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}     # a rounding's half step, relative to the value
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # and the least one, of subnormal values


def blocks(x, page, v):
    """[Hkv, tokens, D] (a multiple of page tokens) as pages [n, Hkv, page/32, D/32, 32, 32] of K, or of V."""
    H, T, D = x.shape
    x = x.reshape(H, T // page, page // 32, 32, D // 32, 32).permute(1, 0, 2, 4, 3, 5)
    return (x.transpose(4, 5) if v else x).contiguous()


def dense(pages, v):
    """The inverse: pages [n, Hkv, page/32, D/32, 32, 32] as [Hkv, tokens, D]."""
    x = pages.transpose(4, 5) if v else pages
    n, H, p32, db = x.shape[:4]
    return x.permute(1, 0, 2, 4, 3, 5).reshape(H, n * p32 * 32, db * 32)


class Case:
    """A cache on the device, and what its sequences hold in fp64 on the CPU.  Pages that no sequence has, and what
    lies behind a sequence's last token, hold NaN and infinities."""

    def __init__(self, dev, lens, Hkv, D, page, dtype, spare=2, extra_pages=1, weights=False, seed=0, mul=1.0, trend=0.0):
        from tokamak_amd import attn
        g = torch.Generator().manual_seed(seed)
        self.B, self.Hkv, self.D, self.page, self.dtype, self.dev = len(lens), Hkv, D, page, dtype, dev
        dt = DT[dtype]
        need = [(n + page - 1) // page for n in lens]
        self.max_pages = max(1, max(need)) + extra_pages
        total = sum(need) + spare
        junk = torch.tensor([float("nan"), float("inf"), -float("inf")])[torch.randint(0, 3, (total, Hkv, page // 32, D // 32, 32, 32), generator=g)]
        k, v = junk.to(dt), junk.flip(0).to(dt)
        table = torch.full((self.B, self.max_pages), -1, dtype=torch.int32)
        perm = torch.randperm(total, generator=g)
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lens):
            x = [(torch.randn(Hkv, n, D, generator=g) * mul).to(dt) for _ in range(2)]
            if trend and n:       # scores that grow along the keys: one direction, longer and longer
                x[0] = (x[0].float() + torch.arange(n)[None, :, None] * trend / n).to(dt)
            self.k.append(x[0].double())
            self.v.append(x[1].double())
            mine = perm[at:at + need[b]]
            at += need[b]
            table[b, :need[b]] = mine.to(torch.int32)
            if n:
                for pool, y, isv in ((k, x[0], False), (v, x[1], True)):
                    d = dense(pool[mine], isv)
                    d[:, :n] = y
                    pool[mine] = blocks(d, page, isv)
        self.free = perm[at:]
        self.lens = list(lens)
        self.weight = torch.rand(self.B, Hkv, self.max_pages * page, generator=g) if weights else None
        self.cache = attn.KvCache(k.to(dev), v.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                                  None if self.weight is None else self.weight.to(dev))

    def held(self, b, cache=None):
        """(K, V) of sequence b as the device holds them, fp64 [Hkv, len, D]."""
        c = cache or self.cache
        n = int(c.kv_len[b])
        t = c.table[b, :(n + self.page - 1) // self.page].long()
        return [dense(x[t].cpu().double(), isv)[:, :n] for x, isv in ((c.k, False), (c.v, True))]


def decode_ref(q, ks, vs, Hkv, scale):
    """q fp64 [B, Hq, D], ks / vs lists of [Hkv, n, D].  Returns o, lse, the weights each position gets (a list of
    [Hkv, n]) and bounds on the error of o's fp32 sums and of lse.

    The bounds: a score is a sum of D products in fp32, off by at most (D + 2) 2^-24 sum |q_i k_i| scale (one
    rounding a term, one of the scale, one of the product with it), its exponential by that relative error and
    4 * 2^-23 of its own, twice: numerator and denominator.  Sums over n keys add n 2^-24 relative to the sum of
    absolute values, P's two halves 2^-21."""
    B, Hq, D = q.shape
    G = Hq // Hkv
    o, lse, w, eo, el = torch.zeros_like(q), torch.full((B, Hq), -math.inf, dtype=torch.float64), [], torch.zeros_like(q), torch.zeros(B, Hq, dtype=torch.float64)
    for b in range(B):
        n = ks[b].shape[1]
        w.append(torch.zeros(Hkv, n, dtype=torch.float64))
        if n == 0:
            continue
        for h in range(Hkv):
            x = q[b, h * G:(h + 1) * G]
            s = x @ ks[b][h].T * scale
            L = torch.logsumexp(s, 1)
            p = torch.exp(s - L[:, None])
            hs = slice(h * G, (h + 1) * G)
            o[b, hs], lse[b, hs] = p @ vs[b][h], L
            w[b][h] = p.sum(0)
            ds = ((D + 2) * 2.0 ** -24 * scale * (x.abs() @ ks[b][h].abs().T) + 2.0 ** -23 * s.abs()).amax(1) + 8 * 2.0 ** -23
            el[b, hs] = ds + n * 2.0 ** -24 + 4 * 2.0 ** -24 * (L.abs() + 16)
            eo[b, hs] = (2 * ds + n * 2.0 ** -23 + 2.0 ** -21)[:, None] * (p @ vs[b][h].abs())
    return o, lse, w, eo, el


def check_decode(case, q, o, lse, Hq, scale=None):
    """Compares the device's o and lse with the 64-bit ones; returns the reference's weights."""
    D = case.D
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    ro, rl, w, eo, el = decode_ref(q.cpu().double().reshape(case.B, Hq, D), case.k, case.v, case.Hkv, scale)
    go, gl = o.cpu().double().reshape(case.B, Hq, D), lse.cpu().double()
    assert torch.isfinite(go).all()
    tol = eo + HALF[case.dtype] * (ro.abs() + eo) + TINY[case.dtype]
    worst = ((go - ro).abs() / tol).max().item()
    some = torch.isfinite(rl)
    assert torch.equal(some, torch.isfinite(gl)) and torch.equal(gl[~some], rl[~some])
    worst_l = ((gl - rl).abs()[some] / el[some]).max().item() if some.any() else 0.0
    print(f"    o {worst:.3f}, lse {worst_l:.3f} of their bounds", flush=True)
    assert worst <= 1.0 and worst_l <= 1.0
    return w


def evict_ref(w, n, budget, sink, recent):
    """Old positions kept of one head, ascending, by one weight after another (w: a list of n floats)."""
    if n <= budget:
        return list(range(n))
    mid = list(range(sink, n - recent))
    best = sorted(mid, key=lambda i: (1, 0.0, i) if math.isnan(w[i]) else (0, -w[i], i))[:budget - sink - recent]
    return list(range(sink)) + sorted(best) + list(range(n - recent, n))
