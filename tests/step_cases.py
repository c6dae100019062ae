"""Shared helpers of the tests of a serving step over the paged cache: the plan by a loop over the sequences, rotary
positions and attention of new rows in 64 bits (angles in 80) on the CPU, with bounds on what the device may be off by."""
import math

import numpy as np
import torch

from kv_cases import HALF, TINY


# ---- the plan -------------------------------------------------------------------------------------


def plan_ref(table, free, n_free, held, want, start, page, num_pages, rows):
    """The plan of lists, one sequence after another; returns all that it writes."""
    table, free, held, B, most = [list(r) for r in table], list(free), list(held), len(want), len(table[0])
    cap, top = most * page, max(0, min(n_free, num_pages))
    held = [max(0, min(h, most)) for h in held]
    ok = [0 <= s <= cap for s in start]
    want = [w if o and 0 < w <= cap - s else 0 for w, s, o in zip(want, start, ok)]
    goal = [-(-(s + w) // page) if o else h for w, s, o, h in zip(want, start, ok, held)]
    for b in range(B):
        for p in range(goal[b], held[b]):
            free[top], table[b][p], top = table[b][p], -1, top + 1
        held[b] = min(held[b], goal[b])
    pool, asked, wanted, n_new, row_start = top, 0, 0, [], [0]
    for b in range(B):
        need = goal[b] - held[b] if want[b] else 0
        asked += need
        n = want[b] if need == 0 or asked <= pool else 0
        wanted += n
        n = n if wanted <= rows else 0
        for _ in range(need if n else 0):
            top -= 1
            table[b][held[b]], held[b] = free[top], held[b] + 1
        n_new.append(n)
        row_start.append(row_start[-1] + n)
    seq = [b for b, n in enumerate(n_new) for _ in range(n)]
    pos = [start[b] + i for b, n in enumerate(n_new) for i in range(n)]
    at = [table[b][p // page] for b, p in zip(seq, pos)]
    slot = [a * page + p % page if 0 <= a < num_pages else -1 for a, p in zip(at, pos)]
    pad = [-1] * (rows - len(seq))
    return {"table": table, "free": free, "n_free": [top], "held": held, "kv_len": [s + n for s, n in zip(start, n_new)],
            "n_new": n_new, "row_start": row_start, "seq": seq + pad, "pos": pos + pad, "slot": slot + pad}


# ---- rotary positions ---------------------------------------------------------------------------------


def freqs_ref(rot, theta, scaling=None, scale=1.0, original=8192.0, low=None, high=None):
    """Frequencies in 80 bits and the scaling's factor, from the header's formulas."""
    L, two_pi = np.longdouble, 2 * np.longdouble("3.14159265358979323846264338327950288")
    theta, s, i = L(theta), L(scale), np.arange(rot // 2).astype(np.longdouble)
    if scaling == "ntk" and rot > 2:
        theta = theta * s ** (L(rot) / (rot - 2))
    f = theta ** (-2 * i / rot)
    if scaling == "linear":
        f = f / s
    if scaling == "bands":
        lo, hi = 1.0 if low is None else low, 4.0 if high is None else high
        t = np.clip((original * f / two_pi - lo) / (L(hi) - lo), 0, 1)
        f = (1 - t) * f / s + t * f
    if scaling == "yarn":
        lo, hi = 1.0 if low is None else low, 32.0 if high is None else high
        a, b = (rot * np.log(L(original) / (two_pi * x)) / (2 * np.log(theta)) for x in (hi, lo))
        a, b = max(np.floor(a), L(0)), min(np.ceil(b), L(rot - 1))
        t = np.clip((i - a) / (b - a if b > a else L(0.001)), 0, 1)
        f = t * f / s + (1 - t) * f
        return f, 0.1 * math.log(scale) + 1.0
    return f, 1.0


def rope_ref(x, pos, freqs, factor, layout, inverse=False):
    """x fp64 [rows, heads, D], pos a list: the rotated rows, and the bound on an fp32 computation of them.

    The bound: an angle is off by 2^-25 of a half circle (its rounding to fp32) and 2^-32 of a circle (the bits that
    are left out), 1e-7 in all; sine and cosine by 4 * 2^-24 of their own; the factor, two products and a sum
    round once each: 4 * 2^-24.  Together below 2^-20 of factor (|x0| + |x1|)."""
    L = np.longdouble
    a = np.array(pos, dtype=np.longdouble)[:, None] * np.asarray(freqs, dtype=np.longdouble)
    a = np.fmod(a, 2 * L("3.14159265358979323846264338327950288")) * (-1 if inverse else 1)
    c, s = (torch.from_numpy((f(a) * factor).astype(np.float64))[:, None] for f in (np.cos, np.sin))
    half = len(freqs)
    i = torch.arange(half)
    i0, i1 = (i, i + half) if layout == "halves" else (2 * i, 2 * i + 1)
    y, e = x.clone(), torch.zeros_like(x)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    e[..., i0] = e[..., i1] = 2.0 ** -20 * factor * (x0.abs() + x1.abs())
    return y, e


def check_rounded(got, ref, e, dtype, what):
    """got (16-bit values as fp64) is ref, off by at most e, rounded once."""
    tol = e + HALF[dtype] * (ref.abs() + e) + TINY[dtype]
    worst = ((got - ref).abs() / tol).max().item() if ref.numel() else 0.0
    print(f"    {what} {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, what


# ---- attention of new rows ------------------------------------------------------------------------------


def visible(length, n, causal, window):
    """[n, length]: which positions each new row sees."""
    j, p = torch.arange(length), length - n + torch.arange(n)[:, None]
    seen = torch.ones(n, length, dtype=torch.bool)
    if causal:
        seen = j <= p
        if window:
            seen &= j > p - window
    return seen


def chunk_ref(q, k, v, seen, Hkv, scale, dtype):
    """q fp64 [n, Hq, D], k and v [Hkv, length, D], seen [n, length]: o, lse and bounds on both.

    The bounds are kv_cases.decode_ref's with P's rounding for the second product in place of its own: one number of
    11 bits in fp16, off by 2^-11 of a P, and by 2^-25 where P is below 2^-14 and the row's sum 2^8 at least; two in
    bf16, 2^-16."""
    n, Hq, D = q.shape
    G, most = Hq // Hkv, seen.shape[1]
    o, lse = torch.zeros_like(q), torch.full((n, Hq), -math.inf, dtype=torch.float64)
    eo, el = torch.zeros_like(q), torch.zeros(n, Hq, dtype=torch.float64)
    part = 2.0 ** -11 if dtype == "f16" else 2.0 ** -16
    some = seen.any(1)
    if not some.any():
        return o, lse, eo, el
    for h in range(Hq):
        kk, vv = k[h // G], v[h // G]
        s = (q[:, h] @ kk.T * scale).masked_fill(~seen, -math.inf)
        top = torch.logsumexp(s, 1)
        p = torch.where(seen, torch.exp(s - torch.where(some, top, 0.0)[:, None]), 0.0)
        o[:, h], lse[:, h] = p @ vv, top
        size = (q[:, h].abs() @ kk.abs().T).masked_fill(~seen, 0.0)
        ds = ((D + 2) * 2.0 ** -24 * scale * size + 2.0 ** -23 * s.masked_fill(~seen, 0.0).abs()).amax(1) + 8 * 2.0 ** -23
        el[:, h] = ds + most * 2.0 ** -24 + 4 * 2.0 ** -24 * (torch.where(some, top, 0.0).abs() + 16)
        eo[:, h] = (2 * ds + most * 2.0 ** -23 + part)[:, None] * (p @ vv.abs()) + 2.0 ** -33 * (seen.double() @ vv.abs())
    return o, lse, eo, el


def check_chunk(case, lens, n_new, q, o, lse, Hq, row_start=None, causal=True, window=0, scale=None, skip=()):
    """Compares the device's packed o and lse with the 64-bit ones, sequence by sequence."""
    D, at = case.D, 0
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q, o, lse = q.cpu().double(), o.cpu().double(), lse.cpu().double()
    worst = worst_l = 0.0
    for b, (length, n) in enumerate(zip(lens, n_new)):
        first = at if row_start is None else row_start[b]
        at += n
        if n == 0 or b in skip:
            continue
        rows = slice(first, first + n)
        ro, rl, eo, el = chunk_ref(q[rows, :Hq * D].reshape(n, Hq, D), case.k[b], case.v[b], visible(length, n, causal, window),
                                   case.Hkv, scale, case.dtype)
        go, gl = o[rows].reshape(n, Hq, D), lse[rows]
        assert torch.isfinite(go).all()
        worst = max(worst, ((go - ro).abs() / (eo + HALF[case.dtype] * (ro.abs() + eo) + TINY[case.dtype])).max().item())
        some = torch.isfinite(rl)
        assert torch.equal(some, torch.isfinite(gl)) and torch.equal(gl[~some], rl[~some])
        if some.any():
            worst_l = max(worst_l, ((gl - rl).abs()[some] / el[some]).max().item())
    print(f"    o {worst:.3f}, lse {worst_l:.3f} of their bounds", flush=True)
    assert worst <= 1.0 and worst_l <= 1.0
