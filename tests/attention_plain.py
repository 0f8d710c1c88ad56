"""Attention over packed sequences and paged caches in 64 bits, one sequence and head at a time, with
bounds on what rounding may do to it.

Bounds.  u is half a step of the tensors' type (eps / 2, relative), e = 2^-24 * 16 * sqrt(dim + n) the
32-bit sums' share: n + dim roundings of at most 2^-24 each, independent in sign, add up to a random walk,
and 16 of its steps are never reached by one value among millions.

* o = sum_j p_j v_j: each weight may be rounded to the type before its product (u), so may the result (u):
  |error| <= (2 u + e) sum_j p_j |v_j|, with a second factor 2 as roundings meet at the end of a binade.
* dv_j = sum_i p_ij do_i likewise with sum_i p_ij |do_i|.
* ds = p (dp - D) is rounded once (u |ds|); D = do . o takes the rounded output (u sum |do| |o|); dp and D
  are 32-bit sums (e sum |do| |v| and e sum |do| |o|).  dq and dk add these up with |k| and |q|, and round once.
"""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# Below the smallest normal value a step no longer shrinks with the value: float16's values under 2^-14 lie
# 2^-24 apart, so that rounding moves them by up to 2^-25 (bfloat16 and float32: 2^-134 and 2^-150, nothing here).
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def e32(n, d):
    return 2.0 ** -24 * 16 * math.sqrt(n + d)


def packed(q, k, v, lens, causal, scale, g=None, start=0):
    """(values, bounds): dicts of out, lse and, with the output's gradient g, dq, dk, dv; float64."""
    dt, u, d = q.dtype, HALF[q.dtype], q.shape[2]
    group = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    val = {"out": torch.zeros_like(q), "lse": torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64,
                                                         device=q.device)}
    tol = {"out": torch.zeros_like(q)}
    if g is not None:
        g = g.double()
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            val[n], tol[n] = torch.zeros_like(x), torch.zeros_like(x)
    at = start
    for n in lens:
        sl = slice(at, at + n)
        at += n
        if n == 0:
            continue
        e = e32(n, d)
        hide = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1) if causal else None
        for h in range(q.shape[1]):
            j = h // group
            s = q[sl, h] @ k[sl, j].T * scale
            if hide is not None:
                s = s.masked_fill(hide, -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            o = p @ v[sl, j]
            val["out"][sl, h], val["lse"][h, sl] = o, lse
            tol["out"][sl, h] = 2 * (2 * u + e) * (p @ v[sl, j].abs())
            if g is None:
                continue
            do = g[sl, h]
            dp = do @ v[sl, j].T
            ds = p * (dp - (do * o).sum(1, keepdim=True))
            val["dv"][sl, j] += p.T @ do
            tol["dv"][sl, j] += 2 * (2 * u + e) * (p.T @ do.abs())
            val["dq"][sl, h] = ds @ k[sl, j] * scale
            val["dk"][sl, j] += ds.T @ q[sl, h] * scale
            a = (do.abs() * o.abs()).sum(1, keepdim=True)
            off = u * ds.abs() + p * (u * a + e * (a + do.abs() @ v[sl, j].abs().T))
            tol["dq"][sl, h] = 2 * scale * (off @ k[sl, j].abs() + (u + e) * (ds.abs() @ k[sl, j].abs()))
            tol["dk"][sl, j] += 2 * scale * (off.T @ q[sl, h].abs() + (u + e) * (ds.abs().T @ q[sl, h].abs()))
    for x in tol.values():
        x += TINY[dt]
    return val, tol


def cached(q, k_pages, v_pages, table, lengths, counts, tree, scale):
    """(out, bound) of attention over a paged cache, float64.  Plain Python lists: lengths, counts."""
    b, n, h, d = q.shape
    kv, page = k_pages.shape[1], k_pages.shape[2]
    u = HALF[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for i in range(b):
        m = lengths[i]
        pre = m - counts[i]
        rows = [(int(table[i][r // page]), r % page) for r in range(m)]
        ok = torch.tensor([0 <= a < k_pages.shape[0] for a, _ in rows], dtype=torch.bool)
        at = torch.tensor([a if f else 0 for (a, _), f in zip(rows, ok.tolist())], dtype=torch.long)
        sl = torch.tensor([s for _, s in rows], dtype=torch.long)
        for c in range(counts[i]):
            see = ok.clone()
            for r in range(pre, m):
                see[r] &= bool(int(tree[i][c]) >> (r - pre) & 1) if tree is not None else r - pre <= c
            use = torch.nonzero(see).flatten()
            if not len(use):
                continue
            for x in range(h):
                y = x // (h // kv)
                kk = k_pages[at[use].to(q.device), y, sl[use].to(q.device)].double()
                vv = v_pages[at[use].to(q.device), y, sl[use].to(q.device)].double()
                p = torch.softmax(kk @ q[i, c, x].double() * scale, 0)
                out[i, c, x] = p @ vv
                tol[i, c, x] = 2 * (2 * u + e32(m, d)) * (p @ vv.abs())
    return out, tol + TINY[q.dtype]


def close(got, want, tol, what=""):
    """Asserts |got - want| <= tol everywhere, finite."""
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - tol
    worst = off.max().item() if off.numel() else 0.0
    if worst > 0:
        i = off.argmax()
        raise AssertionError(f"{what}: {got.flatten()[i]:.9g}, expected {want.flatten()[i]:.9g} "
                             f"within {tol.flatten()[i]:.3g}")
