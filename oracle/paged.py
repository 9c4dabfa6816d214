"""TEST INFRASTRUCTURE ONLY -- paged caches in f64, from the definitions: rotate and append a step's
keys and values, and attend over a sequence's pages.  torch on the CPU; nothing of the package is used."""

from __future__ import annotations

import math

import torch


def rotate(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor | None) -> torch.Tensor:
    """x [T, H, D] f64, rotate-half on the first 2 len(inv_freq) dims by pos * inv_freq."""
    if inv_freq is None or inv_freq.numel() == 0:
        return x
    h = inv_freq.numel()
    ang = pos.double()[:, None, None] * inv_freq.double()
    c, s = ang.cos(), ang.sin()
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def sequence_ok(n: int, c: int, t: int, width: int, page: int) -> bool:
    return n >= 0 and 0 <= c <= t and n + c <= width * page


def append(q, k, v, table, lengths, counts, inv_freq, page: int, n_pages: int, k_scale=None, v_scale=None):
    """(rotated q [B, T, Hq, D] f64, zero in padding; writes: list of (page id, slot, k [H, D], v [H, D]) in
    f64, before the rounding to the pages' type; bad: whether anything was out of range)."""
    B, T = k.shape[:2]
    out = torch.zeros(q.shape, dtype=torch.float64) if q is not None else None
    writes, bad = [], False
    for b in range(B):
        n, c = int(lengths[b]), (T if counts is None else int(counts[b]))
        if not sequence_ok(n, c, T, table.shape[1], page):
            bad = True
            continue
        pos = n + torch.arange(c)
        if q is not None:
            out[b, :c] = rotate(q[b, :c].double(), pos, inv_freq)
        kr, vr = rotate(k[b, :c].double(), pos, inv_freq), v[b, :c].double()
        if k_scale is not None:
            kr, vr = kr / k_scale.double()[:, None], vr / v_scale.double()[:, None]
        for i in range(c):
            pid = int(table[b, (n + i) // page])
            if not 0 <= pid < n_pages:
                bad = True
                continue
            writes.append((pid, (n + i) % page, kr[i], vr[i]))
    return out, writes, bad


def attention(q, k_pages, v_pages, table, lengths, counts=None, scale=None, window=None, k_scale=None, v_scale=None):
    """(o [B, T, Hq, D] f64, lse [B, T, Hq] f64, spread [B, T, Hq, D] = sum_j p_j |v_j|, dots [B, T, Hq] = the
    largest scale * sum_d |q_d k_jd| over the keys seen, bad).  spread and dots size the rounding errors a
    kernel may make."""
    B, T, Hq, D = q.shape
    P, H, page, _ = k_pages.shape
    rep = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    spread = torch.zeros_like(o)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64)
    dots = torch.zeros(B, T, Hq, dtype=torch.float64)
    bad = False
    for b in range(B):
        n, c = int(lengths[b]), (T if counts is None else int(counts[b]))
        if not sequence_ok(n, c, T, table.shape[1], page):
            bad = True
            continue
        for t in range(c):
            end = n + t + 1
            j = torch.arange(max(0, end - window) if window else 0, end)
            pid = table[b].long()[j // page]
            ok = (pid >= 0) & (pid < P)
            bad |= not bool(ok.all())
            pid, slot = pid[ok], (j % page)[ok]
            if pid.numel() == 0:
                continue
            for h in range(Hq):
                k = k_pages[pid, h // rep, slot].double() * (1 if k_scale is None else k_scale[h // rep].double())
                v = v_pages[pid, h // rep, slot].double() * (1 if v_scale is None else v_scale[h // rep].double())
                qd = q[b, t, h].double()
                s = (k @ qd) * scale
                m = s.max()
                e = (s - (0.0 if m == -math.inf else m)).exp()
                z = e.sum()
                lse[b, t, h] = m + z.log()
                dots[b, t, h] = ((k.abs() @ qd.abs()) * abs(scale)).max()
                if z != 0:
                    p = (e / z)[:, None]
                    o[b, t, h] = torch.where(p == 0, 0.0, p * v).sum(0)
                    spread[b, t, h] = torch.where(p == 0, 0.0, p * v.abs()).sum(0)
    return o, lse, spread, dots, bad
